"""Token-side operators without a GPU: refusals, C ABI contract errors, and the differentiable restatements and test oracle
against float64 autograd."""

import ctypes

import pytest
import torch
import torch.nn.functional as F

import token_oracle as O
from theria_amd import _lib
from theria_amd.autograd import hip_embedding, hip_layer_norm, hip_linear_cross_entropy
from theria_amd.models import MHAClassifier


def test_cpu_tensors_are_refused():
    x, ids = torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64)
    for call in (lambda: hip_layer_norm(x), lambda: hip_embedding(ids, x), lambda: hip_linear_cross_entropy(x, x, ids)):
        with pytest.raises(AssertionError, match="requires GPU"):
            call()


def test_model_refuses_unknown_ops():
    with pytest.raises(ValueError, match="ops"):
        MHAClassifier(ops="cuda")


def test_model_loss_is_the_cross_entropy_of_its_logits():
    torch.manual_seed(0)
    model = MHAClassifier()
    tokens, y = torch.randint(0, 32, (4, 10)), torch.randint(0, 5, (4,))
    assert torch.equal(model(tokens, y), F.cross_entropy(model(tokens), y))


def _refused(rc, needle):
    assert rc == _lib.ERR_CONTRACT
    assert needle in _lib.load().theria_last_error().decode()


FAKE = 0x10000  # never dereferenced on the host


def test_layer_norm_contract():
    lib = _lib.load()
    rows = _lib.RowsView(FAKE, 64)

    def fwd(p, x=rows, y=rows, mean=FAKE):
        return lib.theria_layer_norm_fwd(ctypes.byref(p), ctypes.byref(x), None, None, ctypes.byref(y), mean, FAKE, None)

    P = _lib.LayerNormProblem
    _refused(fwd(P(9, 0, 64, 1e-5, 4)), "dtype")
    _refused(fwd(P(2, 1, 64, 1e-5, 4)), "param_dtype")
    _refused(fwd(P(2, 2, 0, 1e-5, 4)), "width")
    _refused(fwd(P(2, 2, 16385, 1e-5, 4)), "width")
    _refused(fwd(P(2, 2, 64, -1.0, 4)), "eps")
    _refused(fwd(P(2, 2, 64, 1e-5, -1)), "rows")
    _refused(fwd(P(2, 2, 64, 1e-5, 4), x=_lib.RowsView(None, 64)), "absent")
    _refused(fwd(P(2, 2, 64, 1e-5, 4), y=_lib.RowsView(FAKE, -64)), "negative stride")
    _refused(fwd(P(2, 2, 64, 1e-5, 4), mean=None), "mean and rstd")
    assert fwd(P(2, 2, 64, 1e-5, 0)) == _lib.OK
    p = ctypes.byref(P(2, 2, 64, 1e-5, 4))
    r = ctypes.byref(rows)
    _refused(lib.theria_layer_norm_bwd(p, r, None, r, FAKE, FAKE, None, FAKE, None, None, None), "workspace")
    _refused(lib.theria_layer_norm_bwd(ctypes.byref(P(2, 2, 64, 1e-5, 0)), r, None, r, FAKE, FAKE, None, FAKE, None, FAKE, None), "rows must be positive")
    _refused(lib.theria_layer_norm_bwd_bwd(p, r, None, r, FAKE, FAKE, None, None, None, None, FAKE, None, None, None), "workspace")
    assert lib.theria_layer_norm_ws_floats(ctypes.byref(P(9, 0, 64, 1e-5, 4))) == 0


def test_embedding_contract():
    lib = _lib.load()
    r = ctypes.byref(_lib.RowsView(FAKE, 64))
    P = _lib.EmbeddingProblem

    def fwd(p, ids=FAKE):
        return lib.theria_embedding_fwd(ctypes.byref(p), ids, r, 0, r, None)

    _refused(fwd(P(5, 1, 64, 1.0, 4, 10, -1)), "dtype")
    _refused(fwd(P(2, 1, 0, 1.0, 4, 10, -1)), "width")
    _refused(fwd(P(2, 1, 64, float("nan"), 4, 10, -1)), "scale")
    _refused(fwd(P(2, 1, 64, 1.0, 4, 2**27 + 1, -1)), "classes")
    _refused(fwd(P(2, 1, 64, 1.0, 4, 10, 10)), "padding")
    _refused(fwd(P(2, 1, 64, 1.0, 4, 10, -1), ids=None), "ids")
    assert fwd(P(2, 1, 64, 1.0, 0, 10, -1)) == _lib.OK
    p = P(2, 1, 64, 1.0, 4, 10, -1)
    _refused(lib.theria_embedding_bwd(ctypes.byref(p), FAKE, r, r, None, None), "workspace")
    _refused(lib.theria_embedding_bwd(ctypes.byref(p), FAKE, r, ctypes.byref(_lib.RowsView(None, 0)), FAKE, None), "absent")
    assert lib.theria_embedding_ws_bytes(ctypes.byref(P(5, 1, 64, 1.0, 4, 10, -1))) == 0
    # pieces' sums of 64 tokens beside four arrays of the tokens and the digits' counts
    assert lib.theria_embedding_ws_bytes(ctypes.byref(P(2, 1, 64, 1.0, 128, 10, -1))) >= 4 * 4 * 128 + 4 * 2 * 64


def test_linear_ce_contract():
    lib = _lib.load()
    rows = _lib.RowsView(FAKE, 64)
    r = ctypes.byref(rows)
    P = _lib.LinearCeProblem

    def fwd(p, loss=FAKE, ws=FAKE, stats=FAKE):
        return lib.theria_linear_ce_fwd(ctypes.byref(p), r, r, None, FAKE, loss, stats, ws, None)

    _refused(fwd(P(7, 1, 1, 64, 4, 10, -100)), "dtype")
    _refused(fwd(P(2, 1, 3, 64, 4, 10, -100)), "reduction")
    _refused(fwd(P(2, 1, 1, 0, 4, 10, -100)), "width")
    _refused(fwd(P(2, 1, 1, 64, 4, 0, -100)), "classes")
    _refused(fwd(P(2, 1, 1, 64, -4, 10, -100)), "n must")
    _refused(fwd(P(2, 1, 1, 64, 4, 2**26 + 1, -100)), "classes")
    _refused(fwd(P(2, 1, 1, 64, 4, 10, -100), loss=None), "loss")
    _refused(fwd(P(2, 1, 1, 64, 4, 10, -100), ws=FAKE + 16), "256-byte-aligned")
    _refused(fwd(P(2, 1, 1, 64, 4, 10, -100), stats=None), "stats")
    p = ctypes.byref(P(2, 1, 1, 64, 4, 10, -100))
    _refused(lib.theria_linear_ce_bwd(p, r, r, None, FAKE, FAKE, None, r, r, None, FAKE, None), "dloss")
    assert lib.theria_linear_ce_ws_bytes(ctypes.byref(P(7, 1, 1, 64, 4, 10, -100)), r, 0, 0, 0, 0) == 0
    for n, v, d in ((0, 1, 1), (0, 10**5, 4096), (1, 1, 1)):  # sizes of nothing divide nothing
        for backward in (0, 1):
            assert lib.theria_linear_ce_ws_bytes(ctypes.byref(P(2, 1, 1, d, n, v, -100)), r, backward, 1, 1, 1) > 0
    # the workspace does not grow with the vocabulary beyond a piece of it: 256 MiB of dz, and what the rows take
    sizes = [lib.theria_linear_ce_ws_bytes(ctypes.byref(P(2, 1, 1, 64, 8192, v, -100)), r, 1, 1, 1, 1) for v in (10**5, 10**7)]
    assert sizes[0] == sizes[1] < (300 << 20)


def test_layer_norm_restatement_and_oracle():
    """The order-three restatement and the oracle's first and second derivatives against autograd of the definition."""
    from theria_amd import _ops

    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    eps = 1e-3
    x, w, b, g, u, a, c = r(4, 11), r(11), r(11), r(4, 11), r(4, 11), r(11), r(11)

    def plain(x, w, b):
        v, m = torch.var_mean(x, -1, correction=0, keepdim=True)
        return (x - m) / torch.sqrt(v + eps) * w + b

    xl, wl, bl, gl = (t.clone().requires_grad_(True) for t in (x, w, b, g))
    y = plain(xl, wl, bl)
    first = torch.autograd.grad(y, (xl, wl, bl), gl, create_graph=True)
    second = torch.autograd.grad(first, (xl, wl, gl), (u, a, c))
    torch.testing.assert_close(O.norm_forward(x, w, b, eps)[0], y.detach())
    for got, want in zip(_ops._host().layer_norm_backward_map(x, w, g, eps), first):
        torch.testing.assert_close(got, want.detach())
    for (got, _), want in zip(O.norm_backward(x, w, g, eps, torch.float32), first):
        torch.testing.assert_close(got, want.detach())
    for (got, _), want in zip(O.norm_second(x, w, g, u, a, c, eps, torch.float32), second):
        torch.testing.assert_close(got, want)


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_linear_ce_restatement_and_oracle(reduction):
    from theria_amd import _ops

    code = {"none": 0, "mean": 1, "sum": 2}[reduction]
    gen = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    x, w, b, g = (t.requires_grad_(True) for t in (r(9, 6), r(5, 6), r(5), r(9)))
    t = torch.tensor([0, 4, -100, 2, 1, -100, 3, 3, 0])
    loss = F.cross_entropy(F.linear(x, w, b), t, reduction=reduction)
    grads = torch.autograd.grad(loss, (x, w, b), g if reduction == "none" else None)
    up = g if reduction == "none" else torch.ones(())
    for got, want in zip(_ops._host().linear_ce_backward_map(x, w, b, t, up, -100, code), grads):
        torch.testing.assert_close(got, want)
    oracle = O.linear_ce(x.float(), w.float(), b.float(), t, -100, reduction, up.detach())
    torch.testing.assert_close(oracle["loss"][0], loss.detach(), rtol=1e-5, atol=1e-6)
    for n, want in zip(("dx", "dw", "db"), grads):
        torch.testing.assert_close(oracle[n][0], want, rtol=1e-5, atol=1e-6)


def test_embedding_oracle():
    gen = torch.Generator().manual_seed(2)
    w = torch.randn(7, 3, generator=gen, dtype=torch.float64, requires_grad=True)
    ids, g = torch.randint(0, 7, (20,), generator=gen), torch.randn(20, 3, generator=gen)
    (dw,) = torch.autograd.grad(F.embedding(ids, w, padding_idx=2) * 1.5, w, g.double())
    torch.testing.assert_close(O.embed_backward(ids, g, 7, 1.5, 2)[0], dw)
