"""hip_embedding on the GPU against float64 sums (tests/token_oracle.py): lookup, gradient by sorted tokens, higher orders."""

import pytest
import torch

import token_oracle as O
from theria_amd.autograd import hip_embedding

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _ids(N, V, kind, seed):
    gen = torch.Generator().manual_seed(seed)
    if kind == "uniform":
        return torch.randint(0, V, (N,), generator=gen)
    if kind == "one":
        return torch.full((N,), V // 2)
    if kind == "rising":
        return torch.arange(N) % V
    return ((torch.rand(N, generator=gen, dtype=torch.float64) * torch.log(torch.tensor(V + 1.0))).exp().long() - 1).clamp(0, V - 1)


def _run(ids, w, g, scale=1.0, padding=None):
    wl = w.detach().requires_grad_(True)
    y = hip_embedding(ids, wl, scale=scale, padding_idx=padding)
    (dw,) = torch.autograd.grad(y, wl, g)
    return y.detach(), dw


def _check(ids, w, g, scale, padding, what):
    y, dw = _run(ids, w, g, scale, padding)
    O.check(y, *O.embed_forward(ids, w, scale), f"{what} rows")
    O.check(dw, *O.embed_backward(ids, g, w.shape[0], scale, padding), f"{what} gradient")


# tokens on both sides of the counting sort's limit (8192) and of a sort tile (4096); tables of one, two and three
# digits; widths of every team, odd and on their borders
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("N,V,D", [(1, 1, 1), (1, 50, 64), (5, 3, 7), (63, 10, 40), (64, 10, 128), (65, 10, 130), (200, 1000, 256), (1000, 32, 64),
                                   (4097, 700, 24), (8192, 50, 16), (8193, 50, 16), (8193, 1023, 33), (9000, 1024, 72), (12289, 40000, 8),
                                   (20000, 1100000, 4), (300, 77, 1032), (500, 20, 2056), (130, 9, 4100), (90, 5, 8200)])
def test_rows_and_gradient_match_float64(dt, N, V, D, hip_device):
    gen = torch.Generator().manual_seed(N + D)
    w = torch.randn(V, D, generator=gen).to(dt).to(hip_device)
    g = torch.randn(N, D, generator=gen).to(dt).to(hip_device)
    for kind in ("uniform", "zipf"):
        print(f"[embedding] {dt} N{N} V{V} D{D} {kind}", flush=True)
        _check(_ids(N, V, kind, N).to(hip_device), w, g, 1.5, None, kind)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N", [1, 63, 64, 65, 255, 256, 257, 511, 512, 513])
@pytest.mark.parametrize("V,D", [(1, 40), (16, 64), (17, 200), (40000, 72), (9000, 520)])
def test_few_tokens(N, V, D, dt, hip_device):
    """On both sides of the gradient in one launch, whose workgroups order their rows' tokens themselves."""
    gen = torch.Generator().manual_seed(N + V)
    w, g = torch.randn(V, D, generator=gen).to(dt).to(hip_device), torch.randn(N, D, generator=gen).to(dt).to(hip_device)
    for kind in ("uniform", "zipf", "one", "rising"):
        _check(_ids(N, V, kind, N).to(hip_device), w, g, 0.5, 0 if V > 1 else None, f"{kind} {N}")
    ids = _ids(N, V, "uniform", 1)
    ids[::3] = torch.tensor([-1, V, 2**40])[torch.arange(len(ids[::3])) % 3]
    _, dw = _run(ids.to(hip_device), w, g)
    known = (ids >= 0) & (ids < V)
    O.check(dw, *O.embed_backward(ids[known], g[known.to(hip_device)], V, 1.0, None), "ids outside the table")


@pytest.mark.parametrize("N,V", [(131072, 3000), (131073, 3000), (200003, 70000)])
def test_many_tokens(N, V, hip_device):
    """On both sides of the radix sort's change to tiles of 4096 tokens."""
    gen = torch.Generator().manual_seed(N)
    w, g = torch.randn(V, 8, generator=gen).to(hip_device), torch.randn(N, 8, generator=gen).to(hip_device)
    for kind in ("uniform", "zipf"):
        _check(_ids(N, V, kind, N).to(hip_device), w, g, 1.0, 1, f"{kind} {N}")


def test_lookup_in_several_launches(hip_device):
    """More ids than a launch takes (2^23)."""
    N = 2**23 + 5
    gen = torch.Generator().manual_seed(1)
    w, ids = torch.randn(100, 3, generator=gen).half().to(hip_device), torch.randint(0, 100, (N,), generator=gen).int().to(hip_device)
    assert torch.equal(hip_embedding(ids, w), w[ids.long()])


@pytest.mark.parametrize("D", [16, 64, 200, 1500, 4096])
@pytest.mark.parametrize("N", [64, 127, 5000, 20001])
def test_one_id_for_every_token_and_rising_ids(N, D, hip_device):
    """The longest runs (pieces of 64 tokens joined) and the shortest."""
    if N * D > 2**26:
        pytest.skip("the float64 reference of this size takes minutes")
    gen = torch.Generator().manual_seed(D)
    w, g = torch.randn(300, D, generator=gen).bfloat16().to(hip_device), torch.randn(N, D, generator=gen).bfloat16().to(hip_device)
    for kind in ("one", "rising"):
        _check(_ids(N, 300, kind, 0).to(hip_device), w, g, 1.0, None, f"{kind} {N} {D}")


@pytest.mark.parametrize("idt", [torch.int32, torch.int64])
def test_shapes_strides_and_id_types(idt, hip_device):
    gen = torch.Generator().manual_seed(4)
    w = torch.randn(40, 50, generator=gen).half().to(hip_device)
    ids = torch.randint(0, 40, (6, 9), generator=gen).to(idt).to(hip_device)
    g = torch.randn(6, 9, 50, generator=gen).half().to(hip_device)
    _check(ids, w, g, 0.25, 3, "3-d")
    _check(ids.t(), w, g.transpose(0, 1), 0.25, None, "transposed ids and gradient")
    wide = torch.randn(40, 64, generator=gen).half().to(hip_device)
    y, dw = _run(ids, wide[:, 3:53], g)
    O.check(y, *O.embed_forward(ids, wide[:, 3:53], 1.0), "rows of a wider table")
    O.check(dw, *O.embed_backward(ids, g, 40, 1.0, None), "its gradient")
    _check(ids, w.t().contiguous().t(), g, 1.0, None, "table stored by columns")
    scalar = hip_embedding(ids[0, 0], w)
    assert torch.equal(scalar, w[ids[0, 0]])
    _check(ids, w, g[:1, :1].expand(6, 9, 50), 1.0, None, "broadcast gradient")
    _check(ids[:0], w, g[:0], 1.0, None, "no ids")


def test_padding_and_ids_outside_the_table(hip_device):
    gen = torch.Generator().manual_seed(5)
    for N in (700, 9000):
        w = torch.randn(30, 72, generator=gen).to(hip_device)
        ids = torch.randint(0, 30, (N,), generator=gen).to(hip_device)
        ids[::3] = 7
        g = torch.randn(N, 72, generator=gen).to(hip_device)
        g[ids == 7] = float("nan")  # the gradients of padding rows are not read
        for pad in (7, 7 - 30):
            y, dw = _run(ids, w, g, 1.0, pad)
            assert torch.equal(y, w[ids]) and torch.isfinite(dw).all() and not dw[7].any()
            O.check(dw, *O.embed_backward(ids, g, 30, 1.0, 7), "gradient beside padding")
        bad = ids.clone()
        bad[::5], bad[1::7] = -1, 30
        bad[2] = 2**40
        out = (bad < 0) | (bad >= 30)
        y, dw = _run(bad, w, torch.where(out.unsqueeze(1), float("nan"), g.nan_to_num()), 1.0, 7)
        assert torch.isnan(y[out]).all() and torch.equal(y[~out], w[bad[~out]])
        O.check(dw, *O.embed_backward(bad, g.nan_to_num(), 30, 1.0, 7), "gradient without the ids outside")


def test_the_same_bits_on_every_run(hip_device):
    gen = torch.Generator().manual_seed(6)
    for N in (6000, 30000):
        w = torch.randn(100, 96, generator=gen).bfloat16().to(hip_device)
        ids, g = _ids(N, 100, "zipf", 1).to(hip_device), torch.randn(N, 96, generator=gen).bfloat16().to(hip_device)
        first = _run(ids, w, g)[1]
        assert all(torch.equal(first, _run(ids, w, g)[1]) for _ in range(4))


def test_higher_orders(hip_device):
    """The gradient is linear: its derivative is a lookup (zero for padding), whose derivative is a gradient again."""
    gen = torch.Generator().manual_seed(8)
    w = torch.randn(25, 40, generator=gen).to(hip_device).requires_grad_(True)
    ids = torch.randint(0, 25, (90,), generator=gen).to(hip_device)
    g = torch.randn(90, 40, generator=gen).to(hip_device).requires_grad_(True)
    u = torch.randn(25, 40, generator=gen).to(hip_device).requires_grad_(True)
    (dw,) = torch.autograd.grad(hip_embedding(ids, w, scale=3.0, padding_idx=2), w, g, create_graph=True)
    (gg,) = torch.autograd.grad(dw, g, u, create_graph=True)
    want = torch.where((ids == 2).unsqueeze(1), 0.0, 3 * u[ids])
    assert torch.equal(gg, want)
    (gu,) = torch.autograd.grad(gg, u, g)
    O.check(gu, *O.embed_backward(ids, g.detach(), 25, 3.0, 2), "third order")


def test_gradient_agrees_with_differences_of_the_lookup(hip_device):
    """The lookup is linear in the table: a difference of it along a direction is exact up to rounding."""
    gen = torch.Generator().manual_seed(9)
    w, d = torch.randn(12, 20, generator=gen).double(), torch.randn(12, 20, generator=gen).double()
    ids, g = torch.randint(0, 12, (50,), generator=gen), torch.randn(50, 20, generator=gen)
    _, dw = _run(ids.to(hip_device), w.float().to(hip_device), g.to(hip_device), 2.0)
    num = (((w + d)[ids] - (w - d)[ids]) * 2.0 / 2 * g.double()).sum()
    bound = (O.embed_backward(ids, g, 12, 2.0, None)[1] * d.abs()).sum()
    assert abs(float((dw.double().cpu() * d).sum() - num)) <= float(bound)


def test_side_streams_and_graph_replays(hip_device):
    gen = torch.Generator().manual_seed(10)
    for N in (3000, 10000):
        w = torch.randn(2000, 64, generator=gen).bfloat16().to(hip_device)
        sets = [(torch.randint(0, 2000, (N,), generator=gen).to(hip_device), torch.randn(N, 64, generator=gen).bfloat16().to(hip_device)) for _ in range(2)]
        ref = [_run(i, w, g) for i, g in sets]
        streams = [torch.cuda.Stream() for _ in sets]
        torch.cuda.synchronize()
        out = []
        for st, (i, g) in zip(streams, sets):
            with torch.cuda.stream(st):
                out.append(_run(i, w, g))
        torch.cuda.synchronize()
        for p, q in zip(out, ref):
            assert torch.equal(p[0], q[0]) and torch.equal(p[1], q[1])
        ids, g = sets[0][0].clone(), sets[0][1].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _run(ids, w, g)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, dw = _run(ids, w, g)
        for k in (1, 0, 1):
            ids.copy_(sets[k][0])
            g.copy_(sets[k][1])
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, ref[k][0]) and torch.equal(dw, ref[k][1])
            _run(*sets[1 - k][:1], w, sets[1 - k][1])


def test_refusals(hip_device):
    w, ids = torch.zeros(5, 8, device=hip_device), torch.zeros(3, dtype=torch.int64, device=hip_device)
    with pytest.raises(AssertionError, match="int32 or int64"):
        hip_embedding(ids.float(), w)
    with pytest.raises(AssertionError, match="ids must be on"):
        hip_embedding(ids.cpu(), w)
    with pytest.raises(AssertionError, match=r"\(V, D\)"):
        hip_embedding(ids, w[0])
    with pytest.raises(AssertionError, match="dtype"):
        hip_embedding(ids, w.double())
    with pytest.raises(AssertionError, match="padding_idx"):
        hip_embedding(ids, w, padding_idx=5)
    with pytest.raises(AssertionError, match="scale"):
        hip_embedding(ids, w, scale=float("inf"))
