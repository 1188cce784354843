"""hip_linear_cross_entropy on the GPU against float64 formulas (tests/token_oracle.py): loss and gradients over every tile
shape, ignored and invalid targets, odd and strided operands, reductions, pieces of the vocabulary, streams and graphs."""

import pytest
import torch

import token_oracle as O
from theria_amd.autograd import hip_linear_cross_entropy

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IGNORE = -100


def _make(N, V, D, dt, dev, seed=0, bias=False, pad=0.0, lean=2.0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    t = torch.randint(0, V, (N,), generator=gen)
    w = r(V, D) / D**0.5
    x = r(N, D) + lean * w[t]
    t[torch.randperm(N, generator=gen)[: int(N * pad)]] = IGNORE
    b = 0.3 * r(V) if bias else None
    return x.to(dt).to(dev), w.to(dt).to(dev), t.to(dev), None if b is None else b.to(dt).to(dev), torch.rand(N, generator=gen).to(dev)


def _run(x, w, t, b=None, reduction="mean", g=None, **kw):
    xl, wl = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    bl = None if b is None else b.detach().requires_grad_(True)
    loss = hip_linear_cross_entropy(xl, wl, t, bl, reduction=reduction, **kw)
    grads = torch.autograd.grad(loss, [a for a in (xl, wl, bl) if a is not None], g)
    return dict(zip(("loss", "dx", "dw", "db"), (loss.detach(), *grads)))


def _check(x, w, t, b, reduction, g, what, ignore=IGNORE):
    got = _run(x, w, t, b, reduction, g, ignore_index=ignore)
    want = O.linear_ce(x, w, b, t, ignore, reduction, torch.ones(()) if g is None else g)
    for n, v in got.items():
        value, tol = want[n]
        O.check(v.reshape(value.shape), value, tol, f"{what} {n}")
    return got


# few classes (up to 16 of 256 or 8 of 512) in one workgroup and in several, and just more of them; few tokens (up to
# 64), tiles of 128 and of 256; widths and vocabularies on and off their multiples; one of each
SIZES = [(1, 1, 1), (1, 2, 8), (3, 5, 64), (25, 5, 64), (64, 8, 512), (65, 8, 511), (300, 8, 513), (700, 16, 256), (90, 9, 257), (333, 13, 100),
         (40, 17, 64), (20000, 3, 65), (5000, 16, 40), (64, 700, 72), (65, 130, 40), (48, 1000, 256), (130, 257, 129), (200, 129, 520), (300, 1031, 65),
         (129, 128, 128), (256, 512, 64), (513, 2050, 96), (1030, 64, 200)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("N,V,D", SIZES)
def test_loss_and_gradients_match_float64(dt, N, V, D, hip_device):
    for reduction, bias, pad in (("mean", False, 0.0), ("none", True, 0.3), ("sum", True, 0.0)):
        print(f"[linear ce] {dt} N{N} V{V} D{D} {reduction} bias={bias} pad={pad}", flush=True)
        x, w, t, b, g = _make(N, V, D, dt, hip_device, seed=N + V, bias=bias, pad=pad)
        _check(x, w, t, b, reduction, g if reduction == "none" else None, f"{reduction} bias={bias}")


@pytest.mark.parametrize("N", [257, 1300, 4100])
@pytest.mark.parametrize("V,D", [(5, 700), (17, 64), (40, 1030), (128, 300), (129, 520), (256, 65), (257, 65)])
def test_float32_of_many_rows_and_few_classes(N, V, D, hip_device):
    x, w, t, b, g = _make(N, V, D, torch.float32, hip_device, seed=N + V, bias=True, pad=0.2)
    _check(x, w, t, b, "none", g, f"{N} {V} {D}")
    _check(x, w, t, None, "mean", None, f"{N} {V} {D} mean")


@pytest.mark.parametrize("dt", DTYPES)
def test_large_tiles(dt, hip_device):
    """Enough tiles for the 256 x 256 shape in all three products (205 and more), with ragged edges."""
    N, V, D = (3850, 3610, 200) if dt != torch.float32 else (3850, 3610, 72)
    x, w, t, b, g = _make(N, V, D, dt, hip_device, seed=1, bias=True, pad=0.1)
    _check(x, w, t, b, "none", g, "large")


@pytest.mark.parametrize("N,V,D", [(3300, 3200, 4040), (4100, 9000, 1024)])
def test_large_tiles_in_both_gradients(N, V, D, hip_device):
    """Tiles of 256 for dx and dw, in one part each (16 x 13 and 13 x 16), and dx in several parts joined in float32."""
    x, w, t, b, _ = _make(N, V, D, torch.bfloat16, hip_device, seed=2)
    got = _run(x, w, t)
    xd, wd = x.double(), w.double()  # on the GPU: the CPU would take a minute
    z = xd @ wd.t()
    p = torch.softmax(z, 1)
    p[torch.arange(N, device=hip_device), t] -= 1
    p /= N
    for n, want, scale in (("dx", p @ wd, p.abs() @ wd.abs()), ("dw", p.t() @ xd, p.abs().t() @ xd.abs())):
        # dz rounded (2^-8 of each entry at most), its logits off by (D + 8) u sum|x w| on both sides, the result rounded
        rel = 2.0**-8 + 4 * (D + 8) * O.U * float((xd.abs() @ wd.abs().t()).max())
        tol = rel * scale + O.half_step(torch.bfloat16) * want.abs()
        off = ((got[n].double() - want).abs() / tol).max()
        assert float(off) <= 1, f"{n}: {float(off):.3g} times the bound"


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("N,V", [(30, 5), (100, 13), (40, 60), (300, 100), (300, 700), (1100, 1030)])
def test_small_losses_keep_their_digits(dt, N, V, hip_device):
    """Rows whose target stands far above the other classes, with logits that every type holds exactly: loss log1p(sum of
    exp(z - top)). The exponent of at most 16 log2(e) = 23.1 has two roundings (its constant's and the product's), 2 * 23.1 ln 2 u
    = 32 u of the exponential, which is good to 2 u itself; V terms are added and log1p good to 4 u: 38 u and V u."""
    gen = torch.Generator().manual_seed(V)
    t = torch.randint(0, V, (N,), generator=gen)
    x = torch.randint(-8, 9, (N, V), generator=gen) / 8.0
    x[torch.arange(N), t] = 3.0
    z = 4.0 * x.double()
    z -= 12.0
    others = torch.exp(z).scatter(1, t.unsqueeze(1), 0.0).sum(1)
    want = torch.log1p(others)
    got = hip_linear_cross_entropy(x.to(dt).to(hip_device), (4.0 * torch.eye(V)).to(dt).to(hip_device), t.to(hip_device), reduction="none")
    off = ((got.double().cpu() - want).abs() / want).max()
    assert float(off) <= (V + 38) * O.U, f"{float(off) / O.U:.3g} u"


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("N", [16384, 16385, 40000])
def test_many_rows_are_listed_by_several_workgroups(dt, N, hip_device):
    """On both sides of the limit of one workgroup; ignored and invalid targets in runs, at both ends, and everywhere."""
    x, w, t, b, g = _make(N, 20, 24, dt, hip_device, seed=4, bias=True, pad=0.3)
    t[:5000], t[-3:] = IGNORE, IGNORE
    t[9000:9100], t[N - 10] = 20, -7
    _check(x, w, t, b, "none", g, f"{N} rows")
    t[:] = IGNORE
    got = _run(x, w, t, b, "sum")
    assert not got["loss"].any() and not got["dx"].any() and not got["dw"].any()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_ignored_rows_are_never_read(dt, reduction, hip_device):
    x, w, t, b, g = _make(300, 200, 72, dt, hip_device, seed=3, bias=True, pad=0.5)
    clean = _run(x, w, t, b, reduction, g if reduction == "none" else None)
    gone = t == IGNORE
    x2, g2 = x.clone(), g.clone()
    x2[gone] = float("nan")
    x2[gone.nonzero()[::2, 0]] = float("inf")
    g2[gone] = float("nan")
    dirty = _run(x2, w, t, b, reduction, g2 if reduction == "none" else None)
    for n in clean:
        assert torch.equal(clean[n], dirty[n]), f"{n} depends on ignored rows"
    assert not clean["dx"][gone].any()
    if reduction == "none":
        assert not clean["loss"][gone].any()


def test_all_rows_ignored_and_no_rows(hip_device):
    for dt in DTYPES:
        x, w, t, b, g = _make(70, 90, 64, dt, hip_device, bias=True, pad=1.0)
        for reduction in ("none", "sum", "mean"):
            got = _run(x, w, t, b, reduction, g if reduction == "none" else None)
            assert torch.isnan(got["loss"]) if reduction == "mean" else not got["loss"].any()
            assert not got["dx"].any() and not got["dw"].any() and not got["db"].any()
        for reduction in ("none", "sum", "mean"):
            got = _run(x[:0], w, t[:0], b, reduction, g[:0] if reduction == "none" else None)
            assert got["dx"].shape == (0, 64) and not got["dw"].any() and not got["db"].any()
            assert got["loss"].shape == ((0,) if reduction == "none" else ())
            if reduction != "none":
                assert torch.isnan(got["loss"]) if reduction == "mean" else not got["loss"].any()


def test_targets_outside_the_vocabulary(hip_device):
    x, w, t, b, g = _make(150, 40, 32, torch.bfloat16, hip_device, bias=True, pad=0.2)
    t[5], t[77], t[140] = 40, -1, 2**40
    got = _check(x, w, t, b, "none", g, "invalid targets")
    assert torch.isnan(got["loss"][[5, 77, 140]]).all() and torch.isnan(got["dx"][[5, 77, 140]]).all()
    assert torch.isfinite(got["dw"]).all()
    assert torch.isnan(_run(x, w, t, b, "mean")["loss"])


@pytest.mark.parametrize("ignore", [0, 7, -1, 10**6])
def test_other_ignored_targets(ignore, hip_device):
    x, w, t, b, g = _make(100, 50, 40, torch.float32, hip_device)
    t[::4] = ignore
    _check(x, w, t, b, "mean", None, f"ignore {ignore}", ignore=ignore)


def test_masked_classes_and_large_logits(hip_device):
    """A bias of minus infinity takes a class out; logits of hundreds stay finite; a row that is NaN stays alone in dx."""
    for dt in DTYPES:
        x, w, t, b, g = _make(90, 300, 64, dt, hip_device, bias=True)
        b[150:] = float("-inf")
        t %= 150
        got = _check(x, w, t, b, "mean", None, f"masked {dt}")
        assert not got["dw"][150:].any() and not got["db"][150:].any()
        _check(x * 40, w, t, None, "mean", None, f"large logits {dt}")
        x[17] = float("nan")
        got = _run(x, w, t, None, "none", g)
        rest = [i for i in range(90) if i != 17]
        assert torch.isnan(got["loss"][17]) and torch.isnan(got["dx"][17]).all()
        assert torch.isfinite(got["loss"][rest]).all() and torch.isfinite(got["dx"][rest]).all()


def test_strides_misaligned_operands_and_leading_dimensions(hip_device):
    for dt in DTYPES:
        x, w, t, b, g = _make(96, 75, 64, dt, hip_device, bias=True)
        want = _run(x, w, t, b, "none", g)
        wide_x, wide_w = torch.zeros(96, 80, dtype=dt, device=hip_device), torch.zeros(75, 72, dtype=dt, device=hip_device)
        wide_x[:, 5:69], wide_w[:, 8:72] = x, w
        off = torch.zeros(75 * 64 + 1, dtype=dt, device=hip_device)
        off[1:] = w.reshape(-1)
        forms = {
            "rows apart": (wide_x[:, 5:69], wide_w[:, 8:72]),
            "weight off 16 bytes": (x, off[1:].view(75, 64)),
            "by columns": (x.t().contiguous().t(), w.t().contiguous().t()),
        }
        for name, (xv, wv) in forms.items():
            got = _run(xv, wv, t, b, "none", g)
            for n in want:
                assert torch.equal(got[n], want[n]), f"{dt} {name} {n}"
        got = _run(x.view(4, 24, 64), w, t.view(4, 24).int(), b, "none", g.view(4, 24))
        assert got["loss"].shape == (4, 24) and torch.equal(got["loss"].view(-1), want["loss"])
        assert got["dx"].shape == (4, 24, 64) and torch.equal(got["dx"].view(96, 64), want["dx"]) and torch.equal(got["dw"], want["dw"])
        one = x[:1].expand(96, 64)
        _check(one, w, t, b, "sum", None, f"{dt} one row for all")


def test_gradients_of_every_size_and_sign(hip_device):
    """Row weights over many orders of magnitude, zero, negative; a row whose own gradient is infinite or NaN."""
    for dt in DTYPES:
        x, w, t, b, g = _make(80, 60, 48, dt, hip_device, bias=True)
        g = (10 ** (g * 4 - 2)) * torch.where(torch.arange(80, device=hip_device) % 3 == 0, -1.0, 1.0)
        g[::7] = 0
        _check(x, w, t, b, "none", g, f"weights {dt}")
        _check(x, w, t, b, "none", torch.zeros_like(g), f"zero weights {dt}")
        bad = g.clone()
        bad[3] = float("inf")
        got = _run(x, w, t, b, "none", bad)
        ref = _run(x, w, t, b, "none", g)
        rest = [i for i in range(80) if i != 3]
        assert torch.equal(got["dx"][rest], ref["dx"][rest]) and not torch.isfinite(got["dx"][3]).any()


def test_only_the_requested_gradients(hip_device):
    x, w, t, b, _ = _make(140, 333, 104, torch.bfloat16, hip_device, bias=True, pad=0.2)
    full = _run(x, w, t, b)
    for i, n in enumerate(("dx", "dw", "db")):
        args = [x, w, b]
        args[i] = args[i].detach().requires_grad_(True)
        (got,) = torch.autograd.grad(hip_linear_cross_entropy(args[0], args[1], t, args[2]), args[i])
        assert torch.equal(got, full[n]), n


def test_pieces_of_the_vocabulary(hip_device):
    """More classes than the backward's workspace holds for these tokens (256 MiB: 16384 of them here), and a float32 weight laid
    out in pieces; dx adds up over the pieces. Checked in float64 on the GPU."""
    for dt, N, V, D in ((torch.bfloat16, 8200, 40000, 64), (torch.float32, 2000, 50000, 1024)):
        x, w, t, b, _ = _make(N, V, D, dt, hip_device, seed=7, bias=True, pad=0.1)
        got = _run(x, w, t, b, "sum")
        keep = t != IGNORE
        xd, wd = torch.where(keep.unsqueeze(1), x.double(), 0), w.double()
        z = xd @ wd.t() + b.double()
        p = torch.softmax(z, 1)
        ti = torch.where(keep, t, 0)
        loss = torch.where(keep, torch.logsumexp(z, 1) - z.gather(1, ti.unsqueeze(1)).squeeze(1), 0).sum()
        del z
        p.scatter_add_(1, ti.unsqueeze(1), torch.full((N, 1), -1.0, device=hip_device, dtype=torch.float64))
        p *= keep.unsqueeze(1)
        big = float((xd.abs() @ wd[:512].abs().t()).max()) * 1.5  # of sum|x w|: other columns are alike
        # dz: half a step of bfloat16; in three planes 2^-24 of each operand and the two larger products left out 2^-24 each.
        # Its logits: sums over D, and at most 12 u where float32 goes as two float16 planes (each rest 2^-22, their product 2^-22)
        rel = (2.0**-8 if dt == torch.bfloat16 else 2.0**-22) + 4 * (D + 16) * O.U * big + (V / 16 + 64) * O.U
        step = O.half_step(dt)
        assert abs(float(got["loss"] - loss)) <= float(loss) * rel
        a = p.abs()
        for n, want, scale in (("dx", p @ wd, a @ wd.abs()), ("dw", p.t() @ xd, a.t() @ xd.abs()), ("db", p.sum(0), a.sum(0))):
            off = ((got[n].double() - want).abs() / ((rel + (V if n == "dx" else N) * O.U) * scale + step * want.abs() + 1e-30)).max()
            assert float(off) <= 1, f"{dt} {n}: {float(off):.3g} times the bound"


def test_second_order_matches_float64_autograd(hip_device):
    """A product with the gradients differentiated again, in float32. The restatement rounds each of its some hundred
    operations by 2^-24; the kernels' first gradients enter through nothing."""
    x, w, t, b, g = _make(30, 17, 24, torch.float32, hip_device, bias=True, pad=0.2)
    gen = torch.Generator().manual_seed(1)
    u, a, c = torch.randn(30, 24, generator=gen), torch.randn(17, 24, generator=gen), torch.randn(17, generator=gen)

    def second(op, x, w, b, g, u, a, c, reduction):
        x, w, b = (v.detach().requires_grad_(True) for v in (x, w, b))
        g = g.detach().requires_grad_(True)
        loss = op(x, w, b, reduction)
        first = torch.autograd.grad(loss, (x, w, b), g if reduction == "none" else None, create_graph=True)
        return torch.autograd.grad(first, (x, w, b) + ((g,) if reduction == "none" else ()), (u, a, c))

    def plain(x, w, b, reduction):
        return torch.nn.functional.cross_entropy(torch.nn.functional.linear(x, w, b), t.cpu(), reduction=reduction)

    for reduction in ("none", "mean", "sum"):
        got = second(lambda x, w, b, r: hip_linear_cross_entropy(x, w, t, b, reduction=r), x, w, b, g, *(v.to(hip_device) for v in (u, a, c)), reduction)
        want = second(plain, *(v.double().cpu() for v in (x, w, b, g, u, a, c)), reduction)
        for p, q in zip(got, want):
            assert float((p.double().cpu() - q).abs().max()) <= 1024 * O.U * float(q.abs().max())


def test_gradient_agrees_with_differences_of_the_loss(hip_device):
    """<gradient, direction> against central differences of the float64 loss (truncation about h^2 = 1e-10)."""
    x, w, t, b, g = _make(40, 33, 20, torch.float32, hip_device, bias=True, pad=0.1)
    got = _run(x, w, t, b, "none", g)
    want = O.linear_ce(x, w, b, t, IGNORE, "none", g)
    gen = torch.Generator().manual_seed(2)
    f = lambda x, w, b: (O.linear_ce(x, w, b, t, IGNORE, "none")["loss"][0] * g.double().cpu()).sum()  # noqa: E731
    args, h = [v.double().cpu() for v in (x, w, b)], 1e-5
    for i, n in enumerate(("dx", "dw", "db")):
        d = torch.randn(args[i].shape, generator=gen, dtype=torch.float64)
        hi, lo = list(args), list(args)
        hi[i], lo[i] = args[i] + h * d, args[i] - h * d
        num = (f(*hi) - f(*lo)) / (2 * h)
        assert abs(float((got[n].double().cpu() * d).sum() - num)) <= float((want[n][1] * d.abs()).sum()) + 1e-7


def test_side_streams_and_graph_replays(hip_device):
    sets = [_make(200, 900, 128, torch.bfloat16, hip_device, seed=s, bias=True, pad=0.1 + 0.5 * s)[:4] for s in (0, 1)]
    ref = [_run(x, w, t, b) for x, w, t, b in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    out = []
    for st, (x, w, t, b) in zip(streams, sets):
        with torch.cuda.stream(st):
            out.append(_run(x, w, t, b))
    torch.cuda.synchronize()
    for p, q in zip(out, ref):
        assert all(torch.equal(p[n], q[n]) for n in q)
    x, w, t, b = (v.clone() for v in sets[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _run(x, w, t, b)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _run(x, w, t, b)
    for k in (1, 0, 1):  # the number of kept rows changes from replay to replay
        for dst, src in zip((x, w, t, b), sets[k]):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(got[n], ref[k][n]) for n in ref[k]), f"replay of set {k}"
        _run(*sets[1 - k])


def test_refusals(hip_device):
    x, w, t, b, _ = _make(6, 9, 16, torch.float32, hip_device, bias=True)
    call = hip_linear_cross_entropy
    with pytest.raises(AssertionError, match="weight"):
        call(x, w[:, :8], t)
    with pytest.raises(AssertionError, match="dtype and device"):
        call(x, w.half(), t)
    with pytest.raises(AssertionError, match="bias"):
        call(x, w, t, b[:4])
    with pytest.raises(AssertionError, match="int32 or int64"):
        call(x, w, t.float())
    with pytest.raises(AssertionError, match="target must have shape"):
        call(x, w, t[:3])
    with pytest.raises(AssertionError, match="target must be on"):
        call(x, w, t.cpu())
    with pytest.raises(AssertionError, match="reduction"):
        call(x, w, t, reduction="median")
    with pytest.raises(AssertionError, match="dtype"):
        call(x.double(), w.double(), t)
