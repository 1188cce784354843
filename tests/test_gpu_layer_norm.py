"""hip_layer_norm on the GPU against float64 formulas (tests/token_oracle.py): forward, backward, double backward and third
order, over every team size, strides, odd widths, empty inputs, streams and graph replays."""

import pytest
import torch

import token_oracle as O
from theria_amd.autograd import hip_layer_norm

pytestmark = pytest.mark.gpu

EPS = 1e-5
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
# every team, 8 lanes to a workgroup of 1024, on and beside the borders; whole and partly filled last vectors
SHAPES = [(1, 1), (3, 7), (5, 16), (17, 64), (1030, 64), (4, 65), (33, 128), (37, 31), (50, 32), (6, 33), (129, 63), (2, 136), (4, 255), (9, 256), (3, 257), (64, 512), (5, 1000),
          (7, 1001), (3, 1024), (2, 2048), (700, 2048), (3, 4096), (2, 4104), (2, 5001), (2, 8192), (2, 16383), (1, 16384), (2100, 8)]


def _make(shape, dt, pt, dev, seed=0, weight=True, bias=True):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    D = shape[-1]
    x = (r(*shape) * 1.5 + r(*shape[:-1], 1)).to(dt).to(dev)
    w = (1 + 0.2 * r(D)).to(pt).to(dev) if weight else None
    b = (0.2 * r(D)).to(pt).to(dev) if bias else None
    g, u = r(*shape).to(dt).to(dev), r(*shape).to(dt).to(dev)
    return x, w, b, g, u, r(D).to(pt).to(dev), r(D).to(pt).to(dev)


def _leaves(*ts):
    return [None if t is None else t.detach().requires_grad_(True) for t in ts]


def _first(x, w, b, g, create=False):
    y = hip_layer_norm(x, w, b, eps=EPS)
    wrt = [t for t in (x, w, b) if t is not None]
    return y, torch.autograd.grad(y, wrt, g, create_graph=create)


def _check_all(x, w, b, g, u, a, c, what):
    pt = (w if w is not None else b).dtype if (w is not None or b is not None) else x.dtype
    xl, wl, bl, gl = _leaves(x, w, b, g)
    y, first = _first(xl, wl, bl, gl, create=True)
    O.check(y, *O.norm_forward(x, w, b, EPS), f"{what} y")
    (dx, dw, db) = O.norm_backward(x, w, g, EPS, pt)
    want = [dx] + ([dw] if w is not None else []) + ([db] if b is not None else [])
    names = ["dx"] + (["dw"] if w is not None else []) + (["db"] if b is not None else [])
    for n, got, (v, t) in zip(names, first, want):
        O.check(got, v, t, f"{what} {n}")
    # the same without a graph to keep
    with torch.no_grad():
        y0 = hip_layer_norm(x, w, b, eps=EPS)
    assert torch.equal(y0, y.detach())
    for got, again in zip(first, _first(xl, wl, bl, g)[1]):
        assert torch.equal(got.detach(), again), f"{what}: gradients differ with and without create_graph"
    cots = [u] + ([a] if w is not None else []) + ([c] if b is not None else [])
    wrt = [xl] + ([wl] if w is not None else []) + [gl]
    second = torch.autograd.grad(first, wrt, cots)
    gx, gw, gg = O.norm_second(x, w, g, u, a if w is not None else None, c if b is not None else None, EPS, pt)
    for n, got, (v, t) in zip(["gx"] + (["gw"] if w is not None else []) + ["gg"], second, [gx] + ([gw] if w is not None else []) + [gg]):
        O.check(got, v, t, f"{what} {n}")


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_every_order_matches_the_formulas(dt, shape, hip_device):
    x, w, b, g, u, a, c = _make(shape, dt, dt, hip_device, seed=shape[1])
    _check_all(x, w, b, g, u, a, c, f"{dt} {shape}")


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(17, 64), (3, 257), (64, 512), (2, 2048), (2, 16384)])
def test_float32_parameters_beside_16_bit_rows(dt, shape, hip_device):
    x, w, b, g, u, a, c = _make(shape, dt, torch.float32, hip_device, seed=3)
    _check_all(x, w, b, g, u, a, c, f"{dt} wide {shape}")


@pytest.mark.parametrize("dt,pt", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("shape", [(40000, 21), (9000, 203), (5000, 1500), (4200, 4101), (600, 8195)])
def test_many_rows_of_odd_widths(dt, pt, shape, hip_device):
    """Teams of every size that walk many rows, the last vector of each partly filled."""
    x, w, b, g, u, a, c = _make(shape, dt, pt, hip_device, seed=shape[1])
    _check_all(x, w, b, g, u, a, c, f"{dt} {shape}")


@pytest.mark.parametrize("weight,bias", [(True, False), (False, True), (False, False)])
def test_parameters_are_optional(weight, bias, hip_device):
    x, w, b, g, u, a, c = _make((12, 96), torch.bfloat16, torch.bfloat16, hip_device, weight=weight, bias=bias)
    _check_all(x, w, b, g, u, a, c, f"weight={weight} bias={bias}")


def test_leading_dimensions_strides_and_misaligned_rows(hip_device):
    for dt in DTYPES:
        base, w, b, g, *_ = _make((4, 6, 96), dt, dt, hip_device, seed=5)
        flat = torch.zeros(4 * 6 * 96 + 1, dtype=dt, device=hip_device)
        flat[1:] = base.reshape(-1)
        wide = torch.zeros(4, 6, 100, dtype=dt, device=hip_device)
        wide[..., :96] = base
        views = {
            "3-d": base,
            "one element off 16 bytes": flat[1:].view(4, 6, 96),
            "rows apart": wide[..., :96],
            "transposed": base.transpose(-1, -2).contiguous().transpose(-1, -2),
            "batches swapped": base.transpose(0, 1).contiguous().transpose(0, 1),
            "broadcast row": base[:1, :1].expand(4, 6, 96),
        }
        for name, x in views.items():
            print(f"[strides] {dt} {name}", flush=True)
            xl, wl, bl = _leaves(x, w, b)
            y, first = _first(xl, wl, bl, g)
            O.check(y, *O.norm_forward(x, w, b, EPS), f"{name} y")
            for n, got, (v, t) in zip(("dx", "dw", "db"), first, O.norm_backward(x, w, g, EPS, dt)):
                O.check(got, v, t, f"{name} {n}")
        # gradients that arrive with strides of their own
        xl, wl, bl = _leaves(base, w, b)
        for gv in (g[:1, :1].expand(4, 6, 96), g.transpose(-1, -2).contiguous().transpose(-1, -2), wide[..., 1:97]):
            for n, got, (v, t) in zip(("dx", "dw", "db"), _first(xl, wl, bl, gv)[1], O.norm_backward(base, w, gv, EPS, dt)):
                O.check(got, v, t, f"strided gradient {n}")


def test_one_row_as_a_vector_and_no_rows(hip_device):
    x, w, b, g, *_ = _make((40,), torch.float32, torch.float32, hip_device)
    O.check(hip_layer_norm(x, w, b, eps=EPS), *O.norm_forward(x, w, b, EPS), "vector")
    xl, wl, bl = _leaves(torch.empty(0, 5, 40, device=hip_device), w, b)
    y = hip_layer_norm(xl, wl, bl)
    assert y.shape == (0, 5, 40)
    gl = torch.empty(0, 5, 40, device=hip_device, requires_grad=True)
    dx, dw, db = torch.autograd.grad(y, (xl, wl, bl), gl, create_graph=True)
    assert dx.shape == (0, 5, 40) and not dw.any() and not db.any()
    gx, gw = torch.autograd.grad((dx, dw, db), (xl, wl), (dx, w, b), allow_unused=True)
    assert gx.shape == (0, 5, 40) and not gw.any()


def test_forward_in_several_launches(hip_device):
    """More rows than a launch takes (2^21)."""
    rows = 2**21 + 3
    x, w, b, g, *_ = _make((rows, 2), torch.float32, torch.float32, hip_device, seed=9)
    xl, wl, bl = _leaves(x, w, b)
    y, first = _first(xl, wl, bl, g)
    O.check(y, *O.norm_forward(x, w, b, EPS), "y")
    for n, got, (v, t) in zip(("dx", "dw", "db"), first, O.norm_backward(x, w, g, EPS, torch.float32)):
        O.check(got, v, t, n)


def test_constant_rows_and_values_far_from_zero(hip_device):
    """A row without variance is all bias; a row around 1000 keeps its variance (no sum of squares)."""
    x = torch.full((3, 130), 7.0, device=hip_device)
    w, b = torch.rand(130, device=hip_device), torch.rand(130, device=hip_device)
    assert torch.equal(hip_layer_norm(x, w, b), b.expand(3, 130))
    far = (1000 + torch.randn(5, 130, generator=torch.Generator().manual_seed(0))).to(hip_device)
    O.check(hip_layer_norm(far, w, b, eps=EPS), *O.norm_forward(far, w, b, EPS), "far rows")


def test_non_finite_rows_stay_in_their_rows(hip_device):
    for bad in (float("nan"), float("inf")):
        x, w, b, g, *_ = _make((9, 300), torch.float32, torch.float32, hip_device)
        clean = x.clone()
        x[4, 17] = bad
        xl, wl, bl = _leaves(x, w, b)
        y, (dx, dw, db) = _first(xl, wl, bl, g)
        others = [i for i in range(9) if i != 4]
        cl, _, _ = _leaves(clean, w, b)
        y0, (dx0, _, db0) = _first(cl, wl, bl, g)
        assert torch.equal(y[others], y0[others]) and torch.equal(dx[others], dx0[others]) and torch.equal(db, db0)
        assert torch.isnan(y[4]).all() and torch.isnan(dx[4]).all() and torch.isnan(dw).all()


def test_gradients_agree_with_differences_of_the_formula(hip_device):
    """<gradient, direction> against central differences of the float64 forward: h = 1e-5 leaves about h^2 of truncation."""
    x, w, b, g, u, a, c = _make((6, 70), torch.float32, torch.float32, hip_device, seed=11)
    xl, wl, bl = _leaves(x, w, b)
    grads = _first(xl, wl, bl, g)[1]
    h = 1e-5
    f = lambda x, w, b: (O.norm_forward(x, w, b, EPS)[0] * g.double().cpu()).sum()  # noqa: E731
    args = [t.double().cpu() for t in (x, w, b)]
    for i, (grad, d) in enumerate(zip(grads, (u, a, c))):
        d = d.double().cpu()
        up, dn = list(args), list(args)
        up[i], dn[i] = args[i] + h * d, args[i] - h * d
        num = (f(*up) - f(*dn)) / (2 * h)
        tol = [t for _, t in O.norm_backward(x, w, g, EPS, torch.float32)][i]
        bound = (tol * d.abs()).sum() + 1e-7 * (grad.double().cpu() * d).abs().sum() + 1e-8
        assert abs(float((grad.double().cpu() * d).sum() - num)) <= float(bound)


def test_third_order_through_the_restatement(hip_device):
    """The gradient of a gradient of a gradient, against float64 autograd on the CPU. Its bound: the same float32 formulas'
    own rounding, 2^-24 times the operations of three derivatives over rows of 24 (some thousands), relative to the
    largest element."""
    x, w, b, g, u, *_ = _make((4, 24), torch.float32, torch.float32, hip_device, seed=2)

    def third(x, w, b, g, u, op):
        x, w, b = _leaves(x, w, b)
        dx, dw, db = torch.autograd.grad(op(x, w, b), (x, w, b), g, create_graph=True)
        s = (dx * u).sum() + (dw * dw).sum() + db.sum()
        (hx, hw) = torch.autograd.grad(s, (x, w), create_graph=True)
        return torch.autograd.grad((hx * u).sum() + (hw * hw).sum(), (x, w))

    def plain(x, w, b):
        v, m = torch.var_mean(x, -1, correction=0, keepdim=True)
        return (x - m) / torch.sqrt(v + EPS) * w + b

    got = third(x, w, b, g, u, lambda *t: hip_layer_norm(*t, eps=EPS))
    want = third(*(t.double().cpu() for t in (x, w, b, g, u)), plain)
    for a, e in zip(got, want):
        assert float((a.double().cpu() - e).abs().max()) <= 4096 * O.U * float(e.abs().max())


def test_only_the_requested_gradients(hip_device):
    x, w, b, g, u, a, c = _make((50, 200), torch.bfloat16, torch.bfloat16, hip_device)
    xl, wl, bl = _leaves(x, w, b)
    full = _first(xl, wl, bl, g)[1]
    assert torch.equal(torch.autograd.grad(hip_layer_norm(xl, w, b, eps=EPS), xl, g)[0], full[0])
    assert torch.equal(torch.autograd.grad(hip_layer_norm(x, wl, b, eps=EPS), wl, g)[0], full[1])
    assert torch.equal(torch.autograd.grad(hip_layer_norm(x, w, bl, eps=EPS), bl, g)[0], full[2])
    # one cotangent at a time through the double backward
    gl = g.clone().requires_grad_(True)
    _, first = _first(xl, wl, bl, gl, create=True)
    for i, (cot, zero) in enumerate(((u, (u, None, None)), (a, (None, a, None)), (c, (None, None, c)))):
        (gg,) = torch.autograd.grad(first[i], gl, cot, retain_graph=True)
        O.check(gg, *O.norm_second(x, w, g, *zero, EPS, torch.bfloat16)[2], f"cotangent {i}")


def test_side_streams_and_two_calls_at_once(hip_device):
    sets = [_make((257, 1000), torch.bfloat16, torch.bfloat16, hip_device, seed=s) for s in (0, 1)]
    ref = [_first(*_leaves(x, w, b), g) for x, w, b, g, *_ in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(3):
        out = []
        for st, (x, w, b, g, *_r) in zip(streams, sets):
            with torch.cuda.stream(st):
                out.append(_first(*_leaves(x, w, b), g))
        torch.cuda.synchronize()
        for (y, gr), (y0, gr0) in zip(out, ref):
            assert torch.equal(y, y0) and all(torch.equal(p, q) for p, q in zip(gr, gr0))


def test_graph_replays_equal_eager(hip_device):
    """Forward, gradients and second order captured together; replays with eager calls in between, on changing inputs."""
    x, w, b, g, u, a, c = _make((130, 320), torch.float32, torch.float32, hip_device)
    xl, wl, bl = _leaves(x, w, b)
    gl = g.clone().requires_grad_(True)

    def step():
        y, first = _first(xl, wl, bl, gl, create=True)
        return [y.detach(), *(t.detach() for t in first), *torch.autograd.grad(first, (xl, wl, gl), (u, a, c))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        with torch.no_grad():
            xl.copy_(x * (1 + 0.1 * i))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for p, q in zip(got, step()):
            assert torch.equal(p, q), f"replay {i}"


def test_refusals(hip_device):
    x = torch.zeros(4, 8, device=hip_device)
    w = torch.ones(8, device=hip_device)
    with pytest.raises(AssertionError, match="dtype"):
        hip_layer_norm(x.double())
    with pytest.raises(AssertionError, match="weight must have shape"):
        hip_layer_norm(x, torch.ones(7, device=hip_device))
    with pytest.raises(AssertionError, match="bias must be on"):
        hip_layer_norm(x, w, torch.ones(8))
    with pytest.raises(AssertionError, match="float32"):
        hip_layer_norm(x.half(), w.bfloat16())
    with pytest.raises(AssertionError, match="one dtype"):
        hip_layer_norm(x.half(), w.half(), w)
    with pytest.raises(AssertionError, match="1 to 16384"):
        hip_layer_norm(torch.zeros(1, 16385, device=hip_device))
    with pytest.raises(AssertionError, match="1 to 16384"):
        hip_layer_norm(torch.zeros(4, 0, device=hip_device))
    with pytest.raises(AssertionError, match="eps"):
        hip_layer_norm(x, w, eps=-1.0)
