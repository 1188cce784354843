"""The token-side operators of a training step as timed cases: layer norm, embedding lookup, linear cross entropy.

Each case is one pass through a public entry point of `theria_amd.autograd` (`own` true), or the same mathematics in
elementary torch operations, in float32 whatever the inputs' type and rounded once at the end (`own` false). A case is
a dict of plain values:

  op      "norm"   layer norm over the last dimension: N rows of D
          "embed"  rows of a (V, D) table looked up by N ids, times a scale
          "loss"   cross entropy of the logits x W^T + b: N rows of D, V classes
  kind    "infer"  forward only, under no_grad
          "train"  forward and every gradient, as in a training step
          "second" norm only: forward, gradients kept differentiable, and the gradient of a product with them, as a
                   meta-gradient takes it
  dtype   of the inputs; wide: the norm's weight and bias are float32 beside 16-bit rows
  pad     share of the ids that are the padding id, of the targets that are ignored
  bias    loss only: the head has a bias
  each    loss only: one loss for each row (reduction "none") with a gradient of its own, instead of the mean
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
_EPS = 1e-5
_PADDING = 0
_IGNORED = -100


def _norm(name, kind, dtype, N, D, wide=False):
    c = {"op": "norm", "kind": kind, "dtype": dtype, "N": N, "D": D, "wide": wide}
    return {"name": name, **c} if name else c


def _embed(name, kind, dtype, N, V, D, pad=0.0):
    c = {"op": "embed", "kind": kind, "dtype": dtype, "N": N, "V": V, "D": D, "pad": pad}
    return {"name": name, **c} if name else c


def _loss(name, kind, dtype, N, V, D, pad=0.0, bias=False, each=False):
    c = {"op": "loss", "kind": kind, "dtype": dtype, "N": N, "V": V, "D": D, "pad": pad, "bias": bias, "each": each}
    return {"name": name, **c} if name else c


def listed():
    return [
        # the meta-learning classifier's norm (25 sequences of 64 tokens, width 64), differentiated twice: latency
        _norm("norm_maml_second_fp32", "second", "fp32", 1600, 64),
        # an ordinary layer of a training step
        _norm("norm_train_bf16", "train", "bf16", 8192, 4096),
        # odd width and row count, float32 parameters beside 16-bit rows, as under mixed precision
        _norm("norm_train_odd_fp16", "train", "fp16", 4999, 1001, wide=True),
        # the largest activation, float32
        _norm("norm_train_large_fp32", "train", "fp32", 65536, 2048),
        # one step of generation: a row for each of 64 sequences
        _embed("embed_step_bf16", "infer", "bf16", 64, 128000, 4096),
        # the classifier's vocabulary of 32: every row of the table gathers hundreds of tokens
        _embed("embed_train_small_vocab_fp32", "train", "fp32", 25600, 32, 64),
        # an ordinary training batch with padding
        _embed("embed_train_bf16", "train", "bf16", 16384, 32000, 2048, pad=0.2),
        # the largest table
        _embed("embed_train_large_bf16", "train", "bf16", 32768, 128000, 4096),
        # the classifier's head: 25 sequences, five classes, a bias
        _loss("loss_head_fp32", "train", "fp32", 25, 5, 64, bias=True),
        # scoring a few sequences' next tokens: bound by reading the weight
        _loss("loss_score_bf16", "infer", "bf16", 48, 128000, 4096, each=True),
        # odd sizes, a third of the tokens ignored, a weight of its own for each of the others
        _loss("loss_train_odd_fp16", "train", "fp16", 3001, 10007, 520, pad=0.33, bias=True, each=True),
        # the largest vocabulary at training size
        _loss("loss_train_large_bf16", "train", "bf16", 8192, 128000, 4096),
    ]


_LARGEST = 6 * 8192 * 128000 * 4096  # flops of loss_train_large_bf16


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width: any size, a multiple of 8 or a multiple of 64."""
    D, step = _log_int(rng, lo, hi), rng.choice([1, 8, 64, 64])
    return max(1, D if D < step else D // step * step)


def draw(rng):
    """One more case of the same ranges, costing at most what the largest listed case does."""
    while True:
        op = rng.choice(["norm", "embed", "loss"])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        N = _log_int(rng, 1, 131072)
        pad = rng.choice([0.0, 0.0, 0.1, 0.5])
        if op == "norm":
            D = _width(rng, 1, 16384)
            if N * D <= 2 ** 27:
                return _norm(None, rng.choice(["infer", "train", "train", "second"]), dtype, N, D,
                             wide=dtype != "fp32" and rng.random() < 0.5)
        elif op == "embed":
            V, D = _log_int(rng, 2, 262144), _width(rng, 1, 8192)
            if N * D <= 2 ** 27 and V * D <= 2 ** 29:
                return _embed(None, rng.choice(["infer", "train", "train"]), dtype, N, V, D, pad)
        else:
            V, D = _log_int(rng, 2, 262144), _width(rng, 8, 8192)
            if 6 * N * V * D <= _LARGEST // 4 and N * V <= 2 ** 30 and V * D <= 2 ** 29 and N * D <= 2 ** 27:
                kind = rng.choice(["infer", "train", "train"])
                return _loss(None, kind, dtype, N, V, D, pad, bias=rng.random() < 0.4, each=rng.random() < 0.3)


def _ignored(c):
    return int(c["N"] * c["pad"])


def work(case):
    c, es = case, _SIZE[case["dtype"]]
    N, D, kind = c["N"], c["D"], c["kind"]
    if c["op"] == "norm":
        ps = 4 if c["wide"] else es
        # rows: x, y; with gradients also g, dx; second order also the cotangent of dx and the gradients of x and g
        rows = {"infer": 2, "train": 4, "second": 7}[kind]
        params = {"infer": 2, "train": 4, "second": 7}[kind]
        return {"bytes": rows * N * D * es + params * D * ps, "flops": {"infer": 8, "train": 24, "second": 60}[kind] * N * D}
    if c["op"] == "embed":
        # ids, the rows read (at most every row once) and written; the gradient's rows read and the table's written
        nbytes = 8 * N + min(N, c["V"]) * D * es + N * D * es
        if kind == "train":
            nbytes += N * D * es + c["V"] * D * es
        return {"bytes": nbytes, "flops": N * D * (2 if kind == "train" else 1)}
    kept, V = N - _ignored(c), c["V"]
    once = 8 * N + kept * D * es + V * D * es + (V * es if c["bias"] else 0) + 4 * (N if c["each"] else 1)
    twice = N * D * es + V * D * es + (V * es if c["bias"] else 0) + 4 * (N if c["each"] else 1)
    return {"bytes": once + (twice if kind == "train" else 0), "flops": (6 if kind == "train" else 2) * kept * V * D}


def _token_ids(gen, N, V, dev):
    """Ids whose frequencies fall as one over their rank, the ranks spread over the table at random."""
    rank = (torch.rand(N, generator=gen, device=dev, dtype=torch.float64) * math.log(V + 1)).exp().long() - 1
    return torch.randperm(V, generator=gen, device=dev)[rank.clamp(0, V - 1)]


def _inputs(c, seed, dev="cuda:0"):
    """The case's tensors from the seed alone."""
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt, N, D = _DTYPES[c["dtype"]], c["N"], c["D"]

    def rand(*shape, std=1.0, mean=0.0, dtype=dt):
        t = torch.empty(*shape, device=dev, dtype=dtype if dtype == torch.float32 or math.prod(shape) > 2 ** 28 else torch.float32)
        return t.normal_(mean, std, generator=gen).to(dtype)

    if c["op"] == "norm":
        pt = torch.float32 if c["wide"] else dt
        # a residual stream: an offset and a spread of its own for each row, a few strong channels
        x = rand(N, D, dtype=torch.float32) * (1 + rand(N, 1, std=0.3, dtype=torch.float32)) + rand(N, 1, std=0.5, dtype=torch.float32)
        x[:, ::97] *= 8
        s = {"x": x.to(dt), "w": rand(D, std=0.1, mean=1.0, dtype=pt), "b": rand(D, std=0.1, dtype=pt)}
        if c["kind"] != "infer":
            s["g"] = rand(N, D)
        if c["kind"] == "second":
            s.update(u=rand(N, D), a=rand(D, dtype=pt), c=rand(D, dtype=pt))
        return s
    pads = torch.randperm(N, generator=gen, device=dev)[:_ignored(c)]
    if c["op"] == "embed":
        ids = _token_ids(gen, N, c["V"], dev)
        ids[pads] = _PADDING
        s = {"ids": ids, "w": rand(c["V"], D, std=0.02)}
        if c["kind"] == "train":
            s["g"] = rand(N, D)
        return s
    # a head with rows of unit-sized products, and rows that lean towards their target's row, as after training
    target = _token_ids(gen, N, c["V"], dev)
    w = rand(c["V"], D, std=1 / math.sqrt(D))
    s = {"x": (rand(N, D, dtype=torch.float32) + 6.0 * w[target].float()).to(dt), "w": w}
    target[pads] = _IGNORED
    s["t"] = target
    if c["bias"]:
        s["b"] = rand(c["V"], std=0.1)
    if c["each"]:
        s["g"] = torch.rand(N, generator=gen, device=dev)
    return s


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if case["kind"] != "infer":
        for n in ("x", "w", "b"):
            if n in state:
                state[n].requires_grad_(True)
        if case["kind"] == "second":
            state["g"].requires_grad_(True)
    return state


def _scale(c):
    return math.sqrt(c["D"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from theria_amd.autograd import hip_embedding, hip_layer_norm, hip_linear_cross_entropy

    c = s["case"]
    kind = c["kind"]
    with torch.set_grad_enabled(kind != "infer"):
        if c["op"] == "norm":
            y = hip_layer_norm(s["x"], s["w"], s["b"], eps=_EPS)
            if kind == "infer":
                return y
            first = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["g"], create_graph=kind == "second")
            if kind == "train":
                return (y, *first)
            second = torch.autograd.grad(first, (s["x"], s["w"], s["g"]), (s["u"], s["a"], s["c"]))
            return (y.detach(), *(t.detach() for t in first), *second)
        if c["op"] == "embed":
            y = hip_embedding(s["ids"], s["w"], scale=_scale(c), padding_idx=_PADDING)
            return y if kind == "infer" else (y, *torch.autograd.grad(y, s["w"], s["g"]))
        loss = hip_linear_cross_entropy(s["x"], s["w"], s["t"], s.get("b"), ignore_index=_IGNORED,
                                        reduction="none" if c["each"] else "mean")
        if kind == "infer":
            return loss
        wrt = [s[n] for n in ("x", "w", "b") if n in s]
        return (loss, *torch.autograd.grad(loss, wrt, s["g"] if c["each"] else None))


# ---------------------------------------------------------------------------------------------------
# plain form
# ---------------------------------------------------------------------------------------------------
@torch.no_grad()
def _run_plain(s):
    return {"norm": _norm_plain, "embed": _embed_plain, "loss": _loss_plain}[s["case"]["op"]](s)


def _norm_plain(s):
    kind, dt, pt = s["case"]["kind"], s["x"].dtype, s["w"].dtype
    x, w, b = s["x"].float(), s["w"].float(), s["b"].float()
    xc = x - x.mean(1, keepdim=True)
    r = 1 / torch.sqrt((xc * xc).mean(1, keepdim=True) + _EPS)
    xh = xc * r
    y = (xh * w + b).to(dt)
    if kind == "infer":
        return y
    g = s["g"].float()
    gw = g * w

    def along(t):  # the derivative of the normalised row, which is symmetric
        return r * (t - t.mean(1, keepdim=True) - xh * (t * xh).mean(1, keepdim=True))

    dx = along(gw)
    first = (dx.to(dt), (g * xh).sum(0).to(pt), g.sum(0).to(pt))
    if kind == "train":
        return (y, *first)
    u, a, c = s["u"].float(), s["a"].float(), s["c"].float()
    pu = along(u)
    h = a * g - r * (u * (gw * xh).mean(1, keepdim=True) + gw * (u * xh).mean(1, keepdim=True))
    gx = along(h) - r * xh * (u * dx).mean(1, keepdim=True)
    return (y, *first, gx.to(dt), (g * pu).sum(0).to(pt), (w * pu + a * xh + c).to(dt))


def _embed_plain(s):
    c, dt = s["case"], s["w"].dtype
    y = (s["w"][s["ids"]].float() * _scale(c)).to(dt)
    if c["kind"] == "infer":
        return y
    g = s["g"].float() * (s["ids"] != _PADDING).unsqueeze(1)
    dw = torch.zeros(c["V"], c["D"], device=g.device).index_add_(0, s["ids"], g)
    return y, (dw * _scale(c)).to(dt)


def _loss_plain(s):
    c, dt = s["case"], s["x"].dtype
    kept = s["t"] != _IGNORED
    t = torch.where(kept, s["t"], 0).unsqueeze(1)
    x, w = torch.where(kept.unsqueeze(1), s["x"].float(), 0.0), s["w"].float()
    z = x @ w.t()
    if "b" in s:
        z += s["b"].float()
    top = z.amax(1, keepdim=True)
    at = z.gather(1, t) - top
    z -= top
    z.exp_()
    total = z.sum(1, keepdim=True)
    each = torch.where(kept, (torch.log(total) - at).squeeze(1), 0.0)
    share = kept / kept.sum()
    loss = each if c["each"] else each.sum() / kept.sum()
    if c["kind"] == "infer":
        return loss
    up = s["g"] * kept if c["each"] else share
    z /= total
    z.scatter_add_(1, t, torch.full_like(at, -1.0))
    z *= up.unsqueeze(1)
    outs = (loss, (z @ w).to(dt), (z.t() @ x).to(dt))
    return (*outs, z.sum(0).to(dt)) if "b" in s else outs


# ---------------------------------------------------------------------------------------------------
# the same outputs in float64, from the definitions
# ---------------------------------------------------------------------------------------------------
def exact(case, seed):
    return {"norm": _norm_exact, "embed": _embed_exact, "loss": _loss_exact}[case["op"]](case, _inputs(case, seed))


def _norm_exact(c, s):
    """Differentiated by autograd, once or twice."""
    x, w, b = (s[n].double().requires_grad_(c["kind"] != "infer") for n in ("x", "w", "b"))
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    y = (x - mean) / (var + _EPS).sqrt() * w + b
    if c["kind"] == "infer":
        return y
    g = s["g"].double().requires_grad_(True)
    first = torch.autograd.grad(y, (x, w, b), g, create_graph=c["kind"] == "second")
    if c["kind"] == "train":
        return (y.detach(), *first)
    second = torch.autograd.grad(first, (x, w, g), [s[n].double() for n in ("u", "a", "c")])
    return (y.detach(), *(t.detach() for t in first), *second)


def _embed_exact(c, s):
    y = torch.index_select(s["w"], 0, s["ids"]).double() * _scale(c)
    if c["kind"] == "infer":
        return y
    ids, order = torch.sort(s["ids"], stable=True)
    live = ids != _PADDING
    dw = torch.zeros(c["V"], c["D"], dtype=torch.float64, device=y.device)
    for i in range(0, c["N"], 8192):  # a piece of the sorted tokens at a time
        k = live[i:i + 8192]
        dw.index_add_(0, ids[i:i + 8192][k], s["g"][order[i:i + 8192][k]].double(), alpha=_scale(c))
    return y, dw


def _loss_exact(c, s):
    N, rows = c["N"], max(1, 2 ** 27 // c["V"])
    w = s["w"].double()
    b = s["b"].double() if "b" in s else 0.0
    count = (s["t"] != _IGNORED).sum().double()
    each = torch.zeros(N, dtype=torch.float64, device=w.device)
    dx = torch.zeros(N, c["D"], dtype=torch.float64, device=w.device)
    dw, db = torch.zeros_like(w), torch.zeros(c["V"], dtype=torch.float64, device=w.device)
    for i in range(0, N, rows):  # a few rows' logits at a time
        at = torch.nonzero(s["t"][i:i + rows] != _IGNORED).squeeze(1) + i
        if not at.numel():
            continue
        x, t = s["x"][at].double(), s["t"][at]
        logp = torch.log_softmax(torch.nn.functional.linear(x, w) + b, dim=1)
        n = torch.arange(at.numel(), device=w.device)
        each[at] = -logp[n, t]
        if c["kind"] == "infer":
            continue
        d = logp.exp_()
        d[n, t] -= 1
        d *= (s["g"][at].double() if c["each"] else 1 / count.expand(at.numel())).unsqueeze(1)
        dx[at] = d @ w
        dw.addmm_(d.t(), x)
        db += d.sum(0)
    loss = each if c["each"] else each.sum() / count
    if c["kind"] == "infer":
        return loss
    return (loss, dx, dw, db) if "b" in s else (loss, dx, dw)
