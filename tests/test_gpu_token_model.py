"""The token-side operators together, as a training step uses them: MHAClassifier with ops="hip" against ops="torch"."""

import copy

import pytest
import torch

from theria_amd.autograd import hip_embedding, hip_layer_norm, hip_linear_cross_entropy, hip_sdpa
from theria_amd.maml import meta_loss_on_tasks
from theria_amd.models import MHAClassifier, MHAConfig
from theria_amd.tasks import sample_token_count_task

pytestmark = pytest.mark.gpu


def _flat(grads):
    return torch.cat([g.reshape(-1) for g in grads]).double()


def _pair(dev):
    torch.manual_seed(0)
    ref = MHAClassifier(MHAConfig(), backend="reference").to(dev)
    hip = copy.deepcopy(ref)
    hip.set_attention_backend("hip")
    hip.set_ops("hip")
    return ref, hip


def test_training_step_matches_the_reference_model(hip_device):
    """Loss and every parameter's gradient of a step. Both sides are float32 with some hundred roundings in a row between
    an embedding and the loss: 2^-24 times a thousand, relative to the whole gradient."""
    ref, hip = _pair(hip_device)
    gen = torch.Generator().manual_seed(1)
    tokens, y = torch.randint(0, 32, (40, 64), generator=gen).to(hip_device), torch.randint(0, 5, (40,), generator=gen).to(hip_device)
    l0, l1 = ref(tokens, y), hip(tokens, y)
    g0 = _flat(torch.autograd.grad(l0, list(ref.parameters())))
    g1 = _flat(torch.autograd.grad(l1, list(hip.parameters())))
    assert abs(float(l0) - float(l1)) <= 1000 * 2**-24 * abs(float(l0))
    assert float((g0 - g1).norm() / g0.norm()) <= 1000 * 2**-24
    assert abs(float(torch.nn.functional.cross_entropy(hip(tokens), y)) - float(l1)) <= 1000 * 2**-24 * abs(float(l1))


def test_full_maml_metagradient_through_the_hip_operators(hip_device):
    """Second order through embedding, norms and attention, at the bar the attention alone is held to (1e-5)."""
    ref, hip = _pair(hip_device)
    gen = torch.Generator().manual_seed(0)
    tasks = [sample_token_count_task(generator=gen, device=hip_device)[0] for _ in range(2)]

    def meta(model):
        loss = meta_loss_on_tasks(model, tasks, inner_lr=0.4, inner_steps=5)
        return _flat(torch.autograd.grad(loss, list(model.parameters())))

    a, b = meta(ref), meta(hip)
    assert float((a - b).norm() / a.norm()) < 1e-5


def test_one_attention_layer_in_bfloat16_end_to_end(hip_device):
    """Embedding, norm, attention, norm and loss in bfloat16, captured with its gradients and replayed."""
    gen = torch.Generator().manual_seed(3)
    V, D, H, B, T = 500, 128, 2, 3, 70
    r = lambda *s: (torch.randn(*s, generator=gen) * 0.1).bfloat16().to(hip_device).requires_grad_(True)  # noqa: E731
    table, qkv, head = r(V, D), r(3 * D, D), r(V, D)
    w1, w2 = (torch.ones(D, device=hip_device, dtype=torch.bfloat16, requires_grad=True) for _ in range(2))
    ids = torch.randint(0, V, (B, T), generator=gen).to(hip_device)
    target = torch.randint(0, V, (B, T), generator=gen).to(hip_device)
    target[:, -10:] = -100
    params = (table, qkv, head, w1, w2)

    def step():
        x = hip_embedding(ids, table, scale=D**0.5)
        q, k, v = (hip_layer_norm(x, w1) @ qkv.t()).view(B, T, 3, H, D // H).permute(2, 0, 3, 1, 4)
        x = x + hip_sdpa(q, k, v, causal=True).transpose(1, 2).reshape(B, T, D)
        loss = hip_linear_cross_entropy(hip_layer_norm(x, w2), head, target)
        return [loss.detach(), *torch.autograd.grad(loss, params)]

    eager = step()
    assert all(torch.isfinite(t).all() for t in eager)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, eager):
            assert torch.equal(a, b), f"replay {i}"
        step()


def _calls(dev):
    x, w = torch.randn(6, 16, device=dev), torch.randn(9, 16, device=dev)
    ids = torch.arange(6, device=dev)
    return x, w, [lambda x, w: hip_layer_norm(x, w[0]).sum(), lambda x, w: hip_embedding(ids, w).sum(), lambda x, w: hip_linear_cross_entropy(x, w, ids)]


def test_transforms_and_forward_mode_are_refused(hip_device):
    """Neither gives a wrong result: both raise."""
    import torch.autograd.forward_ad as fwAD

    x, w, calls = _calls(hip_device)
    for call in calls:
        with pytest.raises(AssertionError, match="torch.func"):
            torch.func.grad(lambda w: call(x, w))(w)
        with pytest.raises(AssertionError, match="torch.func"):
            torch.func.vmap(lambda w: call(x, w))(w.expand(2, 9, 16).contiguous())
        with fwAD.dual_level(), pytest.raises(RuntimeError):
            fwAD.unpack_dual(call(x, fwAD.make_dual(w, torch.ones_like(w)))).tangent.sum()


def test_inference_mode_and_no_grad_give_the_same(hip_device):
    x, w, calls = _calls(hip_device)
    for call in calls:
        ref = call(x, w.clone().requires_grad_(True))
        with torch.no_grad():
            assert torch.equal(call(x, w), ref.detach())
        with torch.inference_mode():
            assert torch.equal(call(x.clone(), w.clone()), ref.detach())


def test_inputs_changed_after_the_forward_are_noticed(hip_device):
    x, w, calls = _calls(hip_device)
    for call, changed in zip(calls[:1] + calls[2:], (x, w)):
        xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        a, b = xl * 1, wl * 1
        loss = call(a, b)
        (a if changed is x else b).add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_accumulated_gradients_and_checkpointing(hip_device):
    """backward() into .grad twice, with a tied table and head, directly and recomputed by torch's checkpointing."""
    from torch.utils.checkpoint import checkpoint

    gen = torch.Generator().manual_seed(5)
    table = torch.randn(50, 32, generator=gen).to(hip_device).requires_grad_(True)
    ids, t = torch.randint(0, 50, (70,), generator=gen).to(hip_device), torch.randint(0, 50, (70,), generator=gen).to(hip_device)
    body = lambda: hip_linear_cross_entropy(hip_layer_norm(hip_embedding(ids, table)), table, t)  # noqa: E731
    body().backward()
    once = table.grad.clone()
    body().backward()
    assert torch.equal(table.grad, 2 * once)
    table.grad = None
    checkpoint(lambda _: body(), torch.zeros(1, device=hip_device, requires_grad=True), use_reentrant=False).backward()
    assert torch.equal(table.grad, once)


def test_a_thread_of_its_own(hip_device):
    """Calls and their backward passes from two Python threads at once, on streams of their own."""
    import threading

    x, w, calls = _calls(hip_device)
    want = []
    for call in calls:
        wl = w.clone().requires_grad_(True)
        want.append(torch.autograd.grad(call(x, wl), wl)[0])
    torch.cuda.synchronize()
    wrong = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                for call, ref in zip(calls, want):
                    wl = w.clone().requires_grad_(True)
                    if not torch.equal(torch.autograd.grad(call(x, wl), wl)[0], ref):
                        wrong.append(call)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work) for _ in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong


def test_views_of_negated_values(hip_device):
    """The imaginary part of a conjugate is a view whose values stand in memory with the other sign."""
    gen = torch.Generator().manual_seed(3)
    part = lambda *shape: torch.complex(torch.zeros(shape), torch.randn(*shape, generator=gen)).to(hip_device).conj().imag  # noqa: E731
    x, w, b, g = part(6, 5), part(5), part(5), part(6, 5)
    assert x.is_neg() and not x.clone().is_neg()
    table, ids, targets = part(7, 5), torch.tensor([0, 6, 3], device=hip_device), torch.tensor([0, 6, 3, 3, 1, 2], device=hip_device)
    up = part(6)
    calls = (
        (lambda x, w, b: hip_layer_norm(x, w, b), (x, w, b), g),
        (lambda t: hip_embedding(ids, t), (table,), g[:3]),
        (lambda x, t: hip_linear_cross_entropy(x, t, targets, reduction="none"), (x, table), up),
    )
    for call, args, cot in calls:
        got = [call(*args)] + list(torch.autograd.grad(call(*(leaves := [a.detach().requires_grad_(True) for a in args])), leaves, cot))
        plain = [a.clone() for a in args]
        want = [call(*plain)] + list(torch.autograd.grad(call(*(leaves := [a.requires_grad_(True) for a in plain])), leaves, cot.clone()))
        for a, e in zip(got, want):
            assert torch.equal(a, e)


def test_forward_mode_is_refused_without_a_graph_too(hip_device):
    import torch.autograd.forward_ad as fwAD

    x, w, calls = _calls(hip_device)
    for call in calls:
        with torch.no_grad(), fwAD.dual_level(), pytest.raises(RuntimeError):
            fwAD.unpack_dual(call(x, fwAD.make_dual(w, torch.ones_like(w)))).tangent.sum()
