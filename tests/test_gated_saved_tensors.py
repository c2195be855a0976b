"""gated_linear under hooks of saved tensors: activation checkpointing, offloading."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint


def test_an_unpack_hook_can_record_a_graph():
    """As a checkpoint's does, whose hook runs the forward pass again with gradients."""
    from vllm_xpu_kernels import ops
    seen = []

    def unpack(t):
        with torch.enable_grad():
            seen.append((torch.ones(2, requires_grad=True) * 2).requires_grad)
        return t

    x, w = (torch.zeros(s, dtype=torch.bfloat16, device="meta").requires_grad_() for s in ((6, 64), (32, 64)))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        out = ops.gated_linear(x, w)
    out.backward(torch.zeros(6, 16, dtype=torch.bfloat16, device="meta"))
    assert len(seen) >= 3 and all(seen)


def _block():
    g = torch.Generator(device="cuda")
    g.manual_seed(7)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, w13, b, w2 = rand(70, 128).to(torch.bfloat16), rand(256, 128) * 0.1, rand(256), rand(128, 128) * 0.1
    return [t.requires_grad_() for t in (x, w13, b, w2)], rand(70, 128).to(torch.bfloat16)


def _feed_forward(x, w13, b, w2):
    from vllm_xpu_kernels import ops
    return torch.nn.functional.linear(ops.gated_linear(x, w13.to(x.dtype), b), w2.to(x.dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("layers", [1, 3])
def test_checkpointed(layers):
    """Blocks whose activations are made again in the backward pass: the bits of the plain step."""
    leaves, d = _block()

    def step(run):
        y = leaves[0]
        for _ in range(layers):
            y = run(y)
        return torch.autograd.grad(y, leaves, d)

    want = step(lambda y: _feed_forward(y, *leaves[1:]))
    got = step(lambda y: checkpoint(_feed_forward, y, *leaves[1:], use_reentrant=False))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_checkpointed_by_a_nested_backward_pass():
    """use_reentrant: the first forward pass records nothing, and the second one is the plain step's."""
    leaves, d = _block()
    _feed_forward(*leaves).backward(d)
    want = [t.grad for t in leaves]
    for t in leaves:
        t.grad = None
    checkpoint(_feed_forward, *leaves, use_reentrant=True).backward(d)
    assert all(torch.equal(t.grad, w) for t, w in zip(leaves, want))


@pytest.mark.gpu
def test_offloaded():
    leaves, d = _block()
    want = torch.autograd.grad(_feed_forward(*leaves), leaves, d)
    with torch.autograd.graph.save_on_cpu():
        out = _feed_forward(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, d), want))
