"""GPU: steps of gated_linear that a graph cannot capture are refused in the forward pass."""
import gc

import pytest
import torch

pytestmark = pytest.mark.gpu

# what a program makes of its leaf before the call
FORMS = {"cast": lambda w: w.to(torch.bfloat16), "slice": lambda w: w.to(torch.bfloat16)[:, :64],
         "joined": lambda w: torch.cat([w[:64].to(torch.bfloat16), w[64:].to(torch.bfloat16)]),
         "scaled": lambda w: (w * 0.5).to(torch.bfloat16), "view": lambda w: w.to(torch.bfloat16).view(-1).view(128, -1)}


def _data():
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")
    return rand(64, 64).to(torch.bfloat16), (rand(128, 64) * 0.1).requires_grad_(), rand(64, 64).to(torch.bfloat16)


def _refused(forward, match):
    """The forward pass alone: its backward is not reached."""
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match=match), torch.cuda.graph(graph):
        forward()
    del graph
    gc.collect()  # (the exception's frames hold what the forward made)


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("what", ["weight", "input", "bias"])
def test_a_leaf_behind_other_operations(form, what):
    """The leaf's graph of an eager step lives: no capture of what is made of the leaf, as a weight, as an input
    or (its first column) as a bias.  Without it the step is captured."""
    from vllm_xpu_kernels import ops
    x, leaf, d = _data()
    w = leaf.detach().to(torch.bfloat16)

    def forward():
        t = FORMS[form](leaf)
        if what == "weight":
            return ops.gated_linear(x, t)
        if what == "input":
            return ops.gated_linear(t[:64], w)
        return ops.gated_linear(x, w, t[:, 0].contiguous())

    run = lambda: torch.autograd.grad(forward(), leaf, d)[0]
    want = run()
    lives = forward()
    _refused(forward, "same leaves")
    del lives
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(run(), want)


def test_an_input_made_before_the_capture():
    """Its graph was made on the default stream, its leaf dead or alive: refused; a detached one is captured."""
    from vllm_xpu_kernels import ops
    x, leaf, d = _data()
    w = leaf.detach().to(torch.bfloat16).requires_grad_()
    made = (x.requires_grad_() * 2.0)
    _refused(lambda: ops.gated_linear(made, w), "default stream")
    made = made.detach()
    want = torch.autograd.grad(ops.gated_linear(made, w), w, d)[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(ops.gated_linear(made, w), w, d)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_eager_steps_and_steps_without_gradients_are_not_refused():
    """Beside a living graph: eager calls on another stream, and captured calls that need no gradient."""
    from vllm_xpu_kernels import ops
    x, leaf, d = _data()
    lives = ops.gated_linear(x, leaf.to(torch.bfloat16))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.gated_linear(x, leaf.to(torch.bfloat16))
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, lives)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        got = ops.gated_linear(x, leaf.to(torch.bfloat16))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, ops.linear(x, leaf.detach().to(torch.bfloat16), activation="silu_and_mul"))
