"""gated_linear_backward of a batch without rows: dx has no elements then, and so no address."""
import ctypes

import pytest
import torch

F32, BF16 = 0, 1


@pytest.mark.parametrize("dx", [None, 16])
def test_the_input_alone(dx):
    """No gradient is left to compute: nothing is read, written or launched."""
    from vllm_xpu_kernels import capi
    a = capi.GatedLinearBackwardArgs(dtype=BF16, dbias_dtype=F32, activation=5, M=0, N=64, K=256, ldx=256, weight=16,
                                     ldw=256, ldd=64, dx=dx, lddx=256, lddw=256)
    assert capi.lib.mi355moe_gated_linear_backward_workspace_size(ctypes.byref(a)) == 0
    assert capi.lib.mi355moe_gated_linear_backward(ctypes.byref(a), None, 0, None) == 0
    a.M = 1
    if dx is None:
        assert capi.lib.mi355moe_gated_linear_backward(ctypes.byref(a), None, 0, None) == -1
        assert b"no gradient is asked for" in capi.lib.mi355moe_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 64), (3, 0, 64), (0, 5, 64)])
@pytest.mark.parametrize("need", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (1, 0, 1), (0, 1, 1), (1, 1, 1)])
def test_any_gradients(shape, need):
    """Frozen weights and biases too: an empty gradient of the input, zeros of the others."""
    from vllm_xpu_kernels import ops
    x, w, b = (torch.ones(s, dtype=torch.bfloat16, device="cuda").requires_grad_(bool(n))
               for s, n in zip((shape, (32, 64), (32,)), need))
    out = ops.gated_linear(x, w, b)
    assert out.shape == shape[:-1] + (16,)
    out.backward(torch.zeros_like(out))
    for t, n in zip((x, w, b), need):
        assert (t.grad is not None) == bool(n)
        if n:
            assert t.grad.shape == t.shape and t.grad.dtype == t.dtype and bool((t.grad == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 64), (3, 0, 64), (0, 5, 64)])
def test_expanded_and_permuted_tensors(shape):
    """A sum's gradient is one number expanded: without rows no strides of it matter, nor those of an input."""
    from vllm_xpu_kernels import ops
    x, w = (torch.ones(s, dtype=torch.bfloat16, device="cuda").requires_grad_() for s in (shape, (32, 64)))
    ops.gated_linear(x, w).sum().backward()
    assert x.grad.shape == shape and bool((w.grad == 0).all())
    out = ops.gated_linear(x, w)
    turned = torch.ones(shape[:-1][::-1] + (16,), dtype=torch.bfloat16, device="cuda").transpose(0, len(shape) - 2)
    for d in (torch.ones(16, 2, dtype=torch.bfloat16, device="cuda").t()[0].expand(out.shape), turned):
        dx, dw = torch.autograd.grad(out, [x, w], d, retain_graph=True)
        assert dx.shape == shape and bool((dw == 0).all())
    with torch.no_grad():
        wide = w.new_ones(1).expand(shape)
        q, s = ops.per_token_int8_quant(wide)
        assert q.shape == shape and s.shape == shape[:-1] + (1,)
        wq, ws = ops.per_token_int8_quant(w.detach())
        assert ops.linear_int8(wide, None, wq, ws).shape == shape[:-1] + (32,)
        assert ops.linear_int8(q, s, wq, ws).shape == shape[:-1] + (32,)
        assert ops.gated_linear(wide, w).shape == ops.linear(wide, w, activation="silu_and_mul").shape == out.shape
