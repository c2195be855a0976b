"""Norm and linear operators without a GPU: what the C ABI refuses before any
device work, what the wrappers refuse, and the ops' registration."""
import ctypes

import pytest
import torch

F32, BF16, F16, I32, E4M3, U8 = 0, 1, 2, 3, 6, 7


@pytest.fixture(scope="module")
def capi():
    from vllm_xpu_kernels import capi
    return capi


def _norm_args(capi, **kw):
    a = capi.RmsNormArgs(dtype=BF16, weight_dtype=BF16, rows=4, cols=256, inner=1, x=16, x_outer=256,
                         weight=16, eps=1e-6, out=16, out_outer=256)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,msg", [
    ({"dtype": I32}, b"input must be float32, bfloat16 or float16"),
    ({"weight_dtype": F16}, b"weight must have the input's type or be float32"),
    ({"cols": 0}, b"invalid shape"),
    ({"rows": -1}, b"invalid shape"),
    ({"inner": 0}, b"invalid shape"),
    ({"residual": 16}, b"residual and residual_out go together"),
    ({"residual_out": 16}, b"residual and residual_out go together"),
    ({"out": None}, b"no output"),
    ({"q": 16, "scales": 16, "group": 48}, b"group_size must be 32, 64 or 128"),
    ({"q": 16, "scales": 16, "group": 128, "cols": 192}, b"divisible by group_size"),
    ({"q": 16, "scales": 16, "group": 128, "scale_dtype": BF16}, b"float32 or e8m0 codes"),
    ({"q": 16, "group": 128}, b"scales missing"),
    ({"x": None}, b"null pointer"),
    ({"weight": None}, b"null pointer"),
])
def test_rms_norm_refuses(capi, kw, msg):
    assert capi.lib.mi355moe_rms_norm(ctypes.byref(_norm_args(capi, **kw)), None) == -1
    assert msg in capi.lib.mi355moe_last_error()


def test_rms_norm_of_no_rows_touches_nothing(capi):
    a = _norm_args(capi, rows=0, x=None, weight=None, out=None)
    assert capi.lib.mi355moe_rms_norm(ctypes.byref(a), None) == 0


def _linear_args(capi, **kw):
    a = capi.LinearArgs(x_dtype=BF16, out_dtype=BF16, bias_dtype=BF16, residual_dtype=BF16,
                        activation=0, M=4, N=64, K=256, x=16, ldx=256, weight=16, ldw=256, out=16,
                        ldo=64)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,msg", [
    ({"x_dtype": F32}, b"x must be bfloat16, float16 or float8_e4m3fn"),
    ({"out_dtype": E4M3}, b"out must be float32, bfloat16 or float16"),
    ({"bias": 16, "bias_dtype": U8}, b"bias must be float32, bfloat16 or float16"),
    ({"residual": 16, "residual_dtype": I32}, b"residual must be float32, bfloat16 or float16"),
    ({"activation": 8}, b"unknown activation"),
    ({"activation": -1}, b"unknown activation"),
    ({"N": 0}, b"invalid shape"),
    ({"K": 0}, b"invalid shape"),
    ({"M": -1}, b"invalid shape"),
    ({"M": 1 << 40}, b"size too large"),
    ({"N": 1 << 40}, b"size too large"),
    ({"K": 1 << 40}, b"size too large"),
    ({"ldx": -256}, b"negative stride"),
    ({"ldo": -64}, b"negative stride"),
    ({"x_dtype": E4M3, "x_scale_row": -2}, b"negative stride"),
    ({"x_dtype": E4M3, "K": 192}, b"K must be divisible by 128"),
    ({"x_dtype": E4M3}, b"scales missing"),
    ({"x": None}, b"null pointer"),
    ({"weight": None}, b"null pointer"),
    ({"out": None}, b"null pointer"),
])
def test_linear_refuses(capi, kw, msg):
    a = _linear_args(capi, **kw)
    assert capi.lib.mi355moe_linear(ctypes.byref(a), None, 0, None) == -1
    assert msg in capi.lib.mi355moe_last_error()
    if msg not in (b"null pointer", b"scales missing"):   # sizes that are refused need no workspace
        assert capi.lib.mi355moe_linear_workspace_size(ctypes.byref(a)) == 0


def test_linear_of_no_rows_touches_nothing(capi):
    a = _linear_args(capi, M=0, x=None, out=None)
    assert capi.lib.mi355moe_linear(ctypes.byref(a), None, 0, None) == 0


def test_null_arguments(capi):
    assert capi.lib.mi355moe_rms_norm(None, None) == -1
    assert capi.lib.mi355moe_linear(None, None, 0, None) == -1
    assert capi.lib.mi355moe_linear_workspace_size(None) == 0


def test_ops_are_registered_and_have_no_cpu_kernel():
    from vllm_xpu_kernels import ops
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError):
        ops.rms_norm(x, torch.ones(128, dtype=torch.bfloat16))
    with pytest.raises(NotImplementedError):
        ops.linear(x, torch.zeros(8, 128, dtype=torch.bfloat16))


def test_wrappers_refuse():
    from vllm_xpu_kernels import ops
    x, w = torch.zeros(2, 128, dtype=torch.bfloat16), torch.zeros(8, 128, dtype=torch.bfloat16)
    g = torch.ones(128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.linear(x, w.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.rms_norm(x, g.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.rms_norm_quant(x.clone().requires_grad_(), g)
    with pytest.raises(ValueError, match="Unsupported activation"):
        ops.linear(x, w, activation="tanh")
    with pytest.raises(ValueError, match="residual_out needs a residual"):
        ops.rms_norm(x, g, residual_out=x)
    with pytest.raises(ValueError, match="residual_out needs a residual"):
        ops.rms_norm_quant(x, g, residual_out=x)
    with pytest.raises(ValueError, match="out must have out_dtype"):
        ops.linear(x, w, out_dtype=torch.float32, out=torch.zeros(2, 8, dtype=torch.bfloat16))


def test_meta_kernels_trace():
    """The ops run on meta tensors (shape propagation without a device)."""
    from vllm_xpu_kernels import ops
    x = torch.zeros(3, 128, dtype=torch.bfloat16, device="meta")
    g = torch.ones(128, dtype=torch.bfloat16, device="meta")
    q, s, n, r = ops.rms_norm_quant(x, g, residual=x, with_norm=True)
    assert q.shape == n.shape == r.shape == (3, 128) and s.shape == (3, 1)
    w = torch.zeros(16, 128, dtype=torch.bfloat16, device="meta")
    assert ops.linear(x, w, activation="silu_and_mul").shape == (3, 8)


def test_linear_workspace_is_checked(capi):
    """A product that splits K refuses a workspace that is missing, too small or
    not aligned, and rows of out that meet, before any device work."""
    a = _linear_args(capi, M=61, N=4096, K=4096, ldx=4096, ldw=4096, ldo=4096, x=1 << 20,
                     weight=1 << 20, out=1 << 20)
    a.x += 2                               # unaligned rows: 64 x 64 tiles, too few without splits
    need = capi.lib.mi355moe_linear_workspace_size(ctypes.byref(a))
    assert need > 0 and need % (61 * 4096 * 4) == 0
    for ws, size in ((None, 0), (None, need), (1 << 20, need - 1)):
        assert capi.lib.mi355moe_linear(ctypes.byref(a), ws, size, None) == -4
        assert b"workspace too small" in capi.lib.mi355moe_last_error()
    assert capi.lib.mi355moe_linear(ctypes.byref(a), (1 << 20) + 4, need, None) == -1
    assert b"workspace must be 16-byte aligned" in capi.lib.mi355moe_last_error()


@pytest.mark.parametrize("kw,msg", [({"N": (1 << 24) + 1, "ldo": 1 << 25}, b"size too large"),
                                    ({"M": 64 * 65535 + 1}, b"size too large"),
                                    ({"ldo": 63}, b"rows of out overlap"),
                                    ({"ldo": 0}, b"rows of out overlap")])
def test_linear_refuses_sizes_beyond_its_grids(capi, kw, msg):
    a = _linear_args(capi, **kw)
    assert capi.lib.mi355moe_linear(ctypes.byref(a), None, 0, None) == -1
    assert msg in capi.lib.mi355moe_last_error()


@pytest.mark.parametrize("group", [0, -128, 48])
def test_rms_norm_quant_refuses_groups(group):
    from vllm_xpu_kernels import ops
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="group_size must be 32, 64, or 128"):
        ops.rms_norm_quant(x, x[0], residual=x, residual_out=x, group_size=group)


def _meta(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype, device="meta")


def _calls(ops, t):
    """Every wrapper, with `t` (a function of the argument's name) choosing each tensor."""
    yield "rms_norm", ("x", "weight", "residual", "residual_out", "out"), lambda: ops.rms_norm(
        t("x", 2, 128), t("weight", 128), residual=t("residual", 2, 128),
        residual_out=t("residual_out", 2, 128), out=t("out", 2, 128))
    yield "rms_norm_quant", ("x", "weight", "residual", "residual_out"), lambda: ops.rms_norm_quant(
        t("x", 2, 128), t("weight", 128), residual=t("residual", 2, 128),
        residual_out=t("residual_out", 2, 128))
    yield "linear", ("x", "weight", "bias", "residual", "out"), lambda: ops.linear(
        t("x", 2, 128), t("weight", 8, 128), t("bias", 8), residual=t("residual", 2, 8), out=t("out", 2, 8))
    f8 = torch.float8_e4m3fn
    yield "linear_fp8", ("x", "x_scale", "weight", "weight_scale", "bias", "residual", "out"), \
        lambda: ops.linear_fp8(
            t("x", 2, 128, dtype=f8), t("x_scale", 2, 1, dtype=torch.float32),
            t("weight", 8, 128, dtype=f8), t("weight_scale", 1, 1, dtype=torch.float32), t("bias", 8),
            residual=t("residual", 2, 8), out=t("out", 2, 8))


def test_wrappers_refuse_every_tensor_that_needs_a_gradient():
    """Inputs and given outputs alike, e4m3 codes cast from a tensor with a gradient too; without
    gradients the same calls run."""
    from vllm_xpu_kernels import ops
    chosen = [None]

    def t(name, *shape, dtype=torch.bfloat16):
        if name != chosen[0]:
            return _meta(*shape, dtype=dtype)
        return _meta(*shape, dtype=torch.float32).requires_grad_().to(dtype) if dtype != torch.float32 \
            else _meta(*shape, dtype=dtype).requires_grad_()

    for op, names, call in _calls(ops, t):
        chosen[0] = None
        call()
        for n in names:
            chosen[0] = n
            with pytest.raises(RuntimeError, match="no gradient"):
                call()
            with torch.no_grad():
                call()


def test_wrappers_refuse_forward_mode_duals():
    """A tangent would be lost, under no_grad too (it does not end forward mode)."""
    import torch.autograd.forward_ad as fw
    from vllm_xpu_kernels import ops
    chosen = [None]

    def t(name, *shape, dtype=torch.bfloat16):
        v = _meta(*shape, dtype=dtype)
        return fw.make_dual(v, _meta(*shape, dtype=dtype)) if name == chosen[0] else v

    with fw.dual_level():
        for op, names, call in _calls(ops, t):
            chosen[0] = None
            call()
            for n in names:
                chosen[0] = n
                with pytest.raises(RuntimeError, match="no gradient"):
                    call()
                with torch.no_grad(), pytest.raises(RuntimeError, match="no gradient"):
                    call()


def test_wrappers_refuse_function_transforms():
    from vllm_xpu_kernels import ops
    w, x = _meta(8, 128), _meta(2, 128)
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.func.grad(lambda v: ops.linear(v, w).float().sum())(x)
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.func.jvp(lambda v: ops.linear(v, w), (x,), (x,))
