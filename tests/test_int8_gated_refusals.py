"""linear_int8, per_token_int8_quant and gated_linear without a GPU: what the C ABI
refuses before any device work, what the wrappers refuse, the ops' registration, and
the gate's derivative against differences."""
import ctypes
import math

import pytest
import torch

F32, BF16, F16, I32, E4M3, I8 = 0, 1, 2, 3, 6, 10


@pytest.fixture(scope="module")
def capi():
    from vllm_xpu_kernels import capi
    return capi


def _linear_args(capi, **kw):
    a = capi.LinearArgs(x_dtype=I8, out_dtype=BF16, bias_dtype=BF16, residual_dtype=BF16, activation=0, M=4, N=64,
                        K=256, x=16, ldx=256, x_scale=16, x_scale_row=1, weight=16, ldw=256, weight_scale=16,
                        weight_scale_row=1, out=16, ldo=64)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,msg", [
    ({"K": 1 << 17}, b"K must be below 131072"),
    ({"x_dtype": BF16, "weight_dtype": I8, "K": 1 << 17}, b"K must be below 131072"),
    ({"x_dtype": BF16, "weight_dtype": F16}, b"weight must have x's type"),
    ({"x_dtype": E4M3, "weight_dtype": I8}, b"weight must have x's type"),
    ({"weight_dtype": BF16}, b"weight must have x's type"),
    ({"x_scale": None}, b"scales missing"),
    ({"weight_scale": None}, b"scales missing"),
    ({"x_dtype": F16, "weight_dtype": I8, "weight_scale": None}, b"scales missing"),
    ({"x_scale_row": -1}, b"negative stride"),
    ({"weight_scale_row": -1}, b"negative stride"),
    ({"activation": 5, "z": 16}, b"z is kept for gated activations of 16-bit operands"),
    ({"x_dtype": BF16, "activation": 0, "z": 16}, b"z is kept for gated activations of 16-bit operands"),
    ({"x_dtype": BF16, "weight_dtype": I8, "activation": 5, "z": 16}, b"z is kept for gated"),
    ({"x_dtype": BF16, "activation": 5, "z": 24}, b"z must be 16-byte aligned"),
    ({"x_dtype": BF16, "activation": 5, "z": 16, "N": (1 << 20) + 1, "ldo": 1 << 21}, b"too large for a backward pass"),
    ({"x_dtype": BF16, "activation": 5, "z": 16, "K": (1 << 24) + 1}, b"too large for a backward pass"),
    ({"x": None}, b"null pointer"),
])
def test_linear_refuses(capi, kw, msg):
    a = _linear_args(capi, **kw)
    assert capi.lib.mi355moe_linear(ctypes.byref(a), None, 0, None) == -1
    assert msg in capi.lib.mi355moe_last_error()


def test_linear_workspace_of_codes_is_checked(capi):
    a = _linear_args(capi, x_dtype=BF16, weight_dtype=I8, x_scale=None, M=5, K=1001, ldx=1001, ldw=1001)
    need = capi.lib.mi355moe_linear_workspace_size(ctypes.byref(a))
    assert need >= 5 * 1008 + 5 * 4
    for ws, size in ((None, 0), (None, need), (1 << 20, need - 1)):
        assert capi.lib.mi355moe_linear(ctypes.byref(a), ws, size, None) == -4
        assert b"workspace too small" in capi.lib.mi355moe_last_error()
    assert capi.lib.mi355moe_linear(ctypes.byref(a), (1 << 20) + 4, need, None) == -1
    assert b"workspace must be 16-byte aligned" in capi.lib.mi355moe_last_error()


@pytest.mark.parametrize("args,msg", [
    ((16, I32, 64, 16, 64, 16, 1, 2, 64), b"input must be float32, bfloat16 or float16"),
    ((16, BF16, 64, 16, 64, 16, 1, 2, 0), b"invalid shape"),
    ((16, BF16, 64, 16, 64, 16, 1, -2, 64), b"invalid shape"),
    ((16, BF16, 64, 16, 64, 16, 1, 2, (1 << 28) + 1), b"size too large"),
    ((16, BF16, -64, 16, 64, 16, 1, 2, 64), b"negative stride"),
    ((16, BF16, 64, 16, 63, 16, 1, 2, 64), b"rows of an output overlap"),
    ((16, BF16, 64, 16, 64, 16, 0, 2, 64), b"rows of an output overlap"),
    ((None, BF16, 64, 16, 64, 16, 1, 2, 64), b"null pointer"),
    ((16, BF16, 64, None, 64, 16, 1, 2, 64), b"null pointer"),
    ((16, BF16, 64, 16, 64, None, 1, 2, 64), b"null pointer"),
])
def test_int8_quant_refuses(capi, args, msg):
    assert capi.lib.mi355moe_int8_quant(*args, None) == -1
    assert msg in capi.lib.mi355moe_last_error()


def test_int8_quant_of_no_rows_touches_nothing(capi):
    assert capi.lib.mi355moe_int8_quant(None, BF16, 64, None, 64, None, 1, 0, 64, None) == 0


def _backward_args(capi, **kw):
    a = capi.GatedLinearBackwardArgs(dtype=BF16, dbias_dtype=BF16, activation=5, M=4, N=64, K=256, x=16, ldx=256,
                                     weight=16, ldw=256, z=16, dout=16, ldd=64, dx=16, lddx=256, dweight=16,
                                     lddw=256, dbias=16)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,msg", [
    ({"dtype": F32}, b"operands must be bfloat16 or float16"),
    ({"activation": 1}, b"the activation must be a gated one"),
    ({"activation": 8}, b"the activation must be a gated one"),
    ({"dbias_dtype": I32}, b"dbias must be float32, bfloat16 or float16"),
    ({"M": -1}, b"invalid shape"),
    ({"N": 0}, b"invalid shape"),
    ({"K": 0}, b"invalid shape"),
    ({"M": 1 << 40}, b"size too large"),
    ({"N": 1 << 40}, b"size too large"),
    ({"K": 1 << 40}, b"size too large"),
    ({"ldx": -1}, b"negative stride"),
    ({"lddx": 255}, b"rows of dx overlap"),
    ({"lddw": 255}, b"rows of dweight overlap"),
    ({"dx": None, "dweight": None, "dbias": None}, b"no gradient is asked for"),
    ({"x": None}, b"null pointer"),
    ({"weight": None}, b"null pointer"),
    ({"z": None}, b"null pointer"),
    ({"dout": None}, b"null pointer"),
])
def test_backward_refuses(capi, kw, msg):
    a = _backward_args(capi, **kw)
    assert capi.lib.mi355moe_gated_linear_backward(ctypes.byref(a), None, 0, None) == -1
    assert msg in capi.lib.mi355moe_last_error()
    if msg != b"null pointer":
        assert capi.lib.mi355moe_gated_linear_backward_workspace_size(ctypes.byref(a)) == 0


def test_backward_workspace_is_checked(capi):
    a = _backward_args(capi)
    need = capi.lib.mi355moe_gated_linear_backward_workspace_size(ctypes.byref(a))
    assert need >= 4 * 128 * 2
    for ws, size in ((None, 0), (None, need), (1 << 20, need - 1)):
        assert capi.lib.mi355moe_gated_linear_backward(ctypes.byref(a), ws, size, None) == -4
        assert b"workspace too small" in capi.lib.mi355moe_last_error()
    assert capi.lib.mi355moe_gated_linear_backward(ctypes.byref(a), (1 << 20) + 4, need, None) == -1
    assert b"workspace must be 16-byte aligned" in capi.lib.mi355moe_last_error()
    assert capi.lib.mi355moe_gated_linear_backward(None, None, 0, None) == -1
    assert capi.lib.mi355moe_gated_linear_backward_workspace_size(None) == 0


def test_ops_have_no_cpu_kernel():
    from vllm_xpu_kernels import ops
    x, w = torch.zeros(2, 128, dtype=torch.bfloat16), torch.zeros(8, 128, dtype=torch.int8)
    s = torch.ones(8)
    with pytest.raises(NotImplementedError):
        ops.linear_int8(x, None, w, s)
    with pytest.raises(NotImplementedError):
        ops.per_token_int8_quant(x)
    with pytest.raises(NotImplementedError):
        ops.gated_linear(x, x.repeat(4, 1))
    with pytest.raises(NotImplementedError):
        ops.gated_linear(x.requires_grad_(), torch.zeros(8, 128, dtype=torch.bfloat16))


def _meta(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype, device="meta")


def test_shapes_without_a_device():
    from vllm_xpu_kernels import ops
    w, s = _meta(16, 128, dtype=torch.int8), _meta(16, dtype=torch.float32)
    assert ops.linear_int8(_meta(3, 5, 128), None, w, s, activation="silu_and_mul").shape == (3, 5, 8)
    q, sc = ops.per_token_int8_quant(_meta(3, 5, 128))
    assert q.shape == (3, 5, 128) and q.dtype == torch.int8 and sc.shape == (3, 5, 1)
    out = ops.linear_int8(q, sc, w, s)
    assert out.shape == (3, 5, 16) and out.dtype == torch.bfloat16
    assert ops.linear_int8(_meta(3, 128, dtype=torch.float16), None, w, s).dtype == torch.float16
    x, w = _meta(3, 5, 128).requires_grad_(), _meta(16, 128).requires_grad_()
    b = _meta(16, dtype=torch.float32).requires_grad_()
    out = ops.gated_linear(x, w, b)
    assert out.shape == (3, 5, 8)
    out.backward(_meta(3, 5, 8))
    for t in (x, w, b):
        assert t.grad.shape == t.shape and t.grad.dtype == t.dtype


def test_wrappers_refuse():
    from vllm_xpu_kernels import ops
    w, s = _meta(16, 128, dtype=torch.int8), _meta(16, dtype=torch.float32)
    x = _meta(2, 128)
    with pytest.raises(ValueError, match="Unsupported activation"):
        ops.linear_int8(x, None, w, s, activation="tanh")
    with pytest.raises(ValueError, match="out must have out_dtype"):
        ops.linear_int8(x, None, w, s, out_dtype=torch.float32, out=_meta(2, 16))
    for bad in (None, "silu", "tanh"):
        with pytest.raises(ValueError, match="Unsupported activation"):
            ops.gated_linear(x, _meta(16, 128), activation=bad)
    for name in ("x", "weight_scale", "bias", "residual", "out"):
        kw = {"x": x, "weight_scale": s, "bias": _meta(16), "residual": _meta(2, 16), "out": _meta(2, 16)}
        kw[name] = kw[name].clone().requires_grad_()
        with pytest.raises(RuntimeError, match="no gradient"):
            ops.linear_int8(kw["x"], None, w, kw["weight_scale"], kw["bias"], None, kw["residual"], out=kw["out"])
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.per_token_int8_quant(x.clone().requires_grad_())


def test_gated_linear_refuses_what_it_has_no_derivative_for():
    import torch.autograd.forward_ad as fw
    from vllm_xpu_kernels import ops
    x, w = _meta(2, 128), _meta(16, 128)
    with fw.dual_level():
        d = fw.make_dual(x, _meta(2, 128))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            ops.gated_linear(d, w)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
            ops.gated_linear(x, fw.make_dual(w, _meta(16, 128)))
    x.requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient of its gradient"):
        torch.autograd.grad(ops.gated_linear(x, w), x, _meta(2, 8), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda v: ops.gated_linear(v, w).float().sum())(_meta(2, 128))


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_the_formula_of_the_gate_against_differences(act):
    """What the kernels compute (f, f') against central differences of f in 64 bits."""
    z = torch.linspace(-8, 8, 4001, dtype=torch.float64)
    c = math.sqrt(2 / math.pi)

    def f(z):
        if act == "silu":
            return z / (1 + torch.exp(-z))
        if act == "gelu":
            return z * (1 + torch.erf(z * math.sqrt(0.5))) / 2
        return z / 2 * (1 + torch.tanh(c * (z + 0.044715 * z ** 3)))

    if act == "silu":
        s = torch.sigmoid(z)
        df = s * (1 + z * (1 - s))
    elif act == "gelu":
        df = (1 + torch.erf(z * math.sqrt(0.5))) / 2 + z * torch.exp(-z * z / 2) * 0.3989422804014327
    else:
        s = torch.sigmoid(1.5957691216057308 * (z + 0.044715 * z ** 3))
        assert float((f(z) - z * s).abs().max()) < 1e-12
        df = s + z * s * (1 - s) * (1.5957691216057308 * (1 + 0.134145 * z * z))
    h = 1e-5
    # |f'''| < 3: the quotient is off by h^2 / 2, and by two roundings of f over 2 h
    assert float(((f(z + h) - f(z - h)) / (2 * h) - df).abs().max()) < 3 * h * h / 6 + 2 ** -52 * 8 / h
