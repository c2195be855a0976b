"""Dense feed-forward operators beside the experts, as a list of measurable cases.

``gated``  out = f(x Wg^T + bg) * (x Wu^T + bu), both projections, the activation and the product in one kernel,
           and its backward pass: the gradients of x, of W = [Wg; Wu] and of the biases from that of out.
           Training steps of a shared expert or a dense layer, and of adapters in front of a frozen one
``int8``   act(x W^T + bias) + residual on 8-bit integers, a scale for each token of x and each row of W; x comes
           as 8-bit integers with its scales, or in 16 bits and is quantised in the call

Sizes are those of the configurations in ``vllm_xpu_kernels/workloads.py`` (hidden 512 to 7168, intermediate 768
to 2880) and generic ones; token counts run from one (a single decode) to 8192, odd ones included.
"""
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.getcwd(), "vllm-xpu-kernels_amd"))

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _gated(m, k, n, dtype="bf16", act="silu_and_mul", bias=False, frozen=False, name=None):
    c = {"op": "gated", "m": m, "k": k, "n": n, "dtype": dtype, "act": act, "bias": bias, "frozen": frozen}
    return dict(c, name=name) if name else c


def _int8(m, k, n, dtype="bf16", act="none", bias=False, residual=False, out="same", given=False, name=None):
    c = {"op": "int8", "m": m, "k": k, "n": n, "dtype": dtype, "act": act, "bias": bias, "residual": residual,
         "out": out, "given": given}
    return dict(c, name=name) if name else c


def listed():
    return [
        # a small expert's step on a few tokens: latency
        _gated(61, 2048, 768, name="gated_train_61"),
        # gradients of the input alone: adapters are trained in front of frozen weights
        _gated(512, 4096, 1024, frozen=True, name="gated_adapter_512"),
        # sizes that no vector divides
        _gated(257, 1001, 515, act="gelu_and_mul", name="gated_odd_257"),
        # a packed batch of no whole tile, biased projections
        _gated(1003, 2880, 2880, "fp16", "gelu_tanh_and_mul", True, name="gated_ragged_1003"),
        # the largest: a shared expert over a full batch
        _gated(8192, 7168, 2048, name="gated_train_8192"),
        # gate and up of one decoded token, the norm's 16-bit output quantised on the way
        _int8(1, 7168, 2048, act="silu_and_mul", name="int8_glu_decode_1"),
        # an output projection of a small decode batch, added to the residual
        _int8(16, 4096, 4096, "fp16", residual=True, name="int8_residual_decode_16"),
        # a biased projection of a decode batch whose tokens were quantised for several products
        _int8(61, 4096, 6144, bias=True, given=True, name="int8_bias_decode_61"),
        # a prefill chunk through a biased projection with an activation, no size a whole tile
        _int8(1003, 2880, 2880, act="gelu_tanh", bias=True, name="int8_bias_gelu_1003"),
        # gate and up over a full prefill batch
        _int8(8192, 7168, 2048, act="silu_and_mul", name="int8_glu_prefill_8192"),
        # the down product over the same batch, added to the routed experts' output
        _int8(8192, 2048, 7168, residual=True, given=True, name="int8_residual_prefill_8192"),
    ]


MOST = 8192 * 7168 * 4096  # multiplications of one product of the largest listed case


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.45:
        m = _log(rng, 32, 8192)
        k = rng.choice([512, 2048, 2880, 4096, 7168, _log(rng, 64, 7168) // 8 * 8, _log(rng, 33, 7168)])
        n = rng.choice([128, 512, 768, 1024, 2048, 2880, _log(rng, 64, 4096) // 8 * 8, _log(rng, 33, 4096)])
        m = max(32, min(m, MOST // (2 * n * k)))
        if k % 8 or n % 8:
            m = min(m, 1024)  # sizes that no vector divides come in small products
        return _gated(m, k, n, rng.choice(["bf16", "bf16", "fp16"]),
                      rng.choice(["silu_and_mul", "silu_and_mul", "gelu_and_mul", "gelu_tanh_and_mul"]),
                      rng.random() < 0.3, rng.random() < 0.25)
    act = rng.choice(["none", "none", "silu", "gelu", "gelu_tanh", "relu2", "silu_and_mul", "silu_and_mul", "gelu_and_mul"])
    m = _log(rng, 1, 8192)
    k = rng.choice([512, 2048, 2880, 4096, 7168, _log(rng, 16, 7168) // 16 * 16, _log(rng, 1, 7168)])
    n = rng.choice([256, 768, 1024, 2048, 2880, 4096, 7168, _log(rng, 1, 7168)])
    rows = 2 * n if act.endswith("_and_mul") else n
    m = max(1, min(m, MOST // (rows * k)))
    if k % 16 or n % 8:
        m = min(m, 1024)
    return _int8(m, k, n, rng.choice(["bf16", "bf16", "fp16"]), act, rng.random() < 0.4, rng.random() < 0.4,
                 "fp32" if rng.random() < 0.2 else "same", rng.random() < 0.5)


# ------------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(1000003 * seed + 11)
    return g


def _codes(x):
    """Rows of x as integers in -127 .. 127 and the scale of each row, in 32 bits."""
    s = x.float().abs().amax(-1, keepdim=True).clamp(min=1e-10) / 127.0
    return torch.round(x.float() / s), s


def prepare(case, seed):
    g = _gen(seed)
    dtype = DTYPES[case["dtype"]]
    M, K, N = case["m"], case["k"], case["n"]
    rows = 2 * N if case["act"].endswith("_and_mul") else N
    # normed activations have channels of different size
    size = torch.exp(0.5 * torch.randn(K, generator=g, device=DEV))
    x = torch.randn(M, K, generator=g, device=DEV).mul_(size).to(dtype)
    w = torch.randn(rows, K, generator=g, device=DEV).mul_(1.0 / math.sqrt(K))
    bias = torch.randn(rows, generator=g, device=DEV).mul_(0.1).to(dtype) if case["bias"] else None
    state = {"case": case, "bias": bias}
    if case["op"] == "gated":
        state["x"], state["weight"] = x.requires_grad_(), w.to(dtype)
        if not case["frozen"]:
            state["weight"].requires_grad_()
            if bias is not None:
                bias.requires_grad_()
        # the loss is scaled, as 16-bit training does
        state["grad"] = torch.randn(M, N, generator=g, device=DEV).to(dtype)
        return state
    out = torch.float32 if case["out"] == "fp32" else dtype
    q, s = _codes(w)
    state["weight"], state["weight_scale"] = q.to(torch.int8), s.squeeze(-1)
    state["x"], state["x_scale"] = x, None
    if case["given"]:
        q, s = _codes(x)
        state["x"], state["x_scale"] = q.to(torch.int8), s
    state["residual"] = torch.randn(M, N, generator=g, device=DEV).to(out) if case["residual"] else None
    state["out_dtype"] = out
    return state


# -------------------------------------------------------------- plain forms

def _f(z, act):
    """The activation of z, and its derivative."""
    name = act.replace("_and_mul", "")
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return z * s, s * (1.0 + z * (1.0 - s))
    if name == "gelu":
        p = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * p, p + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if name == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * z * z)
    if name == "relu2":
        r = z.clamp(min=0.0)
        return r * r, 2.0 * r
    return z, torch.ones_like(z)


@torch.no_grad()
def _plain_gated(state):
    case, dtype = state["case"], state["x"].dtype
    x, w, n = state["x"].float(), state["weight"].float(), case["n"]
    z = x @ w.t()
    if state["bias"] is not None:
        z = z + state["bias"].float()
    gate, up = z[:, :n], z[:, n:]
    f, df = _f(gate, case["act"])
    out = {"out": (f * up).to(dtype)}
    d = state["grad"].float()
    dz = torch.cat([d * up * df, d * f], -1)
    out["dx"] = (dz @ w).to(dtype)
    if not case["frozen"]:
        out["dweight"] = (dz.t() @ x).to(dtype)
        if state["bias"] is not None:
            out["dbias"] = dz.sum(0).to(dtype)
    return out


def _plain_int8(state):
    act, n = state["case"]["act"], state["case"]["n"]
    q, s = (state["x"].float(), state["x_scale"]) if state["x_scale"] is not None else _codes(state["x"])
    z = (q @ state["weight"].float().t()) * s * state["weight_scale"]
    if state["bias"] is not None:
        z = z + state["bias"].float()
    y = _f(z[:, :n], act)[0]
    if act.endswith("_and_mul"):
        y = y * z[:, n:]
    if state["residual"] is not None:
        y = y + state["residual"].float()
    return {"out": y.to(state["out_dtype"])}


def run(state):
    case = state["case"]
    if not own:
        return _plain_gated(state) if case["op"] == "gated" else _plain_int8(state)
    from vllm_xpu_kernels import ops
    if case["op"] == "gated":
        x, w, b = state["x"], state["weight"], state["bias"]
        out = ops.gated_linear(x, w, b, case["act"])
        leaves = {"dx": x}
        if not case["frozen"]:
            leaves["dweight"] = w
            if b is not None:
                leaves["dbias"] = b
        grads = torch.autograd.grad(out, list(leaves.values()), state["grad"])
        return dict(zip(leaves, grads), out=out.detach())
    act = None if case["act"] == "none" else case["act"]
    return {"out": ops.linear_int8(state["x"], state["x_scale"], state["weight"], state["weight_scale"],
                                   state["bias"], act, state["residual"], out_dtype=state["out_dtype"])}


def work(case):
    """Inputs once, outputs once; a product's two operations per multiplication, three products for a step (two where
    the weights are frozen)."""
    b = DTYPES[case["dtype"]].itemsize
    M, K, N = case["m"], case["k"], case["n"]
    rows = 2 * N if case["act"].endswith("_and_mul") else N
    if case["op"] == "gated":
        biases = rows * b if case["bias"] else 0
        read = (M + rows) * K * b + M * N * b + biases
        write = M * N * b + M * K * b + (0 if case["frozen"] else rows * K * b + biases)
        return {"bytes": read + write, "flops": 2.0 * M * rows * K * (2 if case["frozen"] else 3)}
    o = 4 if case["out"] == "fp32" else b
    read = (M * K + 4 * M if case["given"] else M * K * b) + rows * K + 4 * rows
    read += rows * b if case["bias"] else 0
    read += M * N * o if case["residual"] else 0
    return {"bytes": read + M * N * o, "flops": 2.0 * M * rows * K}


# ------------------------------------------------------- the same in 64 bits

def _activation64(z, act):
    if act.startswith("silu"):
        return z * torch.sigmoid(z)
    if act.startswith("gelu_tanh"):
        return torch.nn.functional.gelu(z, approximate="tanh")
    if act.startswith("gelu"):
        return torch.nn.functional.gelu(z)
    return torch.relu(z).square() if act == "relu2" else z


def exact(case, seed):
    state = prepare(case, seed)
    n = case["n"]
    if case["op"] == "gated":
        x, w = state["x"].detach().double(), state["weight"].detach().double()
        z = torch.mm(x, w.t())
        if state["bias"] is not None:
            z += state["bias"].detach().double()
        z.requires_grad_()
        y = _activation64(z[:, :n], case["act"]) * z[:, n:]
        dz, = torch.autograd.grad(y, z, state["grad"].double())
        out = {"out": y.detach(), "dx": torch.mm(dz, w)}
        if not case["frozen"]:
            out["dweight"] = torch.mm(dz.t().contiguous(), x)
            if state["bias"] is not None:
                out["dbias"] = dz.sum(0)
        return out
    x = state["x"].double()
    if state["x_scale"] is None:
        s = torch.maximum(x.abs().amax(1, keepdim=True), x.new_tensor(1e-10)) / 127.0
        x = torch.round(x / s)
    else:
        s = state["x_scale"].double()
    z = torch.mm(x, state["weight"].double().t()) * (s * state["weight_scale"].double()[None, :])
    if state["bias"] is not None:
        z += state["bias"].double()
    y = _activation64(z[:, :n], case["act"])
    if case["act"].endswith("_and_mul"):
        y = y * z[:, n:]
    return {"out": y if state["residual"] is None else y + state["residual"].double()}
