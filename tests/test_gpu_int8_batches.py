"""GPU: an int8 row's result does not depend on the rows beside it, whatever follows its sum."""
import pytest
import torch

pytestmark = pytest.mark.gpu

# (bias, activation, residual, output)
ENDS = [("fp32", None, None, "fp32"), ("bf16", None, None, "fp32"), ("fp32", None, "fp32", "fp32"),
        ("fp16", "silu", "bf16", "fp32"), ("bf16", "gelu", None, "fp32"), ("fp32", "gelu_tanh", "fp32", "fp32"),
        ("fp32", "relu2", "fp32", "fp32"), ("fp32", "silu_and_mul", None, "fp32"), (None, "silu_and_mul", "fp32", "fp32"),
        ("bf16", "gelu_and_mul", "fp16", "fp32"), ("fp32", "gelu_tanh_and_mul", "fp32", "fp32"),
        ("fp32", None, None, "bf16"), ("bf16", "silu_and_mul", "bf16", "bf16"), ("fp16", "relu2", "fp16", "fp16")]
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# K in whole stages, in 16 bytes, and at no alignment; weight rows that end in a tile
@pytest.mark.parametrize("K,rows", [(4096, 1024), (2880, 648), (1001, 1030), (513, 70)])
@pytest.mark.parametrize("given", [True, False])
def test_a_row_with_bias_activation_and_residual_is_the_same_in_every_batch(K, rows, given):
    from vllm_xpu_kernels import ops
    g = torch.Generator(device="cuda")
    g.manual_seed(K + rows)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")
    M = 700
    w = torch.randint(-128, 128, (rows, K), generator=g, device="cuda", dtype=torch.int8)
    ws = (torch.rand(rows, generator=g, device="cuda") - 0.3) * 0.02
    x = rand(M, K).to(torch.bfloat16)
    q, xs = ops.per_token_int8_quant(x) if given else (x, None)
    q[5] = 0  # sums of zero
    for bias, act, res, out in ENDS:
        n = rows // 2 if act and act.endswith("_and_mul") else rows
        b = rand(rows).to(DT[bias]) if bias else None
        r = rand(M, n).to(DT[res]) if res else None
        call = lambda m: ops.linear_int8(q[:m], None if xs is None else xs[:m], w, ws, b, act,
                                         None if r is None else r[:m], out_dtype=DT[out])
        want = call(M)
        for m in (1, 2, 4, 9, 16, 33, 64, 129, 300):
            got = call(m)
            assert torch.equal(got, want[:m]), (bias, act, res, out, m, float((got.double() - want[:m].double()).abs().max()))
