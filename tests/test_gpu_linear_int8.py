"""GPU: linear_int8 and per_token_int8_quant against the formula in 64 bits.

Tolerances.  The products' sums are exact; as a float a sum is off by half a step
of fp32 (U = 2^-24 of it), the scales' product and its product with the sum by
another each: 3 U |z|, and the bias adds U |z|.  The activations' slopes are below
1.13 (relu2: 2 z); their own arithmetic adds 2^-20 of the value (erf, hardware exp2
and reciprocal, and the rounding of the exponent's argument, |z| 2^-24).  The
residual and the output add a rounding each.  Codes and scales of the quantiser
are those of fp32's product and division, bit for bit."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
U = 2.0 ** -24


def _ops():
    from vllm_xpu_kernels import ops
    return ops


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rand(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=_gen(seed), device="cuda") * scale).to(dtype)


def _codes(shape, seed, low=-128):
    return torch.randint(low, 128, shape, generator=_gen(seed), device="cuda", dtype=torch.int8)


def _scales(n, seed, size):
    return (torch.rand(n, generator=_gen(seed), device="cuda") + 0.5) * size


def _quant(x):
    """Scales and codes in fp32 on the CPU, where a division is rounded to nearest."""
    x = x.cpu().float()
    s = x.abs().amax(-1, keepdim=True).clamp(min=1e-10) * torch.tensor(1 / 127, dtype=torch.float32)
    return torch.round(x / s), s


def _f(z, act):
    if act.startswith("silu"):
        return z * torch.sigmoid(z)
    if act.startswith("gelu_tanh"):
        return torch.nn.functional.gelu(z, approximate="tanh")
    if act.startswith("gelu"):
        return torch.nn.functional.gelu(z)
    return torch.relu(z).square() if act == "relu2" else z


def _want(q, xs, w, ws, bias, act, residual):
    """(value, how far fp32 may be off it) in 64 bits."""
    act = act or "none"
    z = (q.double() @ w.double().t()) * (xs.double().reshape(-1, 1) * ws.double().reshape(1, -1))
    e = 3.01 * U * z.abs()
    if bias is not None:
        z = z + bias.double()
        e = e + U * z.abs()
    n = z.shape[-1] // 2 if act.endswith("_and_mul") else z.shape[-1]
    g, eg = z[..., :n], e[..., :n]
    y = _f(g, act)
    slope = 2 * g.abs() + eg if act == "relu2" else (1.0 if act == "none" else 1.13)
    ey = slope * eg + (0 if act == "none" else 2.0 ** -20 * (1 + g.abs()) * y.abs() + 2.0 ** -22 * g.abs())
    if act.endswith("_and_mul"):
        u, eu = z[..., n:], e[..., n:]
        ey = ey * (u.abs() + eu) + y.abs() * eu + U * (y * u).abs()
        y = y * u
    if residual is not None:
        y = y + residual.double()
        ey = ey + U * y.abs()
    return y, ey


def _close(got, y, e):
    info = torch.finfo(got.dtype)
    lim = info.eps / 2 * y.abs() + (1 + info.eps) * e + info.smallest_normal * info.eps / 2
    # a value that may pass the type's largest one rounds to infinity, of its own sign
    over = y.abs() + e >= info.max
    fine = (got.double() - y).abs() <= lim
    assert bool((fine | (over & got.isinf() & (got.double() * y > 0))).all())


ACTS = [None, "silu", "gelu", "gelu_tanh", "relu2", "silu_and_mul", "gelu_and_mul", "gelu_tanh_and_mul"]
# rows x K x outputs: streams, tiles, splits of K, sizes that no vector divides, K of
# one byte, ends inside a stage and inside 16 bytes
SIZES = [(1, 1, 1), (1, 7168, 256), (3, 130, 37), (4, 4096, 4096), (8, 2048, 64), (16, 4096, 512), (17, 7168, 130),
         (61, 4096, 384), (64, 272, 128), (65, 2064, 200), (100, 33, 515), (250, 1001, 257), (300, 4096, 1024),
         (513, 2880, 704), (1100, 144, 1030), (270, 515, 131), (900, 1003, 583), (257, 4099, 515)]


@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("out", ["bf16", "fp16", "fp32"])
def test_codes(M, K, N, out):
    """Every activation, with bias and residual; -128 among the codes."""
    o = _ops()
    for i, act in enumerate(ACTS):
        rows = 2 * N if act and act.endswith("_and_mul") else N
        x, w = _codes((M, K), i), _codes((rows, K), 100 + i)
        xs, ws = _scales(M, 200 + i, 0.02), _scales(rows, 300 + i, 0.7 / (73 * math.sqrt(K)))
        bias = _rand(rows, torch.float32, 400 + i) if i % 2 else None
        res = _rand((M, N), DT[out], 500 + i) if i % 3 else None
        got = o.linear_int8(x, xs[:, None], w, ws, bias, act, res, out_dtype=DT[out])
        assert got.dtype == DT[out] and got.shape == (M, N)
        _close(got, *_want(x, xs, w, ws, bias, act, res))


@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_quantised_in_the_call(M, K, N, dtype):
    o = _ops()
    x = _rand((M, K), DT[dtype], 1) * (1 + 100 * (torch.arange(M, device="cuda") % 7 == 3)).to(DT[dtype])[:, None]
    w, ws = _codes((2 * N, K), 2), _scales(2 * N, 3, 0.7 / (73 * math.sqrt(K)))
    q, s = _quant(x)
    got = o.linear_int8(x, None, w, ws, activation="silu_and_mul")
    assert got.dtype == DT[dtype]
    _close(got, *_want(q.cuda(), s.cuda(), w, ws, None, "silu_and_mul", None))
    # the same bits as quantised before
    q8, s8 = o.per_token_int8_quant(x)
    assert torch.equal(o.linear_int8(q8, s8, w, ws, activation="silu_and_mul", out_dtype=DT[dtype]), got)


def test_sums_are_exact():
    """Products of -128 up to the largest K, where one more would pass 2^31; and of a K past
    fp32's 2^24 with sums that cancel to one."""
    o = _ops()
    one = torch.ones(64, device="cuda")
    for K in (131071, 65536):
        for M in (1, 3, 40, 64):
            x = torch.full((M, K), -128, dtype=torch.int8, device="cuda")
            w = torch.full((64, K), -128, dtype=torch.int8, device="cuda")
            got = o.linear_int8(x, one[:M], w, one, out_dtype=torch.float32)
            assert bool((got == float(torch.tensor(128 * 128 * K, dtype=torch.float32))).all())
            w[:, K // 2:] = 127
            w[:, -1] = 0
            want = 128 * 128 * (K // 2) - 128 * 127 * (K - K // 2 - 1)
            got = o.linear_int8(x, one[:M], w, one, out_dtype=torch.float32)
            assert bool((got == float(torch.tensor(want, dtype=torch.float32))).all())


@pytest.mark.parametrize("K", [4096, 2880, 1001])
def test_a_row_is_the_same_in_every_batch(K):
    """float32 outputs of the bare product: exact sums, the same scaling in every kernel."""
    o = _ops()
    x, w = _codes((700, K), 1), _codes((1024, K), 2)
    xs, ws = _scales(700, 3, 0.02), _scales(1024, 4, 0.01)
    want = o.linear_int8(x, xs, w, ws, out_dtype=torch.float32)
    for m in (1, 4, 9, 16, 33, 64, 129, 300):
        assert torch.equal(o.linear_int8(x[:m], xs[:m], w, ws, out_dtype=torch.float32), want[:m])


def test_strides_shapes_and_alignment():
    o = _ops()
    x3 = _codes((5, 8, 4 * 96), 1)[:, :, 96:192]        # leading dimensions that fold, a slice of the columns
    w = _codes((72, 128), 2)[:, 16:112]
    xs = _scales(80, 3, 0.02).view(5, 8, 2)[:, :, 0]     # a stride of 2
    ws = _scales(72 * 3, 4, 0.01)[::3]
    want, e = _want(x3.reshape(40, 96), xs.reshape(-1), w, ws, None, None, None)
    for s in (xs, xs.unsqueeze(-1), xs.reshape(-1), xs.reshape(-1, 1)):
        got = o.linear_int8(x3, s, w, ws.unsqueeze(-1))
        assert got.shape == (5, 8, 72)
        _close(got.reshape(40, 72), want, e)
    # rows that start anywhere, and an output inside a wider tensor whose rest is left alone
    for off in (1, 2, 8, 15):
        xb, wb = _codes((41 * 200,), 5)[off:off + 40 * 200].view(40, 200), _codes((73 * 200,), 6)[off:off + 72 * 200].view(72, 200)
        s1, s2 = _scales(40, 7, 0.02), _scales(72, 8, 0.01)
        wide = torch.full((40, 100), 7.0, device="cuda")
        out = o.linear_int8(xb, s1, wb, s2, out=wide[:, 3:75])
        assert out.data_ptr() == wide[:, 3:75].data_ptr()
        _close(out, *_want(xb, s1, wb, s2, None, None, None))
        assert bool((wide[:, :3] == 7).all() and (wide[:, 75:] == 7).all())
    # many rows: operands copied to aligned ones, each of them or both
    for off, ld in ((0, 1100), (16, 1104), (3, 1111)):
        xb = _codes((800 * ld + 16,), 5)[off:off + 800 * ld].view(800, ld)[:, :1024]
        wb = _codes((720 * 1032,), 6).view(720, 1032)[:, 8:]
        s1, s2, r = _scales(800, 7, 0.02), _scales(720, 8, 0.002), _rand((800, 721), torch.float16, 9)[:, 1:]
        _close(o.linear_int8(xb, s1, wb, s2, None, "silu_and_mul"), *_want(xb, s1, wb, s2, None, "silu_and_mul", None))
        wide = torch.full((800, 727), 7.0, device="cuda", dtype=torch.float16)
        out = o.linear_int8(xb, s1, wb, s2, residual=r, out=wide[:, 3:723])
        _close(out, *_want(xb, s1, wb, s2, None, None, r))
        assert bool((wide[:, :3] == 7).all() and (wide[:, 723:] == 7).all())
    xb, wb = _codes((40 * 200 + 16,), 5)[15:15 + 40 * 200].view(40, 200), _codes((73 * 200,), 6)[15:15 + 72 * 200].view(72, 200)
    s1, s2 = _scales(40, 7, 0.02), _scales(72, 8, 0.01)
    # in place over the residual
    r = _rand((40, 72), torch.bfloat16, 9)
    want, e = _want(xb, s1, wb, s2, None, None, r)
    assert o.linear_int8(xb, s1, wb, s2, residual=r, out=r).data_ptr() == r.data_ptr()
    _close(r, want, e)


def test_no_rows_and_special_scales():
    o = _ops()
    w, ws = _codes((8, 64), 1), _scales(8, 2, 0.01)
    assert o.linear_int8(_codes((0, 64), 3), _scales(0, 4, 1.0), w, ws).shape == (0, 8)
    assert o.linear_int8(_rand((0, 64), torch.bfloat16, 3), None, w, ws).shape == (0, 8)
    x = _rand((70, 64), torch.bfloat16, 5)
    x[3, 5], x[40, 0], x[41, 63] = float("nan"), float("inf"), float("-inf")
    x[7] = 0
    for m in (8, 70):
        got = o.linear_int8(x[:m], None, w, ws)
        bad = torch.zeros(m, dtype=torch.bool, device="cuda")
        bad[[i for i in (3, 40, 41) if i < m]] = True
        assert torch.equal(got.isnan().all(-1), bad) and torch.equal(got.isnan().any(-1), bad)
        assert bool((got[7] == 0).all())


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 64), (4, 512), (9, 520), (2, 1000), (7, 2048), (5, 2056),
                                       (3, 4096), (900, 7168), (2, 8192), (3, 20000), (2, 32768), (2, 40000)])
def test_quantiser(dtype, rows, cols):
    o = _ops()
    x = _rand((rows, cols), DT[dtype], rows + cols)
    x[0, : cols // 2] *= 1e-3
    if rows > 2:
        x[1] = 0
        x[2] *= 1e-13 if dtype != "fp16" else 1e-4
    q, s = o.per_token_int8_quant(x)
    wq, wsc = _quant(x)
    assert s.shape == (rows, 1) and torch.equal(s.cpu(), wsc)
    assert torch.equal(q.cpu().float(), wq)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_quantiser_at_the_middle_between_codes(dtype):
    """Rows whose maximum is 127 times a value near one, so that quotients lie on and around the
    middles: every 16-bit value's neighbourhood of them, halves to the even code."""
    o = _ops()
    half = torch.arange(-127, 127, device="cuda").float() + 0.5
    steps = torch.arange(-3, 4, device="cuda").float() * torch.finfo(DT[dtype]).eps / 2
    body = (half[:, None] * (1 + steps[None, :])).reshape(-1)
    x = torch.stack([torch.cat([body * k, body.new_tensor([127.0 * k])]) for k in (1.0, 1.0 / 3, 0.37, 1.7, 1e-4)])
    x = x.to(DT[dtype])
    q, s = o.per_token_int8_quant(x)
    wq, wsc = _quant(x)
    assert torch.equal(s.cpu(), wsc) and torch.equal(q.cpu().float(), wq)


def test_quantiser_rows_anywhere():
    o = _ops()
    base = _rand((6, 4, 200), torch.bfloat16, 1)
    for x in (base[:, :, 3:131], base[:, 1], base.view(24, 200)[::2], base[:, :, :1], base[0, 0]):
        q, s = o.per_token_int8_quant(x)
        assert q.shape == x.shape and s.shape == x.shape[:-1] + (1,) and q.is_contiguous()
        wq, wsc = _quant(x)
        assert torch.equal(s.cpu(), wsc) and torch.equal(q.cpu().float(), wq)
    q, s = o.per_token_int8_quant(_rand((0, 64), torch.bfloat16, 1))
    assert q.shape == (0, 64) and s.shape == (0, 1)


def test_captured_and_replayed():
    """Two products quantised in the call in one graph, with new inputs and eager work in between."""
    o = _ops()
    x = _rand((61, 4096), torch.bfloat16, 1)
    w, ws = _codes((512, 4096), 2), _scales(512, 3, 0.0001)
    w2, ws2 = _codes((512, 256), 4), _scales(512, 5, 0.001)
    run = lambda: o.linear_int8(o.linear_int8(x, None, w, ws, activation="silu_and_mul"), None, w2, ws2)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        run()
    torch.cuda.current_stream().wait_stream(st)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = run()
    for seed in (10, 11, 12):
        x.copy_(_rand((61, 4096), torch.bfloat16, seed))
        want = run()
        y.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_many_rows_and_far_offsets():
    """Output elements past 2^31."""
    o = _ops()
    M, N, K = 70000, 32768, 64
    x, w = _codes((M, K), 1), _codes((N, K), 2)
    xs, ws = _scales(M, 3, 0.02), _scales(N, 4, 0.01)
    got = o.linear_int8(x, xs, w, ws)
    for m in (0, 65535, M - 1):
        _close(got[m:m + 1], *_want(x[m:m + 1], xs[m:m + 1], w, ws, None, None, None))


@pytest.mark.parametrize("M,K,N", [(5, 256, 40), (61, 1024, 200), (300, 256, 136), (300, 1001, 131), (515, 512, 1024)])
def test_biases_and_residuals_of_other_types(M, K, N):
    o = _ops()
    x, w = _codes((M, K), 1), _codes((N, K), 2)
    xs, ws = _scales(M, 3, 0.02), _scales(N, 4, 0.7 / (73 * math.sqrt(K)))
    for b in DT.values():
        for r in DT.values():
            for out in DT.values():
                bias, res = _rand(N, b, 5), _rand((M, N), r, 6)
                got = o.linear_int8(x, xs, w, ws, bias, "gelu", res, out_dtype=out)
                _close(got, *_want(x, xs, w, ws, bias, "gelu", res))
    # a residual of rows apart at any address
    res = _rand((M, N + 5), torch.bfloat16, 7)[:, 3:N + 3]
    _close(o.linear_int8(x, xs, w, ws, residual=res), *_want(x, xs, w, ws, None, None, res))


def test_vectors():
    o = _ops()
    w, ws = _codes((24, 64), 1), _scales(24, 2, 0.01)
    x = _rand(64, torch.float16, 3)
    q, s = o.per_token_int8_quant(x)
    assert q.shape == (64,) and s.shape == (1,)
    a, b = o.linear_int8(x, None, w, ws), o.linear_int8(q, s, w, ws, out_dtype=torch.float16)
    assert a.shape == (24,) and torch.equal(a, b)
    _close(a[None], *_want(q[None], s, w, ws, None, None, None))


def test_many_tiles_in_place_on_two_streams():
    """More tiles than workgroups, each stored over the residual that it adds, two products at once."""
    o = _ops()
    M, K, N = 3000, 384, 2320
    x, w, xs, ws = _codes((M, K), 1), _codes((N, K), 2), _scales(M, 3, 0.02), _scales(N, 4, 0.001)
    r = [_rand((M, N), torch.bfloat16, 5 + i) for i in range(2)]
    want = [_want(x, xs, w, ws, None, None, t) for t in r]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in r]
    for st, t in zip(streams, r):
        with torch.cuda.stream(st):
            o.linear_int8(x, xs, w, ws, residual=t, out=t)
    torch.cuda.synchronize()
    for t, v in zip(r, want):
        _close(t, *v)


@pytest.mark.parametrize("bad", ["scale", "no_scale", "weight_scale", "weight", "type", "fp32", "overlap", "columns", "k"])
def test_refusals(bad):
    o = _ops()
    x, w, xs, ws = _codes((6, 64), 1), _codes((32, 64), 2), _scales(6, 3, 1.0), _scales(32, 4, 1.0)
    x16 = _rand((6, 64), torch.bfloat16, 5)
    call = {"scale": lambda: o.linear_int8(x, xs[:5], w, ws), "no_scale": lambda: o.linear_int8(x, None, w, ws),
            "weight_scale": lambda: o.linear_int8(x, xs, w, ws[:31]), "weight": lambda: o.linear_int8(x16, None, x16, ws),
            "type": lambda: o.linear_int8(x16, xs, w, ws), "fp32": lambda: o.linear_int8(x16.float(), None, w, ws),
            "overlap": lambda: o.linear_int8(x16, None, w[:, :64], ws, out=x16[:, :32]),
            "columns": lambda: o.linear_int8(x[:, :32], xs, w, ws),
            "k": lambda: o.linear_int8(_codes((1, 1 << 17), 6), xs[:1], _codes((4, 1 << 17), 7), ws[:4])}[bad]
    with pytest.raises(RuntimeError):
        call()
