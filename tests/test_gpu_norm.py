"""GPU: rms_norm and rms_norm_quant against the formula in 64 bits.

Tolerances.  A 16-bit output is off by half a step of its type at most, on top
of the fp32 arithmetic before it.  The sum of squares has non-negative terms:
every partial sum's rounding is 2^-24 of it at most, and no kernel adds more
than 64 terms in a row before its tree of at most 12 levels, so the sum is off
by 80 * 2^-24 relative, its root by half, and y by that plus the roundings of
h, of the mean, of the root, of the reciprocal and of two products: 48 * 2^-24
in all (FP).  A scale adds three roundings, a code's quotient two more."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

FP = 48 * 2.0 ** -24
EPS = 1e-6
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _ops():
    from vllm_xpu_kernels import ops
    return ops


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rand(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=_gen(seed), device="cuda") * scale).to(dtype)


def _exact(x, w, r=None):
    h = x.double() if r is None else x.double() + r.double()
    y = h / torch.sqrt(h.pow(2).mean(-1, keepdim=True) + EPS) * w.double()
    return h, y


def _close(got, want, fp=FP):
    """got (a rounding of a value within fp of want) against want in 64 bits."""
    info = torch.finfo(got.dtype)
    err = (got.double() - want).abs()
    lim = (info.eps / 2 + fp) * want.abs() * (1 + 1e-6) + info.smallest_normal * info.eps / 2
    assert bool((err <= lim).all()), float((err - lim).max())


def _check_quant(q, s, y, group, ue8m0):
    v = y.view(y.shape[0], -1, group)
    c = torch.maximum(v.abs().amax(-1), torch.full((), 1e-10, dtype=torch.float64, device=y.device))
    c = torch.maximum(c / 448.0, torch.full((), 1 / (448.0 * 512.0), dtype=torch.float64, device=y.device))
    sd = s.double()
    if ue8m0:
        frac, _ = torch.frexp(sd)
        assert bool((frac == 0.5).all())
        assert bool((sd >= c * (1 - 2 * FP)).all()) and bool((sd < 2 * c * (1 + 2 * FP)).all())
    else:
        assert bool(((sd - c).abs() <= (FP + 3 * 2.0 ** -24) * c).all())
    t = (v / sd.unsqueeze(-1)).view(y.shape)
    err = (q.double() - t).abs()
    # half a step of e4m3 (2^-4 relative, 2^-10 below its normal range) of the value that fp32 has
    lim = torch.maximum(t.abs() * 2.0 ** -4, torch.full_like(t, 2.0 ** -10)) + 2 * FP * t.abs()
    assert bool((err <= lim).all()), float((err - lim).max())


SHAPES = [(1, 7168), (3, 512), (61, 4096), (5, 2880), (2, 8), (7, 1), (4, 33), (9, 1001), (130, 128),
          (3, 8192), (2, 8200), (2, 20000), (2, 32776), (2, 40000), (1, 70001), (300, 64), (1025, 80),
          (2049, 2048)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,H", SHAPES)
def test_rms_norm(dev, T, H, dtype):
    x = _rand((T, H), DT[dtype], 1, 3.0)
    w = _rand((H,), DT[dtype], 2) + 1
    out = _ops().rms_norm(x, w, EPS)
    _close(out, _exact(x, w)[1])


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,H", SHAPES)
def test_rms_norm_residual(dev, T, H, dtype):
    x, r = _rand((T, H), DT[dtype], 3), _rand((T, H), DT[dtype], 4, 5.0)
    w = _rand((H,), torch.float32, 5) + 1
    x0, r0 = x.clone(), r.clone()
    out, ro = _ops().rms_norm(x, w, EPS, residual=r)
    h, y = _exact(x, w, r)
    _close(out, y)
    _close(ro, h, 2.0 ** -24)
    assert torch.equal(x, x0) and torch.equal(r, r0)
    # in place: the residual's and the input's own buffers
    _ops().rms_norm(x, w, EPS, residual=r, residual_out=r, out=x)
    assert torch.equal(x, out) and torch.equal(r, ro)


@pytest.mark.parametrize("group,kind", [(128, "f32"), (64, "f32"), (32, "f32"), (128, "ue8m0"),
                                        (32, "e8m0"), (64, "e8m0"), (32, "u8")])
@pytest.mark.parametrize("T,H,dtype,res", [(1, 7168, "bf16", True), (61, 4096, "bf16", True),
                                           (33, 2880, "fp16", False), (5, 128, "bf16", False),
                                           (700, 512, "fp16", True), (3, 9216, "fp32", True),
                                           (2, 33280, "bf16", False), (2, 128 * 330, "bf16", True),
                                           (1030, 2048, "bf16", False)])
def test_rms_norm_quant(dev, T, H, dtype, res, group, kind):
    if H % group:
        H = H // group * group
    x = _rand((T, H), DT[dtype], 6, 2.0)
    r = _rand((T, H), DT[dtype], 7, 4.0) if res else None
    w = _rand((H,), DT[dtype], 8, 0.3) + 1
    sdt = {"f32": torch.float32, "ue8m0": torch.float32, "e8m0": torch.float8_e8m0fnu,
           "u8": torch.uint8}[kind]
    got = _ops().rms_norm_quant(x, w, EPS, residual=r, group_size=group, scale_dtype=sdt,
                                scale_ue8m0=kind == "ue8m0", with_norm=True)
    q, s, n = got[:3]
    h, y = _exact(x, w, r)
    _close(n, y)
    if res:
        _close(got[3], h, 2.0 ** -24)
    sv = torch.exp2(s.double() - 127) if kind == "u8" else s.double()
    _check_quant(q, sv, y, group, kind != "f32")
    # without the 16-bit output, scales transposed: the same codes and scales
    got2 = _ops().rms_norm_quant(x, w, EPS, residual=r, group_size=group, scale_dtype=sdt,
                                 scale_ue8m0=kind == "ue8m0", is_scale_transposed=True)
    assert len(got2) == (3 if res else 2)
    assert torch.equal(got2[0].view(torch.uint8), q.view(torch.uint8))
    assert got2[1].stride(0) == 1 or T == 1
    assert torch.equal(got2[1].double(), s.double())
    if res:   # the residual updated in place
        r2 = r.clone()
        got3 = _ops().rms_norm_quant(x, w, EPS, residual=r2, residual_out=r2, group_size=group,
                                     scale_dtype=sdt, scale_ue8m0=kind == "ue8m0", with_norm=True)
        for a, b in zip(got3, got):
            assert torch.equal(a.double(), b.double())
        assert got3[3] is r2


@pytest.mark.parametrize("T,heads,H,dtype", [(1003, 32, 128, "fp16"), (3, 5, 64, "bf16"),
                                             (17, 3, 80, "bf16"), (1, 8, 128, "fp32"),
                                             (9, 2, 33, "bf16"), (2, 1, 1500, "fp16")])
def test_rms_norm_heads_in_a_packed_projection(dev, T, heads, H, dtype):
    packed = _rand((T, heads + 4, H), DT[dtype], 9)
    w = _rand((H,), DT[dtype], 10) + 1
    x = packed[:, :heads]
    before = packed.clone()
    out = _ops().rms_norm(x, w, EPS)
    assert out.is_contiguous()
    _close(out, _exact(x, w)[1])
    assert torch.equal(packed, before)
    _ops().rms_norm(x, w, EPS, out=x)      # where they lie; the other heads stay
    assert torch.equal(packed[:, :heads], out) and torch.equal(packed[:, heads:], before[:, heads:])
    # into another head range of the same buffer
    if heads <= 4:
        packed.copy_(before)
        _ops().rms_norm(packed[:, :heads], w, EPS, out=packed[:, heads:2 * heads])
        assert torch.equal(packed[:, heads:2 * heads], out)
        assert torch.equal(packed[:, :heads], before[:, :heads])


def test_rms_norm_strides_and_alignment(dev):
    w = _rand((256,), torch.bfloat16, 11) + 1
    buf = _rand((40, 301), torch.bfloat16, 12)
    for x in (buf[:, 3:259], buf[::3, 8:264], _rand((4, 5, 6, 256), torch.bfloat16, 13),
              _rand((256,), torch.bfloat16, 14), _rand((1, 256), torch.bfloat16, 15).expand(7, 256),
              _rand((1 + 7 * 256,), torch.bfloat16, 16)[1:].view(7, 256)):
        got = _ops().rms_norm(x, w, EPS)
        _close(got, _exact(x, w)[1])
        q, s = _ops().rms_norm_quant(x, w, EPS, group_size=64)
        y = _exact(x, w)[1].reshape(-1, 256)
        _check_quant(q.view(-1, 256), s.double(), y, 64, False)
    # rows of an output with a stride of their own: what lies between them stays
    out = torch.full((40, 301), 7.0, dtype=torch.bfloat16, device=dev)
    _ops().rms_norm(buf[:, :256], w, EPS, out=out[:, 5:261])
    _close(out[:, 5:261], _exact(buf[:, :256], w)[1])
    assert bool((out[:, :5] == 7).all()) and bool((out[:, 261:] == 7).all())
    assert _ops().rms_norm(buf[:0, :256], w, EPS).shape == (0, 256)
    assert _ops().rms_norm_quant(buf[:0, :256], w, EPS)[1].shape == (0, 2)


@pytest.mark.parametrize("H", [256, 257, 7168])
def test_rms_norm_special_values(dev, H):
    w = torch.ones(H, dtype=torch.bfloat16, device=dev)
    x = _rand((5, H), torch.bfloat16, 17)
    x[0] = 0                      # eps alone under the root
    x[1, 3] = float("nan")        # the whole row
    x[2, 4] = float("inf")        # 0 everywhere, NaN at the infinity
    x[3] = 1e-30
    out = _ops().rms_norm(x, w, EPS)
    assert bool((out[0] == 0).all()) and bool(out[1].isnan().all())
    assert bool(out[2, 4].isnan()) and int(out[2].isnan().sum()) == 1 and int((out[2] == 0).sum()) == H - 1
    _close(out[3:], _exact(x[3:], w)[1])
    if H % 128 == 0:
        q, s = _ops().rms_norm_quant(x, w, EPS)
        assert bool((s[0] == 1 / (448 * 512)).all()) and bool((q[0].float() == 0).all())
        assert bool(q[1].float().isnan().all()) and bool(q[2, 4].float().isnan())
        assert int(q[2].float().isnan().sum()) == 1
        # a NaN of the weight: its code is NaN, the group's scale comes from the others
        w2 = w.clone()
        w2[7] = float("nan")
        q, s = _ops().rms_norm_quant(x[4:], w2, EPS)
        y = _exact(x[4:], w)[1]
        y[0, 7] = 0
        assert bool(q[0, 7].float().isnan())
        q2 = q.clone()
        q2[0, 7] = 0
        _check_quant(q2, s.double(), y, 128, False)


def test_rms_norm_many_rows(dev):
    """More rows than one grid dimension of 256-thread workgroups holds waves."""
    x = _rand((300000, 16), torch.bfloat16, 18)
    w = _rand((16,), torch.bfloat16, 19) + 1
    _close(_ops().rms_norm(x, w, EPS), _exact(x, w)[1])


def test_rms_norm_large_offsets(dev):
    """Rows whose byte offsets pass 2^32."""
    big = torch.zeros(3, (1 << 30) + 512, dtype=torch.bfloat16, device=dev)
    x = big[:, 8:264]
    x.copy_(_rand((3, 256), torch.bfloat16, 20))
    w = _rand((256,), torch.bfloat16, 21) + 1
    _close(_ops().rms_norm(x, w, EPS), _exact(x, w)[1])


def test_rms_norm_is_deterministic_and_runs_on_the_current_stream(dev):
    x, r = _rand((61, 4096), torch.bfloat16, 22), _rand((61, 4096), torch.bfloat16, 23)
    w = _rand((4096,), torch.bfloat16, 24) + 1
    want = _ops().rms_norm_quant(x, w, EPS, residual=r, with_norm=True)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = _ops().rms_norm_quant(x, w, EPS, residual=r, with_norm=True)
    st.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cap = _ops().rms_norm_quant(x, w, EPS, residual=r, with_norm=True)
    for seed in (30, 31, 32):
        x.copy_(_rand((61, 4096), torch.bfloat16, seed))
        g.replay()
        torch.cuda.synchronize()
        want = _ops().rms_norm_quant(x, w, EPS, residual=r, with_norm=True)
        for a, b in zip(cap, want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_rms_norm_refusals(dev):
    o = _ops()
    x, w = _rand((4, 256), torch.bfloat16, 1), _rand((256,), torch.bfloat16, 2)
    for call, msg in [
        (lambda: o.rms_norm(x, w[:128]), "hidden_size"),
        (lambda: o.rms_norm(x, w.half()), "weight must have the input's type"),
        (lambda: o.rms_norm(x, w.cpu()), "weight must be on a GPU"),
        (lambda: o.rms_norm(x.t(), w[:4].contiguous()), "contiguous in its last dimension"),
        (lambda: o.rms_norm(x, w, residual=x.half()), "residual must have the input's type"),
        (lambda: o.rms_norm(x, w, residual=x[:2]), "residual must have the input's shape"),
        (lambda: o.rms_norm(x.int(), w), "float32, bfloat16 or float16"),
        (lambda: o.rms_norm(x, w, out=x[:1].expand(4, 256)), "must not overlap"),
        (lambda: o.rms_norm(x[:3], w, out=x[1:]), "must not overlap"),
        (lambda: o.rms_norm_quant(x, w, group_size=16), "group_size must be"),
        (lambda: o.rms_norm_quant(x[:, :192], w[:192], group_size=128), "divisible by group_size"),
        (lambda: o.rms_norm_quant(x, w, scale_dtype=torch.bfloat16), "scales must be"),
    ]:
        with pytest.raises(RuntimeError, match=msg):
            call()
    r = torch.zeros_like(x)
    with pytest.raises(RuntimeError, match="must not overlap"):
        o.rms_norm(x, w, residual=r, residual_out=r, out=r)


def test_opcheck(dev):
    """The op's schema, meta kernel and tracing."""
    x, w = _rand((5, 256), torch.bfloat16, 1), _rand((256,), torch.bfloat16, 2)
    op = torch.ops._mi355_C.rms_norm.default
    e = torch.empty_like
    torch.library.opcheck(op, (e(x), None, None, None, x, w, None, EPS))
    torch.library.opcheck(op, (e(x), None, None, e(x), x, w, x.clone(), EPS))
    q = torch.zeros(5, 256, dtype=torch.float8_e4m3fn, device=dev)
    s = torch.zeros(5, 2, device=dev)
    torch.library.opcheck(op, (None, q, s, None, x, w, None, EPS, 128, True),
                          test_utils=("test_autograd_registration", "test_faketensor"))
    op = torch.ops._mi355_C.rms_norm_new.default
    torch.library.opcheck(op, (x, w, None, EPS))
    torch.library.opcheck(op, (x, w, x.clone(), EPS))
    for more in ((True, 128, None, True, False), (False, 32, torch.float8_e8m0fnu, False, True)):
        torch.library.opcheck(op, (x, w, x.clone(), EPS) + more,
                              test_utils=("test_autograd_registration", "test_faketensor"))


def test_traced_by_the_compiler_front_end(dev):
    """A function of the wrapper traces whole (fake tensors, functionalised) and gives the same."""
    x, w = _rand((5, 256), torch.bfloat16, 1), _rand((256,), torch.bfloat16, 2)
    o = _ops()
    f = torch.compile(lambda a, b: o.rms_norm(a, b, EPS), backend="aot_eager", fullgraph=True)
    assert torch.equal(f(x, w), o.rms_norm(x, w, EPS))
    assert math.isfinite(float(x.float().sum()))


def test_rms_norm_leading_dimensions_of_one(dev):
    """Slices that leave a dimension of one element between others: its stride
    does not count."""
    w = _rand((64,), torch.bfloat16, 61) + 1
    buf = _rand((6, 5, 3, 64), torch.bfloat16, 62)
    for x in (buf[:, 2:3], buf[:, 4:, 1:], buf[3:4, :, :2], buf[:, :, 1:2][:, 1:2], buf[2:3, 1:2, 2:]):
        _close(_ops().rms_norm(x, w, EPS), _exact(x, w)[1])
        y = x.contiguous()
        want, wr = _ops().rms_norm(y, w, EPS, residual=y)
        out = torch.full_like(buf, 7.0).as_strided(x.shape, x.stride(), x.storage_offset())
        got, r = _ops().rms_norm(x, w, EPS, residual=x, out=out)
        assert torch.equal(got, want) and torch.equal(r, wr)
    with pytest.raises(RuntimeError, match="do not fold"):
        _ops().rms_norm(buf[:, :2].unsqueeze(2).expand(6, 2, 2, 3, 64), w, EPS)


def _border_case(T, H, dtype, c, group, seed):
    """Rows of +-c under eps 0, so that y = +-weight exactly; the groups' largest weights at
    448 * 2^e, one float32 step (2^-23.8 of it) below and above it, or 1.5 times it.  -> x, weight,
    power-of-two scales"""
    g = torch.Generator().manual_seed(seed)
    n = H // group
    e = torch.randint(-6, 4, (n,), generator=g).double()
    off = torch.tensor([0.0, -2.0 ** -21, 2.0 ** -21, 3.5])[torch.randint(0, 4, (n,), generator=g)].double()
    top = 64.0 * torch.exp2(e) * (7 + off)
    w = top.unsqueeze(1) * (0.25 + 0.5 * torch.rand(n, group, generator=g).double())
    w[torch.arange(n), torch.randint(0, group, (n,), generator=g)] = top
    sign = torch.randint(0, 2, (T, H), generator=g) * 2.0 - 1
    x = (sign * c).to(DT[dtype])
    assert bool((x.double().abs() == c).all()) and bool((w.float().double().amax(1) == top).all())
    return x.cuda(), w.view(H).float().cuda(), torch.exp2(e + (off > 0)).cuda()


@pytest.mark.parametrize("group,kind", [(32, "e8m0"), (64, "ue8m0"), (128, "e8m0"), (128, "ue8m0")])
@pytest.mark.parametrize("H", [96, 384, 512, 768, 896, 2816, 2880, 4096, 6144, 7168, 33280, 40000])
def test_rms_norm_scales_at_powers_of_two(dev, H, group, kind):
    """A power-of-two scale is the least that is no less than max / 448, on the border and one step
    to either side of it, where fp32 cannot tell: not one group may double or halve.  Squares far from
    1 (their fp32 root is coarser than the border) among them."""
    H = max(H // group, 1) * group
    for i, (dtype, c) in enumerate([("bf16", 1.0), ("fp16", 1.5703125), ("fp32", 0.8515625),
                                    ("bf16", 1.5703125 * 2.0 ** 54), ("fp32", 1.2265625 * 2.0 ** -54)]):
        x, w, want = _border_case(7, H, dtype, c, group, 100 * i + H)
        sdt = torch.float8_e8m0fnu if kind == "e8m0" else torch.float32
        for res in (None, torch.zeros_like(x)):
            got = _ops().rms_norm_quant(x, w, 0.0, residual=res, group_size=group, scale_dtype=sdt,
                                        scale_ue8m0=kind == "ue8m0")
            s = got[1].double()
            assert torch.equal(s, want.expand_as(s)), (dtype, c, int((s != want).sum()))


def test_rms_norm_scales_at_powers_of_two_any_alignment(dev):
    """The same where rows start anywhere."""
    for H, group in ((384, 32), (2880, 64), (4096, 128)):
        x, w, want = _border_case(9, H, "bf16", 1.5703125, group, H)
        buf = torch.zeros(9, H + 5, dtype=x.dtype, device=dev)
        buf[:, 3:H + 3] = x
        s = _ops().rms_norm_quant(buf[:, 3:H + 3], w, 0.0, group_size=group,
                                  scale_dtype=torch.float8_e8m0fnu)[1].double()
        assert torch.equal(s, want.expand_as(s))


@pytest.mark.parametrize("quant", [False, True])
def test_rms_norm_more_rows_than_one_launch(dev, quant):
    """Launches take 2^21 rows each: the rows behind the first launch's, whole."""
    T, H = (1 << 21) + 37, 32
    x, r = _rand((T, H), torch.bfloat16, 71), _rand((T, H), torch.bfloat16, 72)
    w = _rand((H,), torch.bfloat16, 73) + 1
    if quant:
        q, s, n, ro = _ops().rms_norm_quant(x, w, EPS, residual=r, group_size=32, with_norm=True)
    else:
        n, ro = _ops().rms_norm(x, w, EPS, residual=r)
    for a in (0, (1 << 21) - 100, T - 1000):
        i = slice(a, a + 1000)
        h, y = _exact(x[i], w, r[i])
        _close(n[i], y)
        _close(ro[i], h, 2.0 ** -24)
        if quant:
            _check_quant(q[i], s[i].double(), y, 32, False)
    # 16 columns, several rows to a wave, without a residual
    x = _rand((T, 16), torch.bfloat16, 74)
    w = _rand((16,), torch.bfloat16, 75) + 1
    out = _ops().rms_norm(x, w, EPS)
    for a in (0, (1 << 21) - 100, T - 1000):
        _close(out[a:a + 1000], _exact(x[a:a + 1000], w)[1])


def test_rms_norm_into_other_heads_of_a_batch(dev):
    """Outputs between the inputs' rows, of any number of leading dimensions that fold: no overlap."""
    w = _rand((64,), torch.bfloat16, 81) + 1
    packed = _rand((2, 3, 10, 64), torch.bfloat16, 82)
    before = packed.clone()
    want, wr = _ops().rms_norm(before[:, :, :4].contiguous(), w, EPS, residual=before[:, :, :4].contiguous())
    got, r = _ops().rms_norm(packed[:, :, :4], w, EPS, residual=packed[:, :, :4],
                             residual_out=packed[:, :, :4], out=packed[:, :, 5:9])
    assert torch.equal(packed[:, :, 5:9], want) and torch.equal(packed[:, :, :4], wr)
    assert torch.equal(packed[:, :, 4], before[:, :, 4]) and torch.equal(packed[:, :, 9], before[:, :, 9])
    # heads that do meet, of one and of several leading dimensions
    for p in (packed, packed[0], packed.view(6, 10, 64)):
        for a, b in ((slice(0, 4), slice(3, 7)), (slice(2, 6), slice(0, 4))):
            with pytest.raises(RuntimeError, match="out must not overlap"):
                _ops().rms_norm(p[..., a, :], w, EPS, out=p[..., b, :])
