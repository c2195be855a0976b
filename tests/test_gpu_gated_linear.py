"""GPU: gated_linear and its gradients against the formula in 64 bits.

Tolerances.  The forward's sums and activation as linear's: an fp32 sum of K products is
off by less than e = 4 (sqrt(K) + 1) 2^-24 sum |x w|; the bias adds a rounding.
dz1 = d z2 f'(z1), dz2 = d f(z1): the errors of z1 and z2 come through |f''| < 1.2 and |f'| <
1.13; f' itself is off by less than 2^-19 (1 + |z|) (1 - sigmoid is off by 2^-23, times
z; the tanh form multiplies that by up to 1.6 (1 + 0.134 z^2) where 1 - sigmoid is not
yet 0, |z| < 5.5: 2^-17), and dz is rounded to x's type: half a step of each of its
values, at most (eps / 2), which every sum over dz carries as eps / 2 sum |dz w|.  The
sums of the products add theirs, and the output its rounding."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ACTS = ["silu_and_mul", "gelu_and_mul", "gelu_tanh_and_mul"]
U = 2.0 ** -24


def _ops():
    from vllm_xpu_kernels import ops
    return ops


def _rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _f(z, act):
    """The activation and its derivative in 64 bits."""
    if act.startswith("silu"):
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * torch.sigmoid(-z))
    if act.startswith("gelu_tanh"):
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return z * (1 + t) / 2, (1 + t) / 2 + z / 2 * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    p = torch.special.ndtr(z)
    return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def _sum_error(n):
    return 4 * (math.sqrt(n) + 1) * U


def _want(x, w, b, act, d):
    """{name: (value, error before the output's rounding)} in 64 bits."""
    half = torch.finfo(x.dtype).eps / 2
    low = torch.finfo(x.dtype).smallest_normal * half   # half of the smallest subnormal step
    x, w, d = x.detach().double(), w.detach().double(), d.double()
    M, K = x.shape
    n = w.shape[0] // 2
    z = x @ w.t()
    ez = _sum_error(K) * (x.abs() @ w.abs().t())
    if b is not None:
        z = z + b.detach().double()
        ez = ez + U * z.abs()
    g, u, eg, eu = z[:, :n], z[:, n:], ez[:, :n], ez[:, n:]
    f, df = _f(g, act)
    ef = 1.13 * eg + 2.0 ** -20 * (1 + g.abs()) * f.abs() + 2.0 ** -22 * g.abs()
    edf = 1.2 * eg + (2.0 ** -17 if act.startswith("gelu_tanh") else 2.0 ** -19 * (1 + g.abs()))
    out = f * u, ef * (u.abs() + eu) + f.abs() * eu + U * (f * u).abs()
    dz = torch.cat([d * u * df, d * f], 1)
    e = torch.cat([d.abs() * (eu * (df.abs() + edf) + u.abs() * edf), d.abs() * ef], 1) + 2 * U * dz.abs()
    r = half * dz.abs() + (1 + half) * e + low
    az = dz.abs() + r
    return {"out": out,
            "dx": (dz @ w, r @ w.abs() + _sum_error(2 * n) * (az @ w.abs())),
            "dw": (dz.t() @ x, r.t() @ x.abs() + _sum_error(M) * (az.t() @ x.abs())),
            "db": (dz.sum(0), e.sum(0) + _sum_error(M) * (dz.abs() + e).sum(0))}


def _close(got, want):
    y, e = want
    info = torch.finfo(got.dtype)
    lim = info.eps / 2 * y.abs() + (1 + info.eps) * e + info.smallest_normal * info.eps / 2
    assert got.shape == y.shape
    assert bool(((got.double() - y).abs() <= lim).all()), float(((got.double() - y).abs() / lim).max())


# rows x K x outputs: one row, few, tiles and their edges, splits, sizes that no vector divides
SIZES = [(1, 8, 8), (1, 1, 1), (2, 33, 5), (16, 512, 128), (17, 100, 33), (61, 2048, 768), (64, 64, 64), (65, 72, 200),
         (130, 1001, 515), (257, 264, 136), (300, 520, 1024), (512, 1024, 256), (1030, 128, 72), (2050, 256, 192), (800, 1003, 327),
         (600, 515, 129), (64, 77, 3), (100, 5003, 515)]


@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("act", ACTS)
def test_gradients(M, K, N, dtype, act):
    o = _ops()
    t = DT[dtype]
    x, w = _rand((M, K), t, 1).requires_grad_(), _rand((2 * N, K), t, 2, 1.5 / math.sqrt(K)).requires_grad_()
    b = _rand(2 * N, torch.float32 if act == ACTS[1] else t, 3).requires_grad_() if act != ACTS[0] else None
    d = _rand((M, N), t, 4)
    want = _want(x, w, b, act, d)
    out = o.gated_linear(x, w, b, act)
    _close(out.detach(), want["out"])
    leaves = [x, w] + ([b] if b is not None else [])
    grads = torch.autograd.grad(out, leaves, d)
    for g, leaf, name in zip(grads, leaves, ("dx", "dw", "db")):
        assert g.dtype == leaf.dtype and g.shape == leaf.shape
        _close(g, want[name])
    # the forward without gradients
    with torch.no_grad():
        _close(o.gated_linear(x, w, b, act), want["out"])


@pytest.mark.parametrize("need", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 1, 1)])
def test_gradients_that_are_not_asked_for(need):
    """Frozen inputs, weights or biases get none, the others theirs."""
    o = _ops()
    x, w, b = (_rand(s, torch.bfloat16, i, c).requires_grad_(bool(n)) for i, (s, n, c) in enumerate(
        zip([(70, 136), (2 * 96, 136), (192,)], need, (1.0, 0.1, 1.0))))
    d = _rand((70, 96), torch.bfloat16, 9)
    want = _want(x, w, b, "silu_and_mul", d)
    o.gated_linear(x, w, b).backward(d)
    for t, n, name in zip((x, w, b), need, ("dx", "dw", "db")):
        assert (t.grad is not None) == bool(n)
        if n:
            _close(t.grad, want[name])


def test_against_differences():
    """The directional derivative along v, from two calls of the forward: off by the roundings of their
    outputs and by what a difference quotient of the formula itself is off."""
    o = _ops()
    act, h = "silu_and_mul", 2.0 ** -5
    for seed in range(3):
        x = _rand((33, 64), torch.float16, seed)
        w, d = _rand((96, 64), torch.float16, seed + 10, 0.1), _rand((33, 48), torch.float16, seed + 20)
        v = torch.sign(_rand((33, 64), torch.float16, seed + 30))
        hi, lo = x + h * v, x - h * v
        step = (hi.double() - lo.double())            # what the rounded points are apart
        outs = [o.gated_linear(p, w, None, act).double() for p in (hi, lo)]
        got = ((outs[0] - outs[1]) * d.double()).sum()
        wants = [_want(p, w, None, act, d) for p in (hi, lo)]
        ref = ((wants[0]["out"][0] - wants[1]["out"][0]) * d.double()).sum()
        half = torch.finfo(torch.float16).eps / 2
        noise = sum((d.double().abs() * (half * t["out"][0].abs() + 2 * t["out"][1] + 2.0 ** -25)).sum() for t in wants)
        assert abs(got - ref) <= noise
        xr = x.clone().requires_grad_()
        dx, = torch.autograd.grad(o.gated_linear(xr, w, None, act), xr, d)
        at = _want(x, w, None, act, d)["dx"]
        lim = ((half * at[0].abs() + 2 * at[1] + 2.0 ** -25) * step.abs()).sum()
        truncation = abs((at[0] * step).sum() - ref)
        slope = (dx.double() * step).sum()
        assert abs(slope - got) <= noise + truncation + lim
        assert abs(slope) > 3 * (noise + truncation + lim) or abs(slope - ref) <= truncation + lim


def test_large_and_special_gates():
    """Gates far to both sides: f' is 0 or 1 there, not NaN; z beyond fp16's range is kept."""
    o = _ops()
    for act in ACTS:
        for big in (30.0, 1e4, 1e18):
            t = torch.bfloat16
            x = torch.ones(20, 8, dtype=t, device="cuda").requires_grad_()
            w = torch.zeros(16, 8, dtype=t, device="cuda")
            w[:4, 0], w[4:8, 0], w[8:, 0] = big, -big, 1.0
            w.requires_grad_()
            out = o.gated_linear(x, w, None, act)
            dx, dw = torch.autograd.grad(out, [x, w], torch.ones_like(out))
            assert bool(dx.isfinite().all() and dw.isfinite().all())
            # dz1 = f': 1 and 0; dz2 = f: big and 0
            assert torch.allclose(dw[:4, 0].float(), torch.full((4,), 20.0, device="cuda"))
            assert bool((dw[4:8, 0].float().abs() < 1e-9).all())
            assert torch.allclose(dw[8:12, 0].double(), w[:4, 0].double() * 20, rtol=2 ** -7)
    x = torch.full((3, 8), 200.0, dtype=torch.float16, device="cuda").requires_grad_()
    w = torch.zeros(4, 8, dtype=torch.float16, device="cuda")
    w[0], w[2] = 100.0, 1e-4                       # gate 160000, factor 0.16
    out = o.gated_linear(x, w, None, "silu_and_mul")
    want = _want(x, w, None, "silu_and_mul", torch.full((3, 2), 2.0 ** -12, dtype=torch.float16, device="cuda"))
    _close(out.detach(), want["out"])
    _close(torch.autograd.grad(out, x, torch.full_like(out, 2.0 ** -12))[0], want["dx"])


def test_infinities_and_nan_stay_in_their_rows():
    o = _ops()
    x, w = _rand((70, 64), torch.bfloat16, 1), _rand((64, 64), torch.bfloat16, 2, 0.2)
    x[5, 3], x[40, 63] = float("nan"), float("inf")
    x.requires_grad_()
    out = o.gated_linear(x, w)
    d = _rand((70, 32), torch.bfloat16, 3)
    d[60, 1] = float("nan")
    dx, = torch.autograd.grad(out, x, d)
    bad = torch.zeros(70, dtype=torch.bool, device="cuda")
    bad[[5, 40, 60]] = True
    assert torch.equal(~dx.isfinite().all(-1), bad)


def test_layouts():
    """Leading dimensions, rows apart and unaligned, expanded and permuted gradients, broadcast inputs."""
    o = _ops()
    act = "silu_and_mul"
    for k0 in (0, 8, 3):
        xb, wb = _rand((6, 7, 160), torch.bfloat16, 1), _rand((80, 160), torch.bfloat16, 2, 0.1)
        x, w = xb[:, :, k0:k0 + 136].detach().requires_grad_(), wb[:, k0:k0 + 136].detach().requires_grad_()
        out = o.gated_linear(x, w)
        assert out.shape == (6, 7, 40)
        grads = {"sum": out.new_ones(1).expand(out.shape), "permuted": _rand((40, 7, 6), torch.bfloat16, 3).permute(2, 1, 0),
                 "apart": _rand((6, 7, 50), torch.bfloat16, 4)[:, :, 5:45],
                 "crossed": _rand((7, 6, 40), torch.bfloat16, 5).transpose(0, 1)}
        for d in grads.values():
            want = _want(x.reshape(42, 136), w, None, act, d.reshape(42, 40))
            dx, dw = torch.autograd.grad(out, [x, w], d, retain_graph=True)
            _close(dx.reshape(42, 136), want["dx"])
            _close(dw, want["dw"])
    # many rows, so that operands are copied where their rows lie anywhere
    for k0, k in ((0, 1000), (8, 1000), (3, 1000), (0, 1003)):
        xb, wb = _rand((700, 1016), torch.float16, 1), _rand((800, 1016), torch.float16, 2, 0.05)
        x, w = xb[:, k0:k0 + k].detach().requires_grad_(), wb[:, k0:k0 + k].detach().requires_grad_()
        d = _rand((700, 400), torch.float16, 3)
        want, out = _want(x, w, None, act, d), o.gated_linear(x, w)
        _close(out.detach(), want["out"])
        for g, name in zip(torch.autograd.grad(out, [x, w], d), ("dx", "dw")):
            _close(g, want[name])
    # one row for all: its gradient is the sum
    row = _rand((1, 64), torch.bfloat16, 6).requires_grad_()
    w = _rand((64, 64), torch.bfloat16, 7, 0.1)
    d = _rand((9, 32), torch.bfloat16, 8)
    got, = torch.autograd.grad(o.gated_linear(row.expand(9, 64), w), row, d)
    full = _want(row.expand(9, 64), w, None, act, d)["dx"]
    y, e = full[0].sum(0, keepdim=True), full[1].sum(0, keepdim=True)
    # (the nine rows' outputs are rounded, and so are torch's partial sums of them)
    _close(got, (y, e + 9 * 2.0 ** -8 * full[0].abs().sum(0, keepdim=True)))


def test_no_rows():
    o = _ops()
    x = _rand((0, 64), torch.bfloat16, 1).requires_grad_()
    w, b = _rand((32, 64), torch.bfloat16, 2).requires_grad_(), _rand(32, torch.bfloat16, 3).requires_grad_()
    out = o.gated_linear(x, w, b)
    dx, dw, db = torch.autograd.grad(out, [x, w, b], torch.zeros_like(out))
    assert out.shape == (0, 16) and dx.shape == (0, 64)
    assert dw.shape == w.shape and bool((dw == 0).all()) and bool((db == 0).all())


def test_same_bits_every_time():
    o = _ops()
    x, w = _rand((777, 640), torch.bfloat16, 1).requires_grad_(), _rand((2 * 328, 640), torch.bfloat16, 2, 0.05).requires_grad_()
    b, d = _rand(656, torch.float32, 3).requires_grad_(), _rand((777, 328), torch.bfloat16, 4)
    first = torch.autograd.grad(o.gated_linear(x, w, b), [x, w, b], d)
    for _ in range(3):
        for a, c in zip(first, torch.autograd.grad(o.gated_linear(x, w, b), [x, w, b], d)):
            assert torch.equal(a, c)


def test_step_captured_and_replayed():
    o = _ops()
    x, w = _rand((200, 256), torch.bfloat16, 1).requires_grad_(), _rand((256, 256), torch.bfloat16, 2, 0.1).requires_grad_()
    b, d = _rand(256, torch.float32, 3).requires_grad_(), _rand((200, 128), torch.bfloat16, 4)
    run = lambda: torch.autograd.grad(o.gated_linear(x, w, b), [x, w, b], d)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        run()
    torch.cuda.current_stream().wait_stream(st)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = run()
    for seed in (10, 11, 12):
        with torch.no_grad():
            x.copy_(_rand((200, 256), torch.bfloat16, seed))
            d.copy_(_rand((200, 128), torch.bfloat16, seed + 100))
        want = run()
        g.replay()
        torch.cuda.synchronize()
        for a, c in zip(got, want):
            assert torch.equal(a, c)


def test_on_another_stream():
    """Two steps at once on streams of their own."""
    o = _ops()
    data = [(_rand((300, 512), torch.bfloat16, i).requires_grad_(), _rand((512, 512), torch.bfloat16, i + 5, 0.05).requires_grad_(),
             _rand((300, 256), torch.bfloat16, i + 9)) for i in range(2)]
    want = [torch.autograd.grad(o.gated_linear(x, w), [x, w], d) for x, w, d in data]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in data], []
    for s, (x, w, d) in zip(streams, data):
        with torch.cuda.stream(s):
            got.append([torch.autograd.grad(o.gated_linear(x, w), [x, w], d) for _ in range(3)])
    torch.cuda.synchronize()
    for g, c in zip(got, want):
        for step in g:
            assert all(torch.equal(a, b) for a, b in zip(step, c))


def test_a_step_of_a_block_and_its_int8_form():
    """As they are used together: a gated feed-forward block's step in 16 bits (the down product torch's),
    then its weights quantised per channel and the block run on int8 products."""
    o = _ops()
    x = _rand((48, 512), torch.bfloat16, 1)
    w13 = _rand((2 * 256, 512), torch.bfloat16, 2, 0.04).requires_grad_()
    w2 = _rand((512, 256), torch.bfloat16, 3, 0.06).requires_grad_()
    g = o.gated_linear(o.rms_norm(x, x.new_ones(512)), w13)
    y = torch.nn.functional.linear(g, w2)
    y.float().square().mean().backward()
    with torch.no_grad():
        w13 -= 0.1 * w13.grad
        w2 -= 0.1 * w2.grad
        h = o.rms_norm(x, x.new_ones(512))
        want = o.linear(o.linear(h, w13, activation="silu_and_mul"), w2).float()
        (q13, s13), (q2, s2) = o.per_token_int8_quant(w13), o.per_token_int8_quant(w2)
        a = o.linear_int8(h, None, q13, s13, activation="silu_and_mul")
        got = o.linear_int8(a, None, q2, s2, residual=x)
    # four quantisations to 127 steps of a row's largest value, some 3.5 times its rms: each
    # adds 3.5 / 127 / sqrt(12) = 0.8 % of a sum's size, the gated product carries three of them
    diff = got.float() - x.float() - want
    assert float(diff.norm() / want.norm()) < 4 * 0.008 + 2 ** -7 * float(x.float().norm() / want.norm())


def test_opcheck():
    """Schemas, autograd registration, fake tensors and AOT dispatch of the operators here and of the int8
    ones; the bits of two calls of one operator agree."""
    from vllm_xpu_kernels import ops
    assert ops
    n = torch.ops._mi355_C
    x, w, b = _rand((5, 64), torch.bfloat16, 1), _rand((32, 64), torch.bfloat16, 2, 0.1), _rand(32, torch.float32, 3)
    q, s = n.per_token_int8_quant(x)
    wq, ws = n.per_token_int8_quant(w)
    out, z = n.gated_linear_keep(x, w, b, 5)
    d = torch.ones_like(out)
    for op, args in (
            (n.per_token_int8_quant, (x,)), (n.linear_int8_new, (q, s, wq, ws, b, None, 0, torch.bfloat16)),
            (n.linear_int8_new, (x, None, wq, ws, None, None, 5, torch.float32)),
            (n.linear_int8, (torch.empty(5, 32, device="cuda"), q, s, wq, ws, None, None, 0)),
            (n.gated_linear_keep, (x, w, b, 6)), (n.gated_linear_backward, (d, x, w, z, 5, torch.float32)),
            (n.gated_linear, (x, w, b, 7)),
            (n.gated_linear, (x.clone().requires_grad_(), w.clone().requires_grad_(), b.clone().requires_grad_(), 5))):
        torch.library.opcheck(op.default, args)


def test_traced_by_aot_autograd():
    """A step of a compiled function (traced forward and backward, run eagerly) is the eager one's."""
    from vllm_xpu_kernels import ops
    x, w = _rand((6, 64), torch.bfloat16, 1).requires_grad_(), _rand((32, 64), torch.bfloat16, 2, 0.1).requires_grad_()
    step = lambda x, w: ops.gated_linear(x, w).float().square().sum()
    want = torch.autograd.grad(step(x, w), [x, w])
    got = torch.autograd.grad(torch.compile(step, backend="aot_eager")(x, w), [x, w])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_changed_input_is_noticed():
    o = _ops()
    x, w = _rand((6, 64), torch.bfloat16, 1), _rand((32, 64), torch.bfloat16, 2, 0.1).requires_grad_()
    out = o.gated_linear(x, w)
    x.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


@pytest.mark.parametrize("bad", ["type", "half", "columns", "strides", "bias", "device"])
def test_refusals(bad):
    o = _ops()
    x, w, b = _rand((6, 64), torch.bfloat16, 1).requires_grad_(), _rand((32, 64), torch.bfloat16, 2), _rand(32, torch.float32, 3)
    change = {"type": lambda: (x.float(), w.float(), b), "half": lambda: (x, w[:31], b[:31]),
              "columns": lambda: (x[:, :32], w, b), "strides": lambda: (x, w.t().contiguous().t(), b),
              "bias": lambda: (x, w, b[:16]), "device": lambda: (x, w.cpu(), b)}[bad]
    with pytest.raises(RuntimeError):
        o.gated_linear(*change())


def test_vectors_and_two_backward_passes():
    o = _ops()
    x, w = _rand(64, torch.bfloat16, 1).requires_grad_(), _rand((48, 64), torch.bfloat16, 2, 0.1).requires_grad_()
    b = _rand(48, torch.float16, 3).requires_grad_()
    out = o.gated_linear(x, w, b)
    assert out.shape == (24,)
    for seed in (4, 5):
        d = _rand(24, torch.bfloat16, seed)
        want = _want(x[None], w, b, ACTS[0], d[None])
        dx, dw, db = torch.autograd.grad(out, [x, w, b], d, retain_graph=True)
        _close(dx[None], want["dx"])
        _close(dw, want["dw"])
        _close(db, want["db"])
        assert db.dtype == torch.float16


def test_one_tensor_as_input_and_weight():
    o = _ops()
    x = _rand((64, 72), torch.bfloat16, 1, 0.3).requires_grad_()
    d = _rand((64, 32), torch.bfloat16, 2)
    want = _want(x, x, None, ACTS[0], d)
    got, = torch.autograd.grad(o.gated_linear(x, x), x, d)
    # (two rounded gradients, and the rounding of their sum)
    half = 2.0 ** -8
    _close(got, (want["dx"][0] + want["dw"][0], want["dx"][1] + want["dw"][1] +
                 half * (want["dx"][0].abs() + want["dw"][0].abs() + want["dx"][1] + want["dw"][1])))


@pytest.mark.parametrize("K,N", [(512, 768), (1000, 520)])
def test_many_tiles(K, N):
    """More tiles than workgroups in each of the three products; and the rows of an expanded weight."""
    o = _ops()
    M = 5000
    x, w = _rand((M, K), torch.bfloat16, 1).requires_grad_(), _rand((2 * N, K), torch.bfloat16, 2, 0.05).requires_grad_()
    d = _rand((M, N), torch.bfloat16, 3)
    want = _want(x, w, None, ACTS[0], d)
    out = o.gated_linear(x, w)
    _close(out.detach(), want["out"])
    dx, dw = torch.autograd.grad(out, [x, w], d)
    _close(dx, want["dx"])
    _close(dw, want["dw"])
    row = _rand((1, K), torch.bfloat16, 4, 0.05)
    wide = row.expand(2 * N, K)
    want = _want(x, wide, None, ACTS[0], d)
    out = o.gated_linear(x, wide)
    _close(out.detach(), want["out"])
    _close(torch.autograd.grad(out, x, d)[0], want["dx"])


def test_a_pass_that_asks_for_less():
    """Gradients of some of the tensors that require one: the same bits, and no tensor for the others."""
    o = _ops()
    x, w = _rand((130, 96), torch.bfloat16, 1).requires_grad_(), _rand((128, 96), torch.bfloat16, 2, 0.1).requires_grad_()
    b, d = _rand(128, torch.float32, 3).requires_grad_(), _rand((130, 64), torch.bfloat16, 4)
    y = o.gated_linear(x, w, b)
    want = torch.autograd.grad(y, [x, w, b], d, retain_graph=True)
    for which in ((0,), (1,), (2,), (0, 2), (1, 2)):
        got = torch.autograd.grad(y, [(x, w, b)[i] for i in which], d, retain_graph=True)
        assert all(torch.equal(g, want[i]) for g, i in zip(got, which))


def test_capture_beside_a_graph_of_the_same_leaves():
    """A step captured while an eager graph of its leaves lives is refused before it records anything; without
    the graph it is captured."""
    o = _ops()
    x, w = _rand((64, 64), torch.bfloat16, 1).requires_grad_(), _rand((128, 64), torch.bfloat16, 2, 0.1).requires_grad_()
    d = _rand((64, 64), torch.bfloat16, 3)
    run = lambda: torch.autograd.grad(o.gated_linear(x, w), [x, w], d)
    want = run()
    lives = o.gated_linear(x, w)
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="same leaves"), torch.cuda.graph(g):
        o.gated_linear(x, w)
    del lives
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = run()
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, run()))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("M,K,N,dtype", [(4323, 8456, 684, torch.bfloat16), (3216, 8960, 2039, torch.float16),
                                         (4078, 8856, 737, torch.bfloat16)])
def test_gradients_together_and_alone(M, K, N, dtype):
    """Sizes at which both products run in one launch: their bits are those of each alone, which a sample of
    rows and columns holds to the formula."""
    o = _ops()
    x, w = _rand((M, K), dtype, 1).requires_grad_(), _rand((2 * N, K), dtype, 2, 0.02).requires_grad_()
    d = _rand((M, N), dtype, 3)
    y = o.gated_linear(x, w)
    dx, dw = torch.autograd.grad(y, [x, w], d, retain_graph=True)
    assert torch.equal(dx, torch.autograd.grad(y, x, d, retain_graph=True)[0])
    assert torch.equal(dw, torch.autograd.grad(y, w, d)[0])
    # the product, and its fp32 sum's error: 2^-24 of the sum of sizes for each of its terms
    both = lambda a, b: (a @ b, a.shape[1] * 2 ** -24 * (a.abs() @ b.abs()))
    with torch.no_grad():
        dz = torch.ops._mi355_C.gated_linear_backward.default(
            d, torch.eye(M, device="cuda", dtype=dtype), None, torch.ops._mi355_C.gated_linear_keep(x, w, None, 5)[1], 5,
            None)[1]  # [2 N, M]: dz itself, which the products take
        rows = torch.tensor([0, 1, 255, 256, M // 2, M - 1], device="cuda")
        _close(dx[rows], both(dz[:, rows].double().t().contiguous(), w.double()))
        cols = torch.tensor([0, 1, N - 1, N, N + 255, 2 * N - 1], device="cuda")
        _close(dw[cols], both(dz[cols].double(), x.double()))
