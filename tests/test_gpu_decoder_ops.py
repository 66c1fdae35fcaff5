"""The decoder-layer operators on fp32 / bf16 / fp16 tensors, on the GPU through the public entry points: rotary positions, the product
with bias, activation and residual, and the expert layer for a few tokens, each against the formula in 64 bits.

Tolerances are sums of roundings: u = half a step of the result's type relative to the value, 2^-24 per fp32 operation of a sum
(times the sum of the magnitudes), and a few 2^-24 for an elementary function."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U24 = 2.0 ** -24
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
HALF_STEP = {"fp32": 2.0 ** -24, "bf16": 2.0 ** -8, "fp16": 2.0 ** -11}      # of the value, for results in the normal range
TINY = {"fp32": 0.0, "bf16": 0.0, "fp16": 2.0 ** -25}                         # half a step below the normal range
ACTS = ("none", "relu", "gelu_erf", "gelu_tanh", "leaky", "silu", "tanh")


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


def rand(gen, *shape, kind="fp32", scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).to(TYPES[kind]).cuda()


def within(got, want, bound, kind, what):
    """|got - want| <= bound + one rounding of the result, elementwise."""
    assert got.dtype == TYPES[kind] and got.shape == want.shape
    bound = bound + HALF_STEP[kind] * (want.abs() + bound) + TINY[kind]
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values off, worst {float((off / bound.clamp_min(1e-300)).max()):.3g} of the bound"


# ---------------------------------------------------------------------------------------------------------------- rotary positions
def rope_exact(x, pos, w, amp, layout, inverse=False):
    """(value, bound) in 64 bits; pos (B, S)."""
    x, rd = x.double(), 2 * w.numel()
    ang = pos.double()[..., None, None] * w
    c, s = ang.cos() * amp, ang.sin() * amp * (-1 if inverse else 1)
    i, j = (slice(0, rd // 2), slice(rd // 2, rd)) if layout == "half" else (slice(0, rd, 2), slice(1, rd, 2))
    a, b, y, e = x[..., i], x[..., j], x.clone(), torch.zeros_like(x)
    y[..., i], y[..., j] = a * c - b * s, b * c + a * s
    # sine and cosine of an fp32 argument, their scaling, two products and a sum; the angle itself to a few 2^-53
    e[..., i] = e[..., j] = (a.abs() + b.abs()) * amp * (6 * U24 + 8 * 2.0 ** -53 * ang.abs())
    return y, e


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("B,S,Hq,Hk,dh,rd,first", [
    (1, 1, 1, 1, 2, 2, 0),                 # the smallest
    (8, 1, 16, 8, 64, 64, 873),            # one token of a batch
    (2, 37, 6, 2, 96, 48, 5),              # part of the head
    (1, 3, 5, 1, 80, 18, 10 ** 6),         # far, widths that fill no vector
    (3, 5, 3, 3, 7, 6, 40),                # odd head width
    (1, 2, 2, 1, 520, 514, 2 ** 31 - 2),   # wide heads, the farthest positions
    (2, 1030, 4, 1, 128, 128, 0),
    (1, 1, 70, 5, 256, 256, 12),           # one token of many heads: several workgroups a token
    (3, 2, 2, 1, 1100, 1030, 9),           # more pieces a head than threads, with a tail
])
def test_rope(dev, kind, layout, B, S, Hq, Hk, dh, rd, first):
    from autodiffusion_amd import ops
    g = torch.Generator().manual_seed(B + S + dh)
    q, k = rand(g, B, S, Hq, dh, kind=kind), rand(g, B, S, Hk, dh, kind=kind)
    w, amp = ops.rope_frequencies(rd, 1e4, "parts" if rd > 2 else None, factor=4.0)
    pos = (first + torch.arange(S).repeat(B, 1) + 3 * torch.arange(B)[:, None]).cuda()
    for inverse in (False, True):
        qo, ko = ops.rope(q, k, pos, w, amp, layout, inverse=inverse)
        for x, y in ((q, qo), (k, ko)):
            within(y, *rope_exact(x, pos, w, amp, layout, inverse), kind, "rope")
            assert torch.equal(y[..., rd:], x[..., rd:])


def test_rope_orders_strides_and_in_place(dev):
    """Heads before tokens, a slice of a fused q / k / v product, packed tokens, shared and integer positions, one tensor, in place: the bits
    of the plain call, and nothing behind the tensors touched."""
    from autodiffusion_amd import ops
    g = torch.Generator().manual_seed(1)
    B, S, Hq, Hk, dh = 2, 33, 4, 2, 64
    w, amp = ops.rope_frequencies(40, 1e6)
    qkv = rand(g, B, S, Hq + 2 * Hk, dh, kind="bf16")
    q, k = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk]
    pos = torch.arange(7, 7 + S).cuda()
    ref = ops.rope(q.contiguous(), k.contiguous(), pos, w, amp)
    for got in (ops.rope(q, k, pos, w, amp), ops.rope(q, k, 7, w, amp), ops.rope(q, k, pos[None].expand(B, S), w, amp)):
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    assert torch.equal(ops.rope(q, None, pos, w, amp)[0], ref[0]) and ops.rope(q, None, pos, w, amp)[1] is None
    hq, hk = q.transpose(1, 2).contiguous(), k.transpose(1, 2).contiguous()                      # (B, H, S, dh) storage
    got = ops.rope(hq.transpose(1, 2), hk.transpose(1, 2), pos, w, amp)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    packed = ops.rope(q.reshape(B * S, Hq, dh), k.reshape(B * S, Hk, dh), pos.repeat(B), w, amp)
    assert torch.equal(packed[0].reshape(q.shape), ref[0]) and torch.equal(packed[1].reshape(k.shape), ref[1])
    keep = qkv.clone()
    ops.rope(q, k, pos, w, amp, inplace=True)
    assert torch.equal(q, ref[0]) and torch.equal(k, ref[1]) and torch.equal(qkv[:, :, Hq + Hk:], keep[:, :, Hq + Hk:])
    odd = rand(g, B, S, Hq, dh + 1, kind="bf16")[..., 1:]                                          # rows that start on no vector
    assert torch.equal(ops.rope(odd, None, pos, w, amp)[0], ops.rope(odd.contiguous(), None, pos, w, amp)[0])
    empty, _ = ops.rope(q[:, :0], None, 0, w, amp)
    assert empty.shape == (B, 0, Hq, dh)
    last = ops.rope(q[..., :40].transpose(2, 3).contiguous().transpose(2, 3), None, pos, w, amp)[0]   # adjacent values are not adjacent in memory
    assert torch.equal(last, ops.rope(q[..., :40].contiguous(), None, pos, w, amp)[0])


def test_rope_frequencies(dev):
    from autodiffusion_amd import ops
    w, a = ops.rope_frequencies(64, 1e4, device="cpu")
    assert a == 1.0 and w.dtype == torch.float64 and float(w[0]) == 1.0 and abs(float(w[16]) - 0.01) < 1e-16
    lin, _ = ops.rope_frequencies(64, 1e4, "linear", 8.0, device="cpu")
    assert torch.equal(lin, w / 8)
    base, _ = ops.rope_frequencies(64, 1e4, "base", 8.0, device="cpu")
    assert float(base[0]) == 1.0 and abs(float(base[-1] / w[-1]) - 1 / 8) < 1e-12
    parts, amp = ops.rope_frequencies(64, 1e4, "parts", 8.0, trained_length=4096, device="cpu")
    turns = 4096 * w / (2 * math.pi)
    assert torch.equal(parts[turns >= 32], w[turns >= 32]) and torch.allclose(parts[turns <= 1], w[turns <= 1] / 8, rtol=1e-15, atol=0)
    assert abs(amp - (0.1 * math.log(8) + 1)) < 1e-15


# ---------------------------------------------------------------------------------------------------------------- product with epilogue
def act64(z, act):
    f = torch.nn.functional
    return {"none": lambda v: v, "relu": f.relu, "gelu_erf": f.gelu, "gelu_tanh": lambda v: f.gelu(v, approximate="tanh"),
            "leaky": lambda v: f.leaky_relu(v, 0.01), "silu": f.silu, "tanh": torch.tanh}[act](z)


def slope64(z, act):
    z = z.detach().requires_grad_()
    with torch.enable_grad():
        return torch.autograd.grad(act64(z, act).sum(), z)[0]


def slope_codes(z, act, kind):
    """The slopes of ``act`` at z in the form the forward keeps them, and their values in 64 bits."""
    d = slope64(z.double(), act)
    if kind == "fp32":
        return d.float(), d.float().double()
    q = (d * 32768 + 8192.5).int()
    return torch.where(q > 32767, q - 65536, q).to(torch.int16), d if act == "leaky" else (q.double() - 8192) / 32768


def slope_values(q, act, kind):
    if kind == "fp32":
        return q.double()
    u = q.int() & 0xFFFF
    d = torch.where(u > 16384, 1.0, 0.01).double() if act == "leaky" else (u.double() - 8192) / 32768
    return torch.where(u == 0, torch.full_like(d, math.nan), d)


def linear_exact(x, w, b, res, act):
    """(y, bound, z, bound of z) in 64 bits."""
    x, w = x.double(), w.double()
    z, mag = x @ w.t(), x.abs() @ w.abs().t()
    if b is not None:
        z, mag = z + b.double(), mag + b.double().abs()
    ez = (x.shape[1] + 2) * U24 * mag
    y = act64(z, act)
    e = ez if act == "none" else 1.13 * ez + 8 * U24 * (z.abs() + 1)          # slopes are at most 1.13
    if res is not None:
        y = y + res.double()
        e = e + 2 * U24 * (y.abs() + res.double().abs())
    return y, e, z, ez


SHAPES = [  # rows, n, k
    (1, 8, 8), (1, 1, 1), (1, 1024, 512), (3, 40, 24), (16, 48, 1000), (17, 100, 36), (33, 16, 72), (64, 130, 257), (24, 520, 96),
    (65, 64, 64), (65, 1, 3), (130, 72, 40), (200, 257, 129), (300, 136, 1000), (257, 640, 264), (1000, 1032, 72), (70, 64, 4096), (129, 127, 2050)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_residual(dev, kind, M, N, K):
    from autodiffusion_amd import ops
    g = torch.Generator().manual_seed(M + 7 * N + K)
    x, w = rand(g, M, K, kind=kind), rand(g, N, K, kind=kind, scale=K ** -0.5)
    b, res = rand(g, N, kind=kind, scale=0.5), rand(g, M, N, kind=kind)
    for i, act in enumerate(ACTS):
        bb, rr = (b, res) if i % 2 == 0 else (None, res) if i == 1 else (b, None)
        y, slope = ops.linear_residual(x, w, bb, rr, act=i, keep_slope=True)
        want, e, z, ez = linear_exact(x, w, bb, rr, act)
        within(y, want, e, kind, f"{act} y")
        # slopes change by at most 1.2 per unit; half a code is 2^-16; the piecewise ones jump where the sum's sign is open
        off = (slope_values(slope, act, kind) - slope64(z, act)).abs()
        bound = 1.2 * ez + 16 * U24 * (z.abs() + 1) ** 2 + (0 if kind == "fp32" else 2.0 ** -16)
        assert ((off <= bound) | ((z.abs() <= ez) & (ACTS[i] in ("relu", "leaky")))).all(), act
        assert torch.equal(y, ops.linear_residual(x, w, bb, rr, act=i))


@pytest.mark.parametrize("kind,M,N,K", [("bf16", 3000, 5000, 512), ("fp16", 4100, 4104, 200), ("fp32", 2100, 2052, 196), ("bf16", 2600, 2600, 300)])
def test_linear_residual_large_tiles(dev, kind, M, N, K):
    """The 256- and 128-wide tiles, ragged at both ends, and a large product whose rows start on no 16 bytes (300 = 37.5 pieces)."""
    from autodiffusion_amd import ops
    g = torch.Generator().manual_seed(M)
    x, w, b, res = rand(g, M, K, kind=kind), rand(g, N, K, kind=kind, scale=K ** -0.5), rand(g, N, kind=kind), rand(g, M, N, kind=kind)
    want, e, _, _ = linear_exact(x, w, b, res, "gelu_erf")
    within(ops.linear_residual(x, w, b, res, act=2), want, e, kind, "large")


def test_linear_residual_strides(dev):
    """Row-strided operands, a residual shared by all rows, leading axes, transposed storage, rows that start on no vector: the bits of the
    contiguous call."""
    from autodiffusion_amd import ops
    g = torch.Generator().manual_seed(2)
    for kind in TYPES:
        for M in (5, 200):
            wide, wwide = rand(g, M, 200, kind=kind), rand(g, 96, 176, kind=kind)
            x, w = wide[:, 8:168], wwide[:, 16:176]
            res = rand(g, 1, 96, kind=kind).expand(M, 96)
            ref = ops.linear_residual(x.contiguous(), w.contiguous(), None, res.contiguous(), act=5)
            assert torch.equal(ops.linear_residual(x, w, None, res, act=5), ref)
            assert torch.equal(ops.linear_residual(x.t().contiguous().t(), w.t().contiguous().t(), None, res, act=5), ref)
            x3 = x.contiguous().reshape(M // 5, 5, 160)
            assert torch.equal(ops.linear_residual(x3, w, None, res.reshape(M // 5, 5, 96), act=5).reshape(M, 96), ref)
            odd = rand(g, M, 161, kind=kind)
            odd[:, 1:] = x
            want, e, _, _ = linear_exact(x, w, None, res, "silu")
            within(ops.linear_residual(odd[:, 1:], w, None, res, act=5), want, e, kind, "odd start")
    assert ops.linear_residual(rand(g, 0, 16), rand(g, 8, 16)).shape == (0, 8)


@pytest.mark.parametrize("kind,M,N,K", [("bf16", 3000, 5000, 64), ("fp16", 2000, 2056, 200), ("fp32", 700, 516, 64), ("bf16", 129, 127, 2050), ("bf16", 100, 64, 8192), ("fp16", 17, 100, 36)])
def test_linear_residual_onto_the_residual(dev, kind, M, N, K):
    """The raw entry with y in place of the residual (every tile size, a split sum, rows that fill no piece): the bits of the call beside it."""
    from autodiffusion_amd import _lib, ops
    g = torch.Generator().manual_seed(M + K)
    x, w, b, res = rand(g, M, K, kind=kind), rand(g, N, K, kind=kind, scale=K ** -0.5), rand(g, N, kind=kind), rand(g, M, N, kind=kind)
    want = ops.linear_residual(x, w, b, res, act=5)
    lib, dt = _lib.load(), _lib.DTYPES[TYPES[kind]]
    need = lib.adx_linear_residual_ws_bytes(M, N, K, dt)
    ws = torch.empty(need + 16, dtype=torch.uint8, device=dev)
    _lib.check(lib.adx_op_linear_residual(x.data_ptr(), K, w.data_ptr(), K, b.data_ptr(), res.data_ptr(), N, None, res.data_ptr(), N, M, N, K, 5, dt, ws.data_ptr(),
                                          need, torch.cuda.current_stream().cuda_stream), "linear_residual")
    assert torch.equal(res, want)


def test_linear_residual_not_finite(dev):
    """An infinity or NaN reaches its own row alone, also through activations and behind ragged ends."""
    from autodiffusion_amd import ops
    g = torch.Generator().manual_seed(3)
    for kind in TYPES:
        for M, N, K in ((3, 40, 100), (100, 72, 100), (80, 72, 104)):
            x, w = rand(g, M, K, kind=kind), rand(g, N, K, kind=kind)
            clean = {i: ops.linear_residual(x, w, act=i) for i in range(7)}
            x2 = x.clone()
            x2[1, K - 1], x2[M - 1, 0] = math.nan, math.inf
            for i in range(7):
                y = ops.linear_residual(x2, w, act=i)
                assert torch.isnan(y[1]).all() and torch.equal(y[2:M - 1], clean[i][2:M - 1]) and torch.equal(y[0], clean[i][0])
                want = act64(x2[M - 1].double() @ w.double().t(), ACTS[i])
                assert torch.equal(torch.isinf(y[M - 1].double()), torch.isinf(want))
                assert torch.equal(torch.isnan(y[M - 1].double()), torch.isnan(want)) or ACTS[i] in ("silu", "gelu_erf", "gelu_tanh")


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_residual_bwd(dev, kind, M, N, K):
    from autodiffusion_amd import ops
    g = torch.Generator().manual_seed(M + 5 * N + K)
    x, w, dy, z = rand(g, M, K, kind=kind), rand(g, N, K, kind=kind, scale=K ** -0.5), rand(g, M, N, kind=kind), rand(g, M, N)
    for i, act in enumerate(ACTS):
        slope, value = (None, torch.ones_like(z).double()) if act == "none" else slope_codes(z, act, kind)
        dx, dw, db = ops.linear_residual_bwd(dy, x, w, slope, act=i)
        dz = dy.double() * value
        ed = torch.zeros_like(dz) if act == "none" else 4 * U24 * dz.abs()                      # as a summand
        e = ed if act == "none" else ed + HALF_STEP[kind] * dz.abs() + TINY[kind]               # as an operand
        aw, ax = w.double().abs(), x.double().abs()
        within(dx, dz @ w.double(), e @ aw + (N + 2) * U24 * (dz.abs() + e) @ aw, kind, f"{act} dx")
        within(dw, dz.t() @ x.double(), e.t() @ ax + (M + 2) * U24 * (dz.abs() + e).t() @ ax, kind, f"{act} dw")
        within(db, dz.sum(0), ed.sum(0) + (M + 2) * U24 * (dz.abs() + ed).sum(0), kind, f"{act} db")
        again = ops.linear_residual_bwd(dy, x, w, slope, act=i)
        assert all(torch.equal(a, b) for a, b in zip((dx, dw, db), again))
    slope, _ = slope_codes(z, "silu", kind)
    only = ops.linear_residual_bwd(dy, x, w, slope, act=5, need_dx=False, need_db=False)
    bias_only = ops.linear_residual_bwd(dy, x, w, slope, act=5, need_dx=False, need_dw=False)
    assert bias_only[0] is None and bias_only[1] is None and torch.equal(bias_only[2], ops.linear_residual_bwd(dy, x, w, slope, act=5)[2])
    assert only[0] is None and only[2] is None and torch.equal(only[1], ops.linear_residual_bwd(dy, x, w, slope, act=5)[1])


def test_linear_residual_gradient_of_rows_that_are_not_finite(dev):
    """A NaN before the activation makes the gradients that depend on it NaN, not others."""
    from autodiffusion_amd import train
    g = torch.Generator().manual_seed(8)
    for kind in TYPES:
        for i in range(1, 7):
            x, w, dy = rand(g, 70, 40, kind=kind), rand(g, 24, 40, kind=kind).requires_grad_(), rand(g, 70, 24, kind=kind)
            x[3, 5] = math.nan
            x.requires_grad_()
            y = train.linear_residual(x, w, act=i)
            dx, dw = torch.autograd.grad(y, (x, w), dy)
            assert torch.isnan(dx[3]).all() and torch.isfinite(dx[:3]).all() and torch.isfinite(dx[4:]).all() and torch.isnan(dw).all()
    with pytest.raises(RuntimeError, match="gradients of gradients"):
        torch.autograd.grad(train.linear_residual(x, w).sum(), w, create_graph=True)


def test_linear_residual_bwd_large(dev):
    from autodiffusion_amd import ops
    g = torch.Generator().manual_seed(9)
    for kind, M, N, K in (("bf16", 3000, 4104, 3600), ("fp32", 1037, 1020, 772), ("fp16", 8200, 264, 200),
                          ("bf16", 3186, 206, 4651), ("fp16", 2051, 2053, 2055), ("fp32", 900, 1021, 771), ("bf16", 700, 1203, 64)):
        x, w, dy = rand(g, M, K, kind=kind), rand(g, N, K, kind=kind, scale=K ** -0.5), rand(g, M, N, kind=kind)
        dx, dw, db = ops.linear_residual_bwd(dy, x, w)
        d, aw, ax = dy.double(), w.double().abs(), x.double().abs()
        within(dx, d @ w.double(), (N + 2) * U24 * d.abs() @ aw, kind, "dx")
        within(dw, d.t() @ x.double(), (M + 2) * U24 * d.abs().t() @ ax, kind, "dw")
        within(db, d.sum(0), (M + 2) * U24 * d.abs().sum(0), kind, "db")


def test_linear_residual_bwd_of_many_rows(dev):
    """More 64-row chunks than a launch has groups (65535): db and dw of 4.2 million rows."""
    from autodiffusion_amd import ops
    M, N, K = 65535 * 64 + 77, 9, 8
    g = torch.Generator(device="cuda").manual_seed(21)
    x, w, dy = (torch.randn(*s, generator=g, device=dev).bfloat16() for s in ((M, K), (N, K), (M, N)))
    y, slope = ops.linear_residual(x, w, act=1, keep_slope=True)
    dx, dw, db = ops.linear_residual_bwd(dy, x, w, slope, act=1)
    dz = dy.double() * slope_values(slope, "relu", "bf16")
    assert torch.equal(slope_values(slope, "relu", "bf16")[-100:], (y[-100:] > 0).double())
    # sums of at most 8200 partial sums of at most 4100 terms each way; relu's slope is 0 or 1: dz is exact
    e = 12300 * U24
    within(dw, dz.t() @ x.double(), e * dz.abs().t() @ x.double().abs(), "bf16", "dw")
    within(db, dz.sum(0), e * dz.abs().sum(0), "bf16", "db")
    within(dx[-200:], dz[-200:] @ w.double(), (N + 2) * U24 * dz[-200:].abs() @ w.double().abs(), "bf16", "dx")


def test_offsets_beyond_32_bits(dev):
    """Tensors of more than 2^31 values: the last rows of the product, of its gradients and of a rotation."""
    from autodiffusion_amd import ops
    g = torch.Generator(device="cuda").manual_seed(23)
    M, N, K = 1_050_001, 2056, 16
    x, w = (torch.randn(*s, generator=g, device=dev).bfloat16() for s in ((M, K), (N, K)))
    y, slope = ops.linear_residual(x, w, act=1, keep_slope=True)
    want, e, _, _ = linear_exact(x[-70:], w, None, None, "relu")
    within(y[-70:], want, e, "bf16", "y")
    assert torch.equal(slope_values(slope[-70:], "relu", "bf16"), (y[-70:] > 0).double())
    dy = y.zero_()
    dy[-70:] = torch.randn(70, N, generator=g, device=dev).bfloat16()
    dx, dw, db = ops.linear_residual_bwd(dy, x, w, slope, act=1)
    dz, xe = dy[-70:].double() * slope_values(slope[-70:], "relu", "bf16"), x[-70:].double()
    within(dx[-70:], dz @ w.double(), (N + 2) * U24 * dz.abs() @ w.double().abs(), "bf16", "dx")
    assert not dx[:-70].any()
    within(dw, dz.t() @ xe, 72 * U24 * dz.abs().t() @ xe.abs(), "bf16", "dw")
    within(db, dz.sum(0), 72 * U24 * dz.abs().sum(0), "bf16", "db")
    del y, slope, dy, dx, x
    tokens, heads, dh = 270_001, 64, 128
    q = torch.empty(tokens, heads, dh, dtype=torch.bfloat16, device=dev)
    q[-9:] = torch.randn(9, heads, dh, generator=g, device=dev).bfloat16()
    freq, amp = ops.rope_frequencies(dh)
    tail = q[-9:].clone()
    ops.rope(q, None, 3, freq, amp, inplace=True)
    assert torch.equal(q[-9:], ops.rope(tail, None, 3 + tokens - 9, freq, amp)[0])


def test_no_gradient_mode(dev):
    """Without gradients the training forms give the same values and record nothing; a rotation in place is seen by a graph that kept the tensor."""
    from autodiffusion_amd import ops, train
    g = torch.Generator().manual_seed(22)
    x, w = rand(g, 70, 64), rand(g, 64, 64).requires_grad_()
    with torch.no_grad():
        y = train.linear_residual(x, w, act=2)
    assert not y.requires_grad and torch.equal(y, train.linear_residual(x, w, act=2).detach())
    freq, _ = ops.rope_frequencies(16)
    kept = rand(g, 1, 5, 4, 16)
    loss = (rand(g, 1, 5, 4, 16).requires_grad_() * kept).sum()
    ops.rope(kept, None, 0, freq, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        t = kept.clone()
        assert torch.equal(ops.rope(t, None, 3, freq, inplace=True)[0], ops.rope(kept, None, 3, freq)[0])


def directional(f, leaves, grads, gen):
    """(<grad, v>, central difference of f along v) in 64 bits for random v."""
    v = [torch.randn(t.shape, generator=gen).double().cuda() for t in leaves]
    h = 1e-5
    up, down = f(*(t + h * d for t, d in zip(leaves, v))), f(*(t - h * d for t, d in zip(leaves, v)))
    return sum(float((a.double() * d).sum()) for a, d in zip(grads, v)), float((up - down) / (2 * h))


@pytest.mark.parametrize("kind", list(TYPES))
def test_linear_residual_autograd(dev, kind):
    """train.linear_residual: gradients against autograd of the formula in 64 bits and, in fp32, against central differences; gradients
    asked for one at a time; an expanded upstream gradient; a residual and a weight shared by two calls."""
    from autodiffusion_amd import train
    g = torch.Generator().manual_seed(4)
    for M, N, K, i in ((40, 72, 56, 2), (130, 64, 96, 5), (7, 33, 19, 3), (96, 40, 64, 0)):
        x, w, b, res, dy = (rand(g, *s, kind=kind, scale=c) for s, c in (((M, K), 1), ((N, K), K ** -0.5), ((N,), 1), ((M, N), 1), ((M, N), 1)))
        leaves = [t.requires_grad_() for t in (x, w, b, res)]
        y = train.linear_residual(*leaves, act=i)
        got = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        d = [t.detach().double().requires_grad_() for t in leaves]
        f = lambda x_, w_, b_, r_: ((act64(x_ @ w_.t() + b_, ACTS[i]) + r_) * dy.double()).sum()  # noqa: E731
        want = torch.autograd.grad(f(*d), d)
        # the slope changes by at most 1.2 per unit of z and is kept to 2^-16, dz is rounded once as an operand
        _, _, z, ez = linear_exact(*[t.detach() for t in (x, w, b)], None, "none")
        dz = (dy.double() * slope64(z, ACTS[i])).abs()
        kept = 1.2 * ez + 16 * U24 * (z.abs() + 1) ** 2 + (0 if kind == "fp32" else 2.0 ** -16)
        e = 0 * dz if i == 0 else dy.double().abs() * kept + HALF_STEP[kind] * dz + TINY[kind]
        bounds = (e @ w.detach().double().abs() + (N + 2) * U24 * (dz + e) @ w.detach().double().abs(),
                  e.t() @ x.detach().double().abs() + (M + 2) * U24 * (dz + e).t() @ x.detach().double().abs(), e.sum(0) + (M + 2) * U24 * (dz + e).sum(0), 0 * dz)
        for a, v, bd, name in zip(got, want, bounds, ("dx", "dw", "db", "dres")):
            within(a, v, bd, kind, name)
        if kind == "fp32":
            lhs, rhs = directional(f, [t.detach().double() for t in leaves], got, g)
            assert abs(lhs - rhs) <= 1e-4 * (abs(rhs) + M ** 0.5 * N ** 0.5)
        for n in range(4):
            sub = [t.detach().requires_grad_(j == n) for j, t in enumerate(leaves)]
            one = torch.autograd.grad(train.linear_residual(*sub, act=i), sub[n], dy)[0]
            assert torch.equal(one, got[n])
        ones = torch.autograd.grad(y, leaves, torch.ones_like(y), retain_graph=True)
        assert all(torch.equal(a, v) for a, v in zip(torch.autograd.grad(y.sum(), leaves), ones))          # an expanded upstream gradient
    # the same weight and residual in two calls: gradients add up
    x1, x2, w, r = (rand(g, *s, kind="fp32").requires_grad_() for s in ((9, 32), (9, 32), (32, 32), (9, 32)))
    h = train.linear_residual(x1, w, None, r, act=5)
    y = train.linear_residual(h, w, None, r + x2, act=2)
    got = torch.autograd.grad(y.square().sum(), (x1, w, r))
    d1, dw, dr, d2 = (t.detach().double().requires_grad_() for t in (x1, w, r, x2))
    hh = act64(d1 @ dw.t(), "silu") + dr
    want = torch.autograd.grad((act64(hh @ dw.t(), "gelu_erf") + dr + d2).square().sum(), (d1, dw, dr))
    for a, v in zip(got, want):
        # a chain of two 32-term products and a square: a few hundred roundings of the largest value
        assert float((a.double() - v).abs().max()) <= 1000 * U24 * float(v.abs().max())


@pytest.mark.parametrize("kind", list(TYPES))
def test_rope_autograd(dev, kind):
    from autodiffusion_amd import ops, train
    g = torch.Generator().manual_seed(5)
    B, S, Hq, Hk, dh = 2, 19, 4, 2, 48
    for layout in ("half", "interleaved"):
        w, amp = ops.rope_frequencies(32, 1e4, "parts", 4.0)
        q, k = rand(g, B, S, Hq, dh, kind=kind).requires_grad_(), rand(g, B, S, Hk, dh, kind=kind).requires_grad_()
        dq, dk = rand(g, B, S, Hq, dh, kind=kind), rand(g, B, S, Hk, dh, kind=kind)
        pos = torch.randint(0, 10 ** 5, (B, S), generator=g).cuda()
        qo, ko = train.rope(q, k, pos, w, amp, layout)
        got = torch.autograd.grad((qo, ko), (q, k), (dq, dk), retain_graph=True)
        for a, up in zip(got, (dq, dk)):
            within(a, *rope_exact(up, pos, w, amp, layout, inverse=True), kind, "gradient")
        # <R x, y> = <x, R^T y>: the gradient is the transpose of the forward map
        if kind == "fp32":
            lhs, rhs = float((qo.detach().double() * dq.double()).sum()), float((q.detach().double() * got[0].double()).sum())
            assert abs(lhs - rhs) <= 20 * U24 * float((q.detach().double().abs() * got[0].double().abs()).sum())
            v = torch.randn(q.shape, generator=g).double().cuda()                     # linear: a difference along v is exact up to rounding
            f = lambda t: float((rope_exact(t, pos, w, amp, layout)[0] * dq.double()).sum())  # noqa: E731
            num = (f(q.detach().double() + v) - f(q.detach().double() - v)) / 2
            assert abs(float((got[0].double() * v).sum()) - num) <= 20 * U24 * float((got[0].double().abs() * v.abs()).sum())
        assert torch.equal(torch.autograd.grad(ko, k, dk, retain_graph=True)[0], got[1])            # only one output used
        assert torch.equal(torch.autograd.grad(qo, q, dq)[0], got[0])
        alone, none = train.rope(q, None, pos, w, amp, layout)
        assert none is None and torch.equal(torch.autograd.grad(alone, q, dq)[0], got[0])


# ---------------------------------------------------------------------------------------------------------------- few-token expert layer
def moe_exact(x, res, router, w13, w2, top_k, parts_err):
    """(y, bound, chosen experts, their weights) in 64 bits: parts_err is what a hidden value may lose as an operand."""
    x, router, w13, w2 = (t.double() for t in (x, router, w13, w2))
    d, inter = x.shape[1], w2.shape[2]
    p = torch.softmax(x @ router.t(), -1)
    val, idx = torch.sort(p, dim=-1, descending=True, stable=True)
    idx, wt = idx[:, :top_k], val[:, :top_k] / val[:, :top_k].sum(-1, keepdim=True)
    y = torch.zeros_like(x) if res is None else res.double()
    e = 2 * U24 * y.abs()
    logit_err = (d + 2) * U24 * (x.abs() @ router.abs().t()).max(-1, keepdim=True).values
    for j in range(top_k):
        a, b = w13[idx[:, j]], w2[idx[:, j]]
        gu, mag = (a @ x[..., None])[..., 0], (a.abs() @ x.abs()[..., None])[..., 0]
        gate, up = gu.chunk(2, -1)
        eg, eu = ((d + 2) * U24 * mag).chunk(2, -1)
        s = gate * torch.sigmoid(gate)
        h = s * up
        eh = (1.1 * eg + 4 * U24 * s.abs()) * up.abs() + s.abs() * eu + (parts_err + 2 * U24) * h.abs()
        o = (b @ h[..., None])[..., 0]
        eo = (b.abs() @ (eh + (inter + 6) * U24 * h.abs())[..., None])[..., 0]
        w = wt[:, j:j + 1]
        y, e = y + w * o, e + w * eo + w * o.abs() * (4 * logit_err + 16 * U24)
    return y, e + 4 * U24 * y.abs(), idx, wt


FEW_TYPES = [("fp32", "fp32"), ("fp32", "bf16"), ("fp32", "bf16x3"), ("fp32", "f16"), ("bf16", "bf16"), ("fp16", "f16")]


def few_weights(g, E, d, inter, precision):
    """(stored w13, stored w2, their values)."""
    from autodiffusion_amd import str_backbone
    w13, w2 = torch.randn(E, 2 * inter, d, generator=g) * d ** -0.5, torch.randn(E, d, inter, generator=g) * inter ** -0.5
    if precision in ("bf16", "f16"):
        t = torch.bfloat16 if precision == "bf16" else torch.float16
        return w13.to(t).cuda(), w2.to(t).cuda(), w13.to(t).cuda(), w2.to(t).cuda()
    s13, s2 = str_backbone.prepare_expert_weights([t[:inter].cuda() for t in w13], [t[inter:].cuda() for t in w13], [t.cuda() for t in w2], precision)
    return s13, s2, w13.cuda(), w2.cuda()


@pytest.mark.parametrize("kind,precision", FEW_TYPES)
@pytest.mark.parametrize("T,d,inter,E,k", [
    (1, 32, 32, 1, 1),           # the smallest, one expert
    (1, 256, 1024, 8, 2),        # one token
    (3, 96, 160, 5, 3),          # widths that fill no piece
    (8, 1024, 512, 8, 2),
    (16, 64, 2080, 64, 8),       # many experts
    (17, 288, 96, 4, 4),         # every expert, two matrix tiles
    (40, 512, 288, 8, 2),
    (64, 160, 352, 2, 1),        # up to 64 tokens in one expert
    (64, 4128, 64, 3, 2),        # the routing in its own kernel
])
def test_moe_few(dev, kind, precision, T, d, inter, E, k):
    from autodiffusion_amd import str_backbone
    g = torch.Generator().manual_seed(T + d + inter + E)
    x, res = rand(g, T, d, kind=kind), rand(g, T, d, kind=kind)
    router = rand(g, E, d, scale=d ** -0.5)
    s13, s2, w13, w2 = few_weights(g, E, d, inter, precision)
    ws = torch.full((1 << 24,), 0x7F, dtype=torch.uint8, device="cuda")                        # a workspace full of anything
    y, idx, wt = str_backbone.moe_few(x, res, router, s13, s2, inter, E, k, precision, workspace=ws, return_routing=True)
    # hidden values in three bf16 parts (2^-25) or two (2^-17, and as much for the product of the low parts)
    want, e, ridx, rwt = moe_exact(x, res, router, w13, w2, k, 2.0 ** -24 if kind == "fp32" else 2.0 ** -15)
    if precision == "bf16x3":                      # weights as two bf16 halves: 2^-17 of every weight, in all three matrices
        h = moe_exact(x, None, router, w13.abs(), w2.abs(), k, 0)[0].abs()
        mag = torch.zeros_like(h)
        for j in range(k):
            a, b = w13.double().abs()[ridx[:, j]], w2.double().abs()[ridx[:, j]]
            gu = (a @ x.double().abs()[..., None])[..., 0]
            gate, up = gu.chunk(2, -1)
            mag = mag + rwt[:, j:j + 1] * (b @ (gate * up * 1.1 + up)[..., None])[..., 0]
        e = e + 4 * 2.0 ** -17 * mag
    assert torch.equal(idx.long(), ridx)
    assert float((wt.double() - rwt).abs().max()) <= 4 * (d + 20) * U24 * float((x.double().abs() @ router.double().abs().t()).max())
    within(y, want, e, kind, "y")
    assert torch.equal(y, str_backbone.moe_few(x, res, router, s13, s2, inter, E, k, precision))          # the order of the sums is fixed
    bare = str_backbone.moe_few(x, None, router, s13, s2, inter, E, k, precision)
    within(bare, want - res.double(), e, kind, "without a residual")
    if T > 2:                                        # a token's result depends on its routing weights and itself alone, to rounding
        first = str_backbone.moe_few(x[:2], res[:2], router, s13, s2, inter, E, k, precision)
        within(first, want[:2], e[:2], kind, "two of the tokens")


def test_moe_few_ties_and_tokens_that_are_not_finite(dev):
    """Equal router logits go to the lowest experts; a token with a NaN or an infinity has a NaN result and leaves the others alone."""
    from autodiffusion_amd import str_backbone
    g = torch.Generator().manual_seed(11)
    E, d, inter, k = 8, 128, 96, 2
    for kind, precision in FEW_TYPES:
        s13, s2, _, _ = few_weights(g, E, d, inter, precision)
        x = rand(g, 6, d, kind=kind)
        router = rand(g, 1, d).expand(E, d).contiguous()
        _, idx, wt = str_backbone.moe_few(x, None, router, s13, s2, inter, E, k, precision, return_routing=True)
        assert torch.equal(idx.cpu(), torch.tensor([[0, 1]] * 6, dtype=torch.int32)) and torch.equal(wt.cpu(), torch.full((6, 2), 0.5))
        router = rand(g, E, d)
        clean = str_backbone.moe_few(x, x, router, s13, s2, inter, E, k, precision)
        x[1, 3], x[4, 0] = math.nan, math.inf
        y, idx, _ = str_backbone.moe_few(x, x, router, s13, s2, inter, E, k, precision, return_routing=True)
        assert torch.isnan(y[1]).all() and torch.isnan(y[4]).all() and int(idx.min()) >= 0 and int(idx.max()) < E
        assert all(torch.isfinite(y[t]).all() for t in (0, 2, 3, 5))
        assert all(torch.allclose(y[t].float(), clean[t].float(), rtol=2 * HALF_STEP[kind] + 1e-5, atol=1e-5) for t in (0, 2, 3, 5))


def test_moe_few_agrees_with_moe_block(dev):
    from autodiffusion_amd import str_backbone
    g = torch.Generator().manual_seed(12)
    for precision, tol in (("fp32", 3e-6), ("bf16x3", 5e-5), ("bf16", 2e-2)):              # the tolerances of moe_block's own test
        s13, s2, _, _ = few_weights(g, 8, 256, 1024, precision)
        x, res, router = rand(g, 24, 256), rand(g, 24, 256), rand(g, 8, 256, scale=1 / 16)
        a, ia, wa = str_backbone.moe_few(x, res, router, s13, s2, 1024, 8, 2, precision, return_routing=True)
        b, ib, wb = str_backbone.moe_block(x, res, router, s13, s2, 1024, 8, 2, precision, return_routing=True)
        assert torch.equal(ia, ib) and torch.allclose(wa, wb, rtol=1e-5, atol=1e-6)
        assert float((a - b).abs().max() / b.abs().max()) < tol


# ---------------------------------------------------------------------------------------------------------------- together, as they are used
def decoder_step(P, x, cache, pos, w, amp, n_head, n_kv, top_k, precision):
    """One token of every item through a decoder layer: fused q / k / v product, rotary positions, attention over the cached keys, out-projection
    with its residual, expert layer with its residual.  x (B, d) of the layer's type."""
    from autodiffusion_amd import ops, str_backbone
    B, d = x.shape
    dh = d // n_head
    qkv = ops.linear_residual(str_backbone.rmsnorm(x, P["n1"], 1e-5).to(x.dtype), P["qkv"], P["qkv_b"]).view(B, 1, n_head + 2 * n_kv, dh)
    q, k = ops.rope(qkv[:, :, :n_head], qkv[:, :, n_head:n_head + n_kv], pos, w, amp)
    v = qkv[:, :, n_head + n_kv:]
    cache[0], cache[1] = torch.cat([cache[0], k], 1), torch.cat([cache[1], v], 1)
    rep = lambda t: t.repeat_interleave(n_head // n_kv, 2).reshape(B, -1, d)  # noqa: E731
    att = ops.attention(q.reshape(B, 1, d), rep(cache[0]), rep(cache[1]), n_head).to(x.dtype).reshape(B, d)
    x = ops.linear_residual(att, P["o"], None, x)
    n2 = str_backbone.rmsnorm(x, P["n2"], 1e-5).to(x.dtype)
    return str_backbone.moe_few(n2, x, P["router"], P["w13"], P["w2"], P["w2"].shape[2], P["router"].shape[0], top_k, precision)


def decoder_step_exact(P, x, cache, pos, w, amp, n_head, n_kv, top_k):
    P = {n: t.double() for n, t in P.items()}
    x = x.double()
    B, d = x.shape
    dh = d // n_head
    norm = lambda t, n: P[n] * t * (t.square().mean(-1, keepdim=True) + 1e-5).rsqrt()  # noqa: E731
    qkv = (norm(x, "n1") @ P["qkv"].t() + P["qkv_b"]).view(B, 1, n_head + 2 * n_kv, dh)
    q, k = (rope_exact(t, pos, w, amp, "half")[0] for t in (qkv[:, :, :n_head], qkv[:, :, n_head:n_head + n_kv]))
    cache[0], cache[1] = torch.cat([cache[0], k], 1), torch.cat([cache[1], qkv[:, :, n_head + n_kv:]], 1)
    K, V = (t.repeat_interleave(n_head // n_kv, 2) for t in cache)
    a = torch.softmax((q * K).sum(-1) * dh ** -0.5, 1)                            # (B, S, H)
    x = x + (a[..., None] * V).sum(1).reshape(B, d) @ P["o"].t()
    return moe_exact(norm(x, "n2"), x, P["router"], P["w13"], P["w2"], top_k, 0)[0]


@pytest.mark.parametrize("kind,precision", [("fp32", "fp32"), ("bf16", "bf16"), ("fp16", "f16")])
def test_decoder_layer_one_token_at_a_time(dev, kind, precision):
    """Five tokens of three items through one decoder layer built of the operators, eager and replayed from a captured graph, against the layer in
    64 bits.  The intermediate tensors of the layer are rounded to its type about eight times, each half a step of values of order one."""
    from autodiffusion_amd import ops
    g = torch.Generator().manual_seed(13)
    B, d, H, Hk, E, inter, k = 3, 256, 8, 4, 8, 512, 2
    dh = d // H
    P = {"n1": rand(g, d).abs() + 0.5, "n2": rand(g, d).abs() + 0.5, "router": rand(g, E, d, scale=1 / 16)}
    for n, shape, c in (("qkv", ((H + 2 * Hk) * dh, d), 1 / 16), ("qkv_b", ((H + 2 * Hk) * dh,), 0.1), ("o", (d, d), 1 / 16), ("w13", (E, 2 * inter, d), 1 / 16),
                        ("w2", (E, d, inter), inter ** -0.5)):
        P[n] = rand(g, *shape, kind=kind, scale=c)
    w, amp = ops.rope_frequencies(dh, 1e6)
    cache = [rand(g, B, 6, Hk, dh, kind=kind), rand(g, B, 6, Hk, dh, kind=kind)]
    cache64 = [t.double() for t in cache]
    for step in range(5):
        x = rand(g, B, d, kind=kind)
        pos = torch.full((B, 1), 6 + step).cuda()
        before = list(cache)
        y = decoder_step(P, x, cache, pos, w, amp, H, Hk, k, precision)
        want = decoder_step_exact(P, x, cache64, pos, w, amp, H, Hk, k)
        rel = float((y.double() - want).norm() / want.norm())
        assert rel <= 8 * HALF_STEP[kind] * (1 if kind != "fp32" else 16), rel
    # the last step captured and replayed, with the program's own work between the replays
    graph, xs, caches = torch.cuda.CUDAGraph(), x.clone(), None
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        decoder_step(P, xs, list(before), pos, w, amp, H, Hk, k, precision)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        caches = list(before)
        out = decoder_step(P, xs, caches, pos, w, amp, H, Hk, k, precision)
    for n in range(4):
        xs.copy_(x if n % 2 == 0 else x.flip(0))
        graph.replay()
        got = out.clone()
        eager = decoder_step(P, xs, list(before), pos, w, amp, H, Hk, k, precision)
        torch.cuda.synchronize()
        assert torch.equal(got, eager)


def test_training_step_captured(dev):
    """Forward and backward of rotary + product under a graph: every replay gives the eager gradients of its inputs."""
    from autodiffusion_amd import ops, train
    g = torch.Generator().manual_seed(14)
    M, d, H = 160, 128, 4
    w, amp = ops.rope_frequencies(32, 1e4)
    inputs = [(rand(g, M, d, kind="bf16"), rand(g, M, d, kind="bf16")) for _ in range(3)]
    wt, b = rand(g, d, d, kind="bf16", scale=d ** -0.5), rand(g, d, kind="bf16")

    def step(x, dy):
        leaves = [t.detach().requires_grad_() for t in (x, wt, b)]
        h = train.linear_residual(*leaves, leaves[0], act=2)
        q, _ = train.rope(h.view(1, M, H, d // H), None, 5, w, amp)
        return [q.detach(), *torch.autograd.grad(q, leaves, dy.view(q.shape))]

    want = [[t.clone() for t in step(*i)] for i in inputs]
    xs, dys = inputs[0][0].clone(), inputs[0][1].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(xs, dys)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(xs, dys)
    for n in (0, 1, 2, 0, 1):
        xs.copy_(inputs[n][0])
        dys.copy_(inputs[n][1])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, v) for a, v in zip(out, want[n])), n
        step(*inputs[(n + 1) % 3])


def test_two_streams_at_once(dev):
    """The operators keep no state between calls: the same work on two streams at a time gives what each gives alone."""
    from autodiffusion_amd import ops, str_backbone
    g = torch.Generator().manual_seed(15)
    s13, s2, _, _ = few_weights(g, 8, 512, 1024, "bf16")
    router = rand(g, 8, 512, scale=0.05)
    xs = [rand(g, 16, 512, kind="bf16") for _ in range(2)]
    big = [rand(g, 700, 2048, kind="bf16") for _ in range(2)]
    w = rand(g, 96, 2048, kind="bf16")

    def work(n):
        return str_backbone.moe_few(xs[n], xs[n], router, s13, s2, 1024, 8, 2, "bf16"), ops.linear_residual(big[n], w, act=5)

    want = [work(0), work(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        got = [None, None]
        for n, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[n] = work(n)
        torch.cuda.synchronize()
        for n in range(2):
            assert all(torch.equal(a, b) for a, b in zip(got[n], want[n]))


def test_key_point_passes_through_the_few_token_layer(dev):
    """MixtralModel with few_token_experts: a prefill and three one-token passes give the default's hidden states (fp32 and split-bf16 operands, whose
    expert layers agree to rounding); the long pass takes the same layer as before, bit for bit."""
    from autodiffusion_amd import str_backbone
    for precision, tol in (("fp32", 1e-5), ("bf16x3", 2e-4)):
        torch.manual_seed(0)
        kw = dict(hidden_size=128, intermediate_size=256, num_hidden_layers=2, num_attention_heads=8, num_key_value_heads=4, vocab_size=8, precision=precision)
        a = str_backbone.MixtralModel(**kw).to(dev)
        b = str_backbone.MixtralModel(few_token_experts=True, **kw).to(dev)
        with torch.no_grad():
            for n, p in a.named_parameters():
                if p.dim() == 2:
                    p.copy_(torch.randn(p.shape) * p.shape[1] ** -0.5)
        b.load_state_dict(a.state_dict())
        emb = torch.randn(4, 40, 128, device=dev)
        ca, cb = a.new_cache(), b.new_cache()
        assert torch.equal(a.extend(emb[:, :37], ca), b.extend(emb[:, :37], cb))                   # 148 tokens: not few
        for i in range(37, 40):
            x, y = a.extend(emb[:, i:i + 1], ca), b.extend(emb[:, i:i + 1], cb)
            # two layers of products of at most 256 terms, agreeing like the two expert layers do
            assert float((x - y).abs().max() / x.abs().max()) < tol
