"""The decoder-layer operators on the GPU where their arguments are extreme: saturated activations, values that are not finite, every tile
of the product, strides; against the formulas in 64 bits.  Tolerances count roundings as in test_gpu_decoder_ops.py."""
import math

import pytest
import torch

from test_gpu_decoder_ops import ACTS, HALF_STEP, TINY, TYPES, U24, act64, dev, few_weights, linear_exact, moe_exact, rand, slope64, within  # noqa: F401

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------------------------- slopes in the tails
def slope_tails(z, act):
    """The slope of ``act`` at z in 64 bits with all its digits in the tails, where 1 + erf and 1 - tanh^2 have none left."""
    q = torch.exp(-2 * z.abs())
    phi = torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    sig, neg = torch.sigmoid(z), torch.sigmoid(-z)
    k, K = math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3), math.sqrt(8 / math.pi) * (1 + 0.134145 * z * z)
    one = torch.ones_like(z)
    return {"none": one, "relu": (z > 0).double(), "leaky": torch.where(z > 0, one, 0.01 * one), "tanh": 4 * q / (1 + q) ** 2,
            "silu": sig * (1 + z * neg), "gelu_erf": 0.5 * torch.erfc(-z * math.sqrt(0.5)) + z * phi,
            "gelu_tanh": torch.sigmoid(k) * (1 + z * torch.sigmoid(-k) * K)}[act]


def slope_error(z, act):
    """What roundings in 32 bits may change of the slope of ``act`` at z (64 bits): relative to the slope wherever that is small."""
    a, d, flushed = z.abs(), slope_tails(z, act).abs(), 1e-35          # single-instruction forms flush results below 2^-126
    if act in ("none", "relu", "leaky"):
        return U24 * d
    if act == "tanh":                          # exp(-2 |z|): two roundings of the argument, 2 for the exponential; a sum, a reciprocal, three products
        return U24 * (4 * a + 16) * d + flushed
    if act == "silu":                          # the sigmoid g likewise; then g (1 + z (1 - g))
        g = torch.sigmoid(z)
        g_err = 2 * a + 5
        return U24 * (g_err * d + g * (4 * (a + 1) + a * torch.minimum(g, 1 - g) * g_err)) + flushed
    if act == "gelu_erf":                      # tail q = exp(-z^2 / 2) times a polynomial; p + z phi
        q, phi = 0.5 * torch.erfc(a * math.sqrt(0.5)), torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
        return U24 * (q * (1.5 * z * z + 52) + a * phi * (1.5 * z * z + 6) + 2 * torch.where(z > 0, 1 - q, q) + d) + flushed
    k = math.sqrt(8 / math.pi)                 # gelu_tanh: g + z g (1 - g) K with the sigmoid g of k z (1 + 0.0447 z^2)
    arg, K = k * a * (1 + 0.044715 * z * z), k * (1 + 0.134145 * z * z)
    g = torch.sigmoid(torch.where(z > 0, arg, -arg))
    return U24 * ((14 * arg + 30) * (g * torch.where(z > 0, 1 - g, torch.ones_like(g)) + a * g * (1 - g) * K) + 3 * a * g * K + 3 * d) + flushed


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M", [64, 192])
def test_slopes_of_saturated_activations(dev, kind, M):
    """fp32 slopes of known arguments (rows of the identity) from -13 to 13: relative accuracy down to the smallest."""
    from autodiffusion_amd import ops
    K, N = 64, 320
    x = torch.eye(K).repeat(M // K, 1).to(TYPES[kind]).cuda()
    w = torch.linspace(-13, 13, N * K).reshape(N, K).to(TYPES[kind]).cuda()
    z = w.double().t().repeat(M // K, 1)
    for i, act in enumerate(ACTS):
        y, slope = ops.linear_residual(x, w, act=i, keep_slope=torch.float32)
        assert slope.dtype == torch.float32 and torch.equal(y, ops.linear_residual(x, w, act=i, keep_slope=True)[0])
        want = slope_tails(z, act)
        assert bool(((slope64(z, act) - want).abs() <= 1e-14 * (1 + z * z)).all())
        off, most = (slope.double() - want).abs(), slope_error(z, act)
        assert bool((off <= most).all()), (act, float((off / most).max()), float(z.flatten()[int((off / most).argmax())]))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("act", ["tanh", "silu", "gelu_erf", "gelu_tanh", "relu", "leaky"])
def test_gradients_of_saturated_units(dev, kind, act):
    """Units that sit at -12 .. -4 and 4 .. 12: their gradients to the accuracy of the type relative to their own small size."""
    from autodiffusion_amd import train
    g = torch.Generator().manual_seed(31)
    M, N, K = 200, 72, 40
    x, w, dy = rand(g, M, K, kind=kind), rand(g, N, K, kind=kind, scale=0.1 * K ** -0.5), rand(g, M, N, kind=kind)
    b = torch.cat([torch.linspace(-12, -4, N // 2), torch.linspace(4, 12, N // 2)]).to(TYPES[kind]).cuda()
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = train.linear_residual(*leaves, act=ACTS.index(act))
    kept = y.grad_fn.saved_tensors[2]
    assert kept.dtype == (torch.int16 if act in ("relu", "leaky") and kind != "fp32" else torch.float32)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    x, w, b = (t.detach() for t in leaves)
    gradients_within(kind, act, x, w, b, dy, (dx, dw, db))
    if kind != "fp16" and act in ("silu", "gelu_erf"):
        assert (db.float().abs()[: N // 2] > 0).all()               # small, not nothing


# ---------------------------------------------------------------------------------------------------------------- every tile of the product
def edges(M, N, K, kind):
    """Edges of the tiles that y, dx and dw are computed in."""
    from autodiffusion_amd import _lib
    return tuple(_lib.load().adx_linear_residual_edge(M, N, K, which, _lib.DTYPES[TYPES[kind]]) for which in range(3))


def gradients_within(kind, act, x, w, b, dy, got, what=""):
    """(dx, dw, db) of the product with its slopes in fp32, elementwise."""
    (M, K), N = x.shape, w.shape[0]
    _, _, z, ez = linear_exact(x, w, b, None, "none")
    d = slope_tails(z, act)
    moved = torch.maximum((slope_tails(z + ez, act) - d).abs(), (slope_tails(z - ez, act) - d).abs())         # what the rounding of z changes
    dz = dy.double() * d
    ed = 0 * dz if act == "none" else dy.double().abs() * (slope_error(z, act) + moved) + U24 * dz.abs()       # as a summand
    e = ed if act == "none" else ed + HALF_STEP[kind] * dz.abs() + TINY[kind]                                  # as an operand
    ax, aw, ad = x.double().abs(), w.double().abs(), dz.abs() + e
    within(got[0], dz @ w.double(), e @ aw + (N + 2) * U24 * ad @ aw, kind, f"{what} dx")
    within(got[1], dz.t() @ x.double(), e.t().contiguous() @ ax + (M + 2) * U24 * ad.t().contiguous() @ ax, kind, f"{what} dw")
    within(got[2], dz.sum(0), ed.sum(0) + (M + 2) * U24 * (dz.abs() + ed).sum(0), kind, f"{what} db")


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M,N,K,edge", [(3590, 3608, 3624, 256), (2500, 2608, 2584, 128), (515, 520, 1032, 64)])
def test_tiles_of_the_training_step(dev, kind, M, N, K, edge):
    """y, dx and dw in tiles of each edge, ragged at both ends and in the summed axis, with an activation."""
    from autodiffusion_amd import train
    assert edges(M, N, K, kind) == (edge,) * 3
    g = torch.Generator().manual_seed(M)
    x, w, b, res, dy = (rand(g, *s, kind=kind, scale=c) for s, c in (((M, K), 1), ((N, K), K ** -0.5), ((N,), 1), ((M, N), 1), ((M, N), 1)))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = train.linear_residual(*leaves, res, act=2)
    got = torch.autograd.grad(y, leaves, dy)
    x, w, b = (t.detach() for t in leaves)
    want, e, _, _ = linear_exact(x, w, b, res, "gelu_erf")
    within(y.detach(), want, e, kind, "y")
    gradients_within(kind, "gelu_erf", x, w, b, dy, got)


@pytest.mark.parametrize("kind,M,N,K,edge", [("fp32", 3590, 3604, 52, 256), ("fp32", 2600, 2500, 44, 128), ("fp16", 3590, 3608, 72, 256), ("fp16", 2600, 2504, 72, 128),
                                             ("bf16", 2600, 2504, 72, 128)])
def test_tiles_of_the_forward(dev, kind, M, N, K, edge):
    """Large tiles over a few steps of the summed axis, with residual, bias and fp32 slopes."""
    from autodiffusion_amd import ops
    assert edges(M, N, K, kind)[0] == edge
    g = torch.Generator().manual_seed(N)
    x, w, b, res = rand(g, M, K, kind=kind), rand(g, N, K, kind=kind, scale=K ** -0.5), rand(g, N, kind=kind), rand(g, M, N, kind=kind)
    y, slope = ops.linear_residual(x, w, b, res, act=5, keep_slope=torch.float32)
    want, e, z, ez = linear_exact(x, w, b, res, "silu")
    within(y, want, e, kind, "y")
    assert bool(((slope.double() - slope_tails(z, "silu")).abs() <= 0.51 * ez + slope_error(z, "silu")).all())          # the slope changes by at most 1 / 2 a unit


@pytest.mark.parametrize("kind,act,M,N,K", [("bf16", "gelu_erf", 1500, 1003, 501), ("fp16", "silu", 700, 999, 1101), ("fp32", "tanh", 900, 1021, 771),
                                            ("bf16", "gelu_tanh", 1030, 515, 1001)])
def test_training_step_laid_out_anew(dev, kind, act, M, N, K):
    """Rows of no whole number of 16-byte pieces in a long product: operands and dz laid out anew, with an activation."""
    from autodiffusion_amd import train
    assert M * N * K >= 2 ** 28 and N % 4 and K % 4
    g = torch.Generator().manual_seed(N)
    leaves = [rand(g, *s, kind=kind, scale=c).requires_grad_() for s, c in (((M, K), 1), ((N, K), K ** -0.5), ((N,), 1))]
    dy = rand(g, M, N, kind=kind)
    y = train.linear_residual(*leaves, act=ACTS.index(act))
    got = torch.autograd.grad(y, leaves, dy)
    x, w, b = (t.detach() for t in leaves)
    want, e, _, _ = linear_exact(x, w, b, None, act)
    within(y.detach(), want, e, kind, "y")
    gradients_within(kind, act, x, w, b, dy, got)


def test_slopes_of_every_path(dev):
    """fp32 slopes of 16-bit tensors from the few-row kernel, unaligned rows, a split sum and odd widths; the gradients from them."""
    from autodiffusion_amd import ops
    g = torch.Generator().manual_seed(32)
    for kind in ("bf16", "fp16"):
        for M, N, K in ((1, 8, 8), (17, 100, 36), (64, 130, 257), (130, 72, 40), (200, 257, 129), (70, 64, 4096), (129, 127, 2050)):
            x, w, b, dy = rand(g, M, K, kind=kind), rand(g, N, K, kind=kind, scale=K ** -0.5), rand(g, N, kind=kind), rand(g, M, N, kind=kind)
            for i, act in enumerate(ACTS):
                if act in ("relu", "leaky"):                     # jump where the sum's sign is open
                    continue
                y, slope = ops.linear_residual(x, w, b, act=i, keep_slope=torch.float32)
                assert torch.equal(y, ops.linear_residual(x, w, b, act=i))
                _, _, z, ez = linear_exact(x, w, b, None, "none")
                moved = torch.maximum((slope_tails(z + ez, act) - slope_tails(z, act)).abs(), (slope_tails(z - ez, act) - slope_tails(z, act)).abs())
                assert bool(((slope.double() - slope_tails(z, act)).abs() <= slope_error(z, act) + moved).all()), act
                got = ops.linear_residual_bwd(dy, x, w, slope, act=i)
                gradients_within(kind, act, x, w, b, dy, got, act)
                shifted = torch.empty(M * N + 1, device=dev)[1:].view(M, N).copy_(slope)             # slopes that start on 4 bytes
                assert all(torch.equal(p, q) for p, q in zip(ops.linear_residual_bwd(dy, x, w, shifted, act=i), got))


# ---------------------------------------------------------------------------------------------------------------- strides of the gradient's operands
@pytest.mark.parametrize("kind", list(TYPES))
def test_gradient_of_strided_operands(dev, kind):
    """x, w, dy and slopes as slices, transposed storage, leading axes and one row for all: the bits of the contiguous call; rows that start on
    no 16 bytes: the formula."""
    from autodiffusion_amd import ops
    g = torch.Generator().manual_seed(33)
    for M in (5, 200):
        x, w, dy = rand(g, M, 200, kind=kind)[:, 8:168], rand(g, 96, 176, kind=kind, scale=0.1)[:, 16:], rand(g, M, 112, kind=kind)[:, 16:]
        _, slope = ops.linear_residual(x, w, act=5, keep_slope=torch.float32)
        want = ops.linear_residual_bwd(dy.contiguous(), x.contiguous(), w.contiguous(), slope, act=5)
        gradients_within(kind, "silu", x, w, None, dy, want)
        turned = [t.t().contiguous().t() for t in (dy, x, w, slope)]
        wide = torch.empty(M, 100, device=dev)
        wide[:, 3:99] = slope
        deep = [t.reshape(M // 5, 5, -1) for t in (dy, x)]
        for got in (ops.linear_residual_bwd(dy, x, w, slope, act=5), ops.linear_residual_bwd(*turned, act=5),
                    ops.linear_residual_bwd(dy, x, w, wide[:, 3:99], act=5), ops.linear_residual_bwd(*deep, w, slope.reshape(M // 5, 5, 96), act=5)):
            assert torch.equal(got[0].reshape(M, 160), want[0]) and torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
        row = dy[:1].expand(M, 96)                                                          # one row for all
        want = ops.linear_residual_bwd(row.contiguous(), x, w, slope, act=5)
        assert all(torch.equal(p, q) for p, q in zip(ops.linear_residual_bwd(row, x, w, slope, act=5), want))
        want = ops.linear_residual_bwd(dy, x[:1].expand(M, 160).contiguous(), w, slope, act=5)
        assert all(torch.equal(p, q) for p, q in zip(ops.linear_residual_bwd(dy, x[:1].expand(M, 160), w, slope, act=5), want))
        odd = [rand(g, t.shape[0], t.shape[1] + 1, kind=kind) for t in (dy, x, w)]
        for o, t in zip(odd, (dy, x, w)):
            o[:, 1:] = t
        odd = [o[:, 1:] for o in odd]
        gradients_within(kind, "silu", x, w, None, dy, ops.linear_residual_bwd(*odd, slope, act=5), "odd start")
        gradients_within(kind, "silu", x[:, :-3], w[:, :-3], None, dy, ops.linear_residual_bwd(odd[0], odd[1][:, :-3], odd[2][:, :-3],
                         ops.linear_residual(x[:, :-3], w[:, :-3], act=5, keep_slope=torch.float32)[1], act=5), "odd width")


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_rows_far_apart(dev, kind):
    """Row strides of 2^21 values and more, whose tiles span more than 32 bits of bytes: forward and gradients."""
    from autodiffusion_amd import ops
    g = torch.Generator().manual_seed(34)
    M, N, K, far = 80, 72, 96, (1 << 21) + 8

    def spread(t):
        flat = torch.empty((t.shape[0] - 1) * far + t.shape[1], dtype=t.dtype, device=dev)
        out = flat.as_strided(t.shape, (far, 1))
        out.copy_(t)
        return out

    x, w, dy, res = rand(g, M, K, kind=kind), rand(g, N, K, kind=kind, scale=0.1), rand(g, M, N, kind=kind), rand(g, M, N, kind=kind)
    want, e, _, _ = linear_exact(x, w, None, res, "silu")
    for a, b in ((spread(x), w), (x, spread(w)), (spread(x), spread(w))):
        y, slope = ops.linear_residual(a, b, None, spread(res), act=5, keep_slope=torch.float32)
        within(y, want, e, kind, "y")
        gradients_within(kind, "silu", x, w, None, dy, ops.linear_residual_bwd(spread(dy), a, b, slope, act=5))
    within(ops.linear_residual(spread(x)[:9], spread(w), None, res[:9], act=5), want[:9], e[:9], kind, "few rows")
    plain = ops.linear_residual_bwd(spread(dy), x, w)                                       # dy itself is the operand
    gradients_within(kind, "none", x, w, None, dy, plain)


# ---------------------------------------------------------------------------------------------------------------- arguments that are not finite, or huge
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M,N", [(5, 16), (80, 16), (70, 11)])
def test_activations_of_extreme_arguments(dev, kind, M, N):
    """What every activation and its slope give for infinities, NaN and the largest finite arguments (as biases of a product of zeros).  silu and the
    gelus are z times a number that is 0 at -inf: NaN, as the formula says."""
    from autodiffusion_amd import ops
    inf, nan = math.inf, math.nan
    top = [1e4, 6e4] if kind == "fp16" else [1e4, 1e18, 1e19, 1e30, 3e38]
    z = torch.tensor(([inf, -inf, nan] + top + [-t for t in top] + [0.0] * 16)[:N]).to(TYPES[kind]).cuda()
    x, w = torch.zeros(M, 24, dtype=TYPES[kind], device=dev), torch.zeros(N, 24, dtype=TYPES[kind], device=dev)
    up, zero, one = torch.where(z > 0, z, 0 * z.abs().nan_to_num()), torch.zeros_like(z), torch.ones_like(z)
    step, sign = (z > 0).to(z.dtype), torch.sign(z)
    lowest = torch.where(z == -inf, z * 0, up)                     # NaN at -inf
    known = torch.where(z.isinf(), z * 0, step)                    # slopes of 1 and 0, NaN at the infinities
    known = torch.where(z == 0, 0.5 * one, known)
    half = torch.where(z == 0, 0.5 * one, step)
    expected = {"none": (z, one), "relu": (up, step), "leaky": (torch.where(z > 0, z, (z.double() * 0.01).to(z.dtype)), torch.where(z > 0, one.float(), 0.01)),
                "silu": (lowest, known), "gelu_erf": (lowest, known), "gelu_tanh": (lowest, half), "tanh": (sign, torch.where(z == 0, one, zero))}
    for i, act in enumerate(ACTS):
        y, slope = ops.linear_residual(x, w, z, act=i, keep_slope=torch.float32)
        value, d = (torch.where(z.isnan(), z, t.to(z.dtype)) if act != "none" else t for t in expected[act])
        for m in (0, M - 1):
            assert torch.allclose(y[m].double(), value.double(), rtol=2 * HALF_STEP[kind], atol=0, equal_nan=True), (act, y[m], value)
            if act != "none":
                d32 = torch.where(z.isnan(), nan, expected[act][1].float())
                assert torch.allclose(slope[m], d32, rtol=60 * U24, atol=0, equal_nan=True), (act, slope[m], d32)


# ---------------------------------------------------------------------------------------------------------------- expert layer
@pytest.mark.parametrize("kind,precision,T,d", [("bf16", "bf16", 40, 160), ("fp32", "fp32", 64, 96), ("fp32", "bf16x3", 17, 32), ("fp16", "f16", 3, 96)])
def test_moe_few_onto_the_residual(dev, kind, precision, T, d):
    """The raw entry with y in place of the residual, widths that end inside a group of 64 output columns: the bits of the call beside it."""
    from autodiffusion_amd import _lib, str_backbone
    g = torch.Generator().manual_seed(T + d)
    x, res, router = rand(g, T, d, kind=kind), rand(g, T, d, kind=kind), rand(g, 8, d, scale=d ** -0.5)
    s13, s2, _, _ = few_weights(g, 8, d, 96, precision)
    want = str_backbone.moe_few(x, res, router, s13, s2, 96, 8, 2, precision)
    lib, dt, prec = _lib.load(), _lib.DTYPES[TYPES[kind]], _lib.PRECISIONS[precision]
    need = lib.adx_moe_few_workspace_bytes(T, d, 96, 8, 2, dt, prec)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    _lib.check(lib.adx_op_moe_few(x.data_ptr(), res.data_ptr(), router.data_ptr(), s13.data_ptr(), s2.data_ptr(), T, d, 96, 8, 2, dt, prec, ws.data_ptr(),
                                  need, res.data_ptr(), torch.cuda.current_stream().cuda_stream), "moe_few")
    assert torch.equal(res, want)


def test_moe_few_of_tensors_that_start_anywhere(dev):
    """Tokens, residual, router and workspace behind a few values of another tensor: the bits of the call on tensors of their own.  Weights off 16
    bytes are refused, not copied on every call."""
    from autodiffusion_amd import _lib, str_backbone
    g = torch.Generator().manual_seed(41)

    def shifted(t, by):
        flat = torch.zeros(t.numel() + by, dtype=t.dtype, device=dev)
        flat[by:] = t.flatten()
        return flat[by:].view(t.shape)

    for kind, precision in (("bf16", "bf16"), ("fp32", "fp32"), ("fp32", "bf16x3")):
        x, res, router = rand(g, 5, 64, kind=kind), rand(g, 5, 64, kind=kind), rand(g, 8, 64)
        s13, s2, _, _ = few_weights(g, 8, 64, 96, precision)
        want = str_backbone.moe_few(x, res, router, s13, s2, 96, 8, 2, precision)
        ws = torch.empty(1 << 22, dtype=torch.uint8, device=dev)[1:]
        for by in (1, 3):
            assert torch.equal(str_backbone.moe_few(shifted(x, by), shifted(res, by), shifted(router, by), s13, s2, 96, 8, 2, precision, workspace=ws), want)
        with pytest.raises(_lib.AdxError, match="aligned"):
            str_backbone.moe_few(x, res, router, shifted(s13, 1), s2, 96, 8, 2, precision)


# ---------------------------------------------------------------------------------------------------------------- captures
@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")
def test_capture_beside_a_live_eager_graph_is_refused(dev):
    """Capturing a step over leaves of an eager graph that is still alive raises, and the program goes on: the eager graph's gradients, then the
    capture, once that graph is gone."""
    from autodiffusion_amd import ops, train
    g = torch.Generator().manual_seed(51)
    freq, amp = ops.rope_frequencies(16)
    x, w, dy = rand(g, 70, 64), rand(g, 64, 64, scale=1 / 8).requires_grad_(), rand(g, 70, 64)
    q, dq = rand(g, 1, 5, 4, 16).requires_grad_(), rand(g, 1, 5, 4, 16)
    forms = ((lambda: train.linear_residual(x, w, act=2), w, dy), (lambda: train.rope(q, None, 3, freq, amp)[0], q, dq))
    for forward, leaf, up in forms:
        want = torch.autograd.grad(forward(), leaf, up)[0].clone()
        alive = forward()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="earlier pass"):
            with torch.cuda.graph(graph):
                forward()
        assert torch.equal(torch.autograd.grad(alive, leaf, up)[0], want)
        del alive
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = torch.autograd.grad(forward(), leaf, up)[0]
        for _ in range(3):
            got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)
            forward()


def test_few_token_layer_of_a_bf16_model(dev, monkeypatch):
    """MixtralModel with few_token_experts under "bf16": its short passes run every expert layer through moe_few, each to the accuracy of the formula on
    the rounded weights; the long pass keeps the bits of the default."""
    from autodiffusion_amd import str_backbone
    torch.manual_seed(0)
    kw = dict(hidden_size=128, intermediate_size=256, num_hidden_layers=2, num_attention_heads=8, num_key_value_heads=4, vocab_size=8, precision="bf16")
    a, b = str_backbone.MixtralModel(**kw).to(dev), str_backbone.MixtralModel(few_token_experts=True, **kw).to(dev)
    with torch.no_grad():
        for n, p in a.named_parameters():
            if p.dim() == 2:
                p.copy_(torch.randn(p.shape) * p.shape[1] ** -0.5)
    b.load_state_dict(a.state_dict())
    calls, plain = [], str_backbone.moe_few

    def recorded(*args):
        out = plain(*args)
        calls.append((args, out))
        return out

    monkeypatch.setattr(str_backbone, "moe_few", recorded)
    emb = torch.randn(4, 40, 128, device=dev)
    ca, cb = a.new_cache(), b.new_cache()
    assert torch.equal(a.extend(emb[:, :37], ca), b.extend(emb[:, :37], cb)) and not calls
    for i in range(37, 40):
        a.extend(emb[:, i:i + 1], ca)
        b.extend(emb[:, i:i + 1], cb)
    assert len(calls) == 2 * 3                          # layers x passes, of the one model
    for (x, res, router, s13, s2, inter, E, k, precision, _, _), y in calls:
        assert precision == "bf16" and x.shape == (4, 128)
        w13, w2 = (t.view(torch.bfloat16).float().reshape(s) for t, s in ((s13, (E, 2 * inter, 128)), (s2, (E, 128, inter))))
        want, e, _, _ = moe_exact(x, res, router, w13, w2, k, 2.0 ** -24)
        within(y, want, e, "fp32", "y")
