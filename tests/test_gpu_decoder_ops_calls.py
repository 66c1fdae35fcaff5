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
    _, _, z, ez = linear_exact(x, w, b, None, "none")
    d = slope_tails(z, act)
    moved = torch.maximum((slope_tails(z + ez, act) - d).abs(), (slope_tails(z - ez, act) - d).abs())         # what the rounding of z changes
    dz = dy.double() * d
    ed = dy.double().abs() * (slope_error(z, act) + moved) + U24 * dz.abs()                            # as a summand
    e = ed + HALF_STEP[kind] * dz.abs() + TINY[kind]                                                   # as an operand
    ax, aw = x.double().abs(), w.double().abs()
    within(db, dz.sum(0), ed.sum(0) + (M + 2) * U24 * (dz.abs() + ed).sum(0), kind, "db")
    within(dw, dz.t() @ x.double(), e.t() @ ax + (M + 2) * U24 * (dz.abs() + e).t() @ ax, kind, "dw")
    within(dx, dz @ w.double(), e @ aw + (N + 2) * U24 * (dz.abs() + e) @ aw, kind, "dx")
    if kind != "fp16" and act in ("silu", "gelu_erf"):
        assert (db.float().abs()[: N // 2] > 0).all()               # small, not nothing


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
