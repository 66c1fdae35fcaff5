"""Calls of the decoder-layer operators that must not lose anything silently, without a GPU: derivatives that are not built and sizes that
do not fit are refused.  Where a call gets as far as the kernels, plain products stand in for them."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from autodiffusion_amd import _lib, ops, str_backbone, train


@pytest.fixture
def plain_product(monkeypatch):
    """``ops.linear_residual`` as a product of host tensors; yields the keep_slope argument of every call."""
    asked = []

    def product(x, w, bias=None, residual=None, act=0, keep_slope=False):
        asked.append(keep_slope)
        y = x @ w.t()
        return (y, torch.ones_like(y)) if keep_slope else y

    monkeypatch.setattr(ops, "linear_residual", product)
    return asked


@pytest.mark.parametrize("enabled", [True, False])
def test_linear_residual_refuses_forward_mode(plain_product, enabled):
    x, w = torch.randn(3, 4), torch.randn(5, 4)
    with torch.set_grad_enabled(enabled), fw.dual_level():
        for args in ((fw.make_dual(x, torch.ones_like(x)), w), (x, fw.make_dual(w, torch.ones_like(w)))):
            with pytest.raises(NotImplementedError, match="forward mode"):
                train.linear_residual(*args, act=5)


def test_linear_residual_keeps_a_slope_only_where_a_graph_is_recorded(plain_product):
    x, w = torch.randn(3, 4), torch.randn(5, 4).requires_grad_()
    with torch.no_grad():
        assert not train.linear_residual(x, w, act=5).requires_grad
    assert not plain_product[-1]
    assert train.linear_residual(x, w, act=5).requires_grad and plain_product[-1]
    assert not train.linear_residual(x, w.detach(), act=5).requires_grad and not plain_product[-1]


def test_rope_refuses_gradients_of_its_frequencies(monkeypatch):
    monkeypatch.setattr(ops, "rope", lambda q, k, positions, inv_freq, amplitude, layout, inverse=False: (q * float(amplitude), None if k is None else k * 1))
    q, k, w = torch.randn(1, 2, 3, 8).requires_grad_(), torch.randn(1, 2, 1, 8), torch.ones(4, dtype=torch.float64)
    for keys in (None, k):
        with pytest.raises(NotImplementedError, match="`inv_freq`"):
            train.rope(q, keys, 0, w.clone().requires_grad_())
        with pytest.raises(NotImplementedError, match="`amplitude`"):
            train.rope(q, keys, 0, w, torch.tensor(1.5, requires_grad=True))
        assert train.rope(q, keys, 0, w, torch.tensor(1.5))[0].requires_grad
        with torch.no_grad():                                        # nothing to lose
            assert torch.equal(train.rope(q, keys, 0, w.clone().requires_grad_(), 2.0)[0], 2 * q)
    for enabled in (True, False):
        with torch.set_grad_enabled(enabled), fw.dual_level(), pytest.raises(NotImplementedError, match="forward mode"):
            train.rope(q.detach(), None, 0, fw.make_dual(w, torch.ones_like(w)))


WRAP = 2 ** 32                                                       # what a C int drops


def huge(*shape, dtype=torch.bfloat16):
    """A tensor of any shape in one value's memory."""
    return torch.zeros(1, dtype=dtype).expand(shape)


def test_sizes_beyond_32_bits_are_refused():
    """Not passed on as their low 32 bits: tokens that nobody would have turned, columns that nobody would have computed."""
    w = torch.ones(1, dtype=torch.float64)
    for q, k in ((huge(WRAP, 1, 2), None), (huge(1, WRAP + 1, 1, 2), None), (huge(WRAP + 1, 1, 1, 2), None), (huge(4, WRAP + 1, 2), None),
                 (huge(4, 1, WRAP + 2), None), (huge(4, 1, 2), huge(4, WRAP + 1, 2)), (huge(2 ** 31, 1, 2), None)):
        with pytest.raises(ValueError, match="2\\^31"):
            ops.rope(q, k, 0, w)
    for first in (2 ** 64 + 5, -2 ** 64):
        with pytest.raises(ValueError, match="int64"):
            ops.rope(huge(4, 1, 2), None, first, w)
    x, wt = huge(5, 16), huge(8, 16)
    for a, b in ((x, huge(WRAP + 128, 16)), (huge(5, WRAP + 16), huge(8, WRAP + 16)), (x, huge((1 << 26) + 1, 16))):
        with pytest.raises(ValueError, match="2\\^26"):
            ops.linear_residual(a, b)
        with pytest.raises(ValueError, match="2\\^26"):
            ops.linear_residual_bwd(huge(5, b.shape[0]), a, b)
    for act in (WRAP, WRAP + 5, 7, -1):
        with pytest.raises(ValueError, match="activation"):
            ops.linear_residual(x, wt, act=act)
        with pytest.raises(ValueError, match="activation"):
            ops.linear_residual_bwd(huge(5, 8), x, wt, huge(5, 8, dtype=torch.int16), act=act)
    ok = dict(x=torch.zeros(4, 32), res=None, router_w=torch.zeros(8, 32), w13=torch.zeros(8, 128, 32), w2=torch.zeros(8, 32, 64), inter=64, n_experts=8, top_k=2)
    for bad in (dict(top_k=WRAP + 2), dict(top_k=2 - WRAP), dict(top_k=0), dict(top_k=9), dict(x=huge(WRAP + 4, 32, dtype=torch.float32))):
        with pytest.raises(ValueError, match="top_k"):
            str_backbone.moe_few(**(ok | bad))


def test_forms_of_the_kept_slope():
    x, w = torch.zeros(5, 16, dtype=torch.bfloat16), torch.zeros(8, 16, dtype=torch.bfloat16)
    for keep in (torch.float16, torch.int16, "fp32", 1):
        with pytest.raises(ValueError, match="keep_slope"):
            ops.linear_residual(x, w, act=2, keep_slope=keep)
    for slope in (torch.zeros(5, 8, dtype=torch.bfloat16), torch.zeros(5, 8, dtype=torch.float64), torch.zeros(5, 7)):
        with pytest.raises(ValueError, match="slope"):
            ops.linear_residual_bwd(torch.zeros(5, 8, dtype=torch.bfloat16), x, w, slope, act=2)
    for slope in (torch.zeros(5, 8, dtype=torch.int16), torch.zeros(5, 8)):
        with pytest.raises(_lib.AdxError, match="device memory"):
            ops.linear_residual_bwd(torch.zeros(5, 8, dtype=torch.bfloat16), x, w, slope, act=2)
    lib, pointer = _lib.load(), 4096                     # refused before it is used
    assert lib.adx_linear_residual_bwd_ws_bytes(100, 64, 64, 2 | _lib.SLOPE_F32, 1) == lib.adx_linear_residual_bwd_ws_bytes(100, 64, 64, 2, 1)
    for act in (7, -1):
        assert lib.adx_op_linear_residual(pointer, 64, pointer, 64, None, None, 0, None, pointer, 64, 100, 64, 64, act | _lib.SLOPE_F32, 1, None, 0, None) == 1
        assert b"activation" in lib.adx_last_error()


def test_capture_over_the_leaves_of_a_live_graph_is_refused():
    """On made-up streams (0: the default one): a pass, then captures while its graph lives and after."""
    class Scaled(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, stream, capturing):
            train._leaves_on(ctx, "scaled", stream, lambda: capturing)
            return 2 * x

        @staticmethod
        def backward(ctx, dy):
            return 2 * dy, None, None

    w = torch.randn(3, requires_grad=True)
    y = Scaled.apply(w, 0, False)
    z = Scaled.apply(w, 2, False)                                    # eager passes on any stream
    with pytest.raises(RuntimeError, match="earlier pass"):
        Scaled.apply(w, 2, True)
    del y
    with pytest.raises(RuntimeError, match="earlier pass"):          # the accumulator is still the first pass's
        Scaled.apply(w, 2, True)
    assert torch.equal(torch.autograd.grad(z.sum(), w)[0], torch.full((3,), 2.0))
    del z
    y = Scaled.apply(w, 2, True)
    z = Scaled.apply(w * 1, 2, True) + Scaled.apply(w, 2, True)      # further passes of the same capture, not only over leaves
    assert torch.equal(torch.autograd.grad((y + z).sum(), w)[0], torch.full((3,), 6.0))
    with torch.no_grad():
        Scaled.apply(w, 3, True)                                     # nothing is recorded
    del y, z
    y = Scaled.apply(w, 4, False)                                    # a warm-up on a side stream whose outputs are still held
    z = Scaled.apply(w, 5, True)
    assert torch.equal(torch.autograd.grad(z.sum(), w)[0], torch.full((3,), 2.0))
