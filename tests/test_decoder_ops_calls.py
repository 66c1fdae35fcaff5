"""Calls of the decoder-layer operators that must not lose anything silently, without a GPU: derivatives that are not built and sizes that
do not fit are refused.  Where a call gets as far as the kernels, plain products stand in for them."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from autodiffusion_amd import ops, train


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
