"""Refusals of the decoder-layer operators, without a GPU: the raw ABI answers before any device work (the pointers below are never
dereferenced) and the Python entry points before they touch the library."""
import ctypes as C

import pytest
import torch

from autodiffusion_amd import _lib, ops, str_backbone, train

FAKE, F32, BF16, F16 = 4096, 0, 1, 2


def refused(rc, word):
    assert rc == 1 and word in _lib.load().adx_last_error(), (rc, _lib.load().adx_last_error())


def test_rope_abi_refusals():
    lib = _lib.load()
    strides = (C.c_int64 * 12)(*([64, 64, 64] * 4))

    def call(q=FAKE, qo=2 * FAKE, hq=1, k=None, ko=None, hk=0, st=strides, freq=FAKE, B=1, S=1, dh=64, rd=64, dt=F32):
        return lib.adx_op_rope(q, qo, hq, k, ko, hk, st, None, 0, 0, 0, freq, 1.0, B, S, dh, rd, 0, 0, dt, None)

    refused(call(q=None), b"null pointer")
    refused(call(k=FAKE), b"null pointer")                          # keys without a place for their result
    refused(call(freq=None), b"null pointer")
    refused(call(st=None), b"null pointer")
    refused(call(dt=3), b"element type")
    for bad in (dict(rd=63), dict(rd=66), dict(rd=0), dict(dh=0), dict(hq=0), dict(hk=2), dict(B=-1), dict(S=-1), dict(k=FAKE, ko=3 * FAKE, hk=0)):
        refused(call(**bad), b"even rotary width")
    refused(call(dh=8192, rd=8192), b"4096")
    refused(call(qo=FAKE, st=(C.c_int64 * 12)(64, 64, 64, 128, 128, 128, 0, 0, 0, 0, 0, 0)), b"in place")
    refused(call(B=1 << 20, S=1 << 20, hq=4096), b"too many tokens")
    assert call(B=0) == 0 and call(S=0) == 0                        # no tokens: nothing to do


def test_linear_residual_abi_refusals():
    lib = _lib.load()

    def call(x=FAKE, w=FAKE, y=FAKE, ldx=64, ldw=64, ldr=0, ldy=64, M=100, N=64, K=64, act=0, dt=BF16, ws=None, n=0):
        return lib.adx_op_linear_residual(x, ldx, w, ldw, None, None, ldr, None, y, ldy, M, N, K, act, dt, ws, n, None)

    for bad in (dict(x=None), dict(w=None), dict(y=None)):
        refused(call(**bad), b"null pointer")
    refused(call(dt=3), b"element type")
    refused(call(act=7), b"activation")
    refused(call(act=-1), b"activation")
    for bad in (dict(M=-1), dict(N=0), dict(K=0), dict(M=(1 << 30) + 1), dict(N=(1 << 26) + 1, ldy=1 << 27), dict(K=(1 << 26) + 1)):
        refused(call(**bad), b"needs 0 <= M")
    refused(call(ldy=63), b"overlap")
    refused(call(ldx=-1), b"negative")
    assert call(M=0) == 0
    need = lib.adx_linear_residual_ws_bytes(100, 64, 8192, BF16)
    assert need > 0                                                  # few tiles, a long sum: split
    refused(call(K=8192, ldx=8192, ldw=8192), b"workspace")
    refused(call(K=8192, ldx=8192, ldw=8192, ws=FAKE, n=need - 1), b"workspace")
    refused(call(K=8192, ldx=8192, ldw=8192, ws=FAKE + 8, n=need), b"workspace")
    assert lib.adx_linear_residual_ws_bytes(0, 64, 64, BF16) == 0 and lib.adx_linear_residual_ws_bytes(8, 64, 64, 9) == 0


def test_linear_residual_bwd_abi_refusals():
    lib = _lib.load()

    def call(dy=FAKE, x=FAKE, w=FAKE, slope=FAKE, dx=FAKE, dw=FAKE, db=FAKE, M=100, N=64, K=64, act=2, dt=BF16, ws=FAKE, n=1 << 40):
        return lib.adx_op_linear_residual_bwd(dy, N, x, K, w, K, slope, dx, dw, db, M, N, K, act, dt, ws, n, None)

    for bad in (dict(dy=None), dict(x=None), dict(w=None), dict(slope=None)):
        refused(call(**bad), b"null pointer")
    refused(call(dt=-1), b"element type")
    refused(call(act=9), b"activation")
    for bad in (dict(M=0), dict(N=(1 << 26) + 1), dict(K=(1 << 26) + 1)):
        refused(call(**bad), b"needs 1 <= M")
    need = lib.adx_linear_residual_bwd_ws_bytes(100, 64, 64, 2, BF16)
    assert need >= 100 * 64 * 2
    refused(call(n=need - 1), b"workspace")
    refused(call(ws=None), b"workspace")


def test_moe_few_abi_refusals():
    lib = _lib.load()

    def call(x=FAKE, router=FAKE, w13=FAKE, w2=FAKE, T=8, d=64, inter=64, E=8, k=2, at=F32, prec=0, ws=FAKE, n=1 << 30, y=FAKE):
        return lib.adx_op_moe_few(x, None, router, w13, w2, T, d, inter, E, k, at, prec, ws, n, y, None)

    for bad in (dict(x=None), dict(router=None), dict(w13=None), dict(w2=None), dict(ws=None), dict(y=None)):
        refused(call(**bad), b"null pointer")
    for bad in (dict(T=0), dict(T=65), dict(d=48), dict(inter=40), dict(E=65), dict(E=0), dict(k=9, E=16), dict(k=0), dict(E=2, k=3), dict(d=0),
                dict(d=1 << 15, inter=(1 << 13) + 32)):
        refused(call(**bad), b"1 <= T <= 64")
    for at, prec in ((BF16, 0), (BF16, 4), (F16, 1), (F16, 0), (F32, 3), (3, 0), (BF16, 2)):
        refused(call(at=at, prec=prec), b"tokens with")
    refused(call(x=FAKE + 4), b"aligned")
    need = lib.adx_moe_few_workspace_bytes(8, 64, 64, 8, 2, F32, 0)
    refused(call(n=need - 1), b"workspace")
    assert lib.adx_moe_few_workspace_bytes(65, 64, 64, 8, 2, F32, 0) == 0 and lib.adx_moe_few_workspace_bytes(8, 64, 64, 8, 2, BF16, 0) == 0


def test_python_refusals():
    q = torch.zeros(2, 3, 4, 64)
    w, amp = ops.rope_frequencies(64, device="cpu")
    for bad in (dict(layout="other"), dict(inv_freq=w.float()), dict(inv_freq=torch.cat([w, w])), dict(k=torch.zeros(2, 3, 4, 32)), dict(k=q.half()),
                dict(q=q.double()), dict(k=torch.zeros(2, 4, 4, 64)), dict(q=q[0, 0]), dict(k=q, inplace=True)):
        args = dict(q=q, k=None, positions=0, inv_freq=w, layout="half", inplace=False) | bad
        with pytest.raises(ValueError):
            ops.rope(args["q"], args["k"], args["positions"], args["inv_freq"], layout=args["layout"], inplace=args["inplace"])
    with pytest.raises(TypeError):
        ops.rope(q, None, 1.5, w)
    with pytest.raises(ValueError, match="gradients"):
        ops.rope(q.clone().requires_grad_(), None, 0, w, inplace=True)
    with pytest.raises(_lib.AdxError, match="device memory"):
        ops.rope(q, None, 0, w)
    for bad in (dict(rotary_dim=7), dict(theta=0.0), dict(factor=0.0), dict(scaling="other"), dict(scaling="base", rotary_dim=2),
                dict(scaling="parts", fast_turns=1.0)):
        with pytest.raises(ValueError):
            ops.rope_frequencies(**(dict(rotary_dim=64, device="cpu") | bad))
    x, wt = torch.zeros(5, 16), torch.zeros(8, 16)
    for args in ((x, wt.half()), (x, torch.zeros(8, 15)), (x.double(), wt.double()), (x, wt, torch.zeros(7)), (x, wt, None, torch.zeros(5, 7)),
                 (x, wt, None, torch.zeros(8)), (x, wt, torch.zeros(8, dtype=torch.bfloat16)), (x, torch.zeros(0, 16))):
        with pytest.raises(ValueError):
            ops.linear_residual(*args)
    with pytest.raises(_lib.AdxError, match="device memory"):
        ops.linear_residual(x, wt)
    with pytest.raises(_lib.AdxError, match="device memory"):
        train.linear_residual(x.requires_grad_(), wt)
    with pytest.raises(ValueError):
        ops.linear_residual_bwd(torch.zeros(5, 8), x, wt, None, act=2)                       # no slope
    with pytest.raises(ValueError):
        ops.linear_residual_bwd(torch.zeros(5, 8), x, wt, torch.zeros(5, 8, dtype=torch.int16), act=2)        # a slope of another type
    with pytest.raises(ValueError):
        ops.linear_residual_bwd(torch.zeros(5, 7), x, wt)
    t, r, w13, w2 = torch.zeros(4, 32), torch.zeros(8, 32), torch.zeros(8, 128, 32), torch.zeros(8, 32, 64)
    ok = dict(x=t, res=None, router_w=r, w13=w13, w2=w2, inter=64, n_experts=8, top_k=2, precision="fp32")
    for bad in (dict(w13=w13[:7]), dict(w2=w2.half()), dict(router_w=r.half()), dict(router_w=r[:4]), dict(res=torch.zeros(4, 31)), dict(x=t.double()),
                dict(precision="bf16"), dict(w13=w13.transpose(1, 2)), dict(x=t[0]), dict(w13=w13.to(torch.int32))):
        with pytest.raises(ValueError):
            str_backbone.moe_few(**(ok | bad))
    with pytest.raises(_lib.AdxError, match="device memory"):
        str_backbone.moe_few(**ok)
    for bad in (dict(hidden_size=48, num_attention_heads=3, num_key_value_heads=3), dict(intermediate_size=80), dict(num_local_experts=65),
                dict(num_local_experts=16, num_experts_per_tok=9)):
        with pytest.raises(ValueError, match="few_token_experts"):
            str_backbone.MixtralModel(**(dict(hidden_size=64, intermediate_size=96, num_hidden_layers=1, num_attention_heads=4, num_key_value_heads=4,
                                              vocab_size=8, few_token_experts=True) | bad))
