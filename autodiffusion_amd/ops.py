"""Operator-level wrappers over the C ABI (one HIP kernel launch each).  Device tensors in, device tensors out."""
from __future__ import annotations

import ctypes as C
import functools
import math
import operator
from typing import Optional, Sequence

import torch

from . import _lib
from ._lib import DTYPES, INT_MAX, StepCoef, check, current_stream, device_of, f32c, on_data_device, ptr, stream_on


def timestep_embedding(t: torch.Tensor, dim: int) -> torch.Tensor:
    lib = _lib.load()
    t = t.to(torch.int64).contiguous()
    out = torch.empty(*t.shape, dim, device=t.device, dtype=torch.float32)
    check(lib.adx_op_timestep_embedding(ptr(t), t.numel(), dim, ptr(out), current_stream()), "timestep_embedding")
    return out


def to_bf16(x: torch.Tensor) -> torch.Tensor:
    lib = _lib.load()
    x = f32c(x)
    y = torch.empty(x.shape, device=x.device, dtype=torch.int16)
    check(lib.adx_op_to_bf16(ptr(x), ptr(y), x.numel(), current_stream()), "to_bf16")
    return y


def to_f16(x: torch.Tensor) -> torch.Tensor:
    """fp32 -> fp16 bit patterns (int16 tensor), saturating at +-65504."""
    x = f32c(x)
    y = torch.empty(x.shape, device=x.device, dtype=torch.int16)
    check(_lib.load().adx_op_to_f16(ptr(x), ptr(y), x.numel(), current_stream()), "to_f16")
    return y


def prepare_weight(w: torch.Tensor, precision: str = "fp32") -> torch.Tensor:
    """The device form of an (N, K) weight that ``adx_op_linear`` reads under ``precision``."""
    prec = _lib.PRECISIONS[precision]
    if prec in (_lib.PREC_F16X2, _lib.PREC_F16):        # operand-plane products only: the weight rounded once to fp16
        return to_f16(w)
    if prec == _lib.PREC_BF16:
        return to_bf16(w)
    if prec == _lib.PREC_BF16X3:
        hi = to_bf16(w)
        hi_f = (hi.to(torch.int32) << 16).view(torch.float32)
        return torch.cat([hi.reshape(-1), to_bf16(f32c(w) - hi_f).reshape(-1)])
    return f32c(w)


def linear(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, act: int = _lib.ACT_NONE,
           precision: str = "fp32", prepared_n: int = 0, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(x w^T + bias)``.  With ``prepared_n`` > 0, ``w`` is already the result of ``prepare_weight`` for N = prepared_n.
    ``workspace`` (a CUDA byte tensor of at least ``linear_stage_bytes`` bytes, bf16 precisions) selects the staged entry."""
    lib = _lib.load()
    x = f32c(x)
    K = x.shape[-1]
    N = prepared_n or w.shape[0]
    M = x.numel() // K
    prec = _lib.PRECISIONS[precision]
    wd = w if prepared_n else prepare_weight(w, precision)
    b = f32c(bias) if bias is not None else None
    y = torch.empty(*x.shape[:-1], N, device=x.device, dtype=torch.float32)
    if workspace is not None:
        check(lib.adx_op_linear_staged(ptr(x), ptr(wd), ptr(b), ptr(y), M, N, K, act, prec, ptr(workspace),
                                       workspace.numel() * workspace.element_size(), current_stream()), "linear_staged")
    else:
        check(lib.adx_op_linear(ptr(x), ptr(wd), ptr(b), ptr(y), M, N, K, act, prec, current_stream()), "linear")
    return y


def stage_planes(x: torch.Tensor, precision: str) -> torch.Tensor:
    """K-blocked bf16 planes of an fp32 (M, K) activation, the X operand form of ``linear_planes``."""
    lib = _lib.load()
    x = f32c(x)
    K = x.shape[-1]
    M = x.numel() // K
    prec = _lib.PRECISIONS[precision]
    out = torch.empty(int(lib.adx_linear_planes_bytes(M, K, prec)), dtype=torch.uint8, device=x.device)
    check(lib.adx_op_stage_planes(ptr(x), M, K, prec, ptr(out), current_stream()), "stage_planes")
    return out


def block_weight(w_prepared: torch.Tensor, N: int, K: int, precision: str) -> torch.Tensor:
    """K-blocked form of a weight that ``prepare_weight`` returned, the W operand form of ``linear_planes``."""
    lib = _lib.load()
    prec = _lib.PRECISIONS[precision]
    out = torch.empty(int(lib.adx_linear_planes_bytes(N, K, prec)), dtype=torch.uint8, device=w_prepared.device)
    check(lib.adx_op_block_weight(ptr(w_prepared), N, K, prec, ptr(out), current_stream()), "block_weight")
    return out


def linear_planes(x_planes: torch.Tensor, w_blocked: torch.Tensor, bias: Optional[torch.Tensor], M: int, N: int, K: int,
                  act: int = _lib.ACT_NONE, precision: str = "bf16x3", out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(x w^T + bias)`` from operands already in the staged kernel's layout: only the product kernel runs."""
    lib = _lib.load()
    b = f32c(bias) if bias is not None else None
    y = out if out is not None else torch.empty(M, N, device=x_planes.device, dtype=torch.float32)
    check(lib.adx_op_linear_planes(ptr(x_planes), ptr(w_blocked), ptr(b), ptr(y), M, N, K, act, _lib.PRECISIONS[precision], current_stream()),
          "linear_planes")
    return y


def mlp256(x: torch.Tensor, w1_blocked: torch.Tensor, b1: Optional[torch.Tensor], act1: int, w2_blocked: torch.Tensor,
           b2: Optional[torch.Tensor], act2: int = _lib.ACT_NONE, gate: Optional[torch.Tensor] = None, res: Optional[torch.Tensor] = None,
           precision: str = "bf16x3", out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``res + gate * act2(act1(x w1^T + b1) w2^T + b2)`` for x (M, 256) in one kernel; weights in ``block_weight`` form."""
    lib = _lib.load()
    x = f32c(x)
    M = x.shape[0]
    planes = 2 if precision == "bf16x3" else 1
    nbytes = w1_blocked.numel() * w1_blocked.element_size()
    N1 = nbytes // (256 * 2 * planes)                   # bf16 elements, one or two planes
    if N1 * 256 * 2 * planes != nbytes or w2_blocked.numel() * w2_blocked.element_size() != nbytes or x.shape[-1] != 256:
        raise ValueError("mlp256: x must be (M, 256) and both weights the block_weight form of (N1, 256) / (256, N1) matrices")
    for t, n in ((b1, N1), (b2, 256), (gate, M * 256), (res, M * 256), (out, M * 256)):
        if t is not None and t.numel() != n:
            raise ValueError("mlp256: operand of the wrong size")
    b1 = f32c(b1) if b1 is not None else None
    b2 = f32c(b2) if b2 is not None else None
    gate = f32c(gate) if gate is not None else None
    res = f32c(res) if res is not None else None
    y = out if out is not None else torch.empty(M, 256, device=x.device, dtype=torch.float32)
    check(lib.adx_op_mlp256(ptr(x), ptr(w1_blocked), ptr(b1), int(act1), ptr(w2_blocked), ptr(b2), int(act2), ptr(gate), ptr(res), ptr(y),
                            M, N1, _lib.PRECISIONS[precision], current_stream()), "adx_op_mlp256")
    return y


def linear_stage_bytes(M: int, N: int, K: int, precision: str) -> int:
    return int(_lib.load().adx_linear_stage_bytes(int(M), int(N), int(K), _lib.PRECISIONS[precision]))


def layernorm(x: torch.Tensor, gamma=None, beta=None, shift=None, scale=None, eps: float = 1e-5, relu: bool = False) -> torch.Tensor:
    lib = _lib.load()
    x = f32c(x)
    d = x.shape[-1]
    rows = x.numel() // d
    ld_mod = 0
    if shift is not None:
        shift, scale = f32c(shift), f32c(scale)
        ld_mod = d
    y = torch.empty_like(x)
    check(lib.adx_op_layernorm(ptr(x), ptr(f32c(gamma)) if gamma is not None else None, ptr(f32c(beta)) if beta is not None else None,
                               ptr(shift), ptr(scale), ld_mod, eps, int(relu), rows, d, ptr(y), current_stream()), "layernorm")
    return y


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, n_head: int, scale: Optional[float] = None,
              mask_off: int = -1, precision: str = "fp32") -> torch.Tensor:
    """q (B,Sq,H*dh), k (B,Skv,H*dh), v (B,Skv,H*dv) -> (B,Sq,H*dv)."""
    lib = _lib.load()
    q, k, v = f32c(q), f32c(k), f32c(v)
    B, Sq, Skv = q.shape[0], q.shape[1], k.shape[1]
    dh, dv = q.shape[2] // n_head, v.shape[2] // n_head
    if scale is None:
        scale = dh ** -0.5
    o = torch.empty(B, Sq, n_head * dv, device=q.device, dtype=torch.float32)
    check(lib.adx_op_attention_prec(ptr(q), ptr(k), ptr(v), ptr(o), B, n_head, Sq, Skv, dh, dv, float(scale), mask_off,
                                    _lib.PRECISIONS[precision], current_stream()), "attention")
    return o


def normalize(x: torch.Tensor) -> torch.Tensor:
    lib = _lib.load()
    x = f32c(x)
    y = torch.empty_like(x)
    check(lib.adx_op_normalize(ptr(x), ptr(y), x.numel() // x.shape[-1], x.shape[-1], current_stream()), "normalize")
    return y


def denormalize(y: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    lib = _lib.load()
    y = f32c(y)
    r = f32c(residual) if residual is not None else None
    x = torch.empty_like(y)
    check(lib.adx_op_denormalize(ptr(y), ptr(r), ptr(x), y.numel() // y.shape[-1], y.shape[-1], current_stream()), "denormalize")
    return x


def sched_step(x: torch.Tensor, model_out: torch.Tensor, z: Optional[torch.Tensor], row: Sequence[float], want_x0: bool = False):
    lib = _lib.load()
    x, model_out = f32c(x), f32c(model_out)
    z = f32c(z) if z is not None else None
    coef = torch.tensor([float(v) for v in row], dtype=torch.float32, device=x.device)
    xn = torch.empty_like(x)
    x0 = torch.empty_like(x) if want_x0 else None
    check(lib.adx_op_sched_step(ptr(x), ptr(model_out), ptr(z), ptr(xn), ptr(x0), x.numel(), ptr(coef), current_stream()), "sched_step")
    return (xn, x0) if want_x0 else xn


def select_modes(traj: torch.Tensor, k: int, em_iter: int = 25):
    """(B, M, L, D) sampled trajectories -> (modes (B, k, L, D), weights (B, k)), weights descending."""
    lib = _lib.load()
    traj = f32c(traj)
    B, M, L, D = traj.shape
    modes = torch.empty(B, k, L, D, device=traj.device, dtype=torch.float32)
    weights = torch.empty(B, k, device=traj.device, dtype=torch.float32)
    check(lib.adx_op_select_modes(ptr(traj), B, M, L, D, int(k), int(em_iter), ptr(modes), ptr(weights), current_stream()), "select_modes")
    return modes, weights


def q_sample(x0: torch.Tensor, noise: torch.Tensor, t: torch.Tensor, sqrt_acp: torch.Tensor, sqrt_1m_acp: torch.Tensor,
             want_v: bool = False):
    """x_t = sqrt_acp[t] x0 + sqrt_1m_acp[t] noise with a timestep per batch row (dim 0); also v = sqrt_acp[t] noise -
    sqrt_1m_acp[t] x0 when ``want_v``.  Returns (x_t, v or None)."""
    lib = _lib.load()
    x0, noise = f32c(x0), f32c(noise)
    t = t.to(device=x0.device, dtype=torch.int64).contiguous()
    sa, s1 = f32c(sqrt_acp).to(x0.device), f32c(sqrt_1m_acp).to(x0.device)
    n_rows = x0.shape[0]
    row_len = x0.numel() // n_rows
    xt = torch.empty_like(x0)
    v = torch.empty_like(x0) if want_v else None
    check(lib.adx_op_q_sample(ptr(x0), ptr(noise), ptr(t), ptr(sa), ptr(s1), ptr(xt), ptr(v), n_rows, row_len, current_stream()), "q_sample")
    return xt, v


def weighted_mse(out: torch.Tensor, target: torch.Tensor, t: torch.Tensor, weight: torch.Tensor):
    """(loss_rows (B,), loss_mean ()): loss_rows[b] = weight[t[b]] * mean((out[b] - target[b])**2)."""
    lib = _lib.load()
    out, target = f32c(out), f32c(target)
    t = t.to(device=out.device, dtype=torch.int64).contiguous()
    w = f32c(weight).to(out.device)
    n_rows = out.shape[0]
    row_len = out.numel() // n_rows
    rows = torch.empty(n_rows, device=out.device, dtype=torch.float32)
    mean = torch.empty(1, device=out.device, dtype=torch.float32)
    check(lib.adx_op_weighted_mse(ptr(out), ptr(target), ptr(t), ptr(w), ptr(rows), ptr(mean), n_rows, row_len, current_stream()), "weighted_mse")
    return rows, mean.reshape(())


def randn(n_lead: int, batch: int, row_len: int, seed: int, row0: int = 0, device="cuda") -> torch.Tensor:
    """(n_lead, batch, row_len) N(0,1) values from the library's counter-based generator (Philox4x32-10 + Box-Muller): the value of
    element e of batch row b under leading index l depends only on (seed, row0 + b, l, e // 4)."""
    lib = _lib.load()
    out = torch.empty(n_lead, batch, row_len, device=device, dtype=torch.float32)
    ctl = torch.empty(2, device=out.device, dtype=torch.int64)
    check(lib.adx_op_randn(ptr(out), n_lead, batch, row_len, int(seed) & 0xFFFFFFFFFFFFFFFF, int(row0), ptr(ctl), current_stream()), "randn")
    return out


# ------------------------------------------------------------------------------------------------ fp32 / bf16 / fp16 tensors
_Strides = C.c_int64 * 12


def rope_frequencies(rotary_dim: int, theta: float = 1e4, scaling: Optional[str] = None, factor: float = 1.0, trained_length: int = 4096,
                     fast_turns: float = 32.0, slow_turns: float = 1.0, device="cuda"):
    """(inv_freq, amplitude) for ``rope``: radians a position of every rotated pair, fp64 (rotary_dim / 2,), and the factor on its outputs.
    ``scaling`` None: theta^(-2 j / rotary_dim).  For positions beyond ``trained_length``: "linear" slows every pair by ``factor``;
    "base" raises theta so that the slowest pair is slowed by ``factor`` and the fastest by nothing; "parts" slows the pairs that make less than
    ``slow_turns`` turns in the trained length, keeps those that make more than ``fast_turns``, blends those between, and raises the
    amplitude to 0.1 ln(factor) + 1."""
    if rotary_dim <= 0 or rotary_dim % 2 or theta <= 0 or factor <= 0:
        raise ValueError("rope_frequencies: an even rotary width, positive theta and factor")
    if scaling not in (None, "linear", "base", "parts"):
        raise ValueError(f"rope_frequencies: unknown scaling {scaling!r}")
    if scaling == "base":
        if rotary_dim == 2:
            raise ValueError("rope_frequencies: scaling 'base' needs more than one pair")
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    inv = theta ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    amplitude = 1.0
    if scaling == "linear":
        inv = inv / factor
    elif scaling == "parts":
        if not fast_turns > slow_turns or trained_length <= 0:
            raise ValueError("rope_frequencies: fast_turns above slow_turns and a positive trained length")
        keep = ((trained_length * inv / (2 * math.pi) - slow_turns) / (fast_turns - slow_turns)).clamp(0, 1)
        inv = inv * keep + inv / factor * (1 - keep)
        amplitude = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    return inv.to(device), amplitude


@on_data_device
def rope(q: torch.Tensor, k: Optional[torch.Tensor], positions, inv_freq: torch.Tensor, amplitude: float = 1.0, layout: str = "half",
         inverse: bool = False, inplace: bool = False):
    """Rotary positions of q (B, S, Hq, dh) and k (B, S, Hk, dh) -- or (N, H, dh) for packed tokens -- in one launch -> (q', k').

    ``positions``: an int (token s of every item at positions + s) or an int64 tensor that broadcasts to the token axes; ``inv_freq`` (rd / 2,)
    fp64 and ``amplitude`` as ``rope_frequencies`` gives them: the first rd <= dh values of a head are rotated, the others copied.  ``layout``:
    "half" pairs (j, j + rd / 2), "interleaved" (2 j, 2 j + 1).  fp32, bf16 or fp16; any strides with adjacent values in a head (a slice of
    a fused q / k / v product, heads before tokens as a transposed view); every axis below 2^31.  ``inverse`` applies the transpose -- the gradient.
    ``inplace`` writes into q and k, which must not overlap each other."""
    if layout != "half" and layout != "interleaved":
        raise ValueError(f"rope: unknown layout {layout!r}")
    dtype, shape = q.dtype, q.shape
    dt, axes = DTYPES.get(dtype), len(shape)
    if dt is None or (k is not None and k.dtype != dtype):
        raise ValueError("rope: q and k are fp32, bf16 or fp16, both the same")
    if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError("rope: inv_freq is a contiguous fp64 vector (rope_frequencies)")
    if axes not in (3, 4) or (k is not None and (k.shape[:-2] != shape[:-2] or k.shape[-1] != shape[-1])):
        raise ValueError("rope: q (B, S, Hq, dh) and k (B, S, Hk, dh), or (N, Hq, dh) and (N, Hk, dh)")
    hq, dh, rd = shape[-2], shape[-1], 2 * inv_freq.shape[0]
    hk = 0 if k is None else k.shape[-2]
    if rd > dh or rd == 0 or hq == 0 or (k is not None and hk == 0):
        raise ValueError(f"rope: {rd} rotated values of heads of {dh}, and at least one head")
    if shape[0] > INT_MAX or shape[-3] > INT_MAX or hq > INT_MAX or hk > INT_MAX or dh > INT_MAX:
        raise ValueError("rope: items, tokens, heads and head width are below 2^31 each")
    pos = positions if isinstance(positions, torch.Tensor) else None
    first = operator.index(positions) if pos is None else 0
    if not -(1 << 62) <= first <= 1 << 62:
        raise ValueError("rope: positions are int64")
    if pos is not None and pos.dtype != torch.int64:
        raise ValueError("rope: positions are int64")
    if inplace:
        for t in (q, k):
            if t is not None and dh > 1 and t.stride(-1) != 1:
                raise ValueError("rope: in place needs adjacent values in a head")
            if t is not None and any(n > 1 and st == 0 for n, st in zip(t.shape, t.stride())):
                raise ValueError("rope: in place needs a tensor without repeated elements")
            if t is not None and t.requires_grad and torch.is_grad_enabled():
                raise ValueError("rope: in place is not recorded for gradients (train.rope)")
        if k is not None and k.numel() and k.data_ptr() == q.data_ptr():
            raise ValueError("rope: q and k in place are the same memory")
    stream = stream_on(device_of("rope", q, k, pos, inv_freq))
    if inplace:
        qo, ko = q, k
        for t in (q, k):
            if t is not None and not t.is_inference():
                torch.autograd.graph.increment_version(t)        # a graph that kept the old values notices
    else:
        if dh > 1 and q.stride(-1) != 1:
            q = q.contiguous()
        if k is not None and dh > 1 and k.stride(-1) != 1:
            k = k.contiguous()
        qo, ko = q.new_empty(shape), None if k is None else k.new_empty(k.shape)
    S = shape[-3]
    B = shape[0] if axes == 4 else 1
    if B * S == 0:
        return qo, ko
    pb = ps = 0
    if pos is not None:
        if pos.shape != shape[:-2]:
            pos = pos.expand(shape[:-2])
        ps = pos.stride(-1)
        pb = pos.stride(0) if axes == 4 else 0
    outer = (0,) if axes == 3 else ()
    st = outer + q.stride()[:-1] + outer + qo.stride()[:-1]
    st += (0,) * 6 if k is None else outer + k.stride()[:-1] + outer + ko.stride()[:-1]
    check(_lib.load().adx_op_rope(q.data_ptr(), qo.data_ptr(), hq, None if k is None else k.data_ptr(), None if k is None else ko.data_ptr(), hk,
                                  _Strides(*st), None if pos is None else pos.data_ptr(), pb, ps, first,
                                  inv_freq.data_ptr(), amplitude, B, S, dh, rd, layout == "interleaved", inverse, dt, stream), "rope")
    return qo, ko


def _rows(t: torch.Tensor):
    """(tensor, row stride) of t viewed as rows of its last axis, copied only where its strides do not allow the view."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    rows, width = t.shape
    if width > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, (t.stride(0) if rows > 1 else width)


_SLOPE = (torch.float32, torch.int16, torch.int16)       # by DTYPES code


def _on_pieces(t: torch.Tensor, ld: int):
    """(tensor, row stride) with rows that start on 16 bytes, if whole 16-byte pieces make up a row (else the library lays it out anew)."""
    size, width = t.element_size(), t.shape[1]
    if width * size % 16 == 0 and (ld * size % 16 or t.data_ptr() % 16):
        t, ld = t.clone(memory_format=torch.contiguous_format), width
    return t, ld


_MOST_WIDE = 1 << 26


@functools.lru_cache(maxsize=4096)
def _linear_residual_bytes(M: int, N: int, K: int, dt: int, act: int = -1) -> int:
    lib = _lib.load()
    return int(lib.adx_linear_residual_ws_bytes(M, N, K, dt) if act < 0 else lib.adx_linear_residual_bwd_ws_bytes(M, N, K, act, dt))


@on_data_device
def linear_residual(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
                    act: int = _lib.ACT_NONE, keep_slope=False):
    """``act(x w^T + bias) + residual`` in the tensors' own type (fp32, bf16 or fp16, all the same; fp32 sums, one rounding): x (..., K),
    w (N, K), bias (N,), residual (..., N).  ``act``: ACT_NONE .. ACT_TANH.  ``keep_slope`` also returns the activation's slope, which
    ``linear_residual_bwd`` needs: with torch.float32 in fp32; with True fp32 for fp32 tensors and 16-bit codes (see adx.h) in an int16 tensor
    otherwise -- exact for ACT_RELU and ACT_LEAKY, while slopes of the smooth activations below 2^-16 vanish.  Rows of x, w and residual may be
    strided (adjacent values in a row)."""
    dtype = x.dtype
    dt = DTYPES.get(dtype)
    if dt is None or w.dtype != dtype or (bias is not None and bias.dtype != dtype) or (residual is not None and residual.dtype != dtype):
        raise ValueError("linear_residual: x, w, bias and residual are fp32, bf16 or fp16, all the same")
    if w.dim() != 2 or x.dim() < 1:
        raise ValueError("linear_residual: x (..., K) and w (N, K)")
    N, K = w.shape
    if x.shape[-1] != K or N == 0 or K == 0:
        raise ValueError("linear_residual: x (..., K) and w (N, K)")
    if N > _MOST_WIDE or K > _MOST_WIDE or not 0 <= act <= _lib.ACT_TANH:
        raise ValueError(f"linear_residual: widths {N} and {K} of at most 2^26, activation code {act} of ACT_NONE .. ACT_TANH")
    wide = keep_slope is torch.float32
    if keep_slope is not False and keep_slope is not True and not wide:
        raise ValueError("linear_residual: keep_slope is False, True or torch.float32")
    out_shape = (*x.shape[:-1], N)
    if (bias is not None and bias.shape != (N,)) or (residual is not None and residual.shape != out_shape):
        raise ValueError("linear_residual: bias (N,) and residual of the output's shape")
    stream = stream_on(device_of("linear_residual", x, w, bias, residual))
    y = x.new_empty(out_shape)
    slope = x.new_empty(out_shape, dtype=keep_slope if wide else _SLOPE[dt]) if keep_slope else None
    x2, ldx = _rows(x)
    M = x2.shape[0]
    if M:
        w2, ldw = _rows(w)
        if M > 64:                                       # fewer rows are read where they lie
            (x2, ldx), (w2, ldw) = _on_pieces(x2, ldx), _on_pieces(w2, ldw)
        b = None if bias is None else bias.contiguous()
        r2, ldr = (None, 0) if residual is None else _rows(residual)
        need = _linear_residual_bytes(M, N, K, dt)
        ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
        check(_lib.load().adx_op_linear_residual(x2.data_ptr(), ldx, w2.data_ptr(), ldw, None if b is None else b.data_ptr(),
                                                 None if r2 is None else r2.data_ptr(), ldr, None if slope is None else slope.data_ptr(), y.data_ptr(), N,
                                                 M, N, K, act | _lib.SLOPE_F32 if wide else act, dt, None if ws is None else ws.data_ptr(), need, stream), "linear_residual")
    return (y, slope) if keep_slope else y


@on_data_device
def linear_residual_bwd(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, slope: Optional[torch.Tensor] = None, act: int = _lib.ACT_NONE,
                        need_dx: bool = True, need_dw: bool = True, need_db: bool = True):
    """(dx, dw, db) of ``linear_residual`` from the gradient of its output, its operands and (unless act is ACT_NONE) the slope that
    the forward kept; None for those not asked for.  The gradient of the residual is dy."""
    dtype = dy.dtype
    dt = DTYPES.get(dtype)
    if dt is None or x.dtype != dtype or w.dtype != dtype:
        raise ValueError("linear_residual_bwd: dy, x and w are fp32, bf16 or fp16, all the same")
    wide = slope is not None and slope.dtype == torch.float32
    if slope is not None and not wide and slope.dtype != _SLOPE[dt]:
        raise ValueError("linear_residual_bwd: slope is what linear_residual returned with keep_slope")
    if w.dim() != 2 or x.dim() < 1:
        raise ValueError("linear_residual_bwd: x (..., K), w (N, K), dy and slope (..., N)")
    N, K = w.shape
    if x.shape[-1] != K or dy.shape != (*x.shape[:-1], N) or (slope is not None and slope.shape != dy.shape):
        raise ValueError("linear_residual_bwd: x (..., K), w (N, K), dy and slope (..., N)")
    if N > _MOST_WIDE or K > _MOST_WIDE or not 0 <= act <= _lib.ACT_TANH:
        raise ValueError(f"linear_residual_bwd: widths {N} and {K} of at most 2^26, activation code {act} of ACT_NONE .. ACT_TANH")
    if act != _lib.ACT_NONE and slope is None:
        raise ValueError("linear_residual_bwd: the activation's gradient needs slope (linear_residual with keep_slope)")
    stream = stream_on(device_of("linear_residual_bwd", dy, x, w, slope))
    g, ldd = _rows(dy)
    M = g.shape[0]
    dx = x.new_empty(x.shape) if need_dx else None
    dw = w.new_empty((N, K)) if need_dw else None
    db = w.new_empty((N,)) if need_db else None
    if M == 0:                                           # sums over no rows
        for t in (dw, db):
            if t is not None:
                t.zero_()
    elif need_dx or need_dw or need_db:
        (x2, ldx), (w2, ldw), (g, ldd) = _on_pieces(*_rows(x)), _on_pieces(*_rows(w)), _on_pieces(g, ldd)
        z = None if slope is None else slope.contiguous()
        need = _linear_residual_bytes(M, N, K, dt, act)
        ws = torch.empty(need, dtype=torch.uint8, device=x.device)
        check(_lib.load().adx_op_linear_residual_bwd(g.data_ptr(), ldd, x2.data_ptr(), ldx, w2.data_ptr(), ldw, None if z is None else z.data_ptr(),
                                                     None if dx is None else dx.data_ptr(), None if dw is None else dw.data_ptr(),
                                                     None if db is None else db.data_ptr(), M, N, K, act | _lib.SLOPE_F32 if wide else act, dt, ws.data_ptr(), need, stream),
              "linear_residual_bwd")
    return dx, dw, db
