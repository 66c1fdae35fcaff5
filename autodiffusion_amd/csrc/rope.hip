// Rotary positions of queries and keys: every pair (a, b) of a head's first `rd` values is turned by the angle p * w_j of its
// token's position p and its own frequency w_j and scaled by an amplitude A,
//     (a, b) -> A (a cos - b sin, b cos + a sin),
// with pairs (j, j + rd / 2) ("half") or (2 j, 2 j + 1) ("interleaved"); the values behind the first rd are copied.  The map is
// linear and orthogonal up to A, so its transpose -- the gradient -- is the same map with the angle negated (inverse != 0).
//
// Angles.  p * w reaches 10^6 radians at far positions, where fp32 keeps two digits of the turn: product and reduction run in 64
// bits (turns = p * w / 2 pi, quarter turns taken off), sine and cosine of the rest, |x| <= pi / 4, in 32.  They cost as much as
// moving a few hundred bytes, so a workgroup computes each (token, pair) once, keeps it in LDS and applies it to every head of
// both tensors.
//
// Bound: memory.  One item = V pairs of one head = two 16-byte loads and stores (V = 8 for 16-bit types); q and k share the launch.
// 671 MB moved (bf16, 8 x 4096 tokens, 32 + 8 heads of 128): 135 us, 4.97 of the 5.1 TB/s of a large copy.  One token of 32 + 8
// heads: 3.0 us, 3.6 with one workgroup a token; of 128 + 8 heads of 256 fp32 values 3.8 and 12.9.
#include "adx_ops.h"
#include "engine.h"
#include "typed.h"

namespace adx {
namespace {

constexpr int ROPE_THREADS = 256;
constexpr int ROPE_LDS = 2048;               // (token, pair) angles of one workgroup: 16 KB

struct RopeTensor {
    const void* x; void* y;
    int64_t xb, xs, xh, yb, ys, yh;          // element strides of batch item, token, head (the last axis is contiguous)
    int heads;
};

struct RopeArgs {
    RopeTensor t[2];
    const int64_t* pos; int64_t pb, ps, pos0;        // position of token (b, s): pos[b pb + s ps], or pos0 + s without `pos`
    const double* inv_freq;
    float amplitude;
    int64_t tokens; int S;
    int pairs, tail;                          // rd / 2, dh - rd (0 where the outputs are the inputs: the tail stays as it is)
    int per_group;                            // tokens of one workgroup
    float sign;                               // -1: the transpose
};

// sin and cos of 2 pi r
__device__ __forceinline__ void turn(double r, float* s, float* c) {
    r -= rint(r);
    const double q = rint(4.0 * r);
    float sn, cn;
    sincospif((float)((4.0 * r - q) * 0.5), &sn, &cn);           // |argument| <= 1/4
    const int k = (int)q & 3;
    const float a = (k & 1) ? cn : sn, b = (k & 1) ? sn : cn;
    *s = (k & 2) ? -a : a;
    *c = (k == 1 || k == 2) ? -b : b;
}

template <typename T, int V, bool INTER>
__global__ __launch_bounds__(ROPE_THREADS) void rope_kernel(const RopeArgs a) {
    __shared__ float2 angle[ROPE_LDS];                            // (A cos, +-A sin) of (token, pair)
    const int tid = threadIdx.x, P = a.pairs, per = a.per_group;
    const int64_t tok0 = (int64_t)blockIdx.x * per;
    const int n_tok = (int)(a.tokens - tok0 < per ? a.tokens - tok0 : per);
    for (int i = tid; i < n_tok * P; i += ROPE_THREADS) {
        const int tk = i / P, j = i - tk * P;
        const int64_t n = tok0 + tk, b = n / a.S, s = n - b * a.S;
        const double p = (double)(a.pos ? a.pos[b * a.pb + s * a.ps] : a.pos0 + s);
        float sn, cn;
        turn(p * (a.inv_freq[j] * 0.15915494309189533577), &sn, &cn);
        angle[i] = make_float2(a.amplitude * cn, a.sign * a.amplitude * sn);
    }
    __syncthreads();
    const int heads = a.t[0].heads + a.t[1].heads;
    const int turned = P / V, chunks = turned + (a.tail + 2 * V - 1) / (2 * V);
    // a thread keeps its chunk and walks (token, head) rows; chunks beyond the workgroup's width take another round
    for (int c0 = 0; c0 < chunks; c0 += ROPE_THREADS) {
        const int width = min(chunks - c0, ROPE_THREADS), rows = ROPE_THREADS / width;
        const int r0 = tid / width, c = c0 + tid - r0 * width;
        if (r0 >= rows) continue;
        const bool is_tail = c >= turned;
        const int at = is_tail ? 2 * P + (c - turned) * 2 * V : INTER ? 2 * c * V : c * V;
        const int at2 = is_tail || INTER ? at + V : at + P;
        const bool two = !is_tail || (c - turned) * 2 * V + V < a.tail;
        int tk = 0, h = (int)blockIdx.y * rows + r0;
        const int step = rows * (int)gridDim.y;
        while (h >= heads) { h -= heads; ++tk; }
        while (tk < n_tok) {
            const RopeTensor& t = a.t[h >= a.t[0].heads];
            const int hh = h >= a.t[0].heads ? h - a.t[0].heads : h;
            const int64_t n = tok0 + tk, b = n / a.S, s = n - b * a.S;
            const T* x = static_cast<const T*>(t.x) + b * t.xb + s * t.xs + hh * t.xh;
            T* y = static_cast<T*>(t.y) + b * t.yb + s * t.ys + hh * t.yh;
            typedef Pack<T, V> P_t;
            P_t u = *reinterpret_cast<const P_t*>(x + at), v = u;
            if (two) v = *reinterpret_cast<const P_t*>(x + at2);
            if (!is_tail) {
                const float2* w = angle + tk * P + c * V;
                if (INTER) {
                    T buf[2 * V];
#pragma unroll
                    for (int e = 0; e < V; ++e) { buf[e] = u.v[e]; buf[V + e] = v.v[e]; }
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float p = (float)buf[2 * e], q = (float)buf[2 * e + 1];
                        buf[2 * e] = (T)(p * w[e].x - q * w[e].y);
                        buf[2 * e + 1] = (T)(q * w[e].x + p * w[e].y);
                    }
#pragma unroll
                    for (int e = 0; e < V; ++e) { u.v[e] = buf[e]; v.v[e] = buf[V + e]; }
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float p = (float)u.v[e], q = (float)v.v[e];
                        u.v[e] = (T)(p * w[e].x - q * w[e].y);
                        v.v[e] = (T)(q * w[e].x + p * w[e].y);
                    }
                }
            }
            *reinterpret_cast<P_t*>(y + at) = u;
            if (two) *reinterpret_cast<P_t*>(y + at2) = v;
            h += step;
            while (h >= heads) { h -= heads; ++tk; }
        }
    }
}

template <typename T, int V>
void launch_rope(const RopeArgs& a, bool inter, dim3 grid, hipStream_t s) {
    if (inter) hipLaunchKernelGGL((rope_kernel<T, V, true>), grid, dim3(ROPE_THREADS), 0, s, a);
    else hipLaunchKernelGGL((rope_kernel<T, V, false>), grid, dim3(ROPE_THREADS), 0, s, a);
}

}  // namespace
}  // namespace adx

using namespace adx;

#define ADX_API extern "C" __attribute__((visibility("default")))

ADX_API int adx_op_rope(const void* q, void* q_out, int heads_q, const void* k, void* k_out, int heads_k, const int64_t* strides_host,
                        const int64_t* positions, int64_t pos_stride_b, int64_t pos_stride_s, int64_t pos0, const double* inv_freq, float amplitude,
                        int B, int S, int dh, int rotary_dim, int interleaved, int inverse, int dtype, void* stream) {
    if (!q || !q_out || !strides_host || !inv_freq || (!k != !k_out)) { set_error("rope: null pointer"); return ADX_EINVAL; }
    if (!dtype_ok(dtype)) { set_error("rope: unknown element type"); return ADX_EINVAL; }
    if (B < 0 || S < 0 || heads_q <= 0 || (k ? heads_k <= 0 : heads_k != 0) || dh <= 0 || rotary_dim <= 0 || (rotary_dim & 1) || rotary_dim > dh) {
        set_error("rope: needs heads, an even rotary width of at most the head width, and no heads without a tensor"); return ADX_EINVAL;
    }
    if (rotary_dim > 2 * ROPE_LDS || (int64_t)heads_q + heads_k > (1 << 20)) { set_error("rope: at most 4096 rotated values a head and 2^20 heads"); return ADX_EINVAL; }
    const int64_t tokens = (int64_t)B * S;
    if (tokens == 0) return ADX_OK;
    RopeArgs a;
    const bool in_place = q == q_out && (!k || k == k_out);
    const int64_t* st = strides_host;
    a.t[0] = RopeTensor{q, q_out, st[0], st[1], st[2], st[3], st[4], st[5], heads_q};
    a.t[1] = RopeTensor{k, k_out, st[6], st[7], st[8], st[9], st[10], st[11], heads_k};
    for (int i = 0; i < (k ? 2 : 1); ++i) {
        const RopeTensor& t = a.t[i];
        if (t.x == t.y && (t.xb != t.yb || t.xs != t.ys || t.xh != t.yh)) { set_error("rope: an output in place of its input needs the input's strides"); return ADX_EINVAL; }
    }
    a.pos = positions; a.pb = pos_stride_b; a.ps = pos_stride_s; a.pos0 = pos0;
    a.inv_freq = inv_freq; a.amplitude = amplitude; a.tokens = tokens; a.S = S;
    a.pairs = rotary_dim / 2; a.tail = in_place ? 0 : dh - rotary_dim;
    a.sign = inverse ? -1.f : 1.f;
    // widest vector that every row start, every stride, the pair count and the tail are multiples of
    const int size = dtype_bytes(dtype);
    int V = 16 / size;
    uintptr_t ptrs = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(k_out);
    int64_t steps = a.pairs | a.tail;
    for (int i = 0; i < (k ? 12 : 6); ++i) steps |= st[i];
    while (V > 1 && ((ptrs & (uintptr_t)(V * size - 1)) || (steps & (V - 1)))) V >>= 1;
    if (V == 4 && size == 2) V = 2;
    // tokens of a workgroup: about eight items a thread, within the angle table; few tokens: one each, its heads spread over the CUs that would idle
    const int chunks = a.pairs / V + (a.tail + 2 * V - 1) / (2 * V);
    const int64_t items = (int64_t)chunks * (heads_q + heads_k);
    int64_t per = (8 * ROPE_THREADS + items - 1) / items;
    per = per < ROPE_LDS / a.pairs ? per : ROPE_LDS / a.pairs;
    const int64_t spread = (tokens + 1023) / 1024;
    per = per < spread ? per : spread;
    a.per_group = (int)(per > 1 ? per : 1);
    const int64_t groups = (tokens + a.per_group - 1) / a.per_group;
    if (groups >= 1 << 24) { set_error("rope: too many tokens for one launch"); return ADX_EINVAL; }
    const int64_t rounds = (items * a.per_group + ROPE_THREADS - 1) / ROPE_THREADS, idle = groups < 256 ? 256 / groups : 1;
    const dim3 grid((unsigned)groups, (unsigned)(rounds < idle ? rounds : idle));
    hipStream_t s = (hipStream_t)stream;
    if (size == 4) {
        if (V == 4) launch_rope<float, 4>(a, interleaved != 0, grid, s);
        else if (V == 2) launch_rope<float, 2>(a, interleaved != 0, grid, s);
        else launch_rope<float, 1>(a, interleaved != 0, grid, s);
    } else if (dtype == DT_BF16) {
        if (V == 8) launch_rope<__bf16, 8>(a, interleaved != 0, grid, s);
        else if (V == 2) launch_rope<__bf16, 2>(a, interleaved != 0, grid, s);
        else launch_rope<__bf16, 1>(a, interleaved != 0, grid, s);
    } else {
        if (V == 8) launch_rope<_Float16, 8>(a, interleaved != 0, grid, s);
        else if (V == 2) launch_rope<_Float16, 2>(a, interleaved != 0, grid, s);
        else launch_rope<_Float16, 1>(a, interleaved != 0, grid, s);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? ADX_OK : hip_fail(e, "rope");
}
