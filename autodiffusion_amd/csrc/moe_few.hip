// The whole sparse expert layer for a few tokens (one key point of a batch of scenarios: 1 .. 64), in two kernels:
//     y[t] = res[t] + sum_j w_j W2_{e_j} (silu(W1_{e_j} x[t]) * W3_{e_j} x[t]),   (e_j, w_j) = the top_k largest of softmax(R x[t]),
//     renormalised to sum one (ties: lowest expert index).
// With so few tokens the layer is one pass over the chosen experts' weights: 16 rows of a weight matrix meet all tokens of its expert
// in one matrix instruction, so the arithmetic is hidden and only the rate of the weight loads counts.  Nothing is staged: fragments
// go from global memory to registers, every wave of a workgroup takes its own pieces of the summed axis.
//   1. up    workgroup = (chosen expert, 16 hidden columns): routing, gate and up products, silu(g) u -> hidden rows;
//   2. down  workgroup = (16 output columns, a share of the (expert, K piece) units): weighted products added per token; with more than
//            one share the last workgroup of a column group to finish adds the shares in order -- the order of the sums never depends
//            on timing.
// The routing of all tokens is computed by every workgroup of `up` itself while that costs less than a launch (ROUTE_INSIDE below),
// otherwise by a kernel of its own in front.
//
// Precision.  Sums are fp32.  The hidden values stay at fp32 accuracy: they are kept as two (16-bit outputs, 2^-17) or three (fp32
// outputs, 2^-25) bf16 parts, each an operand of the second product.  fp32 tokens meet 16-bit weights in three parts, fp16 tokens in
// two (exact); fp16 weights are split exactly into two bf16 parts as they are loaded (11 bits = 8 + 3): hidden values beyond
// the fp16 range stay finite.
#include "adx_ops.h"
#include "engine.h"
#include "fastmath.h"
#include "typed.h"

#include <type_traits>

namespace adx {
namespace {

constexpr int FEW_MAX_T = 64, FEW_MAX_K = 8, FEW_MAX_E = 64;
constexpr int WAVES = 8;                                  // of a workgroup of either product
enum : int { P_F32 = 0, P_BF16 = 1, P_BF16X3 = 2, P_F16 = 4 };         // the ADX_PREC_* codes

struct FewArgs {
    const void* x; const void* res; const float* router;
    const void* w13; const void* w2;
    int T, d, inter, E, top_k;
    int* idx; float* wts;                                 // [T][top_k]
    int* table; int active;                               // `up` -> `down`: [active] rows of {expert or -1, count, entries (token * top_k + slot)[T]}
    void* h; int64_t h_plane;                             // hidden rows [part][T top_k][inter]; elements of one part
    float* part; int* arrived;                            // shares > 1: [shares][T][d], [d / 16]
    int shares, k_splits;
    void* y;
};

// Reductions over a wave by data-parallel moves: pairs and quads, the mirrored halves of 8 and 16 lanes, then the row and half swaps --
// vector instructions of a few cycles each, where a shuffle is a round trip through the LDS crossbar.
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false));
}
constexpr int QUAD_SWAP1 = 0xB1, QUAD_SWAP2 = 0x4E, HALF_MIRROR = 0x141, MIRROR = 0x140;
__device__ __forceinline__ float wave_sum(float v) {
    v += dpp<QUAD_SWAP1>(v);
    v += dpp<QUAD_SWAP2>(v);
    v += dpp<HALF_MIRROR>(v);
    v += dpp<MIRROR>(v);
    return xor32_add(xor16_add(v));
}
__device__ __forceinline__ float xor16_max(float x) {
    const unsigned u = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, dpp<QUAD_SWAP1>(v));
    v = fmaxf(v, dpp<QUAD_SWAP2>(v));
    v = fmaxf(v, dpp<HALF_MIRROR>(v));
    v = fmaxf(v, dpp<MIRROR>(v));
    return xor32_max(xor16_max(v));
}

// ------------------------------------------------------------------------------------------------------------- operand fragments
// Eight (fp32 weights: four) consecutive values of the summed axis a lane.  A weight fragment is PW bf16 parts, a token
// fragment PX parts; their product is the sum of the part products whose orders matter.
__device__ __forceinline__ unsigned high_halves(float a, float b) {        // truncated bf16 of two values, packed
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
__device__ __forceinline__ float high_value(float a) { return __uint_as_float(__float_as_uint(a) & 0xFFFF0000u); }

// parts by truncation: each takes 8 significant bits, the remainder is exact
template <int N> __device__ __forceinline__ void split8(const float (&v)[8], uint4 (&p)[N]) {
    float r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = v[e];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        p[i] = make_uint4(high_halves(r[0], r[1]), high_halves(r[2], r[3]), high_halves(r[4], r[5]), high_halves(r[6], r[7]));
        if (i + 1 < N) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float hi = high_value(r[e]);
                r[e] = __builtin_isfinite(r[e]) ? r[e] - hi : 0.f;       // an infinity or NaN lives in the first part alone
            }
        }
    }
}

typedef Pack<__bf16, 8> bf8;
typedef Pack<_Float16, 8> h8;

__device__ __forceinline__ f32x4_t mfma_bf(const uint4& w, const uint4& x, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, w), __builtin_bit_cast(bf16x8_t, x), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4_t mfma_h(const uint4& w, const uint4& x, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, w), __builtin_bit_cast(f16x8_t, x), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4_t mfma_f(const uint4& w, const uint4& x, f32x4_t c) {
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w.x), __uint_as_float(x.x), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w.y), __uint_as_float(x.y), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w.z), __uint_as_float(x.z), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w.w), __uint_as_float(x.w), c, 0, 0, 0);
}

// What one lane loads of a weight row (CE values), and its bf16 parts
template <int P> struct Weight {
    static constexpr int CE = P == P_F32 ? 4 : 8, SZ = P == P_F32 ? 4 : 2;
    static constexpr int RAW = P == P_BF16X3 ? 2 : 1, PARTS = P == P_BF16X3 || P == P_F16 ? 2 : 1;
    uint4 raw[RAW];
    // `at`: element index of the first value; `low`: elements between the high and the low plane
    __device__ __forceinline__ void load(const void* w, int64_t at, int64_t low) {
        const unsigned char* p = static_cast<const unsigned char*>(w) + at * SZ;
        raw[0] = *reinterpret_cast<const uint4*>(p);
        if constexpr (RAW == 2) raw[1] = *reinterpret_cast<const uint4*>(p + low * SZ);
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < RAW; ++i) raw[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    __device__ __forceinline__ void parts(uint4 (&p)[PARTS]) const {
        if constexpr (P == P_F16) {
            const h8 h = __builtin_bit_cast(h8, raw[0]);
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = (float)h.v[e];
            split8<2>(v, p);
        } else {
#pragma unroll
            for (int i = 0; i < PARTS; ++i) p[i] = raw[i];
        }
    }
};

// sum over part products of order < ORDER
template <int PW, int PX, int ORDER>
__device__ __forceinline__ f32x4_t mfma_parts(const uint4 (&w)[PW], const uint4 (&x)[PX], f32x4_t c) {
#pragma unroll
    for (int i = PX - 1; i >= 0; --i)
#pragma unroll
        for (int j = PW - 1; j >= 0; --j)
            if (i + j < ORDER) c = mfma_bf(w[j], x[i], c);               // the small terms first
    return c;
}

// ------------------------------------------------------------------------------------------------------------- routing
// The routing of tokens t0 .. t0 + n - 1 by a whole workgroup: every wave takes its part of the summed axis of one token and eight
// experts, so that the loads of a logit are one round trip; then the choice, one token a wave.  `part`: n ceil(E / 8) * 64 floats of LDS.
constexpr int ROUTE_GROUPS = 8;                           // tokens times groups of eight experts a call may hold in LDS
template <typename A>
__device__ __forceinline__ void route(const FewArgs& a, int t0, int n, float* part, int* idx, float* wts) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int groups = (a.E + 7) / 8;
    for (int p = 0; p < n * groups; ++p) {
        const int t = p / groups, e0 = (p - t * groups) * 8;
        const A* x = static_cast<const A*>(a.x) + (int64_t)(t0 + t) * a.d;
        float s[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) s[q] = 0.f;
        for (int i = threadIdx.x * 4; i < a.d; i += 256 * WAVES) {      // d is a multiple of 32
            const Pack<A, 4> xv = *reinterpret_cast<const Pack<A, 4>*>(x + i);
            float4 wv[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) wv[q] = *reinterpret_cast<const float4*>(a.router + (int64_t)min(e0 + q, a.E - 1) * a.d + i);
#pragma unroll
            for (int q = 0; q < 8; ++q) s[q] += (float)xv.v[0] * wv[q].x + (float)xv.v[1] * wv[q].y + (float)xv.v[2] * wv[q].z + (float)xv.v[3] * wv[q].w;
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            s[q] = wave_sum(s[q]);
            if (lane == 0) part[(p * WAVES + wave) * 8 + q] = s[q];
        }
    }
    __syncthreads();
    for (int t = wave; t < n; t += WAVES) {
        float mine = -INFINITY;
        if (lane < a.E) {
            const float* l = part + (t * groups + (lane >> 3)) * WAVES * 8 + (lane & 7);
            mine = 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) mine += l[w * 8];
        }
        const float mx = wave_max(mine);
        const float ex = lane < a.E ? expf(mine - mx) : 0.f;
        const float p = ex / wave_sum(ex);
        // NaN probabilities (a token that is not finite) count as the largest, so that the choice is always an expert
        float key = lane < a.E ? (p != p ? INFINITY : p) : -1.f, total = 0.f, chosen_p = 0.f;
        int chosen = 0;
        for (int j = 0; j < a.top_k; ++j) {
            const float best = wave_max(key);
            const int e = __ffsll((long long)__ballot(key == best)) - 1;       // lowest index among equals
            const float pe = __shfl(p, e, 64);
            if (lane == j) { chosen = e; chosen_p = pe; }
            total += pe;
            if (lane == e) key = -1.f;
        }
        if (lane < a.top_k) {
            idx[t * a.top_k + lane] = chosen;
            wts[t * a.top_k + lane] = chosen_p / total;
        }
    }
    __syncthreads();
}

template <typename A>
__global__ __launch_bounds__(64 * WAVES) void few_route_kernel(const FewArgs a) {
    __shared__ float part[ROUTE_GROUPS * WAVES * 8];
    const int t = blockIdx.x;
    route<A>(a, t, 1, part, a.idx + t * a.top_k, a.wts + t * a.top_k);
}

// The `rank`-th expert (by index) that any token chose, -1 if there are fewer; its entries (token * top_k + slot) in token order
struct Chosen {
    int entry[FEW_MAX_T];
    unsigned used[2];
    int count;
};
__device__ __forceinline__ int chosen_expert(const int* idx, int n, int rank, unsigned* used) {
    if (threadIdx.x < 2) used[threadIdx.x] = 0u;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += 64 * WAVES) atomicOr(&used[idx[i] >> 5], 1u << (idx[i] & 31));       // LDS; the result does not depend on the order
    __syncthreads();
    unsigned long long m = (unsigned long long)used[1] << 32 | used[0];
    for (int i = 0; i < rank && m; ++i) m &= m - 1;
    return m ? __ffsll((long long)m) - 1 : -1;
}
// the entries of expert e (a token chooses an expert once: at most T); executed by the whole workgroup
__device__ __forceinline__ void entries_of(const int* idx, int n, int e, Chosen& c) {
    __syncthreads();
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x;
        int base = 0;
        for (int i0 = 0; i0 < n; i0 += 64) {
            const bool hit = i0 + lane < n && idx[i0 + lane] == e;
            const unsigned long long m = __ballot(hit);
            if (hit) c.entry[base + __popcll(m & ((1ull << lane) - 1ull))] = i0 + lane;
            base += __popcll(m);
        }
        if (lane == 0) c.count = base;
    }
    __syncthreads();
}

// ------------------------------------------------------------------------------------------------------------- gate and up
// Tokens of an expert are taken 16 MT at a time; a second pass finds the weights in the L2.
template <typename A, int P, int MT, bool INSIDE>
__global__ __launch_bounds__(64 * WAVES, (P == P_F32 || sizeof(A) == 2) ? 4 : 2) void few_up_kernel(const FewArgs a) {
    typedef Weight<P> W;
    constexpr int CE = W::CE, PIECE = 8 * CE;                            // 128 bytes of a 16-bit or fp32 row
    constexpr bool RAW_X = P == P_F32 || sizeof(A) == 2;                 // token values go into the matrix instruction as they are
    constexpr int PX = RAW_X ? 1 : 3, PH = P == P_F32 ? 1 : sizeof(A) == 4 ? 3 : 2;
    __shared__ float sums[WAVES][2 * MT][64][4];
    __shared__ int idx_s[FEW_MAX_T * FEW_MAX_K];
    __shared__ float wts_s[INSIDE ? FEW_MAX_T * FEW_MAX_K : 1];
    __shared__ Chosen ch;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r16 = lane & 15, g = lane >> 4;
    const int n = a.T * a.top_k;
    if constexpr (INSIDE) {
        static_assert(ROUTE_GROUPS * WAVES * 8 <= WAVES * 2 * 64 * 4, "the routing's sums fit");
        route<A>(a, 0, a.T, &sums[0][0][0][0], idx_s, wts_s);
        if (blockIdx.x == 0 && blockIdx.y == 0)
            for (int i = tid; i < n; i += 64 * WAVES) { a.idx[i] = idx_s[i]; a.wts[i] = wts_s[i]; }
    } else {
        for (int i = tid; i < n; i += 64 * WAVES) idx_s[i] = a.idx[i];
    }
    if (blockIdx.x == 0 && blockIdx.y == 0 && a.shares > 1)
        for (int i = tid; i < a.d / 16; i += 64 * WAVES) a.arrived[i] = 0;
    __syncthreads();
    const int e = chosen_expert(idx_s, n, blockIdx.y, ch.used);
    int* row_of_table = a.table + (int64_t)blockIdx.y * (a.T + 2);
    if (e < 0) {
        if (blockIdx.x == 0 && tid == 0) row_of_table[0] = -1;
        return;
    }
    entries_of(idx_s, n, e, ch);
    const int count = ch.count, col0 = blockIdx.x * 16;
    if (blockIdx.x == 0) {
        if (tid < count) row_of_table[2 + tid] = ch.entry[tid];
        if (tid == 0) { row_of_table[0] = e; row_of_table[1] = count; }
    }
    const int64_t low = (int64_t)a.E * 2 * a.inter * a.d;
    const int64_t gate = ((int64_t)e * 2 * a.inter + col0 + r16) * a.d + g * CE, up = gate + (int64_t)a.inter * a.d;
    for (int m0 = 0; m0 < count; m0 += 16 * MT) {
        const A* x[MT];
        bool live[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            live[t] = m0 + t * 16 + r16 < count;
            x[t] = static_cast<const A*>(a.x) + (int64_t)(live[t] ? ch.entry[m0 + t * 16 + r16] / a.top_k : 0) * a.d + g * CE;
        }
        f32x4_t acc[2][MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[0][t] = acc[1][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        constexpr int U = 2;                                              // pieces in flight a wave
        const int K = a.d - g * CE;
        for (int k = wave * PIECE; k < a.d; k += U * WAVES * PIECE) {
            W w[2 * U][2];
            uint4 xv[2 * U][MT][RAW_X ? 1 : 2];
#pragma unroll
            for (int q = 0; q < 2 * U; ++q) {
                const int kq = k + (q >> 1) * WAVES * PIECE + (q & 1) * 4 * CE;
                const bool ok = kq < K;
                if (ok) { w[q][0].load(a.w13, gate + kq, low); w[q][1].load(a.w13, up + kq, low); }
                else { w[q][0].clear(); w[q][1].clear(); }
#pragma unroll
                for (int t = 0; t < MT; ++t) {
#pragma unroll
                    for (int z = 0; z < (RAW_X ? 1 : 2); ++z)
                        xv[q][t][z] = ok && live[t] ? *reinterpret_cast<const uint4*>(reinterpret_cast<const unsigned char*>(x[t] + kq) + 16 * z) : make_uint4(0u, 0u, 0u, 0u);
                }
            }
#pragma unroll
            for (int q = 0; q < 2 * U; ++q) {
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    if constexpr (P == P_F32) {
                        acc[0][t] = mfma_f(w[q][0].raw[0], xv[q][t][0], acc[0][t]);
                        acc[1][t] = mfma_f(w[q][1].raw[0], xv[q][t][0], acc[1][t]);
                    } else if constexpr (RAW_X && P == P_BF16) {
                        acc[0][t] = mfma_bf(w[q][0].raw[0], xv[q][t][0], acc[0][t]);
                        acc[1][t] = mfma_bf(w[q][1].raw[0], xv[q][t][0], acc[1][t]);
                    } else if constexpr (RAW_X) {
                        acc[0][t] = mfma_h(w[q][0].raw[0], xv[q][t][0], acc[0][t]);
                        acc[1][t] = mfma_h(w[q][1].raw[0], xv[q][t][0], acc[1][t]);
                    } else {
                        const float v[8] = {__uint_as_float(xv[q][t][0].x), __uint_as_float(xv[q][t][0].y), __uint_as_float(xv[q][t][0].z), __uint_as_float(xv[q][t][0].w),
                                            __uint_as_float(xv[q][t][1].x), __uint_as_float(xv[q][t][1].y), __uint_as_float(xv[q][t][1].z), __uint_as_float(xv[q][t][1].w)};
                        uint4 px[PX], pw[W::PARTS];
                        split8<PX>(v, px);
#pragma unroll
                        for (int z = 0; z < 2; ++z) {
                            w[q][z].parts(pw);
                            acc[z][t] = mfma_parts<W::PARTS, PX, 3>(pw, px, acc[z][t]);
                        }
                    }
                }
            }
        }
        __syncthreads();                                                  // what `sums` held before has been read
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            *reinterpret_cast<f32x4_t*>(sums[wave][2 * t][lane]) = acc[0][t];
            *reinterpret_cast<f32x4_t*>(sums[wave][2 * t + 1][lane]) = acc[1][t];
        }
        __syncthreads();
        // result layout of the 16x16 product: column (token) = lane & 15, row (hidden column) = 4 (lane >> 4) + reg
        const int rows = min(count - m0, 16 * MT);
        for (int i = tid; i < rows * 16; i += 64 * WAVES) {
            const int m = i >> 4, c = i & 15, t = m >> 4, l = (c >> 2) * 16 + (m & 15);
            float vg = 0.f, vu = 0.f;
#pragma unroll
            for (int s = 0; s < WAVES; ++s) { vg += sums[s][2 * t][l][c & 3]; vu += sums[s][2 * t + 1][l][c & 3]; }
            float v = vg / (1.f + expf(-vg)) * vu;
            const int64_t at = (int64_t)ch.entry[m0 + m] * a.inter + col0 + c;
            if constexpr (P == P_F32) static_cast<float*>(a.h)[at] = v;
            else {
#pragma unroll
                for (int p = 0; p < PH; ++p) {
                    const __bf16 b = (__bf16)v;
                    static_cast<__bf16*>(a.h)[p * a.h_plane + at] = b;
                    v = __builtin_isfinite((float)b) ? v - (float)b : 0.f;
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------------------- down
template <typename A, int P, int MT>
__global__ __launch_bounds__(64 * WAVES, (P == P_F32 || sizeof(A) == 2) ? 4 : 2) void few_down_kernel(const FewArgs a) {
    typedef Weight<P> W;
    constexpr int CE = W::CE, PIECE = 8 * CE, PH = P == P_F32 ? 1 : sizeof(A) == 4 ? 3 : 2;
    constexpr int ROWS = MT == 1 ? 16 : FEW_MAX_T;                        // tokens the launch may have
    __shared__ float ysum[WAVES][ROWS][16 + 1];
    __shared__ int last;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r16 = lane & 15, g = lane >> 4;
    const int col0 = blockIdx.x * 16;
    for (int i = lane; i < ROWS * 17; i += 64) (&ysum[wave][0][0])[i] = 0.f;
    __syncthreads();
    const int64_t low = (int64_t)a.E * a.inter * a.d;
    // unit u = (chosen expert u / k_splits, part u % k_splits of the hidden axis); this workgroup takes every shares-th
    const int piece_len = (a.inter + a.k_splits * PIECE - 1) / (a.k_splits * PIECE) * PIECE;
    for (int u = blockIdx.y; u < a.active * a.k_splits; u += a.shares) {
        const int* row_of_table = a.table + (int64_t)(u / a.k_splits) * (a.T + 2);
        const int e = row_of_table[0];
        if (e < 0) break;
        const int count = row_of_table[1], k_lo = (u % a.k_splits) * piece_len, k_hi = min(k_lo + piece_len, a.inter);
        const int64_t row = ((int64_t)e * a.d + col0 + r16) * a.inter + g * CE;
        for (int m0 = 0; m0 < count; m0 += 16 * MT) {
            int64_t h[MT];
            int entry[MT];
            float wt[MT];
            bool live[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                live[t] = m0 + t * 16 + r16 < count;
                entry[t] = live[t] ? row_of_table[2 + m0 + t * 16 + r16] : 0;
                wt[t] = a.wts[entry[t]];
                h[t] = (int64_t)entry[t] * a.inter + g * CE;
            }
            f32x4_t acc[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
            constexpr int U = W::RAW + MT * PH > 4 ? 1 : W::RAW + MT * PH > 2 ? 2 : 4;    // pieces in flight a wave, by registers
            const int K = k_hi - g * CE;
            for (int k = k_lo + wave * PIECE; k < k_hi; k += U * WAVES * PIECE) {
                W w[2 * U];
                uint4 hv[2 * U][MT][PH];
#pragma unroll
                for (int q = 0; q < 2 * U; ++q) {
                    const int kq = k + (q >> 1) * WAVES * PIECE + (q & 1) * 4 * CE;
                    const bool ok = kq < K;
                    if (ok) w[q].load(a.w2, row + kq, low);
                    else w[q].clear();
#pragma unroll
                    for (int t = 0; t < MT; ++t)
#pragma unroll
                        for (int p = 0; p < PH; ++p)
                            hv[q][t][p] = ok && live[t] ? *reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(a.h) + (p * a.h_plane + h[t] + kq) * W::SZ)
                                                        : make_uint4(0u, 0u, 0u, 0u);
                }
#pragma unroll
                for (int q = 0; q < 2 * U; ++q) {
                    uint4 pw[W::PARTS];
                    if constexpr (P != P_F32) w[q].parts(pw);
#pragma unroll
                    for (int t = 0; t < MT; ++t) {
                        if constexpr (P == P_F32) acc[t] = mfma_f(w[q].raw[0], hv[q][t][0], acc[t]);
                        else acc[t] = mfma_parts<W::PARTS, PH, PH>(pw, hv[q][t], acc[t]);
                    }
                }
            }
            // a token chooses an expert once: the lanes of a wave add to different rows
#pragma unroll
            for (int t = 0; t < MT; ++t)
                if (live[t]) {
                    const int tok = entry[t] / a.top_k;
#pragma unroll
                    for (int q = 0; q < 4; ++q) ysum[wave][tok][4 * g + q] += wt[t] * acc[t][q];
                }
        }
    }
    __syncthreads();
    const A* res = static_cast<const A*>(a.res);
    A* y = static_cast<A*>(a.y);
    if (a.shares == 1) {
        for (int i = tid; i < a.T * 16; i += 64 * WAVES) {
            const int t = i >> 4, c = i & 15;
            float v = 0.f;
#pragma unroll
            for (int s = 0; s < WAVES; ++s) v += ysum[s][t][c];
            const int64_t at = (int64_t)t * a.d + col0 + c;
            if (res) v += (float)res[at];
            y[at] = (A)v;
        }
        return;
    }
    for (int i = tid; i < a.T * 16; i += 64 * WAVES) {
        const int t = i >> 4, c = i & 15;
        float v = 0.f;
#pragma unroll
        for (int s = 0; s < WAVES; ++s) v += ysum[s][t][c];
        __hip_atomic_store(&a.part[((int64_t)blockIdx.y * a.T + t) * a.d + col0 + c], v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    // The last workgroup of this column group adds the shares.  Nobody waits: the others have left.  The shares are written and read
    // by device-scope accesses, which go past the L2 of an XCD; every wave waits for its own to arrive before the workgroup is counted.
    // (A device-scope fence does the same by writing back the whole L2: 40 us for one token of width 512.)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) last = __hip_atomic_fetch_add(&a.arrived[blockIdx.x], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.shares - 1;
    __syncthreads();
    if (!last) return;
    for (int i = tid; i < a.T * 16; i += 64 * WAVES) {
        const int t = i >> 4, c = i & 15;
        const int64_t at = (int64_t)t * a.d + col0 + c;
        float v = res ? (float)res[at] : 0.f;
        float s = 0.f;
        for (int p0 = 0; p0 < a.shares; p0 += 8) {                        // eight loads in flight, added in order
            float f[8];
#pragma unroll
            for (int p = 0; p < 8; ++p) f[p] = __hip_atomic_load(&a.part[(int64_t)min(p0 + p, a.shares - 1) * a.T * a.d + at], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
            for (int p = 0; p < 8; ++p) s += p0 + p < a.shares ? f[p] : 0.f;
        }
        y[at] = (A)(s + v);
    }
}

// ------------------------------------------------------------------------------------------------------------- host
inline size_t up256(size_t v) { return (v + 255) / 256 * 256; }

struct FewPlan { int shares, k_splits, active; size_t idx, wts, table, h, part, arrived, bytes; int64_t h_plane; };

FewPlan few_plan(int T, int d, int inter, int E, int top_k, int act_type, int precision) {
    FewPlan p;
    const int n = T * top_k, piece = precision == P_F32 ? 32 : 64;
    p.active = n < E ? n : E;                                             // experts that can have been chosen
    // enough workgroups to keep the whole card loading, each with at least a piece of the hidden axis for every wave
    const int groups = d / 16;
    int want = (512 + groups - 1) / groups;
    const int most_k = inter / (piece * WAVES) > 1 ? inter / (piece * WAVES) : 1;
    p.k_splits = 1;
    if (want > p.active) p.k_splits = (want + p.active - 1) / p.active;
    if (p.k_splits > most_k) p.k_splits = most_k;
    // as many units each: an uneven share is a second round for all
    const int units = p.active * p.k_splits, per = units > want ? units / want : 1;
    p.shares = (units + per - 1) / per;
    p.h_plane = (int64_t)n * inter;
    size_t off = 0;
    auto take = [&](size_t b) { const size_t at = off; off += up256(b); return at; };
    p.idx = take((size_t)n * 4);
    p.wts = take((size_t)n * 4);
    p.table = take((size_t)p.active * (T + 2) * 4);
    p.h = take((size_t)p.h_plane * (precision == P_F32 ? 4 : act_type == DT_F32 ? 6 : 4));
    p.part = take(p.shares > 1 ? (size_t)p.shares * T * d * 4 : 0);
    p.arrived = take((size_t)groups * 4);
    p.bytes = off;
    return p;
}

bool few_shape_ok(int T, int d, int inter, int E, int top_k) {
    return T >= 1 && T <= FEW_MAX_T && d >= 32 && d % 32 == 0 && d <= (1 << 16) && inter >= 32 && inter % 32 == 0 && inter <= (1 << 18) && E >= 1 && E <= FEW_MAX_E && top_k >= 1 &&
           top_k <= FEW_MAX_K && top_k <= E;
}

bool few_types_ok(int act_type, int precision) {
    if (act_type == DT_F32) return precision == P_F32 || precision == P_BF16 || precision == P_BF16X3 || precision == P_F16;
    return (act_type == DT_BF16 && precision == P_BF16) || (act_type == DT_F16 && precision == P_F16);
}

// tokens times groups of eight experts up to which `up` routes by itself
constexpr int ROUTE_INSIDE = 2;
static_assert(ROUTE_INSIDE <= ROUTE_GROUPS, "fits LDS");

template <typename A, int P, int MT>
void launch_few_layer(const FewArgs& a, const FewPlan& p, hipStream_t s) {
    const dim3 up((unsigned)(a.inter / 16), (unsigned)p.active), down((unsigned)(a.d / 16), (unsigned)p.shares), block(64 * WAVES);
    if (a.T * ((a.E + 7) / 8) <= ROUTE_INSIDE) {
        hipLaunchKernelGGL((few_up_kernel<A, P, MT, true>), up, block, 0, s, a);
    } else {
        hipLaunchKernelGGL(few_route_kernel<A>, dim3((unsigned)a.T), block, 0, s, a);
        hipLaunchKernelGGL((few_up_kernel<A, P, MT, false>), up, block, 0, s, a);
    }
    hipLaunchKernelGGL((few_down_kernel<A, P, MT>), down, block, 0, s, a);
}

template <typename A, int P>
void launch_by_tokens(const FewArgs& a, const FewPlan& p, hipStream_t s) {
    if (a.T <= 16) launch_few_layer<A, P, 1>(a, p, s);
    else launch_few_layer<A, P, 2>(a, p, s);
}

}  // namespace
}  // namespace adx

using namespace adx;

#define ADX_API extern "C" __attribute__((visibility("default")))

ADX_API size_t adx_moe_few_workspace_bytes(int T, int d, int inter, int E, int top_k, int act_type, int precision) {
    if (!few_shape_ok(T, d, inter, E, top_k) || !few_types_ok(act_type, precision)) return 0;
    return few_plan(T, d, inter, E, top_k, act_type, precision).bytes;
}

ADX_API int adx_op_moe_few(const void* x, const void* res, const float* router_w, const void* w13, const void* w2, int T, int d, int inter, int E,
                           int top_k, int act_type, int precision, void* workspace, size_t workspace_bytes, void* y, void* stream) {
    if (!x || !router_w || !w13 || !w2 || !workspace || !y) { set_error("moe_few: null pointer"); return ADX_EINVAL; }
    if (!few_shape_ok(T, d, inter, E, top_k)) {
        set_error("moe_few: needs 1 <= T <= 64 tokens, 1 <= top_k <= min(E, 8), E <= 64, and hidden (<= 65536) / expert (<= 262144) widths that are multiples of 32"); return ADX_EINVAL;
    }
    if (!few_types_ok(act_type, precision)) {
        set_error("moe_few: fp32 tokens with fp32, bf16, bf16x3 or f16 weights, bf16 tokens with bf16 weights, fp16 tokens with f16 weights"); return ADX_EINVAL;
    }
    if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(res) | reinterpret_cast<uintptr_t>(router_w) |
         reinterpret_cast<uintptr_t>(w13) | reinterpret_cast<uintptr_t>(w2) | reinterpret_cast<uintptr_t>(workspace)) & 15) {
        set_error("moe_few: pointers must be 16-byte aligned"); return ADX_EINVAL;
    }
    const FewPlan p = few_plan(T, d, inter, E, top_k, act_type, precision);
    if (workspace_bytes < p.bytes) { set_error("moe_few: workspace smaller than adx_moe_few_workspace_bytes"); return ADX_EINVAL; }
    unsigned char* base = static_cast<unsigned char*>(workspace);
    FewArgs a;
    a.x = x; a.res = res; a.router = router_w; a.w13 = w13; a.w2 = w2; a.T = T; a.d = d; a.inter = inter; a.E = E; a.top_k = top_k;
    a.idx = reinterpret_cast<int*>(base + p.idx); a.wts = reinterpret_cast<float*>(base + p.wts);
    a.table = reinterpret_cast<int*>(base + p.table); a.active = p.active;
    a.h = base + p.h; a.h_plane = p.h_plane; a.part = reinterpret_cast<float*>(base + p.part); a.arrived = reinterpret_cast<int*>(base + p.arrived);
    a.shares = p.shares; a.k_splits = p.k_splits; a.y = y;
    hipStream_t s = (hipStream_t)stream;
    if (act_type == DT_BF16) launch_by_tokens<__bf16, P_BF16>(a, p, s);
    else if (act_type == DT_F16) launch_by_tokens<_Float16, P_F16>(a, p, s);
    else if (precision == P_F32) launch_by_tokens<float, P_F32>(a, p, s);
    else if (precision == P_BF16) launch_by_tokens<float, P_BF16>(a, p, s);
    else if (precision == P_BF16X3) launch_by_tokens<float, P_BF16X3>(a, p, s);
    else launch_by_tokens<float, P_F16>(a, p, s);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? ADX_OK : hip_fail(e, "moe_few");
}
