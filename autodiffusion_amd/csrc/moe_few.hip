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

// Sizes of the launches, each the best of a sweep on 1 .. 64 tokens of widths 256 .. 1536: `up` at most so many workgroups; `down` at
// least so many, and enough that none reads more than so many KB of weights
constexpr int UP_BLOCKS = 768, DOWN_BLOCKS = 256, DOWN_KB = 192;

struct FewArgs {
    const void* x; const void* res; const float* router;
    const void* w13; const void* w2;
    int T, d, inter, E, top_k;
    int* idx; float* wts;                                 // [T][top_k]
    int* table;                                           // `up` -> `down`: how many experts were chosen, and a row {expert, count, entries (token * top_k + slot)[T]} each
    void* h; int64_t h_plane;                             // hidden rows [part][T top_k][inter]; elements of one part
    float* part;                                          // [k_splits][T top_k][d]
    int* arrived; int arrivals;                           // workgroups of `down` that are done, a column group
    int wk, k_splits;
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

__device__ __forceinline__ unsigned wave_or(unsigned v) {
    v |= __float_as_uint(dpp<QUAD_SWAP1>(__uint_as_float(v)));
    v |= __float_as_uint(dpp<QUAD_SWAP2>(__uint_as_float(v)));
    v |= __float_as_uint(dpp<HALF_MIRROR>(__uint_as_float(v)));
    v |= __float_as_uint(dpp<MIRROR>(__uint_as_float(v)));
    auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = r[0] | r[1];
    r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return r[0] | r[1];
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
    // `base`: the same for the whole wave; `at`: byte offset of the lane's first value; `low`: bytes between the high and the low plane
    __device__ __forceinline__ void load(const unsigned char* base, unsigned at, int64_t low) {
        raw[0] = *reinterpret_cast<const uint4*>(base + at);
        if constexpr (RAW == 2) raw[1] = *reinterpret_cast<const uint4*>(base + low + at);
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
// Sums of eight values a lane over the wave: lanes 0 .. 3 return value 4 (lane & 1) + 2 (lane >> 1) + i in r[i].  The first two steps
// halve the values instead of keeping eight sums a lane.
constexpr int ROTATE4 = 0x124, ROTATE8 = 0x128;            // rotations within 16 lanes
__device__ __forceinline__ void wave_sum8(const float (&s)[8], int lane, float (&r)[2]) {
    float p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = ((lane & 1) ? s[i + 4] : s[i]) + dpp<QUAD_SWAP1>((lane & 1) ? s[i] : s[i + 4]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float v = ((lane & 2) ? p[i + 2] : p[i]) + dpp<QUAD_SWAP2>((lane & 2) ? p[i] : p[i + 2]);
        v += dpp<ROTATE4>(v);
        v += dpp<ROTATE8>(v);
        r[i] = xor32_add(xor16_add(v));
    }
}

// The routing of tokens t0 .. t0 + n - 1 by a whole workgroup.  The waves spread over groups of eight experts and parts of the summed
// axis; a wave reads its piece of the router once for all tokens.  Then the choice, one token a wave.  `part`: n ROUTE_WAVE floats of LDS.
constexpr int ROUTE_TOKENS = 4, ROUTE_WAVE = WAVES * 8;           // tokens of one round
template <typename A, int N>
__device__ __forceinline__ void route(const FewArgs& a, int t0, int n, float* part, int* idx, float* wts) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int groups = (a.E + 7) / 8, parts = WAVES / groups, e0 = wave / parts * 8;        // WAVES >= 8 >= groups; waves beyond groups * parts rest
    if (wave < groups * parts) {
        float s[N][8];
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
            for (int q = 0; q < 8; ++q) s[t][q] = 0.f;
        for (int i = (wave % parts * 64 + lane) * 4; i < a.d; i += 256 * parts) {          // d is a multiple of 32
            float4 wv[8];
            Pack<A, 4> xv[N];
#pragma unroll
            for (int q = 0; q < 8; ++q) wv[q] = *reinterpret_cast<const float4*>(a.router + (int64_t)min(e0 + q, a.E - 1) * a.d + i);
#pragma unroll
            for (int t = 0; t < N; ++t) xv[t] = *reinterpret_cast<const Pack<A, 4>*>(static_cast<const A*>(a.x) + (int64_t)(t0 + min(t, n - 1)) * a.d + i);
#pragma unroll
            for (int t = 0; t < N; ++t)
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    s[t][q] += (float)xv[t].v[0] * wv[q].x + (float)xv[t].v[1] * wv[q].y + (float)xv[t].v[2] * wv[q].z + (float)xv[t].v[3] * wv[q].w;
        }
#pragma unroll
        for (int t = 0; t < N; ++t) {
            float r[2];
            wave_sum8(s[t], lane, r);
            if (lane < 4 && t < n) *reinterpret_cast<float2*>(part + t * ROUTE_WAVE + wave * 8 + 4 * (lane & 1) + 2 * (lane >> 1)) = make_float2(r[0], r[1]);
        }
    }
    __syncthreads();
    for (int t = wave; t < n; t += WAVES) {
        float mine = -INFINITY;
        if (lane < a.E) {
            const float* l = part + t * ROUTE_WAVE + (lane >> 3) * parts * 8 + (lane & 7);
            mine = 0.f;
            for (int w = 0; w < parts; ++w) mine += l[w * 8];
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
    __shared__ __attribute__((aligned(16))) float part[ROUTE_WAVE];
    const int t = blockIdx.x;
    route<A, 1>(a, t, 1, part, a.idx + t * a.top_k, a.wts + t * a.top_k);
}

// The `rank`-th expert (by index) that any token chose, -1 if there are fewer; `chosen`: how many there are.  Every wave finds it by itself.
__device__ __forceinline__ int chosen_expert(const int* idx, int n, int rank, int lane, int* chosen) {
    unsigned lo = 0, hi = 0;
    for (int i = lane; i < n; i += 64) {
        const int e = idx[i];
        if (e < 32) lo |= 1u << e; else hi |= 1u << (e - 32);
    }
    unsigned long long used = (unsigned long long)wave_or(hi) << 32 | wave_or(lo);
    *chosen = __popcll(used);
    for (int i = 0; i < rank && used; ++i) used &= used - 1;
    return used ? __ffsll((long long)used) - 1 : -1;
}
// The entries (token * top_k + slot) of expert e in token order -- a token chooses an expert once: at most T -- and their number.  Every wave
// writes the whole list (the same values) and so may read it without a barrier.
__device__ __forceinline__ int entries_of(const int* idx, int n, int e, int lane, int* list) {
    int count = 0;
    for (int i0 = 0; i0 < n; i0 += 64) {
        const bool hit = i0 + lane < n && idx[i0 + lane] == e;
        const unsigned long long m = __ballot(hit);
        if (hit) list[count + __popcll(m & ((1ull << lane) - 1ull))] = i0 + lane;
        count += __popcll(m);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    return count;
}

// ------------------------------------------------------------------------------------------------------------- gate and up
// A wave multiplies 16 NT gate rows and 16 NT up rows with 16 MT tokens over its part of the summed axis; `wk` waves share a group
// of rows, WAVES / wk groups a workgroup.  Tokens of an expert are taken 16 MT at a time; a second pass finds the weights in the L2.
// With many tokens NT = 2: every row group reads all tokens again from the L2, which costs as much as the weights at NT = 1
// (64 tokens, width 1536, 8 experts of 6144: 85 us).
template <typename A, int P, int MT, int NT, bool INSIDE>
__global__ __launch_bounds__(64 * WAVES, P == P_F32 || sizeof(A) == 2 ? 4 : 2) void few_up_kernel(const FewArgs a) {
    typedef Weight<P> W;
    constexpr int CE = W::CE, PIECE = 8 * CE;                            // 128 bytes of a 16-bit or fp32 row
    constexpr bool RAW_X = P == P_F32 || sizeof(A) == 2;                 // token values go into the matrix instruction as they are
    constexpr int PX = RAW_X ? 1 : 3, PH = P == P_F32 ? 1 : sizeof(A) == 4 ? 3 : 2;
    __shared__ __attribute__((aligned(16))) float sums[WAVES][2 * MT * NT][64][4];
    __shared__ int idx_s[FEW_MAX_T * FEW_MAX_K];
    __shared__ float wts_s[INSIDE ? FEW_MAX_T * FEW_MAX_K : 1];
    __shared__ int list[FEW_MAX_T];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r16 = lane & 15, g = lane >> 4;
    const int n = a.T * a.top_k;
    if constexpr (INSIDE) {
        static_assert(ROUTE_TOKENS * ROUTE_WAVE <= WAVES * 2 * 64 * 4, "the routing's sums fit");
        if (a.T == 1) route<A, 1>(a, 0, 1, &sums[0][0][0][0], idx_s, wts_s);
        else
            for (int t0 = 0; t0 < a.T; t0 += ROUTE_TOKENS)
                route<A, ROUTE_TOKENS>(a, t0, min(ROUTE_TOKENS, a.T - t0), &sums[0][0][0][0], idx_s + t0 * a.top_k, wts_s + t0 * a.top_k);
        if (blockIdx.x == 0 && blockIdx.y == 0)
            for (int i = tid; i < n; i += 64 * WAVES) { a.idx[i] = idx_s[i]; a.wts[i] = wts_s[i]; }
    } else {
        for (int i = tid; i < n; i += 64 * WAVES) idx_s[i] = a.idx[i];
    }
    __syncthreads();
    int chosen;
    const int e = chosen_expert(idx_s, n, blockIdx.y, lane, &chosen);
    int* row_of_table = a.table + 1 + (int64_t)blockIdx.y * (a.T + 2);
    if (blockIdx.x == 0 && blockIdx.y == 0) {
        if (tid == 0) a.table[0] = chosen;
        for (int i = tid; i < a.arrivals; i += 64 * WAVES) a.arrived[i] = 0;
    }
    if (e < 0) return;
    const int count = entries_of(idx_s, n, e, lane, list);
    if (blockIdx.x == 0 && wave == 0) {
        if (lane < count) row_of_table[2 + lane] = list[lane];
        if (tid == 0) { row_of_table[0] = e; row_of_table[1] = count; }
    }
    const int col0 = ((int)blockIdx.x * (WAVES / a.wk) + wave / a.wk) * 16 * NT, kw = wave % a.wk;
    // a wave-uniform base and 32-bit byte offsets a lane (the host limits an expert's matrix to 2^31 bytes)
    const int64_t low = (int64_t)a.E * 2 * a.inter * a.d * W::SZ;
    const unsigned char* gate = static_cast<const unsigned char*>(a.w13) + (int64_t)e * 2 * a.inter * a.d * W::SZ;
    const unsigned char* up = gate + (int64_t)a.inter * a.d * W::SZ;
    unsigned row[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) row[j] = ((unsigned)min(col0 + 16 * j + r16, a.inter - 1) * (unsigned)a.d + g * CE) * W::SZ;
    for (int m0 = 0; m0 < count; m0 += 16 * MT) {
        unsigned x[MT];
        bool live[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            live[t] = m0 + t * 16 + r16 < count;
            x[t] = ((unsigned)(live[t] ? list[m0 + t * 16 + r16] / a.top_k : 0) * (unsigned)a.d + g * CE) * sizeof(A);
        }
        f32x4_t acc[NT][2][MT];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[j][0][t] = acc[j][1][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        constexpr int U = MT * NT > 1 ? 1 : 2;                            // pieces in flight a wave
        const int K = a.d - g * CE;
        const int stride = U * a.wk * PIECE;
        W w[2 * U][NT][2];
        uint4 xv[2 * U][MT][RAW_X ? 1 : 2];
        auto load = [&](int q, int k) {                                   // half piece q of the round that starts at k; zero past the end
            const int kq = k + (q >> 1) * a.wk * PIECE + (q & 1) * 4 * CE;
            const bool ok = kq < K;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                if (ok) { w[q][j][0].load(gate, row[j] + kq * W::SZ, low); w[q][j][1].load(up, row[j] + kq * W::SZ, low); }
                else { w[q][j][0].clear(); w[q][j][1].clear(); }
            }
#pragma unroll
            for (int t = 0; t < MT; ++t) {
#pragma unroll
                for (int z = 0; z < (RAW_X ? 1 : 2); ++z)
                    xv[q][t][z] = ok && live[t] ? *reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(a.x) + (unsigned)(x[t] + kq * sizeof(A) + 16 * z)) : make_uint4(0u, 0u, 0u, 0u);
            }
        };
        for (int k = kw * PIECE; k < a.d; k += stride) {
#pragma unroll
            for (int q = 0; q < 2 * U; ++q) load(q, k);
#pragma unroll
            for (int q = 0; q < 2 * U; ++q) {
                uint4 px[MT][PX];
                if constexpr (!RAW_X) {
#pragma unroll
                    for (int t = 0; t < MT; ++t) {
                        const float v[8] = {__uint_as_float(xv[q][t][0].x), __uint_as_float(xv[q][t][0].y), __uint_as_float(xv[q][t][0].z), __uint_as_float(xv[q][t][0].w),
                                            __uint_as_float(xv[q][t][1].x), __uint_as_float(xv[q][t][1].y), __uint_as_float(xv[q][t][1].z), __uint_as_float(xv[q][t][1].w)};
                        split8<PX>(v, px[t]);
                    }
                }
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        uint4 pw[W::PARTS];
                        if constexpr (!RAW_X) w[q][j][z].parts(pw);
#pragma unroll
                        for (int t = 0; t < MT; ++t) {
                            if constexpr (P == P_F32) acc[j][z][t] = mfma_f(w[q][j][z].raw[0], xv[q][t][0], acc[j][z][t]);
                            else if constexpr (RAW_X && P == P_BF16) acc[j][z][t] = mfma_bf(w[q][j][z].raw[0], xv[q][t][0], acc[j][z][t]);
                            else if constexpr (RAW_X) acc[j][z][t] = mfma_h(w[q][j][z].raw[0], xv[q][t][0], acc[j][z][t]);
                            else acc[j][z][t] = mfma_parts<W::PARTS, PX, 3>(pw, px[t], acc[j][z][t]);
                        }
                    }
            }
        }
        __syncthreads();                                                  // what `sums` held before has been read
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                *reinterpret_cast<f32x4_t*>(sums[wave][(j * MT + t) * 2][lane]) = acc[j][0][t];
                *reinterpret_cast<f32x4_t*>(sums[wave][(j * MT + t) * 2 + 1][lane]) = acc[j][1][t];
            }
        __syncthreads();
        // result layout of the 16x16 product: column (token) = lane & 15, row (hidden column) = 4 (lane >> 4) + reg
        const int rows = min(count - m0, 16 * MT), cols = 16 * NT * (WAVES / a.wk), left = (int)blockIdx.x * cols;
        for (int i = tid; i < rows * cols; i += 64 * WAVES) {
            const int m = i / cols, c = i - m * cols, w0 = c / (16 * NT) * a.wk, cc = c % (16 * NT);
            if (left + c >= a.inter) continue;
            const int t = ((cc >> 4) * MT + (m >> 4)) * 2, l = ((cc & 15) >> 2) * 16 + (m & 15);
            float vg = 0.f, vu = 0.f;
            for (int s = 0; s < a.wk; ++s) { vg += sums[w0 + s][t][l][c & 3]; vu += sums[w0 + s][t + 1][l][c & 3]; }
            float v = vg / (1.f + expf(-vg)) * vu;
            const int64_t at = (int64_t)list[m0 + m] * a.inter + left + c;
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
// A workgroup multiplies 16 NT rows of one expert's matrix with that expert's hidden rows over one of k_splits parts of the hidden
// axis (its waves share the part) and leaves the sums of every (token, slot) entry; the last workgroup of a group of output columns
// adds a token's entries, weighted, slot by slot and part by part.
template <typename A, int P, int MT, int NT>
__global__ __launch_bounds__(64 * WAVES, P == P_F32 || (P == P_BF16 && sizeof(A) == 2) ? 4 : 2) void few_down_kernel(const FewArgs a) {
    typedef Weight<P> W;
    constexpr int CE = W::CE, PIECE = 8 * CE, PH = P == P_F32 ? 1 : sizeof(A) == 4 ? 3 : 2, COLS = 16 * NT;
    __shared__ __attribute__((aligned(16))) float sums[WAVES][MT * NT][64][4];
    __shared__ int last;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r16 = lane & 15, g = lane >> 4;
    const int col0 = blockIdx.x * COLS, chosen = a.table[0], n = a.T * a.top_k;
    const int rank = blockIdx.y / a.k_splits, part = blockIdx.y % a.k_splits;
    if (rank >= chosen) return;
    const int* row_of_table = a.table + 1 + (int64_t)rank * (a.T + 2);
    const int e = row_of_table[0], count = row_of_table[1];
    const int64_t low = (int64_t)a.E * a.inter * a.d * W::SZ;
    const unsigned char* w2 = static_cast<const unsigned char*>(a.w2) + (int64_t)e * a.inter * a.d * W::SZ;
    const unsigned char* hidden[PH];
#pragma unroll
    for (int p = 0; p < PH; ++p) hidden[p] = static_cast<const unsigned char*>(a.h) + p * a.h_plane * W::SZ;
    const int len = (a.inter + a.k_splits * PIECE - 1) / (a.k_splits * PIECE) * PIECE, k_lo = part * len, k_hi = min(k_lo + len, a.inter);
    unsigned row[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) row[j] = ((unsigned)min(col0 + 16 * j + r16, a.d - 1) * (unsigned)a.inter + g * CE) * W::SZ;
    for (int m0 = 0; m0 < count; m0 += 16 * MT) {
        unsigned h[MT];
        bool live[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int m = m0 + t * 16 + r16, entry = row_of_table[2 + min(m, a.T - 1)];     // read before `count` is known: one round trip
            live[t] = m < count;
            h[t] = ((unsigned)(live[t] ? entry : 0) * (unsigned)a.inter + g * CE) * W::SZ;
        }
        f32x4_t acc[NT][MT];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[j][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        constexpr int REGS = NT * W::RAW + MT * PH, U = REGS <= 2 ? 4 : REGS <= 4 ? 2 : 1;    // pieces in flight a wave, by registers
        const int K = k_hi - g * CE;
        constexpr int STRIDE = U * WAVES * PIECE;
        W w[2 * U][NT];
        uint4 hv[2 * U][MT][PH];
        auto load = [&](int q, int k) {                                   // half piece q of the round that starts at k; zero past the end
            const int kq = k + (q >> 1) * WAVES * PIECE + (q & 1) * 4 * CE;
            const bool ok = kq < K;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                if (ok) w[q][j].load(w2, row[j] + kq * W::SZ, low);
                else w[q][j].clear();
            }
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int p = 0; p < PH; ++p)
                    hv[q][t][p] = ok && live[t] ? *reinterpret_cast<const uint4*>(hidden[p] + (unsigned)(h[t] + kq * W::SZ)) : make_uint4(0u, 0u, 0u, 0u);
        };
        for (int k = k_lo + wave * PIECE; k < k_hi; k += STRIDE) {
#pragma unroll
            for (int q = 0; q < 2 * U; ++q) load(q, k);
#pragma unroll
            for (int q = 0; q < 2 * U; ++q) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    uint4 pw[W::PARTS];
                    if constexpr (P != P_F32) w[q][j].parts(pw);
#pragma unroll
                    for (int t = 0; t < MT; ++t) {
                        if constexpr (P == P_F32) acc[j][t] = mfma_f(w[q][j].raw[0], hv[q][t][0], acc[j][t]);
                        else acc[j][t] = mfma_parts<W::PARTS, PH, PH>(pw, hv[q][t], acc[j][t]);
                    }
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int t = 0; t < MT; ++t) *reinterpret_cast<f32x4_t*>(sums[wave][j * MT + t][lane]) = acc[j][t];
        __syncthreads();
        const int rows = min(count - m0, 16 * MT);
        for (int i = tid; i < rows * COLS; i += 64 * WAVES) {
            const int m = i / COLS, c = i % COLS;
            if (col0 + c >= a.d) continue;
            const int t = (c >> 4) * MT + (m >> 4), l = ((c & 15) >> 2) * 16 + (m & 15);
            float v = 0.f;
#pragma unroll
            for (int s = 0; s < WAVES; ++s) v += sums[s][t][l][c & 3];
            __hip_atomic_store(&a.part[((int64_t)part * n + row_of_table[2 + m0 + m]) * a.d + col0 + c], v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
    // The last workgroup of this column group joins.  Nobody waits: the others have left.  The sums are written and read by device-scope
    // accesses, which go past the L2 of an XCD; every wave waits for its own to arrive before the workgroup is counted.
    // (A device-scope fence does the same by writing back the whole L2: 40 us for one token of width 512.)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) last = __hip_atomic_fetch_add(&a.arrived[blockIdx.x], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == chosen * a.k_splits - 1;
    __syncthreads();
    if (!last) return;
    // Two columns an item, two items and eight terms at a time: a thread's loads are in flight together, for the tail of the launch is their latency.
    const A* res = static_cast<const A*>(a.res);
    const int terms = a.top_k * a.k_splits, items = a.T * (COLS / 2);
    typedef unsigned long long u64;
    constexpr int J = 2, C = 8;
    for (int i0 = tid; i0 < items; i0 += J * 64 * WAVES) {
        float s0[J], s1[J];
        int t[J], c[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int i = min(i0 + j * 64 * WAVES, items - 1);
            t[j] = i / (COLS / 2);
            c[j] = min(col0 + i % (COLS / 2) * 2, a.d - 2);               // columns behind d load the last two again
            s0[j] = s1[j] = 0.f;
        }
        for (int q0 = 0; q0 < terms; q0 += C) {
            u64 f[J][C];
            float wt[J][C];
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int p = 0; p < C; ++p) {
                    const int q = min(q0 + p, terms - 1), slot = q / a.k_splits, entry = t[j] * a.top_k + slot;
                    wt[j][p] = a.wts[entry];
                    f[j][p] = __hip_atomic_load(reinterpret_cast<const u64*>(a.part + ((int64_t)(q - slot * a.k_splits) * n + entry) * a.d + c[j]), __ATOMIC_RELAXED,
                                                __HIP_MEMORY_SCOPE_AGENT);
                }
#pragma unroll
            for (int p = 0; p < C; ++p)
                if (q0 + p < terms) {
#pragma unroll
                    for (int j = 0; j < J; ++j) {
                        s0[j] += wt[j][p] * __uint_as_float((unsigned)f[j][p]);
                        s1[j] += wt[j][p] * __uint_as_float((unsigned)(f[j][p] >> 32));
                    }
                }
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int i = i0 + j * 64 * WAVES;
            if (i >= items) break;
            if (col0 + i % (COLS / 2) * 2 >= a.d) continue;               // stored once: y may be the residual
            const int64_t at = (int64_t)t[j] * a.d + c[j];
            Pack<A, 2> r, o;
            if (res) r = *reinterpret_cast<const Pack<A, 2>*>(res + at);
            o.v[0] = (A)(s0[j] + (res ? (float)r.v[0] : 0.f));
            o.v[1] = (A)(s1[j] + (res ? (float)r.v[1] : 0.f));
            *reinterpret_cast<Pack<A, 2>*>(static_cast<A*>(a.y) + at) = o;
        }
    }
}

// ------------------------------------------------------------------------------------------------------------- host
inline size_t up256(size_t v) { return (v + 255) / 256 * 256; }

// Row groups of a wave: one while the tokens fit one matrix tile, else as many as make the tokens' reads small against the weights'
inline int up_nt(int T) { return T <= 16 ? 1 : 2; }
inline int down_nt(int T) { return T <= 16 ? 1 : 4; }

struct FewPlan { int active, wk, up_blocks, k_splits, down_blocks; size_t idx, wts, table, h, part, arrived, bytes; int64_t h_plane; };

FewPlan few_plan(int T, int d, int inter, int E, int top_k, int act_type, int precision) {
    FewPlan p;
    const int n = T * top_k, piece = precision == P_F32 ? 32 : 64;
    p.active = n < E ? n : E;                                             // experts that can have been chosen
    // `up`: within UP_BLOCKS by the number of waves that share a row group ...
    const int groups = (inter + 16 * up_nt(T) - 1) / (16 * up_nt(T));
    p.wk = WAVES;
    while (p.wk > 1 && (groups + WAVES / p.wk - 1) / (WAVES / p.wk) * p.active > UP_BLOCKS) p.wk /= 2;
    p.up_blocks = (groups + WAVES / p.wk - 1) / (WAVES / p.wk);
    // ... `down`: DOWN_BLOCKS and DOWN_KB by the number of parts of the hidden axis, each with a piece for every wave
    p.down_blocks = (d + 16 * down_nt(T) - 1) / (16 * down_nt(T));
    const int64_t bytes = (int64_t)p.active * d * inter * (precision == P_F32 ? 4 : 2) / DOWN_KB >> 10;
    const int want = (int)((bytes > DOWN_BLOCKS ? bytes : DOWN_BLOCKS) / (p.down_blocks * p.active)), most = inter / (piece * WAVES);
    p.k_splits = want < most ? want : most;
    if (p.k_splits < 1) p.k_splits = 1;
    p.h_plane = (int64_t)n * inter;
    size_t off = 0;
    auto take = [&](size_t b) { const size_t at = off; off += up256(b); return at; };
    p.idx = take((size_t)n * 4);
    p.wts = take((size_t)n * 4);
    p.table = take((1 + (size_t)p.active * (T + 2)) * 4);
    p.h = take((size_t)p.h_plane * (precision == P_F32 ? 4 : act_type == DT_F32 ? 6 : 4));
    p.part = take((size_t)p.k_splits * n * d * 4);
    p.arrived = take((size_t)p.down_blocks * 4);
    p.bytes = off;
    return p;
}

bool few_shape_ok(int T, int d, int inter, int E, int top_k) {
    return T >= 1 && T <= FEW_MAX_T && d >= 32 && d % 32 == 0 && d <= (1 << 16) && inter >= 32 && inter % 32 == 0 && inter <= (1 << 18) && E >= 1 && E <= FEW_MAX_E && top_k >= 1 &&
           top_k <= FEW_MAX_K && top_k <= E && (int64_t)d * inter <= 1 << 28;
}

bool few_types_ok(int act_type, int precision) {
    if (act_type == DT_F32) return precision == P_F32 || precision == P_BF16 || precision == P_BF16X3 || precision == P_F16;
    return (act_type == DT_BF16 && precision == P_BF16) || (act_type == DT_F16 && precision == P_F16);
}

// Tokens up to which `up` routes by itself: as long as all fit one round (the launch it saves costs 4 us, a second round 5)
constexpr int ROUTE_INSIDE = ROUTE_TOKENS;
template <typename A, int P, int MT, int UP_NT, int DOWN_NT>
void launch_few_layer(const FewArgs& a, const FewPlan& p, hipStream_t s) {
    const dim3 up((unsigned)p.up_blocks, (unsigned)p.active), down((unsigned)p.down_blocks, (unsigned)(p.active * p.k_splits)), block(64 * WAVES);
    bool inside = false;
    if constexpr (MT == 1) {
        inside = a.T <= ROUTE_INSIDE;
        if (inside) hipLaunchKernelGGL((few_up_kernel<A, P, 1, UP_NT, true>), up, block, 0, s, a);
    }
    if (!inside) {
        hipLaunchKernelGGL(few_route_kernel<A>, dim3((unsigned)a.T), block, 0, s, a);
        hipLaunchKernelGGL((few_up_kernel<A, P, MT, UP_NT, false>), up, block, 0, s, a);
    }
    hipLaunchKernelGGL((few_down_kernel<A, P, MT, DOWN_NT>), down, block, 0, s, a);
}

template <typename A, int P>
void launch_by_tokens(const FewArgs& a, const FewPlan& p, hipStream_t s) {
    if (a.T <= 16) launch_few_layer<A, P, 1, 1, 1>(a, p, s);
    else launch_few_layer<A, P, 2, 2, 4>(a, p, s);
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
        set_error("moe_few: needs 1 <= T <= 64 tokens, 1 <= top_k <= min(E, 8), E <= 64, and hidden (<= 65536) / expert (<= 262144) widths that are multiples of 32 with d * inter <= 2^28"); return ADX_EINVAL;
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
    a.table = reinterpret_cast<int*>(base + p.table);
    a.h = base + p.h; a.h_plane = p.h_plane; a.part = reinterpret_cast<float*>(base + p.part); a.arrived = reinterpret_cast<int*>(base + p.arrived);
    a.arrivals = p.down_blocks; a.wk = p.wk; a.k_splits = p.k_splits; a.y = y;
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
