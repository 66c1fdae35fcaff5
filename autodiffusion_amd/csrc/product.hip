// y = act(x w^T + bias) + residual on fp32, bf16 or fp16 tensors, and its gradients.  All three products of a training step are
//     C[i][j] = sum_k A(i, k) B(j, k)
// with either operand stored with k contiguous ("row": x and w of the forward) or with its own index contiguous ("column"): the
// data gradient dx[m][k] = sum_n dz[m][n] w[n][k] has a column B, the weight gradient dw[n][k] = sum_m dz[m][n] x[m][k] two column
// operands.  Sums are fp32; bias, activation and residual are applied to the fp32 sum and the result is rounded once.
#include "adx_ops.h"
#include "engine.h"
#include "fastmath.h"
#include "typed.h"

#include <type_traits>

namespace adx {
namespace {

constexpr int ACT_TANH_ = 6;

__device__ __align__(16) unsigned char zero_chunk[16];            // what copies past the end of the summed axis read

// ------------------------------------------------------------------------------------------------------------- activations
// Phi(-|z|), the smaller tail of the normal distribution, and e = exp(-z^2 / 2): e times a polynomial in t = 1 / (1 + 0.35 |z|), fitted to
// Phi(-|z|) / (t e) for |z| <= 13 (relative error 8e-8; in fp32 4e-7 up to |z| = 2, then about 6e-8 z^2, 8e-6 at 13, from the roundings of the exponent;
// absolute at most 1.5e-7; 1 - erf would have no digits left in the tail).  The slope shares the exponential: the activation of a 256 x 256 tile is as long as a quarter of its products at k = 1024.
__device__ __forceinline__ float normal_tail(float z, float& e) {
    e = exp2_fast(-0.72134752044448170f * z * z);
    const float t = rcp_fast(1.f + 0.35f * fabsf(z));
    float p = -0.029108895f;
    p = p * t + 0.14378804f; p = p * t - 0.255326897f; p = p * t + 0.158721581f; p = p * t - 0.0227904506f;
    p = p * t + 0.105369069f; p = p * t + 0.11986912f; p = p * t + 0.139856696f; p = p * t + 0.139621705f;
    return p * t * e;
}
__device__ __forceinline__ float sigmoid_fast(float z) { return rcp_fast(1.f + exp2_fast(-1.44269504088896341f * z)); }
// z + 0.044715 z^3 scaled so that its sigmoid is (1 + tanh(sqrt(2 / pi) (z + 0.044715 z^3))) / 2
__device__ __forceinline__ float gelu_tanh_arg(float z) { return 1.59576912160573071f * z * (1.f + 0.044715f * z * z); }

// act(z) in place and, with SLOPE, act'(z) from the same exponentials
template <typename T, int V, bool SLOPE> __device__ __forceinline__ void apply_act(float (&v)[V], float (&d)[V], int act) {
    switch (act) {                                                 // uniform: one branch for all values
        case ACT_RELU:
#pragma unroll
            for (int e = 0; e < V; ++e) { if (SLOPE) d[e] = v[e] > 0.f ? 1.f : v[e] == v[e] ? 0.f : v[e]; v[e] = v[e] < 0.f ? 0.f : v[e]; }      // NaN stays
            break;
        case ACT_LEAKY:
#pragma unroll
            for (int e = 0; e < V; ++e) { if (SLOPE) d[e] = v[e] > 0.f ? 1.f : v[e] == v[e] ? 0.01f : v[e]; v[e] = v[e] > 0.f ? v[e] : 0.01f * v[e]; }
            break;
        case ACT_SILU:
#pragma unroll
            for (int e = 0; e < V; ++e) { const float g = sigmoid_fast(v[e]); if (SLOPE) d[e] = g * (1.f + v[e] * (1.f - g)); v[e] *= g; }
            break;
        case ACT_TANH_:
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if (SLOPE) {                                       // 1 - tanh^2 as 4 q / (1 + q)^2, q = exp(-2 |z|): the difference has no digits left beyond |z| = 9
                    const float q = exp2_fast(-2.88539008177792682f * fabsf(v[e])), r = rcp_fast(1.f + q);
                    d[e] = 4.f * q * r * r;
                }
                v[e] = tanhf(v[e]);
            }
            break;
        case ACT_GELU_ERF:
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float g;
                const float q = normal_tail(v[e], g), p = v[e] > 0.f ? 1.f - q : q;
                if (SLOPE) d[e] = p + v[e] * 0.39894228040143268f * g;
                v[e] *= p;
            }
            break;
        case ACT_GELU_TANH:
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float g = sigmoid_fast(gelu_tanh_arg(v[e]));
                if (SLOPE) {
                    const float c = fminf(fmaxf(v[e], -30.f), 30.f);            // beyond 30 the slope is 0 or 1
                    d[e] = v[e] == v[e] ? g + c * g * (1.f - g) * 1.59576912160573071f * (1.f + 0.134145f * c * c) : v[e];
                }
                v[e] *= g;
            }
            break;
        default:
            if (SLOPE)
#pragma unroll
                for (int e = 0; e < V; ++e) d[e] = 1.f;
    }
}

// What the forward keeps for the gradient is the activation's slope, not its argument: the backward needs no exponentials.  In fp32
// a slope has its relative accuracy down to the smallest ones: a unit in saturation (GELU at -5: -7e-6) learns from those alone.  16-bit tensors
// may keep codes of half the size instead: q stands for (q - 8192) / 32768, 0 for NaN (what the conversion of one gives), and LeakyReLU's
// two for 1 and 0.01 themselves -- exact for ReLU and LeakyReLU; of the smooth activations slopes below 2^-16 vanish.
template <typename T> struct Code { typedef unsigned short type; };
template <> struct Code<float> { typedef float type; };
__device__ __forceinline__ void set_code(float d, float& q) { q = d; }
__device__ __forceinline__ void set_code(float d, unsigned short& q) { q = (unsigned short)(unsigned)(d * 32768.f + 8192.5f); }
__device__ __forceinline__ float slope_value(float q, int act) { return q; }
__device__ __forceinline__ float slope_value(unsigned short q, int act) {
    const float d = act == ACT_LEAKY ? (q > 16384 ? 1.f : 0.01f) : (float)((int)q - 8192) * (1.f / 32768.f);
    return q ? d : __builtin_nanf("");
}

// ------------------------------------------------------------------------------------------------------------- the problem
struct ProductArgs {
    const void* A; int64_t lda;              // element strides of the axis that is not contiguous
    const void* B; int64_t ldb;
    int64_t M; int N; int64_t K;             // C is M x N, K is summed
    int64_t own_a; int own_b;                // column operands: values of their own index that may be read (M, N, or padded to whole pieces)
    const void* bias; const void* res; int64_t ldr;
    void* slope; bool slope_f32;             // [M][N]: the activation's slope (for the gradient), fp32 or Code<T>
    void* y; int64_t ldy;
    int act;
    int splits; int64_t k_split;             // K range of one split (a multiple of the K step)
    float* part;                             // splits > 1: [splits][M][N] partial sums
    bool vec;                                // 16-byte epilogue
    int tiles_m, tiles_n;
};

// V consecutive columns of one row, all of them inside it and V-aligned: bias, activation (and slope), residual, one rounding, store
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> residual_at(const ProductArgs& a, int64_t m, int n) {
    return *reinterpret_cast<const Pack<T, V>*>(static_cast<const T*>(a.res) + m * a.ldr + n);
}
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> bias_at(const ProductArgs& a, int n) {
    return *reinterpret_cast<const Pack<T, V>*>(static_cast<const T*>(a.bias) + n);
}
template <typename S, int V>
__device__ __forceinline__ void put_slopes(const ProductArgs& a, int64_t m, int n, const float (&d)[V]) {
    Pack<S, V> q;
#pragma unroll
    for (int e = 0; e < V; ++e) set_code(d[e], q.v[e]);
    *reinterpret_cast<Pack<S, V>*>(static_cast<S*>(a.slope) + m * a.N + n) = q;
}
template <typename T, int V>
__device__ __forceinline__ void activate(const ProductArgs& a, int64_t m, int n, float (&v)[V], const Pack<T, V>& b) {
    if (a.bias) {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] += (float)b.v[e];
    }
    float d[V];
    if (a.slope) {
        apply_act<T, V, true>(v, d, a.act);
        if (a.slope_f32) put_slopes<float, V>(a, m, n, d);
        else put_slopes<typename Code<T>::type, V>(a, m, n, d);
    } else apply_act<T, V, false>(v, d, a.act);
}
template <typename T, int V>
__device__ __forceinline__ void put(const ProductArgs& a, int64_t m, int n, const float (&v)[V]) {
    typedef Pack<T, V> P;
    P o;
#pragma unroll
    for (int e = 0; e < V; ++e) o.v[e] = (T)v[e];
    *reinterpret_cast<P*>(static_cast<T*>(a.y) + m * a.ldy + n) = o;
}
template <typename T, int V>
__device__ __forceinline__ void finish(const ProductArgs& a, int64_t m, int n, float (&v)[V]) {
    Pack<T, V> b{};
    if (a.bias) b = bias_at<T, V>(a, n);
    activate<T, V>(a, m, n, v, b);
    if (a.res) {
        const Pack<T, V> r = residual_at<T, V>(a, m, n);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] += (float)r.v[e];
    }
    put<T, V>(a, m, n, v);
}

// ------------------------------------------------------------------------------------------------------------- large tiles
typedef __attribute__((address_space(3))) void* lds_ptr;

// 64 x 16 bytes from per-lane global addresses to 1 KB of LDS.  Issued from inline assembly: the compiler would make every later LDS
// read wait for all copies it knows of; the kernel orders them itself with counted waits and barriers.
__device__ __forceinline__ void copy_1k_lanes(const void* g, unsigned lds_uniform) {
    unsigned keep;          // m0 is restored: the compiler does not expect inline assembly to change it
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "s"(lds_uniform), "v"(g) : "memory");
}
// the same with a wave-uniform base and a 32-bit byte offset a lane: no vector arithmetic
__device__ __forceinline__ void copy_1k(const void* base_uniform, unsigned lane_offset, unsigned lds_uniform) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "s"(lds_uniform), "v"(lane_offset), "s"(base_uniform) : "memory");
}
template <int N> __device__ __forceinline__ void wait_copies() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// One operand's part of a K step: ROWS of its own index x 64 bytes of k, an image in LDS.
//   row:    [ROWS][64 B]; 16-byte chunk c of row r sits at c ^ ((r >> 2) & 3): 16 rows of one chunk (a quarter of a fragment read) meet
//           every bank once
//   column: [KE][ROWS]; the 16-bit fragment read is the transposing LDS read (4 k-rows x 16 own indices a 16-lane group): 32-byte unit
//           u of k-row k sits at u ^ f(k) so that the k-rows of one read lie in different banks; fp32 reads 32 consecutive values
template <typename T, bool COL, int ROWS, int KB> struct Side {
    static constexpr int SZ = sizeof(T), CE = 16 / SZ, KE = KB / SZ;
    static constexpr int BYTES = ROWS * KB, SLABS = BYTES / 1024, RB = ROWS * SZ;
    static __device__ __forceinline__ int row_swizzle(int r) { return KB == 64 ? (r >> 2) & 3 : (r >> 1) & 7; }
    static __device__ __forceinline__ int unit_swizzle(int k) {
        if constexpr (SZ == 2) { constexpr int mask = RB / 32 - 1; return (((k & 3) | (((k >> 3) & 1) << 2)) & mask) << 5; }
        else return ((k >> 2) & 1) << 7;
    }
    // own index and first k (relative to the tile) of the 16 bytes that lane `lane` copies to slab `slab`
    static __device__ __forceinline__ void source(int slab, int lane, int& row, int& k) {
        if constexpr (!COL) {
            constexpr int CPR = KB / 16;                       // chunks of a row
            row = slab * (64 / CPR) + lane / CPR;
            k = ((lane & (CPR - 1)) ^ row_swizzle(row)) * CE;
        } else {
            const int at = slab * 1024 + lane * 16;
            k = at / RB;
            row = ((at % RB) ^ unit_swizzle(k)) / SZ;
        }
    }
    // 16 bytes of k for own index base + (lane & 31): k = kk * 2 CE + CE * (lane >> 5) + 0 .. CE - 1
    static __device__ __forceinline__ uint4 fragment(const unsigned char* img, int base, int kk, int lane) {
        if constexpr (!COL) {
            const int r = base + (lane & 31), c = 2 * kk + (lane >> 5);
            return *reinterpret_cast<const uint4*>(img + r * KB + ((c ^ row_swizzle(r)) << 4));
        } else if constexpr (SZ == 2) {
            typedef short s4 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) s4* s4p;
            const int k = kk * 16 + 8 * (lane >> 5) + ((lane & 15) >> 2), own = (base + 16 * ((lane >> 4) & 1) + (lane & 3) * 4) * 2;
            union { s4 h[2]; uint4 u; } f;
            f.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s4p)(img + k * RB + (own ^ unit_swizzle(k))));
            f.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s4p)(img + (k + 4) * RB + (own ^ unit_swizzle(k + 4))));
            return f.u;
        } else {
            const int k = kk * 8 + 4 * (lane >> 5), own = (base + (lane & 31)) * 4;
            uint4 u;
            u.x = *reinterpret_cast<const unsigned*>(img + k * RB + (own ^ unit_swizzle(k)));
            u.y = *reinterpret_cast<const unsigned*>(img + (k + 1) * RB + (own ^ unit_swizzle(k)));
            u.z = *reinterpret_cast<const unsigned*>(img + (k + 2) * RB + (own ^ unit_swizzle(k)));
            u.w = *reinterpret_cast<const unsigned*>(img + (k + 3) * RB + (own ^ unit_swizzle(k)));
            return u;
        }
    }
};

template <typename T> __device__ __forceinline__ f32x16_t mfma32(const uint4& a, const uint4& b, f32x16_t c) {
    if constexpr (std::is_same<T, __bf16>::value) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    } else if constexpr (std::is_same<T, _Float16>::value) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
    } else {
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.x), __uint_as_float(b.x), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.y), __uint_as_float(b.y), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.z), __uint_as_float(b.z), c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.w), __uint_as_float(b.w), c, 0, 0, 0);
    }
}

// Epilogue of a wave's 32 FI x 32 FJ results: 32 rows at a time through LDS, so that a row's columns are stored as whole lines.
// Result layout of the 32x32 product: column = lane & 31, row = (q & 3) + 8 (q >> 2) + 4 (lane >> 5).
template <typename T, int FI, int FJ>
__device__ __forceinline__ void store_tile(const ProductArgs& a, f32x16_t (&acc)[FI][FJ], unsigned char* smem, int64_t m_wave, int n_wave, int wave, int lane) {
    constexpr int NW = FJ * 32, EP_LD = NW + 4, V = 16 / sizeof(T), LPR = NW / V, RPI = 64 / LPR;   // lanes of a row, rows of one pass
    float* patch = reinterpret_cast<float*>(smem) + wave * 32 * EP_LD;
    const int n = n_wave + (lane % LPR) * V;
    // Loads are waited for with every store issued before them, so none stands between stores: the bias of the lane's columns and the residual of the
    // first 64 rows are in registers (the fragments' are free) before the first store, later rows follow 64 behind.  With both read where they are
    // used (the residual a pass of 8 rows ahead) 6984 x 4096 x 1024 bf16 takes 97 us instead of 80.
    // Activated sums go back to LDS, so that only the addition of the residual is unrolled, not the activations.
    constexpr int PASSES = 32 / RPI, HELD = FI <= 2 ? FI : 2;
    const bool with_res = a.res && a.vec && a.splits <= 1;
    Pack<T, V> held[HELD][PASSES];
    const int64_t m_last = a.M - 1;
    auto hold = [&](int i) {                                   // 32 rows of the wave's tile; past the end of the tensor: the last row
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            const int64_t m = m_wave + i * 32 + p * RPI + lane / LPR;
            held[i % HELD][p] = residual_at<T, V>(a, m < m_last ? m : m_last, n < a.N ? n : 0);
        }
    };
    auto sums = [&](int r) { return patch + r * EP_LD + (lane % LPR) * V; };
    auto get = [&](int r, float (&v)[V]) {
#pragma unroll
        for (int e = 0; e < V; e += 4) {
            const float4 f = *reinterpret_cast<const float4*>(sums(r) + e);
            v[e] = f.x; v[e + 1] = f.y; v[e + 2] = f.z; v[e + 3] = f.w;
        }
    };
    Pack<T, V> bias{};
    if (a.bias && a.vec) bias = bias_at<T, V>(a, n < a.N ? n : 0);
    if (with_res)
#pragma unroll
        for (int i = 0; i < HELD; ++i) hold(i);
#pragma unroll
    for (int i = 0; i < FI; ++i) {
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < FJ; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<float4*>(patch + (lane & 31) * EP_LD + j * 32 + 8 * q + 4 * (lane >> 5)) =
                    make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
        wait_lds();
        __builtin_amdgcn_wave_barrier();
        if (!a.vec) {                                          // rows that hold no whole pieces: a lane a column, so that stores stay side by side
            constexpr int STEP = NW < 64 ? NW : 64, ROWS = 64 / STEP;
#pragma unroll 1
            for (int c0 = 0; c0 < NW; c0 += STEP)
#pragma unroll 1
                for (int p = 0; p < 32 / ROWS; ++p) {
                    const int r = p * ROWS + lane / STEP, c = n_wave + c0 + lane % STEP;
                    const int64_t m = m_wave + i * 32 + r;
                    float v[1] = {patch[r * EP_LD + c0 + lane % STEP]};
                    if (m < a.M && c < a.N) {
                        if (a.splits > 1) a.part[((int64_t)blockIdx.y * a.M + m) * a.N + c] = v[0];
                        else finish<T, 1>(a, m, c, v);
                    }
                }
            wait_lds();
            continue;
        }
        if (!with_res) {
#pragma unroll 1
            for (int p = 0; p < PASSES; ++p) {
                const int r = p * RPI + lane / LPR;
                const int64_t m = m_wave + i * 32 + r;
                float v[V];
                get(r, v);
                if (m < a.M && n < a.N) {
                    if (a.splits > 1) {
                        float* o = a.part + ((int64_t)blockIdx.y * a.M + m) * a.N + n;
#pragma unroll
                        for (int e = 0; e < V; e += 4) *reinterpret_cast<float4*>(o + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
                    } else {
                        activate<T, V>(a, m, n, v, bias);
                        put<T, V>(a, m, n, v);
                    }
                }
            }
        } else {
#pragma unroll 1
            for (int p = 0; p < PASSES; ++p) {                 // the activated sums go back to where this lane read them
                const int r = p * RPI + lane / LPR;
                const int64_t m = m_wave + i * 32 + r;
                float v[V];
                get(r, v);
                if (m < a.M && n < a.N) activate<T, V>(a, m, n, v, bias);
#pragma unroll
                for (int e = 0; e < V; e += 4) *reinterpret_cast<float4*>(sums(r) + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
            }
#pragma unroll
            for (int p = 0; p < PASSES; ++p) {
                const int r = p * RPI + lane / LPR;
                const int64_t m = m_wave + i * 32 + r;
                float v[V];
                get(r, v);
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] += (float)held[i % HELD][p].v[e];
                if (m < a.M && n < a.N) put<T, V>(a, m, n, v);
            }
            if (i + HELD < FI) hold(i + HELD);
        }
        wait_lds();
    }
}

// Workgroup tile BM x BN, WM x WN waves, a K step of KB bytes a row, a ring of R LDS slots.  Copies go straight from global memory to
// LDS and are R - 1 steps ahead.  One barrier a step: a wave passes it when it holds the step's last fragments in registers and
// its copies of the next step have landed; behind it the step's slot is refilled and the next step is read, both under the step's
// last products.  Fragments are read under the products before theirs, all of them in front of the first half of those.
template <typename T, bool ACOL, bool BCOL, int BM, int BN, int WM, int WN, int KB, int R>
__global__ __launch_bounds__(64 * WM * WN, 2) void product_kernel(const ProductArgs a) {
    typedef Side<T, ACOL, BM, KB> SA;
    typedef Side<T, BCOL, BN, KB> SB;
    constexpr int W = WM * WN, KE = SA::KE, SZ = sizeof(T);
    constexpr int FI = BM / WM / 32, FJ = BN / WN / 32, NW = BN / WN, NKK = KB / 32;
    constexpr int SLOT = SA::BYTES + SB::BYTES, PA = SA::SLABS / W, PB = SB::SLABS / W, P = PA + PB;
    constexpr int EP_LD = NW + 4;
    static_assert(SA::SLABS % W == 0 && SB::SLABS % W == 0, "slabs spread evenly over the waves");
    static_assert(W * 32 * EP_LD * 4 <= R * SLOT, "the epilogue's patches fit the slots");
    static_assert((R & (R - 1)) == 0 && (R - 1) * P < 64, "slot of a step by mask; counted waits");
    __shared__ __attribute__((aligned(1024))) unsigned char smem[R * SLOT];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // XCD x (blockIdx % 8) walks a contiguous range of an order of column panels eight tiles wide, so that the workgroups that
    // run on an XCD at one time share rows and columns in its L2
    const int n_tiles = a.tiles_m * a.tiles_n, per_xcd = (n_tiles + 7) / 8;
    const int lin = (int)(blockIdx.x & 7) * per_xcd + (int)(blockIdx.x >> 3);
    if (lin >= n_tiles) return;
    const int panel = lin / (a.tiles_m * 8), width = min(8, a.tiles_n - panel * 8), in = lin - panel * a.tiles_m * 8;
    const int64_t m0 = (int64_t)(in / width) * BM;
    const int n0 = (panel * 8 + in % width) * BN;
    const int64_t k_lo = (int64_t)blockIdx.y * a.k_split, k_len = (k_lo + a.k_split < a.K ? k_lo + a.k_split : a.K) - k_lo;
    const int nk = (int)((k_len + KE - 1) / KE);
    const int wm = wave / WN, wn = wave % WN;

    // Sources: a wave-uniform base that advances by a step, a constant 32-bit byte offset a lane (the host checks that tiles span less
    // than 2^31 bytes).  Own indices past the end repeat the last valid ones (those results are not stored); k past the end reads zeros.
    const unsigned lds0 = (unsigned)(uintptr_t)(lds_ptr)smem;
    unsigned oa[PA], ob[PB];
    int ka[PA], kb[PB];
    const int64_t row_end = (ACOL ? a.own_a : a.M) - m0, col_end = (BCOL ? a.own_b : a.N) - n0;
#pragma unroll
    for (int i = 0; i < PA; ++i) {
        int row;
        SA::source(wave + i * W, lane, row, ka[i]);
        const int last = (int)(row_end < BM ? row_end : BM) - (ACOL ? SA::CE : 1);
        row = min(row, last);
        oa[i] = (unsigned)((ACOL ? (int64_t)ka[i] * a.lda + row : (int64_t)row * a.lda + ka[i]) * SZ);
    }
#pragma unroll
    for (int i = 0; i < PB; ++i) {
        int row;
        SB::source(wave + i * W, lane, row, kb[i]);
        const int last = (int)(col_end < BN ? col_end : BN) - (BCOL ? SB::CE : 1);
        row = min(row, last);
        ob[i] = (unsigned)((BCOL ? (int64_t)kb[i] * a.ldb + row : (int64_t)row * a.ldb + kb[i]) * SZ);
    }
    const unsigned char* base_a = static_cast<const unsigned char*>(a.A) + (ACOL ? k_lo * a.lda + m0 : m0 * a.lda + k_lo) * SZ;
    const unsigned char* base_b = static_cast<const unsigned char*>(a.B) + (BCOL ? k_lo * a.ldb + n0 : (int64_t)n0 * a.ldb + k_lo) * SZ;
    const int64_t step_a = (ACOL ? a.lda * KE : KE) * SZ, step_b = (BCOL ? a.ldb * KE : KE) * SZ;
    int left = (int)k_len;                                     // valid k from the next step to copy on
    // the i-th of this wave's copies of the next step, into its slot
    auto copy_a = [&](int i, unsigned slot) {
        const unsigned at = lds0 + slot + (unsigned)(wave + i * W) * 1024u;
        if (left >= KE) copy_1k(base_a, oa[i], at);
        else copy_1k_lanes(ka[i] < left ? base_a + oa[i] : zero_chunk, at);
    };
    auto copy_b = [&](int i, unsigned slot) {
        const unsigned at = lds0 + slot + SA::BYTES + (unsigned)(wave + i * W) * 1024u;
        if (left >= KE) copy_1k(base_b, ob[i], at);
        else copy_1k_lanes(kb[i] < left ? base_b + ob[i] : zero_chunk, at);
    };
    auto advance = [&]() { base_a += step_a; base_b += step_b; left -= KE; };

    f32x16_t acc[FI][FJ];
#pragma unroll
    for (int i = 0; i < FI; ++i)
#pragma unroll
        for (int j = 0; j < FJ; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.f;

#pragma unroll
    for (int t = 0; t < R; ++t) {
#pragma unroll
        for (int i = 0; i < PA; ++i) copy_a(i, t * SLOT);
#pragma unroll
        for (int i = 0; i < PB; ++i) copy_b(i, t * SLOT);
        advance();
    }
    wait_copies<(R - 1) * P>();
    barrier();
    uint4 fa[2][FI], fb[2][FJ];
#pragma unroll
    for (int j = 0; j < FJ; ++j) fb[0][j] = SB::fragment(smem + SA::BYTES, wn * NW + j * 32, 0, lane);
#pragma unroll
    for (int i = 0; i < FI; ++i) fa[0][i] = SA::fragment(smem, wm * (BM / WM) + i * 32, 0, lane);
    for (int kt = 0; kt < nk; ++kt) {
        const unsigned slot = (unsigned)(kt & (R - 1)) * SLOT, next = (unsigned)((kt + 1) & (R - 1)) * SLOT;
#pragma unroll
        for (int kk = 0; kk < NKK; ++kk) {
            const bool turn = kk == NKK - 1;
            if (turn) {
                wait_lds();                                    // this wave has read all of the step ...
                wait_copies<(R - 2) * P>();                    // ... and its copies of the next one have landed
                barrier();
            }
            const unsigned char* img = smem + (turn ? next : slot);
            const int to = (kk + 1) & 1, at = turn ? 0 : kk + 1;
#pragma unroll
            for (int i = 0; i < FI; ++i) {
                if (i == 0) {
#pragma unroll
                    for (int j = 0; j < FJ; ++j) fb[to][j] = SB::fragment(img + SA::BYTES, wn * NW + j * 32, at, lane);
                }
                if (2 * i < FI) {
#pragma unroll
                    for (int r = 2 * i; r < min(2 * i + 2, FI); ++r) fa[to][r] = SA::fragment(img, wm * (BM / WM) + r * 32, at, lane);
                }
                if (turn) {
#pragma unroll
                    for (int p = i * PA / FI; p < (i + 1) * PA / FI; ++p) copy_a(p, slot);
#pragma unroll
                    for (int p = i * PB / FI; p < (i + 1) * PB / FI; ++p) copy_b(p, slot);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < FJ; ++j) acc[i][j] = mfma32<T>(fb[kk & 1][j], fa[kk & 1][i], acc[i][j]);      // rows of the result: n; columns: m
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        advance();
    }
    wait_copies<0>();
    wait_lds();
    barrier();

    store_tile<T, FI, FJ>(a, acc, smem, m0 + wm * (BM / WM), n0 + wn * NW, wave, lane);
}

// The first min(left, 16 / size) values from p, which need not lie on 16 bytes, zeros behind them
template <typename T> __device__ __forceinline__ uint4 unaligned_chunk(const T* p, int64_t left) {
    constexpr int CE = 16 / sizeof(T);
    union { T v[CE]; uint4 u; } f;
    f.u = make_uint4(0u, 0u, 0u, 0u);
    if (left >= CE) __builtin_memcpy(&f.u, p, 16);
    else {
#pragma unroll
        for (int e = 0; e < CE; ++e) if (e < left) f.v[e] = p[e];
    }
    return f.u;
}

// Operands whose rows start on no 16 bytes and that nobody has laid out anew: loads through registers into the same images, 64 x 64
// tiles, one slot.
template <typename T, bool ACOL, bool BCOL>
__global__ __launch_bounds__(256) void product_any_kernel(const ProductArgs a) {
    typedef Side<T, ACOL, 64, 64> SA;
    typedef Side<T, BCOL, 64, 64> SB;
    constexpr int KE = SA::KE, CE = SA::CE;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[4 * 32 * 36 * 4];             // two images, then the epilogue's patches
    static_assert(sizeof(smem) >= SA::BYTES + SB::BYTES, "images fit");
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave >> 1, wn = wave & 1;
    const int64_t m0 = (int64_t)(blockIdx.x / a.tiles_n) * 64;
    const int n0 = (int)(blockIdx.x % a.tiles_n) * 64;
    const int64_t k_lo = (int64_t)blockIdx.y * a.k_split, k_hi = k_lo + a.k_split < a.K ? k_lo + a.k_split : a.K;
    auto gather = [&](const void* base, int64_t ld, bool col, int64_t own, int64_t own_end, int64_t k, unsigned at) {
        const int64_t left = col ? (k < k_hi ? own_end - own : 0) : (own < own_end ? k_hi - k : 0);
        *reinterpret_cast<uint4*>(smem + at) = unaligned_chunk(static_cast<const T*>(base) + (col ? k * ld + own : own * ld + k), left);
    };
    f32x16_t acc[1][1];
#pragma unroll
    for (int q = 0; q < 16; ++q) acc[0][0][q] = 0.f;
    int ra, ka, rb, kb;
    SA::source(wave, lane, ra, ka);
    SB::source(wave, lane, rb, kb);
    for (int64_t k = k_lo; k < k_hi; k += KE) {
        gather(a.A, a.lda, ACOL, m0 + ra, a.M, k + ka, tid * 16);
        gather(a.B, a.ldb, BCOL, n0 + rb, a.N, k + kb, SA::BYTES + tid * 16);
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
            acc[0][0] = mfma32<T>(SB::fragment(smem + SA::BYTES, wn * 32, kk, lane), SA::fragment(smem, wm * 32, kk, lane), acc[0][0]);
        __syncthreads();
    }
    store_tile<T, 1, 1>(a, acc, smem, m0 + wm * 32, n0 + wn * 32, wave, lane);
}

// the partial sums of a split product, added in split order, and the epilogue
template <typename T, int V>
__global__ __launch_bounds__(256) void product_join_kernel(const ProductArgs a) {
    const int per_row = a.N / V;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= a.M * per_row) return;
    const int64_t m = i / per_row;
    const int n = (int)(i - m * per_row) * V;
    float v[V];
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = 0.f;
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) {
        const Pack<float, V> f = *reinterpret_cast<const Pack<float, V>*>(a.part + ((int64_t)s * a.M + m) * a.N + n);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] += f.v[e];
    }
    finish<T, V>(a, m, n, v);
}

// ------------------------------------------------------------------------------------------------------------- few rows
// M <= 64: the weights are read once and nothing is staged.  A workgroup owns 16 rows of w (and reads all rows of x: 24 x 6144 x 1536
// moves 28 MB of x from the L2s beside 19 MB of w); its waves take 128-byte pieces of K in turn, load fragments of both operands from global memory into registers (16 rows x 16 bytes a
// quarter wave) and add up in LDS at the end.
template <typename T> __device__ __forceinline__ f32x4_t mfma16(const uint4& a, const uint4& b, f32x4_t c) {
    if constexpr (std::is_same<T, __bf16>::value) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    } else if constexpr (std::is_same<T, _Float16>::value) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
    } else {
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.x), __uint_as_float(b.x), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.y), __uint_as_float(b.y), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.z), __uint_as_float(b.z), c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.w), __uint_as_float(b.w), c, 0, 0, 0);
    }
}

// 16 bytes from element k of a row of K elements; zero past its end
template <typename T, bool ALIGNED>
__device__ __forceinline__ uint4 row_chunk(const T* row, int64_t k, int64_t K) {
    if constexpr (ALIGNED) return k < K ? *reinterpret_cast<const uint4*>(row + k) : make_uint4(0u, 0u, 0u, 0u);
    else return unaligned_chunk(row + k, K - k);
}

template <typename T, int MT, int NWAVES, bool ALIGNED>
__global__ __launch_bounds__(64 * NWAVES) void product_few_kernel(const ProductArgs a) {
    constexpr int CE = 16 / sizeof(T), UNIT = 8 * CE;
    __shared__ float sums[NWAVES][MT][64][4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n0 = blockIdx.x * 16, r16 = lane & 15, g = lane >> 4;
    const T *w = static_cast<const T*>(a.B) + (int64_t)min(n0 + r16, a.N - 1) * a.ldb + g * CE, *x[MT];
    bool live[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        live[t] = t * 16 + r16 < a.M;
        x[t] = static_cast<const T*>(a.A) + (int64_t)(live[t] ? t * 16 + r16 : 0) * a.lda + g * CE;
    }
    f32x4_t acc[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    const int64_t K = a.K - g * CE;
    constexpr int U = MT >= 4 ? 2 : 4;                             // pieces in flight a wave
    for (int64_t k = (int64_t)wave * UNIT; k < a.K; k += (int64_t)U * NWAVES * UNIT) {
        uint4 fw[2 * U], fx[2 * U][MT];
#pragma unroll
        for (int h = 0; h < 2 * U; ++h) {
            const int64_t kh = k + (int64_t)(h >> 1) * NWAVES * UNIT + (h & 1) * 4 * CE;
            fw[h] = row_chunk<T, ALIGNED>(w, kh, K);
#pragma unroll
            for (int t = 0; t < MT; ++t) fx[h][t] = live[t] ? row_chunk<T, ALIGNED>(x[t], kh, K) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int h = 0; h < 2 * U; ++h)
#pragma unroll
            for (int j = 0; j < MT; ++j) acc[j] = mfma16<T>(fw[h], fx[h][j], acc[j]);
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) *reinterpret_cast<f32x4_t*>(sums[wave][j][lane]) = acc[j];
    __syncthreads();
    // result layout of the 16x16 product: column (m) = lane & 15, row (n) = 4 (lane >> 4) + reg
    for (int i = tid; i < MT * 256; i += 64 * NWAVES) {
        const int nn = i % 16, m = i / 16, n = n0 + nn;
        if (m >= a.M || n >= a.N) continue;
        const int t = m >> 4, l = (nn >> 2) * 16 + (m & 15), q = nn & 3;
        float v[1] = {0.f};
#pragma unroll
        for (int s = 0; s < NWAVES; ++s) v[0] += sums[s][t][l][q];
        finish<T, 1>(a, m, n, v);
    }
}

// ------------------------------------------------------------------------------------------------------------- gradient of the epilogue
// dz = dy act'(z), rounded to the operand type of the products that follow, and per chunk of rows the fp32 column sums of the
// unrounded dz (joined in chunk order: no atomics).  Bound: memory; 8192 x 4096 bf16 with fp32 slopes moves 268 MB in 48 us, with codes 201 MB in 42.
constexpr int SLOPE_ROWS = 64;

template <typename T, typename S, bool VEC>
__global__ __launch_bounds__(256) void slope_kernel(const void* dy_, int64_t ldd, const void* slope_, void* dz_, int ldz, float* part, void* db, int64_t M, int N, int act) {
    constexpr int V = VEC ? 16 / sizeof(T) : 1, ROWS = V == 8 ? 2 : 4;
    __shared__ float sums[4][64 * V];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = (blockIdx.x * 64 + lane) * V;
    typedef Pack<T, V> P;
    for (int64_t chunk = blockIdx.y; chunk * SLOPE_ROWS < M; chunk += gridDim.y) {
        const int64_t r0 = chunk * SLOPE_ROWS, r1 = r0 + SLOPE_ROWS < M ? r0 + SLOPE_ROWS : M;
        float sum[V];
#pragma unroll
        for (int e = 0; e < V; ++e) sum[e] = 0.f;
        if (n < N) {
            for (int64_t m = r0 + wave; m < r1; m += 4 * ROWS) {        // loads do not pass the stores: 1037 x 1020 fp32 took 3 us more one by one
                P d[ROWS];
                Pack<S, V> q[ROWS];
#pragma unroll
                for (int i = 0; i < ROWS; ++i) {
                    const int64_t mi = m + 4 * i < r1 ? m + 4 * i : m;
                    d[i] = *reinterpret_cast<const P*>(static_cast<const T*>(dy_) + mi * ldd + n);
                    if (act != ACT_NONE) q[i] = *reinterpret_cast<const Pack<S, V>*>(static_cast<const S*>(slope_) + mi * N + n);
                }
#pragma unroll
                for (int i = 0; i < ROWS; ++i) {
                    if (m + 4 * i >= r1) break;
                    P o = d[i];                                         // without an activation: laid out anew
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        float g = (float)d[i].v[e];
                        if (act != ACT_NONE) { g *= slope_value(q[i].v[e], act); o.v[e] = (T)g; }
                        sum[e] += g;
                    }
                    if (dz_) *reinterpret_cast<P*>(static_cast<T*>(dz_) + (m + 4 * i) * ldz + n) = o;
                }
            }
        } else if (!VEC && dz_ && n < ldz) {                       // zeros up to whole pieces
            for (int64_t m = r0 + wave; m < r1; m += 4) static_cast<T*>(dz_)[m * ldz + n] = (T)0.f;
        }
        if (!part) continue;
        __syncthreads();                                            // the chunk before has been read
#pragma unroll
        for (int e = 0; e < V; ++e) sums[wave][lane * V + e] = sum[e];
        __syncthreads();
        for (int i = threadIdx.x; i < 64 * V; i += 256) {
            const int col = blockIdx.x * 64 * V + i;
            if (col >= N) continue;
            const float s = (sums[0][i] + sums[1][i]) + (sums[2][i] + sums[3][i]);
            if (db) static_cast<T*>(db)[col] = (T)s;                // all rows in one chunk
            else part[chunk * N + col] = s;
        }
    }
}

// Rows of `cols` values, `ld` apart, laid out anew in whole 16-byte pieces with zeros behind them: a tile's copies go by such pieces.
template <typename T>
__global__ __launch_bounds__(256) void product_pack_kernel(const void* x, int64_t ld, int64_t rows, int cols, void* out) {
    constexpr int CE = 16 / sizeof(T);
    const int per_row = (cols + CE - 1) / CE;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * per_row; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / per_row;
        const int c = (int)(i - r * per_row) * CE;
        static_cast<uint4*>(out)[i] = unaligned_chunk(static_cast<const T*>(x) + r * ld + c, cols - c);
    }
}

constexpr int JOIN_WAVES = 16;
template <typename T>
__global__ __launch_bounds__(64 * JOIN_WAVES) void colsum_join_kernel(const float* part, int64_t chunks, int N, void* out) {
    __shared__ float sums[JOIN_WAVES][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = blockIdx.x * 64 + lane;
    float s = 0.f;
    if (n < N) {
#pragma unroll 4
        for (int64_t c = wave; c < chunks; c += JOIN_WAVES) s += part[c * N + n];
    }
    sums[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && n < N) {
        s = 0.f;
#pragma unroll
        for (int w = 0; w < JOIN_WAVES; ++w) s += sums[w][lane];
        static_cast<T*>(out)[n] = (T)s;
    }
}

// ------------------------------------------------------------------------------------------------------------- host
struct Plan { int tile; int splits; int64_t k_split; size_t part_bytes; };       // tile: 0 few rows, else its edge

// Few rows: the streaming kernel.  Else the largest tile that still gives most CUs one (256: one workgroup a CU, 200 of 256 CUs; 128 and
// 64: several a CU hide each other's waits).  Both sides of the borders (us a call, gelu and residual):
//   64 rows    bf16 x 1024 x 1024: 8 - 64 rows 9 here, 14 in tiles; x 6144 x 1536: 24 rows 9.9 / 13.3, 32 rows 11 / 13.6, 64 rows 17 / 13.8; fp32
//              x 4096 x 4096: 16 rows 22 / 26, 32 rows 30 / 27, 64 rows 49 / 29 -- above 32 rows the tiles win where w is large
//   tiles(128) bf16, K = 1024: 2304^2 (324) 25.5 in 128, 29.8 in 64; 2560^2 (400) 26 / 34; K = 4096: 1280^2 (100) 52 / 43, 1792^2 (196) 53 / 68, 2304^2
//              63 / 97, 2560^2 67 / 115; fp32: 2304^2 140 / 126, 2560^2 141 / 140, 2816^2 142 / 145 -- right for fp32, late for bf16
//   tiles(256) bf16, K = 1024: 3328^2 (169) 41 in 256, 44 in 128; 3840^2 (225) 44 / 51; 4352^2 (289: a second round) 81 / 67; fp32: 3328^2 264 / 220,
//              3584^2 (196) 267 / 280, 3840^2 268 / 282, 4352^2 524 / 360 -- the second round of a few tiles is not seen
// Tiles of 64 split the summed axis up to four workgroups a CU as long as each keeps 20
// steps of 128 bytes (8 where the tiles alone leave half of the card idle): 1024 x 1024 x 4096 bf16 26 us in one part, 23 in three; the join
// costs 5 us, so that 1037 x 1024 x 1024 takes 11 us in one part and 15 in two.
Plan plan_product(int64_t M, int N, int64_t K, int dt, bool acol, bool bcol) {
    Plan p{0, 1, K, 0};
    if (!acol && !bcol && M <= 64) return p;
    const int64_t ke = 128 / dtype_bytes(dt);                 // K step of the tiles
    auto tiles = [&](int64_t t) { return ((M + t - 1) / t) * ((N + t - 1) / t); };
    p.tile = tiles(256) >= 200 ? 256 : tiles(128) >= 400 ? 128 : 64;
    const int64_t steps = (K + ke - 1) / ke;
    p.k_split = steps * ke;
    if (p.tile == 64) {
        const int64_t n = tiles(64), most = steps / (n < 128 ? 8 : 20);
        int64_t want = 1024 / n;
        want = want < most ? want : most;
        if (want > 1) {
            const int64_t per = (steps + want - 1) / want;
            p.splits = (int)((steps + per - 1) / per);
            p.k_split = per * ke;
            if (p.splits > 1) p.part_bytes = (size_t)p.splits * (size_t)M * (size_t)N * 4;
        }
    }
    return p;
}

template <typename T, bool ACOL, bool BCOL, int EDGE>
void launch_tile(const ProductArgs& a, hipStream_t s) {
    const int n_tiles = a.tiles_m * a.tiles_n;
    const dim3 grid((unsigned)((n_tiles + 7) / 8 * 8), (unsigned)a.splits);
    // 256: 238 us for 8192 x 4096 x 4096 bf16 (the products alone) with steps of 128 bytes in two slots, 250 - 270 with 64 in four, 279 with four waves of 128 x 128;
    // 64: 26 us for 1024 x 1024 x 4096 with 64 in four, 34 with 128 in two
    constexpr int WN = EDGE == 256 ? 4 : 2, KB = EDGE == 64 ? 64 : 128, R = EDGE == 64 ? 4 : 2;
    hipLaunchKernelGGL((product_kernel<T, ACOL, BCOL, EDGE, EDGE, 2, WN, KB, R>), grid, dim3(128 * WN), 0, s, a);
}

template <typename T, int MT, int NWAVES>
void launch_few(const ProductArgs& a, bool aligned, hipStream_t s) {
    const dim3 grid((unsigned)((a.N + 15) / 16));
    if (aligned) hipLaunchKernelGGL((product_few_kernel<T, MT, NWAVES, true>), grid, dim3(64 * NWAVES), 0, s, a);
    else hipLaunchKernelGGL((product_few_kernel<T, MT, NWAVES, false>), grid, dim3(64 * NWAVES), 0, s, a);
}

inline bool on(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }
inline bool on16(const void* p) { return on(p, 16); }
constexpr int SLOPE_F32 = 0x100;             // ADX_SLOPE_F32

inline int whole(int64_t n, int dt) { const int V = 16 / dtype_bytes(dt); return (int)((n + V - 1) / V * V); }      // up to whole 16-byte pieces

void pack_rows(const void* x, int64_t ld, int64_t rows, int cols, int dt, void* out, hipStream_t s) {
    const int64_t n = rows * (whole(cols, dt) / (16 / dtype_bytes(dt))), blocks = (n + 255) / 256;
    with_dtype(dt, [&](auto t) { hipLaunchKernelGGL(product_pack_kernel<decltype(t)>, dim3((unsigned)(blocks < (1 << 22) ? blocks : 1 << 22)), dim3(256), 0, s, x, ld, rows, cols, out); });
}

// packed: row operands have zeros behind their K values up to whole pieces
hipError_t product(ProductArgs a, int dt, bool acol, bool bcol, bool packed, void* part, hipStream_t s) {
    const int V = 16 / dtype_bytes(dt);
    Plan p = plan_product(a.M, a.N, a.K, dt, acol, bcol);
    a.vec = a.N % V == 0 && a.ldy % V == 0 && on16(a.y) && on16(a.bias) && (!a.res || (on16(a.res) && a.ldr % V == 0)) && on(a.slope, V * (a.slope_f32 ? 4 : 2));
    // operands by 16-byte pieces: rows start on 16 bytes and whole pieces make up the contiguous axis
    const bool pieces = on16(a.A) && on16(a.B) && a.lda % V == 0 && a.ldb % V == 0 && (acol ? a.own_a % V == 0 : packed || a.K % V == 0) &&
                        (bcol ? a.own_b % V == 0 : packed || a.K % V == 0);
    const bool near = a.lda < (1 << 21) && a.ldb < (1 << 21);  // a tile's 256 rows span less than 2^31 bytes
    if (p.tile == 0) {
        with_dtype(dt, [&](auto t) {
            typedef decltype(t) T;
            if (a.M <= 16) launch_few<T, 1, 8>(a, pieces, s);
            else if (a.M <= 32) launch_few<T, 2, 8>(a, pieces, s);
            else launch_few<T, 4, 8>(a, pieces, s);
        });
        return hipGetLastError();
    }
    const bool any = !pieces || !near;
    if (any) p.tile = 64;
    a.splits = p.splits; a.k_split = p.k_split; a.part = static_cast<float*>(part);
    a.tiles_m = (int)((a.M + p.tile - 1) / p.tile); a.tiles_n = (a.N + p.tile - 1) / p.tile;
    if ((int64_t)a.tiles_m * a.tiles_n > (1 << 23) - 8) return hipErrorInvalidValue;           // 2^32 threads a launch
    with_dtype(dt, [&](auto t) {
        typedef decltype(t) T;
        auto by_tile = [&](auto ac, auto bc) {
            constexpr bool AC = decltype(ac)::value, BC = decltype(bc)::value;
            if (any) hipLaunchKernelGGL((product_any_kernel<T, AC, BC>), dim3((unsigned)(a.tiles_m * a.tiles_n), (unsigned)a.splits), dim3(256), 0, s, a);
            else if (p.tile == 256) launch_tile<T, AC, BC, 256>(a, s);
            else if (p.tile == 128) launch_tile<T, AC, BC, 128>(a, s);
            else launch_tile<T, AC, BC, 64>(a, s);
        };
        if (acol) by_tile(std::true_type{}, std::true_type{});
        else if (bcol) by_tile(std::false_type{}, std::true_type{});
        else by_tile(std::false_type{}, std::false_type{});
        if (a.splits > 1) {
            constexpr int JV = 16 / sizeof(T);
            const int64_t n = a.M * (a.vec ? a.N / JV : a.N);
            if (a.vec) hipLaunchKernelGGL((product_join_kernel<T, JV>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a);
            else hipLaunchKernelGGL((product_join_kernel<T, 1>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a);
        }
    });
    return hipGetLastError();
}

inline size_t up256(size_t v) { return (v + 255) / 256 * 256; }

// Operands whose rows are no whole number of 16-byte pieces are laid out anew (two more launches and passes over them) where the
// product is long: loads through registers take three times as long (bf16 3186 x 206 x 4651, forward and backward: 445 us against 149), but a
// short product is over before the launches would be.  Few rows are read where they lie.
inline bool worth_packing(int64_t M, int64_t N, int64_t K) { return (double)M * N * K >= (1 << 28); }

struct FwdWorkspace { size_t part, x, w, bytes; bool pack; };

FwdWorkspace fwd_workspace(int64_t M, int N, int64_t K, int dt) {
    FwdWorkspace f;
    const Plan p = plan_product(M, N, K, dt, false, false);
    const int Kp = whole(K, dt);
    f.pack = p.tile && Kp != K && worth_packing(M, N, K);
    size_t off = 0;
    f.part = off; off += up256(p.part_bytes);
    f.x = off; off += f.pack ? up256((size_t)M * Kp * dtype_bytes(dt)) : 0;
    f.w = off; off += f.pack ? up256((size_t)N * Kp * dtype_bytes(dt)) : 0;
    f.bytes = off;
    return f;
}

struct BwdWorkspace { size_t dz, sums, part, x, w, bytes; int64_t chunks; bool store_dz, pack; };

BwdWorkspace bwd_workspace(int64_t M, int N, int64_t K, int act, int dt) {
    BwdWorkspace w;
    const int Np = whole(N, dt), Kp = whole(K, dt);
    w.chunks = (M + SLOPE_ROWS - 1) / SLOPE_ROWS;
    w.store_dz = act != ACT_NONE || (Np != N && worth_packing(M, N, K));
    w.pack = Kp != K && worth_packing(M, N, K);
    size_t off = 0;
    w.dz = off; off += w.store_dz ? up256((size_t)M * Np * dtype_bytes(dt)) : 0;
    w.sums = off; off += up256((size_t)w.chunks * N * 4);
    const size_t pa = plan_product(M, (int)K, N, dt, false, true).part_bytes, pb = plan_product(N, (int)K, M, dt, true, true).part_bytes;
    w.part = off; off += up256(pa > pb ? pa : pb);
    w.x = off; off += w.pack ? up256((size_t)M * Kp * dtype_bytes(dt)) : 0;
    w.w = off; off += w.pack ? up256((size_t)N * Kp * dtype_bytes(dt)) : 0;
    w.bytes = off;
    return w;
}

// widths: 16 rows of w a workgroup of 512 threads, 2^32 threads a launch
bool shape_ok(int64_t M, int N, int K) { return M >= 0 && N > 0 && K > 0 && M <= (int64_t)1 << 30 && N <= 1 << 26 && K <= 1 << 26; }

}  // namespace
}  // namespace adx

using namespace adx;

#define ADX_API extern "C" __attribute__((visibility("default")))

ADX_API int adx_linear_residual_edge(int64_t M, int N, int K, int which, int dtype) {
    if (!shape_ok(M, N, K) || M == 0 || !dtype_ok(dtype)) return -1;
    if (which == 0) return plan_product(M, N, K, dtype, false, false).tile;
    if (which == 1) return plan_product(M, K, N, dtype, false, true).tile;
    return which == 2 ? plan_product(N, K, M, dtype, true, true).tile : -1;
}

ADX_API size_t adx_linear_residual_ws_bytes(int64_t M, int N, int K, int dtype) {
    if (!shape_ok(M, N, K) || !dtype_ok(dtype) || M == 0) return 0;
    return fwd_workspace(M, N, K, dtype).bytes;
}

ADX_API int adx_op_linear_residual(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* res, int64_t ldr, void* slope,
                                   void* y, int64_t ldy, int64_t M, int N, int K, int act, int dtype, void* workspace, size_t workspace_bytes,
                                   void* stream) {
    if (!dtype_ok(dtype)) { set_error("linear_residual: unknown element type"); return ADX_EINVAL; }
    const bool slope_f32 = (act & SLOPE_F32) || dtype == DT_F32;
    act &= ~SLOPE_F32;
    if (act < ACT_NONE || act > ACT_TANH_) { set_error("linear_residual: unknown activation"); return ADX_EINVAL; }
    if (!shape_ok(M, N, K)) { set_error("linear_residual: needs 0 <= M <= 2^30 and 0 < N, K <= 2^26"); return ADX_EINVAL; }
    if (M == 0) return ADX_OK;
    if (!x || !w || !y) { set_error("linear_residual: null pointer"); return ADX_EINVAL; }
    if (ldx < 0 || ldw < 0 || ldr < 0 || ldy < N) { set_error("linear_residual: negative row stride, or output rows that overlap"); return ADX_EINVAL; }
    const FwdWorkspace ws = fwd_workspace(M, N, K, dtype);
    if (ws.bytes && (!workspace || workspace_bytes < ws.bytes || !on16(workspace))) {
        set_error("linear_residual: needs a 16-byte aligned workspace of adx_linear_residual_ws_bytes bytes"); return ADX_EINVAL;
    }
    hipStream_t s = (hipStream_t)stream;
    unsigned char* base = static_cast<unsigned char*>(workspace);
    ProductArgs a{};
    a.A = x; a.lda = ldx; a.B = w; a.ldb = ldw; a.M = M; a.N = N; a.K = K; a.bias = bias; a.res = res; a.ldr = ldr; a.slope = slope; a.y = y; a.ldy = ldy;
    a.act = act; a.slope_f32 = slope_f32;
    if (ws.pack) {
        pack_rows(x, ldx, M, K, dtype, base + ws.x, s);
        pack_rows(w, ldw, N, K, dtype, base + ws.w, s);
        a.A = base + ws.x; a.B = base + ws.w; a.lda = a.ldb = whole(K, dtype);
    }
    const hipError_t e = product(a, dtype, false, false, ws.pack, base + ws.part, s);
    return e == hipSuccess ? ADX_OK : hip_fail(e, "linear_residual");
}

ADX_API size_t adx_linear_residual_bwd_ws_bytes(int64_t M, int N, int K, int act, int dtype) {
    if (!shape_ok(M, N, K) || !dtype_ok(dtype) || M == 0) return 0;
    return bwd_workspace(M, N, K, act & ~SLOPE_F32, dtype).bytes;
}

ADX_API int adx_op_linear_residual_bwd(const void* dy, int64_t ldd, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* slope, void* dx,
                                       void* dw, void* db, int64_t M, int N, int K, int act, int dtype, void* workspace, size_t workspace_bytes,
                                       void* stream) {
    if (!dtype_ok(dtype)) { set_error("linear_residual_bwd: unknown element type"); return ADX_EINVAL; }
    const bool slope_f32 = (act & SLOPE_F32) || dtype == DT_F32;
    act &= ~SLOPE_F32;
    if (act < ACT_NONE || act > ACT_TANH_) { set_error("linear_residual_bwd: unknown activation"); return ADX_EINVAL; }
    if (!shape_ok(M, N, K) || M == 0) { set_error("linear_residual_bwd: needs 1 <= M <= 2^30 and 0 < N, K <= 2^26"); return ADX_EINVAL; }
    if (!dy || (dx && !w) || (dw && !x) || (act != ACT_NONE && !slope)) { set_error("linear_residual_bwd: null pointer"); return ADX_EINVAL; }
    if (ldd < 0 || ldx < 0 || ldw < 0) { set_error("linear_residual_bwd: negative row stride"); return ADX_EINVAL; }
    const BwdWorkspace ws = bwd_workspace(M, N, K, act, dtype);
    if (!workspace || workspace_bytes < ws.bytes || !on16(workspace)) {
        set_error("linear_residual_bwd: needs a 16-byte aligned workspace of adx_linear_residual_bwd_ws_bytes bytes"); return ADX_EINVAL;
    }
    hipStream_t s = (hipStream_t)stream;
    unsigned char* base = static_cast<unsigned char*>(workspace);
    void* dz = base + ws.dz;
    float* sums = reinterpret_cast<float*>(base + ws.sums);
    const int V = 16 / dtype_bytes(dtype);
    const bool store = ws.store_dz && (dx || dw);
    const int Np = whole(N, dtype), Kp = whole(K, dtype);
    if (store || db) {
        const bool vec = N % V == 0 && ldd % V == 0 && on16(dy) && on(slope, V * (slope_f32 ? 4 : 2));
        with_dtype(dtype, [&](auto t) {
            typedef decltype(t) T;
            const int cols = vec ? 64 * V : 64, width = store ? Np : N;
            const dim3 grid((unsigned)((width + cols - 1) / cols), (unsigned)(ws.chunks < 65535 ? ws.chunks : 65535));
            void* to = store ? dz : nullptr;
            float* part = db ? sums : nullptr;
            void* whole_db = ws.chunks == 1 ? db : nullptr;
            auto by_slope = [&](auto kept) {
                typedef decltype(kept) S;
                if (vec) hipLaunchKernelGGL((slope_kernel<T, S, true>), grid, dim3(256), 0, s, dy, ldd, slope, to, Np, part, whole_db, M, N, act);
                else hipLaunchKernelGGL((slope_kernel<T, S, false>), grid, dim3(256), 0, s, dy, ldd, slope, to, Np, part, whole_db, M, N, act);
            };
            if (slope_f32) by_slope(float{});
            else by_slope(typename Code<T>::type{});
            if (db && ws.chunks > 1) hipLaunchKernelGGL(colsum_join_kernel<T>, dim3((unsigned)((N + 63) / 64)), dim3(64 * JOIN_WAVES), 0, s, sums, ws.chunks, N, db);
        });
    }
    const void* g = store ? dz : dy;
    const int64_t ldg = store ? Np : ldd;
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && dx) {
        ProductArgs a{};
        a.A = g; a.lda = ldg; a.B = w; a.ldb = ldw; a.own_b = K; a.M = M; a.N = K; a.K = N; a.y = dx; a.ldy = K;
        if (ws.pack) { pack_rows(w, ldw, N, K, dtype, base + ws.w, s); a.B = base + ws.w; a.ldb = a.own_b = Kp; }
        e = product(a, dtype, false, true, store, base + ws.part, s);
    }
    if (e == hipSuccess && dw) {
        ProductArgs a{};
        a.A = g; a.lda = ldg; a.own_a = store ? Np : N; a.B = x; a.ldb = ldx; a.own_b = K; a.M = N; a.N = K; a.K = M; a.y = dw; a.ldy = K;
        if (ws.pack) { pack_rows(x, ldx, M, K, dtype, base + ws.x, s); a.B = base + ws.x; a.ldb = a.own_b = Kp; }
        e = product(a, dtype, true, true, false, base + ws.part, s);
    }
    return e == hipSuccess ? ADX_OK : hip_fail(e, "linear_residual_bwd");
}
