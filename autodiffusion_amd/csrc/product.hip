// y = act(x w^T + bias) + residual on fp32, bf16 or fp16 tensors, and its gradients.  All three products of a training step are
//     C[i][j] = sum_k A(i, k) B(j, k)
// with either operand stored with k contiguous ("row": x and w of the forward) or with its own index contiguous ("column"): the
// data gradient dx[m][k] = sum_n dz[m][n] w[n][k] has a column B, the weight gradient dw[n][k] = sum_m dz[m][n] x[m][k] two column
// operands.  Sums are fp32; bias, activation and residual are applied to the fp32 sum and the result is rounded once.
#include "adx_ops.h"
#include "engine.h"
#include "typed.h"

#include <type_traits>

namespace adx {
namespace {

constexpr int ACT_TANH_ = 6;

__device__ __align__(16) unsigned char zero_chunk[16];            // what copies past the end of the summed axis read

// ------------------------------------------------------------------------------------------------------------- activations
template <int V> __device__ __forceinline__ void apply_act(float (&v)[V], int act) {
    switch (act) {                                                 // uniform: one branch for all values
        case ACT_RELU:
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = v[e] < 0.f ? 0.f : v[e];          // NaN stays
            break;
        case ACT_LEAKY:
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = v[e] > 0.f ? v[e] : 0.01f * v[e];
            break;
        case ACT_SILU:
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = v[e] / (1.f + expf(-v[e]));
            break;
        case ACT_TANH_:
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = tanhf(v[e]);
            break;
        case ACT_GELU_ERF:
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = 0.5f * v[e] * (1.f + erff(v[e] * 0.70710678118654752f));
            break;
        case ACT_GELU_TANH:
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = 0.5f * v[e] * (1.f + tanhf(0.79788456080286536f * (v[e] + 0.044715f * v[e] * v[e] * v[e])));
            break;
        default: break;
    }
}

__device__ __forceinline__ float act_slope(float z, int act) {
    switch (act) {
        case ACT_RELU: return z > 0.f ? 1.f : 0.f;
        case ACT_LEAKY: return z > 0.f ? 1.f : 0.01f;
        case ACT_SILU: { const float g = 1.f / (1.f + expf(-z)); return g * (1.f + z * (1.f - g)); }
        case ACT_TANH_: { const float t = tanhf(z); return 1.f - t * t; }
        case ACT_GELU_ERF: return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * 0.39894228040143268f * expf(-0.5f * z * z);
        case ACT_GELU_TANH: {
            const float t = tanhf(0.79788456080286536f * (z + 0.044715f * z * z * z));
            return 0.5f * (1.f + t) + 0.5f * z * (1.f - t * t) * 0.79788456080286536f * (1.f + 0.134145f * z * z);
        }
        default: return 1.f;
    }
}

// ------------------------------------------------------------------------------------------------------------- the problem
struct ProductArgs {
    const void* A; int64_t lda;              // element strides of the axis that is not contiguous
    const void* B; int64_t ldb;
    int64_t M; int N; int64_t K;             // C is M x N, K is summed
    const void* bias; const void* res; int64_t ldr;
    void* pre;                               // [M][N]: the value before the activation (for the gradient)
    void* y; int64_t ldy;
    int act;
    int splits; int64_t k_split;             // K range of one split (a multiple of the K step)
    float* part;                             // splits > 1: [splits][M][N] partial sums
    bool vec;                                // 16-byte epilogue
    int tiles_m, tiles_n;
};

// V consecutive columns of one row: bias, activation, residual, one rounding, store
template <typename T, int V>
__device__ __forceinline__ void finish(const ProductArgs& a, int64_t m, int n, float (&v)[V], bool vec) {
    T* y = static_cast<T*>(a.y) + m * a.ldy + n;
    const T* bias = static_cast<const T*>(a.bias);
    const T* res = static_cast<const T*>(a.res) + (a.res ? m * a.ldr + n : 0);
    T* pre = static_cast<T*>(a.pre) + (a.pre ? m * a.N + n : 0);
    typedef Pack<T, V> P;
    if (vec) {
        if (bias) {
            const P b = *reinterpret_cast<const P*>(bias + n);
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] += (float)b.v[e];
        }
        P o;
        if (a.pre) {
#pragma unroll
            for (int e = 0; e < V; ++e) o.v[e] = (T)v[e];
            *reinterpret_cast<P*>(pre) = o;
        }
        apply_act<V>(v, a.act);
        if (a.res) {
            const P r = *reinterpret_cast<const P*>(res);
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] += (float)r.v[e];
        }
#pragma unroll
        for (int e = 0; e < V; ++e) o.v[e] = (T)v[e];
        *reinterpret_cast<P*>(y) = o;
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if (n + e >= a.N) break;
            if (bias) v[e] += (float)bias[n + e];
            if (a.pre) pre[e] = (T)v[e];
        }
        apply_act<V>(v, a.act);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if (n + e >= a.N) break;
            if (a.res) v[e] += (float)res[e];
            y[e] = (T)v[e];
        }
    }
}

// ------------------------------------------------------------------------------------------------------------- large tiles
typedef const __attribute__((address_space(3))) void* lds_cptr;
typedef __attribute__((address_space(3))) void* lds_ptr;

// 64 x 16 bytes from per-lane global addresses to 1 KB of LDS.  Issued from inline assembly: the compiler would make every later LDS
// read wait for all copies it knows of; the kernel orders them itself with counted waits and barriers.
__device__ __forceinline__ void copy_1k(const void* g, unsigned lds_uniform) {
    unsigned keep;          // m0 is restored: the compiler does not expect inline assembly to change it
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "s"(lds_uniform), "v"(g) : "memory");
}
template <int N> __device__ __forceinline__ void wait_copies() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// One operand's part of a tile: ROWS of its own index x 128 bytes of k, in one of two LDS images.
//   row:    [ROWS][128 B]; 16-byte chunk c of row r sits at c ^ ((r >> 1) & 7): the fragment read (32 rows x one chunk) meets
//           every bank once
//   column: [KE][ROWS]; the 16-bit fragment read is the transposing LDS read (4 k-rows x 16 own indices a 16-lane group): 32-byte unit
//           u of k-row k sits at u ^ f(k) so that the k-rows of one read lie in different banks; fp32 reads 32 consecutive values
template <typename T, bool COL, int ROWS> struct Side {
    static constexpr int SZ = sizeof(T), CE = 16 / SZ, KE = 128 / SZ;
    static constexpr int BYTES = ROWS * 128, SLABS = BYTES / 1024, RB = ROWS * SZ;
    static __device__ __forceinline__ int unit_swizzle(int k) {
        if constexpr (SZ == 2) { constexpr int mask = RB / 32 - 1; return (((k & 3) | (((k >> 3) & 1) << 2)) & mask) << 5; }
        else return ((k >> 2) & 1) << 7;
    }
    // own index and first k (relative to the tile) of the 16 bytes that lane `lane` copies to slab `slab`
    static __device__ __forceinline__ void source(int slab, int lane, int& row, int& k) {
        if constexpr (!COL) {
            row = slab * 8 + (lane >> 3);
            k = ((lane & 7) ^ ((row >> 1) & 7)) * CE;
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
            return *reinterpret_cast<const uint4*>(img + r * 128 + ((c ^ ((r >> 1) & 7)) << 4));
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

// Workgroup tile BM x BN, WM x WN waves, a K step of 128 bytes a row, two LDS slots.  DMA: copies from global memory straight to
// LDS (operands whose rows start on 16 bytes); otherwise element loads through registers into the same images.
template <typename T, bool ACOL, bool BCOL, int BM, int BN, int WM, int WN, bool DMA>
__global__ __launch_bounds__(64 * WM * WN) void product_kernel(const ProductArgs a) {
    typedef Side<T, ACOL, BM> SA;
    typedef Side<T, BCOL, BN> SB;
    constexpr int W = WM * WN, KE = SA::KE, CE = SA::CE, SZ = sizeof(T);
    constexpr int FI = BM / WM / 32, FJ = BN / WN / 32, NW = BN / WN;
    constexpr int SLOT = SA::BYTES + SB::BYTES, PA = SA::SLABS / W, PB = SB::SLABS / W;
    constexpr int EP_LD = NW + 4;
    static_assert(SA::SLABS % W == 0 && SB::SLABS % W == 0, "slabs spread evenly over the waves");
    static_assert(W * 32 * EP_LD * 4 <= 2 * SLOT, "the epilogue's patches fit the slots");
    __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * SLOT];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // XCD x (blockIdx % 8) walks a contiguous range of an order of column panels eight tiles wide, so that the workgroups that
    // run on an XCD at one time share rows and columns in its L2
    const int n_tiles = a.tiles_m * a.tiles_n, per_xcd = (n_tiles + 7) / 8;
    const int lin = (int)(blockIdx.x & 7) * per_xcd + (int)(blockIdx.x >> 3);
    if (lin >= n_tiles) return;
    const int panel = lin / (a.tiles_m * 8), width = min(8, a.tiles_n - panel * 8), in = lin - panel * a.tiles_m * 8;
    const int64_t m0 = (int64_t)(in / width) * BM;
    const int n0 = (panel * 8 + in % width) * BN;
    const int64_t k_lo = (int64_t)blockIdx.y * a.k_split, k_hi = k_lo + a.k_split < a.K ? k_lo + a.k_split : a.K;
    const int nk = (int)((k_hi - k_lo + KE - 1) / KE);
    const int wm = wave / WN, wn = wave % WN;

    const unsigned lds0 = (unsigned)(uintptr_t)(lds_ptr)smem;
    const unsigned char *pa[PA], *pb[PB];                     // this lane's source of its slabs, K step 0
    int ka[PA], kb[PB];                                        // its k relative to the step
    int64_t ra[PA], rb[PB];
#pragma unroll
    for (int i = 0; i < PA; ++i) {
        int row;
        SA::source(wave + i * W, lane, row, ka[i]);
        ra[i] = m0 + row;
        // a row image repeats its last row past the end (those results are not stored); a column image has chunks past the end,
        // which are not read
        if constexpr (!ACOL) { if (ra[i] > a.M - 1) ra[i] = a.M - 1; }
        pa[i] = static_cast<const unsigned char*>(a.A) + (ACOL ? (k_lo + ka[i]) * a.lda + ra[i] : ra[i] * a.lda + k_lo + ka[i]) * SZ;
        if (ACOL && ra[i] >= a.M) ka[i] = 1 << 30;
    }
#pragma unroll
    for (int i = 0; i < PB; ++i) {
        int row;
        SB::source(wave + i * W, lane, row, kb[i]);
        rb[i] = n0 + row;
        if constexpr (!BCOL) { if (rb[i] > a.N - 1) rb[i] = a.N - 1; }
        pb[i] = static_cast<const unsigned char*>(a.B) + (BCOL ? (k_lo + kb[i]) * a.ldb + rb[i] : rb[i] * a.ldb + k_lo + kb[i]) * SZ;
        if (BCOL && rb[i] >= a.N) kb[i] = 1 << 30;
    }
    const int64_t step_a = (ACOL ? a.lda * KE : KE) * SZ, step_b = (BCOL ? a.ldb * KE : KE) * SZ;
    auto issue = [&](int kt) {                                 // K step kt -> slot kt & 1; what lies past the end is zero
        const unsigned slot = (unsigned)(kt & 1) * SLOT;
        const int left = (int)(k_hi - k_lo < (int64_t)(kt + 1) * KE ? k_hi - k_lo - (int64_t)kt * KE : KE);      // valid k of this step (<= 0 past the end)
        if constexpr (DMA) {
#pragma unroll
            for (int i = 0; i < PA; ++i) {
                copy_1k(ka[i] < left ? pa[i] : zero_chunk, lds0 + slot + (unsigned)(wave + i * W) * 1024u);
                pa[i] += step_a;
            }
#pragma unroll
            for (int i = 0; i < PB; ++i) {
                copy_1k(kb[i] < left ? pb[i] : zero_chunk, lds0 + slot + SA::BYTES + (unsigned)(wave + i * W) * 1024u);
                pb[i] += step_b;
            }
        } else {
            auto gather = [&](const unsigned char* p, int k, int64_t own, int64_t own_end, bool col, unsigned at) {
                T v[CE];
#pragma unroll
                for (int e = 0; e < CE; ++e) {
                    const bool ok = col ? (k < left && own + e < own_end) : (k + e < left);
                    v[e] = ok ? reinterpret_cast<const T*>(p)[e] : (T)0.f;
                }
                *reinterpret_cast<Pack<T, CE>*>(smem + at + lane * 16) = *reinterpret_cast<Pack<T, CE>*>(v);
            };
#pragma unroll
            for (int i = 0; i < PA; ++i) { gather(pa[i], ka[i], ra[i], a.M, ACOL, slot + (wave + i * W) * 1024); pa[i] += step_a; }
#pragma unroll
            for (int i = 0; i < PB; ++i) { gather(pb[i], kb[i], rb[i], a.N, BCOL, slot + SA::BYTES + (wave + i * W) * 1024); pb[i] += step_b; }
        }
    };

    f32x16_t acc[FI][FJ];
#pragma unroll
    for (int i = 0; i < FI; ++i)
#pragma unroll
        for (int j = 0; j < FJ; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.f;

    issue(0);
    issue(1);
    for (int kt = 0; kt < nk; ++kt) {
        wait_copies<PA + PB>();                                // this wave's copies of step kt have landed ...
        if constexpr (!DMA) wait_lds();
        barrier();                                             // ... and everybody's
        const unsigned char* img = smem + (kt & 1) * SLOT;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            uint4 fa[FI], fb[FJ];
#pragma unroll
            for (int j = 0; j < FJ; ++j) fb[j] = SB::fragment(img + SA::BYTES, wn * NW + j * 32, kk, lane);
#pragma unroll
            for (int i = 0; i < FI; ++i) fa[i] = SA::fragment(img, wm * (BM / WM) + i * 32, kk, lane);
#pragma unroll
            for (int i = 0; i < FI; ++i)
#pragma unroll
                for (int j = 0; j < FJ; ++j) acc[i][j] = mfma32<T>(fb[j], fa[i], acc[i][j]);      // rows of the result: n; columns: m
        }
        wait_lds();
        barrier();                                             // nobody reads the slot any more
        issue(kt + 2);
    }
    wait_copies<0>();
    if constexpr (!DMA) wait_lds();
    barrier();

    // Epilogue: 32 rows x NW columns at a time through LDS, so that a row's columns are stored as whole lines.  Result layout of the
    // 32x32 product: column = lane & 31, row = (q & 3) + 8 (q >> 2) + 4 (lane >> 5).
    constexpr int V = 16 / SZ, LPR = NW / V, RPI = 64 / LPR;   // lanes of a row, rows of one pass
    float* patch = reinterpret_cast<float*>(smem) + wave * 32 * EP_LD;
    const int n = n0 + wn * NW + (lane % LPR) * V;
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
#pragma unroll 1
        for (int p = 0; p < 32 / RPI; ++p) {
            const int r = p * RPI + lane / LPR;
            const int64_t m = m0 + wm * (BM / WM) + i * 32 + r;
            float v[V];
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                const float4 f = *reinterpret_cast<const float4*>(patch + r * EP_LD + (lane % LPR) * V + e);
                v[e] = f.x; v[e + 1] = f.y; v[e + 2] = f.z; v[e + 3] = f.w;
            }
            if (m < a.M && n < a.N) {
                if (a.splits > 1) {
                    float* o = a.part + ((int64_t)blockIdx.y * a.M + m) * a.N + n;
                    if (a.vec) {
#pragma unroll
                        for (int e = 0; e < V; e += 4) *reinterpret_cast<float4*>(o + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
                    } else {
#pragma unroll
                        for (int e = 0; e < V; ++e) if (n + e < a.N) o[e] = v[e];
                    }
                } else finish<T, V>(a, m, n, v, a.vec);
            }
        }
        wait_lds();
    }
}

// the partial sums of a split product, added in split order, and the epilogue
template <typename T>
__global__ __launch_bounds__(256) void product_join_kernel(const ProductArgs a) {
    constexpr int V = 16 / sizeof(T);
    const int per_row = (a.N + V - 1) / V;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= a.M * per_row) return;
    const int64_t m = i / per_row;
    const int n = (int)(i - m * per_row) * V;
    float v[V];
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = 0.f;
    for (int s = 0; s < a.splits; ++s) {
        const float* p = a.part + ((int64_t)s * a.M + m) * a.N + n;
        if (a.vec) {
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                const float4 f = *reinterpret_cast<const float4*>(p + e);
                v[e] += f.x; v[e + 1] += f.y; v[e + 2] += f.z; v[e + 3] += f.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) if (n + e < a.N) v[e] += p[e];
        }
    }
    finish<T, V>(a, m, n, v, a.vec);
}

// ------------------------------------------------------------------------------------------------------------- few rows
// M <= 64: the weights are read once and everything else is small, so nothing is staged.  A workgroup owns 16 NT rows of w; its
// waves take 128-byte pieces of K in turn, load fragments of both operands from global memory into registers (16 rows x 16 bytes a
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
    constexpr int CE = 16 / sizeof(T);
    if constexpr (ALIGNED) return k < K ? *reinterpret_cast<const uint4*>(row + k) : make_uint4(0u, 0u, 0u, 0u);
    else {
        union { T v[CE]; uint4 u; } f;
        f.u = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int e = 0; e < CE; ++e) if (k + e < K) f.v[e] = row[k + e];
        return f.u;
    }
}

template <typename T, int MT, int NT, int NWAVES, bool ALIGNED>
__global__ __launch_bounds__(64 * NWAVES) void product_few_kernel(const ProductArgs a) {
    constexpr int CE = 16 / sizeof(T), UNIT = 8 * CE;
    __shared__ float sums[NWAVES][MT * NT][64][4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n0 = blockIdx.x * 16 * NT, r16 = lane & 15, g = lane >> 4;
    const T *w[NT], *x[MT];
    bool live[MT];
#pragma unroll
    for (int t = 0; t < NT; ++t) w[t] = static_cast<const T*>(a.B) + (int64_t)min(n0 + t * 16 + r16, a.N - 1) * a.ldb + g * CE;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        live[t] = t * 16 + r16 < a.M;
        x[t] = static_cast<const T*>(a.A) + (int64_t)(live[t] ? t * 16 + r16 : 0) * a.lda + g * CE;
    }
    f32x4_t acc[NT][MT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    const int64_t K = a.K - g * CE;
    constexpr int U = MT * NT >= 4 ? 2 : 4;                        // pieces in flight a wave
    for (int64_t k = (int64_t)wave * UNIT; k < a.K; k += (int64_t)U * NWAVES * UNIT) {
        uint4 fw[2 * U][NT], fx[2 * U][MT];
#pragma unroll
        for (int h = 0; h < 2 * U; ++h) {
            const int64_t kh = k + (int64_t)(h >> 1) * NWAVES * UNIT + (h & 1) * 4 * CE;
#pragma unroll
            for (int t = 0; t < NT; ++t) fw[h][t] = row_chunk<T, ALIGNED>(w[t], kh, K);
#pragma unroll
            for (int t = 0; t < MT; ++t) fx[h][t] = live[t] ? row_chunk<T, ALIGNED>(x[t], kh, K) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int h = 0; h < 2 * U; ++h)
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < MT; ++j) acc[i][j] = mfma16<T>(fw[h][i], fx[h][j], acc[i][j]);
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) *reinterpret_cast<f32x4_t*>(sums[wave][i * MT + j][lane]) = acc[i][j];
    __syncthreads();
    // result layout of the 16x16 product: column (m) = lane & 15, row (n) = 4 (lane >> 4) + reg
    for (int i = tid; i < MT * NT * 256; i += 64 * NWAVES) {
        const int nn = i % (16 * NT), m = i / (16 * NT), n = n0 + nn;
        if (m >= a.M || n >= a.N) continue;
        const int t = (nn >> 4) * MT + (m >> 4), l = ((nn & 15) >> 2) * 16 + (m & 15), q = nn & 3;
        float v[1] = {0.f};
#pragma unroll
        for (int s = 0; s < NWAVES; ++s) v[0] += sums[s][t][l][q];
        finish<T, 1>(a, m, n, v, true);
    }
}

// ------------------------------------------------------------------------------------------------------------- gradient of the epilogue
// dz = dy act'(z), rounded to the operand type of the products that follow, and per chunk of rows the fp32 column sums of the
// unrounded dz (joined in chunk order: no atomics).
constexpr int SLOPE_ROWS = 64;

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void slope_kernel(const void* dy_, int64_t ldd, const void* pre_, void* dz_, float* part, int64_t M, int N, int act) {
    constexpr int V = VEC ? 16 / sizeof(T) : 1;
    __shared__ float sums[4][64 * V];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = (blockIdx.x * 64 + lane) * V;
    const int64_t r0 = (int64_t)blockIdx.y * SLOPE_ROWS, r1 = r0 + SLOPE_ROWS < M ? r0 + SLOPE_ROWS : M;
    typedef Pack<T, V> P;
    float sum[V];
#pragma unroll
    for (int e = 0; e < V; ++e) sum[e] = 0.f;
    if (n < N) {
        for (int64_t m = r0 + wave; m < r1; m += 4) {
            const P d = *reinterpret_cast<const P*>(static_cast<const T*>(dy_) + m * ldd + n);
            P o;
            if (act != ACT_NONE) {
                const P z = *reinterpret_cast<const P*>(static_cast<const T*>(pre_) + m * N + n);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float g = (float)d.v[e] * act_slope((float)z.v[e], act);
                    sum[e] += g;
                    o.v[e] = (T)g;
                }
                *reinterpret_cast<P*>(static_cast<T*>(dz_) + m * N + n) = o;
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) sum[e] += (float)d.v[e];
            }
        }
    }
    if (!part) return;
#pragma unroll
    for (int e = 0; e < V; ++e) sums[wave][lane * V + e] = sum[e];
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * V; i += 256) {
        const int col = blockIdx.x * 64 * V + i;
        if (col < N) part[(int64_t)blockIdx.y * N + col] = (sums[0][i] + sums[1][i]) + (sums[2][i] + sums[3][i]);
    }
}

template <typename T>
__global__ __launch_bounds__(256) void colsum_join_kernel(const float* part, int64_t chunks, int N, void* out) {
    __shared__ float sums[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = blockIdx.x * 64 + lane;
    float s = 0.f;
    if (n < N)
        for (int64_t c = wave; c < chunks; c += 4) s += part[c * N + n];
    sums[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && n < N) static_cast<T*>(out)[n] = (T)((sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]));
}

// ------------------------------------------------------------------------------------------------------------- host
struct Plan { int tile; int splits; int64_t k_split; size_t part_bytes; };       // tile: 0 few rows, else its edge

Plan plan_product(int64_t M, int N, int64_t K, int dt, bool acol, bool bcol) {
    Plan p{0, 1, K, 0};
    if (!acol && !bcol && M <= 64) return p;
    const int64_t ke = 128 / dtype_bytes(dt);
    auto tiles = [&](int64_t t) { return ((M + t - 1) / t) * ((N + t - 1) / t); };
    p.tile = (dt != DT_F32 && tiles(256) >= 200) ? 256 : tiles(128) >= 200 ? 128 : 64;
    const int64_t steps = (K + ke - 1) / ke;
    p.k_split = steps * ke;
    if (p.tile == 64 && tiles(64) < 256) {
        int64_t want = 512 / tiles(64);
        const int64_t most = steps / 8;
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
void launch_tile(const ProductArgs& a, bool dma, hipStream_t s) {
    constexpr int WM = 2, WN = EDGE == 256 ? 4 : 2;
    const int n_tiles = a.tiles_m * a.tiles_n;
    const dim3 grid((unsigned)((n_tiles + 7) / 8 * 8), (unsigned)a.splits);
    if (dma) hipLaunchKernelGGL((product_kernel<T, ACOL, BCOL, EDGE, EDGE, WM, WN, true>), grid, dim3(64 * WM * WN), 0, s, a);
    else if constexpr (EDGE == 64) hipLaunchKernelGGL((product_kernel<T, ACOL, BCOL, EDGE, EDGE, WM, WN, false>), grid, dim3(64 * WM * WN), 0, s, a);
}

template <typename T, int MT, int NT, int NWAVES>
void launch_few(const ProductArgs& a, bool aligned, hipStream_t s) {
    const dim3 grid((unsigned)((a.N + 16 * NT - 1) / (16 * NT)));
    if (aligned) hipLaunchKernelGGL((product_few_kernel<T, MT, NT, NWAVES, true>), grid, dim3(64 * NWAVES), 0, s, a);
    else hipLaunchKernelGGL((product_few_kernel<T, MT, NT, NWAVES, false>), grid, dim3(64 * NWAVES), 0, s, a);
}

inline bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

hipError_t product(ProductArgs a, int dt, bool acol, bool bcol, void* part, hipStream_t s) {
    const int V = 16 / dtype_bytes(dt);
    Plan p = plan_product(a.M, a.N, a.K, dt, acol, bcol);
    a.vec = a.N % V == 0 && a.ldy % V == 0 && on16(a.y) && on16(a.bias) && (!a.res || (on16(a.res) && a.ldr % V == 0)) && on16(a.pre);
    // operands by 16-byte pieces: rows start on 16 bytes and whole pieces make up the contiguous axis
    const bool pieces = on16(a.A) && on16(a.B) && a.lda % V == 0 && a.ldb % V == 0 && (acol ? a.M : a.K) % V == 0 && (bcol ? a.N : a.K) % V == 0;
    if (p.tile == 0) {
        with_dtype(dt, [&](auto t) {
            typedef decltype(t) T;
            if (a.M <= 16) launch_few<T, 1, 1, 8>(a, pieces, s);
            else if (a.M <= 32) launch_few<T, 2, 1, 8>(a, pieces, s);
            else launch_few<T, 4, 1, 8>(a, pieces, s);
        });
        return hipGetLastError();
    }
    if (!pieces && p.tile != 64) p.tile = 64;                  // operands that need element loads: the small tile, as many splits as planned (none)
    a.splits = p.splits; a.k_split = p.k_split; a.part = static_cast<float*>(part);
    a.tiles_m = (int)((a.M + p.tile - 1) / p.tile); a.tiles_n = (a.N + p.tile - 1) / p.tile;
    if ((int64_t)a.tiles_m * a.tiles_n > 0x3FFFFFFF) return hipErrorInvalidValue;
    with_dtype(dt, [&](auto t) {
        typedef decltype(t) T;
        auto by_tile = [&](auto ac, auto bc) {
            constexpr bool AC = decltype(ac)::value, BC = decltype(bc)::value;
            if (p.tile == 256) { if constexpr (sizeof(T) == 2) launch_tile<T, AC, BC, 256>(a, pieces, s); }
            else if (p.tile == 128) launch_tile<T, AC, BC, 128>(a, pieces, s);
            else launch_tile<T, AC, BC, 64>(a, pieces, s);
        };
        if (acol) by_tile(std::true_type{}, std::true_type{});
        else if (bcol) by_tile(std::false_type{}, std::true_type{});
        else by_tile(std::false_type{}, std::false_type{});
        if (a.splits > 1) {
            const int64_t n = a.M * ((a.N + V - 1) / V);
            hipLaunchKernelGGL(product_join_kernel<T>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a);
        }
    });
    return hipGetLastError();
}

inline size_t up256(size_t v) { return (v + 255) / 256 * 256; }

struct BwdWorkspace { size_t dz, sums, part, bytes; int64_t chunks; };

BwdWorkspace bwd_workspace(int64_t M, int N, int64_t K, int act, int dt) {
    BwdWorkspace w;
    w.chunks = (M + SLOPE_ROWS - 1) / SLOPE_ROWS;
    size_t off = 0;
    w.dz = off; off += act != ACT_NONE ? up256((size_t)M * N * dtype_bytes(dt)) : 0;
    w.sums = off; off += up256((size_t)w.chunks * N * 4);
    const size_t pa = plan_product(M, (int)K, N, dt, false, true).part_bytes, pb = plan_product(N, (int)K, M, dt, true, true).part_bytes;
    w.part = off; off += up256(pa > pb ? pa : pb);
    w.bytes = off;
    return w;
}

bool shape_ok(int64_t M, int N, int K) { return M >= 0 && N > 0 && K > 0 && M <= (int64_t)1 << 30; }

}  // namespace
}  // namespace adx

using namespace adx;

#define ADX_API extern "C" __attribute__((visibility("default")))

ADX_API size_t adx_linear_residual_ws_bytes(int64_t M, int N, int K, int dtype) {
    if (!shape_ok(M, N, K) || !dtype_ok(dtype) || M == 0) return 0;
    return plan_product(M, N, K, dtype, false, false).part_bytes;
}

ADX_API int adx_op_linear_residual(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* res, int64_t ldr, void* pre,
                                   void* y, int64_t ldy, int64_t M, int N, int K, int act, int dtype, void* workspace, size_t workspace_bytes,
                                   void* stream) {
    if (!dtype_ok(dtype)) { set_error("linear_residual: unknown element type"); return ADX_EINVAL; }
    if (act < ACT_NONE || act > ACT_TANH_) { set_error("linear_residual: unknown activation"); return ADX_EINVAL; }
    if (!shape_ok(M, N, K)) { set_error("linear_residual: needs 0 <= M <= 2^30 and positive N, K"); return ADX_EINVAL; }
    if (M == 0) return ADX_OK;
    if (!x || !w || !y) { set_error("linear_residual: null pointer"); return ADX_EINVAL; }
    if (ldx < 0 || ldw < 0 || ldr < 0 || ldy < N) { set_error("linear_residual: negative row stride, or output rows that overlap"); return ADX_EINVAL; }
    const size_t need = plan_product(M, N, K, dtype, false, false).part_bytes;
    if (need && (!workspace || workspace_bytes < need || !on16(workspace))) {
        set_error("linear_residual: needs a 16-byte aligned workspace of adx_linear_residual_ws_bytes bytes"); return ADX_EINVAL;
    }
    ProductArgs a{};
    a.A = x; a.lda = ldx; a.B = w; a.ldb = ldw; a.M = M; a.N = N; a.K = K; a.bias = bias; a.res = res; a.ldr = ldr; a.pre = pre; a.y = y; a.ldy = ldy;
    a.act = act;
    const hipError_t e = product(a, dtype, false, false, workspace, (hipStream_t)stream);
    return e == hipSuccess ? ADX_OK : hip_fail(e, "linear_residual");
}

ADX_API size_t adx_linear_residual_bwd_ws_bytes(int64_t M, int N, int K, int act, int dtype) {
    if (!shape_ok(M, N, K) || !dtype_ok(dtype) || M == 0) return 0;
    return bwd_workspace(M, N, K, act, dtype).bytes;
}

ADX_API int adx_op_linear_residual_bwd(const void* dy, int64_t ldd, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* pre, void* dx,
                                       void* dw, void* db, int64_t M, int N, int K, int act, int dtype, void* workspace, size_t workspace_bytes,
                                       void* stream) {
    if (!dtype_ok(dtype)) { set_error("linear_residual_bwd: unknown element type"); return ADX_EINVAL; }
    if (act < ACT_NONE || act > ACT_TANH_) { set_error("linear_residual_bwd: unknown activation"); return ADX_EINVAL; }
    if (!shape_ok(M, N, K) || M == 0) { set_error("linear_residual_bwd: needs 1 <= M <= 2^30 and positive N, K"); return ADX_EINVAL; }
    if (!dy || (dx && !w) || (dw && !x) || (act != ACT_NONE && !pre)) { set_error("linear_residual_bwd: null pointer"); return ADX_EINVAL; }
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
    if (act != ACT_NONE || db) {
        if (ws.chunks > 65535) { set_error("linear_residual_bwd: more than 4 million rows"); return ADX_EINVAL; }
        const bool vec = N % V == 0 && ldd % V == 0 && on16(dy) && on16(pre);
        with_dtype(dtype, [&](auto t) {
            typedef decltype(t) T;
            const int cols = vec ? 64 * V : 64;
            const dim3 grid((unsigned)((N + cols - 1) / cols), (unsigned)ws.chunks);
            if (vec) hipLaunchKernelGGL((slope_kernel<T, true>), grid, dim3(256), 0, s, dy, ldd, pre, dz, db ? sums : nullptr, M, N, act);
            else hipLaunchKernelGGL((slope_kernel<T, false>), grid, dim3(256), 0, s, dy, ldd, pre, dz, db ? sums : nullptr, M, N, act);
            if (db) hipLaunchKernelGGL(colsum_join_kernel<T>, dim3((unsigned)((N + 63) / 64)), dim3(256), 0, s, sums, ws.chunks, N, db);
        });
    }
    const void* g = act != ACT_NONE ? dz : dy;
    const int64_t ldg = act != ACT_NONE ? N : ldd;
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && dx) {
        ProductArgs a{};
        a.A = g; a.lda = ldg; a.B = w; a.ldb = ldw; a.M = M; a.N = K; a.K = N; a.y = dx; a.ldy = K;
        e = product(a, dtype, false, true, base + ws.part, s);
    }
    if (e == hipSuccess && dw) {
        ProductArgs a{};
        a.A = g; a.lda = ldg; a.B = x; a.ldb = ldx; a.M = N; a.N = K; a.K = M; a.y = dw; a.ldy = K;
        e = product(a, dtype, true, true, base + ws.part, s);
    }
    return e == hipSuccess ? ADX_OK : hip_fail(e, "linear_residual_bwd");
}
