// ude_gated.h -- matrix products of the gated feed-forward block (ude_gated.hip) on the matrix cores.
//
//   forward    h = act(x Wg^T) .* (x Wu^T)          two products of one operand, joined in the epilogue
//              y = h Wd^T
//   pullback   dh = dy Wd -> dg = dh u act'(g), du = dh act(g), h = act(g) u       (epilogue of the product)
//              dx = dg Wg + du Wu                    one product over the concatenated axis 2 F
//              dWg = dg^T x, dWu = du^T x, dWd = dy^T h
// Rows are samples (x: T x D row-major = the ABI's D x T column-major).  Every product is C[m, n] = sum_k A(m, k) B(n, k) with each
// operand stored either with consecutive k adjacent ("K") or with consecutive rows adjacent ("R"): that covers both weight orders.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/udecore.h"

namespace gated {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

struct F32 {
    typedef float E;
    static __device__ float to(float x) { return x; }
    static __device__ E from(float x) { return x; }
};
struct F16 {
    typedef short E;  // 16-bit patterns: loads, LDS and the matrix instructions do not look at them
    static __device__ float to(E x) { return (float)__builtin_bit_cast(_Float16, x); }
    static __device__ E from(float x) { return __builtin_bit_cast(E, (_Float16)x); }
    static __device__ f4 mfma(s8 a, s8 b, f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    }
};
struct BF16 {
    typedef short E;
    static __device__ float to(E x) { return __builtin_bit_cast(float, (unsigned)(unsigned short)x << 16); }
    static __device__ E from(float x) { return __builtin_bit_cast(E, (__bf16)x); }
    static __device__ f4 mfma(s8 a, s8 b, f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
    }
};

// act(g) and act'(g) in Float32
static __device__ inline float gate_act(int act, float g, float* slope) {
    switch (act) {
        case UDE_GATE_TANH: {
            const float t = tanhf(g);
            *slope = 1.f - t * t;
            return t;
        }
        case UDE_GATE_RBF: {
            const float e = expf(-g * g);
            *slope = -2.f * g * e;
            return e;
        }
        case UDE_GATE_RELU:
            *slope = g > 0.f ? 1.f : 0.f;
            return g > 0.f ? g : g * 0.f;  // (NaN stays NaN)
        case UDE_GATE_SIGMOID: {
            const float s = 1.f / (1.f + expf(-g));
            *slope = s * (1.f - s);
            return s;
        }
        case UDE_GATE_SWISH: {
            const float s = 1.f / (1.f + expf(-g));
            *slope = s * (1.f + g * (1.f - s));
            return g * s;
        }
        case UDE_GATE_GELU_TANH: {
            const float c = 0.7978845608028654f, q = 0.044715f;
            const float t = tanhf(c * (g + q * g * g * g));
            *slope = 0.5f * (1.f + t) + 0.5f * g * (1.f - t * t) * c * (1.f + 3.f * q * g * g);
            return 0.5f * g * (1.f + t);
        }
        case UDE_GATE_GELU_ERF: {
            const float p = 0.5f * (1.f + erff(g * 0.7071067811865476f));
            *slope = p + g * 0.3989422804014327f * expf(-0.5f * g * g);
            return g * p;
        }
        default:
            *slope = 1.f;
            return g;
    }
}

enum { EPI_STORE = 0, EPI_GATE = 1, EPI_PULL = 2 };

struct Args {
    const void* A[2];
    const void* B[2];
    void* C[2];
    int64_t lda, ldb[2], ldc[2];
    int M, N, K;
    int nseg;      // EPI_STORE: products summed into one output, C[0] = sum_s A[s] B[s]^T
    int act;
    int vecA, vecB;  // 16-byte loads allowed: base and leading dimension aligned
    float *gate, *up;        // EPI_GATE: stored if not NULL; EPI_PULL: read; leading dimension N
    void *dg, *du, *h;       // EPI_PULL: dg and du with leading dimension ldc[0], h with ldc[1]
};

// 8 consecutive elements along the stored axis of a tile; elements outside are zero
template <class E>
static __device__ inline void load8(const E* p, int64_t left, bool row, int vec, E* o) {
    if (row && vec && left >= 8) {
        typedef E V __attribute__((ext_vector_type(16 / sizeof(E))));
#pragma unroll
        for (int i = 0; i < (int)sizeof(E) / 2; ++i) {
            const V v = ((const V*)p)[i];
#pragma unroll
            for (int j = 0; j < (int)(16 / sizeof(E)); ++j) o[i * (16 / sizeof(E)) + j] = v[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = (row && i < left) ? p[i] : (E)0;
    }
}

// One 64 x 64 tile of C by four wavefronts, 32 x 32 each, K in steps of 32 through LDS, loads checked element by element where a row is
// not 16-byte aligned or a tile reaches over an edge: right for every size, stride and alignment.
// The operands of a matrix instruction are swapped (B first): a lane then holds four CONSECUTIVE n of one row m.
template <class T, int EPI, bool AK, bool BKc>
__global__ __launch_bounds__(256) void gemm_any(const Args a) {
    typedef typename T::E E;
    constexpr int BM = 64, BN = 64, KS = 32, LD = KS + 16 / (int)sizeof(E);
    __shared__ __attribute__((aligned(16))) E sA[BM * LD];
    __shared__ __attribute__((aligned(16))) E sB[BN * LD];
    const int tid = threadIdx.x, lane = tid & 63, wm = (tid >> 6) & 1, wn = tid >> 7;
    const int nm = (a.M + BM - 1) / BM;
    constexpr int NT = EPI == EPI_GATE ? BN / 2 : BN;  // output columns of a tile
    const int m0 = (int)(blockIdx.x % nm) * BM, n0 = (int)(blockIdx.x / nm) * NT;
    const int z = blockIdx.z;
    f4 acc[2][2] = {};
    for (int seg = 0; seg < a.nseg; ++seg) {
        const E* A = (const E*)a.A[a.nseg > 1 ? seg : z];
        const int bi = a.nseg > 1 ? seg : z;
        for (int k0 = 0; k0 < a.K; k0 += KS) {
            E va[8], vb[8];
            int ra, ka, rb, kb;
            if (AK) {
                ra = tid >> 2, ka = (tid & 3) * 8;
                load8(A + (int64_t)(m0 + ra) * a.lda + k0 + ka, a.K - k0 - ka, m0 + ra < a.M, a.vecA, va);
            } else {
                ka = tid >> 3, ra = (tid & 7) * 8;
                load8(A + (int64_t)(k0 + ka) * a.lda + m0 + ra, a.M - m0 - ra, k0 + ka < a.K, a.vecA, va);
            }
            // EPI_GATE: rows 0..31 of the tile come from Wg, 32..63 from Wu
            if (BKc) {
                rb = tid >> 2, kb = (tid & 3) * 8;
                const int half = EPI == EPI_GATE ? rb / NT : 0, n = n0 + rb - half * NT;
                load8((const E*)a.B[EPI == EPI_GATE ? half : bi] + (int64_t)n * a.ldb[EPI == EPI_GATE ? half : bi] + k0 + kb, a.K - k0 - kb, n < a.N, a.vecB, vb);
            } else {
                kb = tid >> 3, rb = (tid & 7) * 8;
                const int half = EPI == EPI_GATE ? rb / NT : 0, n = n0 + rb - half * NT;
                load8((const E*)a.B[EPI == EPI_GATE ? half : bi] + (int64_t)(k0 + kb) * a.ldb[EPI == EPI_GATE ? half : bi] + n, a.N - n, k0 + kb < a.K, a.vecB, vb);
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 8; ++i) sA[AK ? ra * LD + ka + i : (ra + i) * LD + ka] = va[i];
#pragma unroll
            for (int i = 0; i < 8; ++i) sB[BKc ? rb * LD + kb + i : (rb + i) * LD + kb] = vb[i];
            __syncthreads();
            const int r = lane & 15, g = lane >> 4;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const E* pa = sA + (wm * 32 + i * 16 + r) * LD;
                    const E* pb = sB + (EPI == EPI_GATE ? j * 32 + wn * 16 + r : wn * 32 + j * 16 + r) * LD;
                    if constexpr (sizeof(E) == 2) {
                        acc[i][j] = T::mfma(*(const s8*)(pb + g * 8), *(const s8*)(pa + g * 8), acc[i][j]);
                    } else {  // (a step of four k: the same k of both operands in every lane group, in any order)
#pragma unroll
                        for (int kk = 0; kk < KS; kk += 16) {
                            const f4 x = *(const f4*)(pb + kk + g * 4), w = *(const f4*)(pa + kk + g * 4);
#pragma unroll
                            for (int s = 0; s < 4; ++s) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[s], w[s], acc[i][j], 0, 0, 0);
                        }
                    }
                }
        }
    }
    const int r = lane & 15, g = lane >> 4;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int m = m0 + wm * 32 + i * 16 + r;
        if (m >= a.M) continue;
        if constexpr (EPI == EPI_GATE) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int n = n0 + wn * 16 + g * 4 + q;
                if (n >= a.N) continue;
                float slope;
                const float gv = acc[i][0][q], uv = acc[i][1][q];
                ((E*)a.C[0])[(int64_t)m * a.ldc[0] + n] = T::from(gate_act(a.act, gv, &slope) * uv);
                if (a.gate) {
                    a.gate[(int64_t)m * a.N + n] = gv;
                    a.up[(int64_t)m * a.N + n] = uv;
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int n = n0 + wn * 32 + j * 16 + g * 4 + q;
                    if (n >= a.N) continue;
                    const float c = acc[i][j][q];
                    if constexpr (EPI == EPI_STORE) {
                        ((E*)a.C[z])[(int64_t)m * a.ldc[z] + n] = T::from(c);
                    } else {
                        const int64_t at = (int64_t)m * a.N + n;
                        const float gv = a.gate[at], uv = a.up[at];
                        float slope;
                        const float av = gate_act(a.act, gv, &slope);
                        const int64_t to = (int64_t)m * a.ldc[0] + n;
                        ((E*)a.dg)[to] = T::from(c * uv * slope);
                        ((E*)a.du)[to] = T::from(c * av);
                        ((E*)a.h)[(int64_t)m * a.ldc[1] + n] = T::from(av * uv);
                    }
                }
        }
    }
}

}  // namespace gated
