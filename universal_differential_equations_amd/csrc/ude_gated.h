// ude_gated.h -- matrix products of the gated feed-forward block (ude_gated.hip) on the matrix cores.
//
//   forward    h = act(x Wg^T) .* (x Wu^T)          two products of one operand, joined in the epilogue
//              y = h Wd^T
//   pullback   dh = dy Wd -> dg = dh u act'(g), du = dh act(g), h = act(g) u       (epilogue of the product)
//              dx = dg Wg + du Wu                    one product over the concatenated axis 2 F
//              dWg = dg^T x, dWu = du^T x, dWd = dy^T h
// Rows are samples (x: T x D row-major = the ABI's D x T column-major).  Every product is C[m, n] = sum_k A(m, k) B(n, k) with each
// operand stored either with consecutive k adjacent ("K") or with consecutive rows adjacent ("R"): that covers both weight orders.
// h, dg and du are rounded to the block's type, because an operand of a 16-bit matrix instruction has 16 bits: the error of y against Float64 is
// sqrt 2 of one rounding's (0.0024 of its norm in BFloat16, 0.00029 in Float16, against 0.0017 and 0.0002 with h in Float32).  h as the sum of two 16-bit
// values would take that back for twice the instructions of every product that it enters: a third more for the forward call, five sixths (with dg and du) for the pullback.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

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
    // 16 k: four steps of four.  Which k a lane group feeds does not matter where both operands do the same.
    static __device__ f4 mfma(s8 a, s8 b, f4 c) {
        const f4 x = __builtin_bit_cast(f4, a), y = __builtin_bit_cast(f4, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], y[i], c, 0, 0, 0);
        return c;
    }
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

// act(g) and act'(g) in Float32.  QUICK (16-bit kinds): the hardware's exponential and reciprocal, a few 2^-22 of the value off, far below
// the rounding of the result; Float32 calls the accurate functions.  Sums that would cancel are written as what they are equal to:
// (1 + tanh z) / 2 = sigmoid(2 z), (1 + erf z) / 2 = erfc(-z) / 2.
template <bool QUICK>
static __device__ inline float sigmoid(float x) {
    return QUICK ? __builtin_amdgcn_rcpf(1.f + __expf(-x)) : 1.f / (1.f + expf(-x));
}
template <bool QUICK, int ACT>
static __device__ inline float gate_act(float g, float* slope) {
    if constexpr (ACT == UDE_GATE_TANH) {
        const float t = tanhf(g);
        *slope = 1.f - t * t;
        return t;
    } else if constexpr (ACT == UDE_GATE_RBF) {
        const float e = QUICK ? __expf(-g * g) : expf(-g * g);
        *slope = -2.f * g * e;
        return e;
    } else if constexpr (ACT == UDE_GATE_RELU) {
        *slope = g > 0.f ? 1.f : 0.f;
        return g > 0.f ? g : g == g ? 0.f : g;  // (NaN stays NaN)
    } else if constexpr (ACT == UDE_GATE_SIGMOID) {
        const float s = sigmoid<QUICK>(g);
        *slope = s * (1.f - s);
        return s;
    } else if constexpr (ACT == UDE_GATE_SWISH) {
        const float s = sigmoid<QUICK>(g);
        *slope = s * (1.f + g * (1.f - s));
        return g * s;
    } else if constexpr (ACT == UDE_GATE_GELU_TANH) {
        const float c = 1.5957691216057308f, q = 0.044715f;  // 2 sqrt(2 / pi)
        const float x = fabsf(g) > 100.f ? copysignf(100.f, g) : g;  // (s is 0 or 1 there, and the cube would overflow)
        const float s = sigmoid<QUICK>(c * (x + q * x * x * x));
        *slope = s + x * s * (1.f - s) * c * (1.f + 3.f * q * x * x);
        return g * s;
    } else if constexpr (ACT == UDE_GATE_GELU_ERF) {
        const float p = 0.5f * erfcf(g * -0.7071067811865476f), x = -0.5f * g * g;
        *slope = p + g * 0.3989422804014327f * (QUICK ? __expf(x) : expf(x));
        return g * p;
    } else {
        *slope = 1.f;
        return g;
    }
}
// n values at once, so that the choice of act is made once and the values' chains overlap
template <bool QUICK, int N, int ACT>
static __device__ inline void gate_acts(const float* g, float* act, float* slope) {
#pragma unroll
    for (int i = 0; i < N; ++i) act[i] = gate_act<QUICK, ACT>(g[i], slope + i);
}
template <bool QUICK, int N>
static __device__ inline void gate_acts(int which, const float* g, float* act, float* slope) {
    switch (which) {
        case UDE_GATE_TANH: gate_acts<QUICK, N, UDE_GATE_TANH>(g, act, slope); break;
        case UDE_GATE_RBF: gate_acts<QUICK, N, UDE_GATE_RBF>(g, act, slope); break;
        case UDE_GATE_RELU: gate_acts<QUICK, N, UDE_GATE_RELU>(g, act, slope); break;
        case UDE_GATE_SIGMOID: gate_acts<QUICK, N, UDE_GATE_SIGMOID>(g, act, slope); break;
        case UDE_GATE_SWISH: gate_acts<QUICK, N, UDE_GATE_SWISH>(g, act, slope); break;
        case UDE_GATE_GELU_TANH: gate_acts<QUICK, N, UDE_GATE_GELU_TANH>(g, act, slope); break;
        case UDE_GATE_GELU_ERF: gate_acts<QUICK, N, UDE_GATE_GELU_ERF>(g, act, slope); break;
        default: gate_acts<QUICK, N, UDE_GATE_IDENTITY>(g, act, slope);
    }
}

enum { EPI_STORE = 0, EPI_GATE = 1, EPI_PULL = 2 };

// One product C[m, n] = sum_k A(m, k) B(n, k)
struct Product {
    const void *A, *B;
    void* C;
    int64_t lda, ldb, ldc;
    int M, N;
    int vecA, vecB;  // rows begin on 16-byte boundaries (few_rows)
    int vecC;        // rows of C begin on a multiple of so many elements: 4, 2 or 1
};
struct Args {
    Product p[3];  // EPI_STORE: nprod of them side by side, or (nseg = 2) p[0] + p[1] into p[0].C; EPI_GATE: B of p[0] and p[1]
    int K, nprod, nseg;
    int act;
    // gemm_tile: the tiles from `first` on; tm, tn (not 0): a piece of such a larger tile each, in the order of those; split > 1: each a part
    // of K, the sums of tile t and part s go to part[(t * split + s) * tile size] and join_parts adds them up
    int first, tm, tn, split, tiles;  // tiles: of this launch
    float* part;
    int64_t room;  // bytes there
    float *gate, *up;     // EPI_GATE: stored if not NULL; EPI_PULL: read; leading dimension N
    int vecG;             // ... whose rows begin on a multiple of so many elements
    void *dg, *du, *h;    // EPI_PULL: dg and du with leading dimension p[0].ldc, h with ldh
    int64_t ldh;
};

// Kernel arguments lie in memory that the scalar cache has to fetch line by line, about a microsecond each when a kernel begins; read where
// they are first used, one after the other, they cost a small product more than its arithmetic.  This asks for all lines at once.
template <class A>
static __device__ inline void touch(const A& a) {
    const int* p = (const int*)&a;
    static_assert(sizeof(A) > 64 * 4 && sizeof(A) <= 64 * 6, "one word of each line");
    asm volatile("" ::"s"(p[0]), "s"(p[16]), "s"(p[32]), "s"(p[48]), "s"(p[64]), "s"(p[sizeof(A) / 4 - 1]));
}

// 8 consecutive elements along the stored axis of a tile; elements outside are zero.  (Vector memory takes any address that an element may have:
// one or two loads also where rows are not aligned.)
template <class E>
static __device__ inline void load8(const E* p, int64_t left, bool row, E* o) {
    if (row && left >= 8) {
        __builtin_memcpy(o, p, 8 * sizeof(E));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = (row && i < left) ? p[i] : (E)0;
    }
}

// What a kernel does with N times four consecutive columns n[].. of rows m[] (v: Wu's products for EPI_GATE)
// Rows begin on a multiple of `vec` elements (4, 2 or 1); left = columns from here on
template <class T>
static __device__ inline void store4(typename T::E* to, const float* x, int left, int vec) {
    typedef typename T::E E;
    typedef E E4 __attribute__((ext_vector_type(4)));
    typedef E E2 __attribute__((ext_vector_type(2)));
    const E4 o = {T::from(x[0]), T::from(x[1]), T::from(x[2]), T::from(x[3])};
    if (vec == 4 && left >= 4) {
        *(E4*)to = o;
    } else if (vec >= 2 && left >= 4) {
        ((E2*)to)[0] = E2{o[0], o[1]};
        ((E2*)to)[1] = E2{o[2], o[3]};
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (q < left) to[q] = o[q];
    }
}
static __device__ inline void load4(const float* p, float* o, int left, int vec) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    if (vec == 4 && left >= 4) {
        const f4 x = *(const f4*)p;
#pragma unroll
        for (int q = 0; q < 4; ++q) o[q] = x[q];
    } else if (vec >= 2 && left >= 4) {
        const f2 x = ((const f2*)p)[0], y = ((const f2*)p)[1];
        o[0] = x[0], o[1] = x[1], o[2] = y[0], o[3] = y[1];
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) o[q] = q < left ? p[q] : 0.f;
    }
}
template <class T, int EPI, int N>
static __device__ inline void finish(const Args& a, const Product& p, const int* m, const int* n, const f4* c, const f4* v) {
    typedef typename T::E E;
    constexpr bool QUICK = sizeof(E) == 2;
    if constexpr (EPI == EPI_STORE) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (m[i] < p.M && n[i] < p.N) store4<T>((E*)p.C + (int64_t)m[i] * p.ldc + n[i], (const float*)&c[i], p.N - n[i], p.vecC);
    } else if constexpr (EPI == EPI_GATE) {
        float act[4 * N], slope[4 * N];
        gate_acts<QUICK, 4 * N>(a.act, (const float*)c, act, slope);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (m[i] < p.M && n[i] < p.N) {
                float h[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) h[q] = act[4 * i + q] * v[i][q];
                store4<T>((E*)p.C + (int64_t)m[i] * p.ldc + n[i], h, p.N - n[i], p.vecC);
                if (a.gate) {
                    const int64_t at = (int64_t)m[i] * p.N + n[i];
                    store4<F32>(a.gate + at, (const float*)&c[i], p.N - n[i], a.vecG);
                    store4<F32>(a.up + at, (const float*)&v[i], p.N - n[i], a.vecG);
                }
            }
    } else {
        float g[4 * N], u[4 * N], act[4 * N], slope[4 * N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int64_t at = (int64_t)m[i] * p.N + n[i];
            const int left = m[i] < p.M ? p.N - n[i] : 0;
            load4(a.gate + at, g + 4 * i, left, a.vecG);
            load4(a.up + at, u + 4 * i, left, a.vecG);
        }
        gate_acts<QUICK, 4 * N>(a.act, g, act, slope);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (m[i] < p.M && n[i] < p.N) {
                float dg[4], du[4], h[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    dg[q] = c[i][q] * u[4 * i + q] * slope[4 * i + q];
                    du[q] = c[i][q] * act[4 * i + q];
                    h[q] = act[4 * i + q] * u[4 * i + q];
                }
                const int64_t to = (int64_t)m[i] * p.ldc + n[i];
                store4<T>((E*)a.dg + to, dg, p.N - n[i], p.vecC);
                store4<T>((E*)a.du + to, du, p.N - n[i], p.vecC);
                store4<T>((E*)a.h + (int64_t)m[i] * a.ldh + n[i], h, p.N - n[i], p.vecC);
            }
    }
}

// One 64 x 64 tile of C by four wavefronts, 32 x 32 each, K in steps of 32 through registers and LDS, loads checked element by element where a tile
// reaches over an edge: right for every size, stride and alignment.  Bound by the way of one step's loads: forward and pullback of 233 x 667 x 6283 in
// BFloat16 take 611 us = 29 TFLOP/s (with loads of single elements where rows are not aligned: 1017).
// The operands of a matrix instruction are swapped (B first): a lane then holds four CONSECUTIVE n of one row m.
template <class T, int EPI, bool AK, bool BKc>
__global__ __launch_bounds__(256) void gemm_any(const Args a) {
    typedef typename T::E E;
    constexpr int BM = 64, BN = 64, KS = 32, LD = KS + 16 / (int)sizeof(E);
    __shared__ __attribute__((aligned(16))) E sA[BM * LD];
    __shared__ __attribute__((aligned(16))) E sB[BN * LD];
    const int tid = threadIdx.x, lane = tid & 63, wm = (tid >> 6) & 1, wn = tid >> 7;
    const Product& q = a.p[blockIdx.z];
    const int nm = (q.M + BM - 1) / BM;
    if ((int)blockIdx.x >= nm * ((q.N + (EPI == EPI_GATE ? BN / 2 : BN) - 1) / (EPI == EPI_GATE ? BN / 2 : BN))) return;  // (the grid is that of the largest)
    constexpr int NT = EPI == EPI_GATE ? BN / 2 : BN;  // output columns of a tile
    const int m0 = (int)(blockIdx.x % nm) * BM, n0 = (int)(blockIdx.x / nm) * NT;
    f4 acc[2][2] = {};
    for (int seg = 0; seg < a.nseg; ++seg) {
        const Product& s = a.p[a.nseg > 1 ? seg : blockIdx.z];
        const E* A = (const E*)s.A;
        for (int k0 = 0; k0 < a.K; k0 += KS) {
            E va[8], vb[8];
            int ra, ka, rb, kb;
            if (AK) {
                ra = tid >> 2, ka = (tid & 3) * 8;
                load8(A + (int64_t)(m0 + ra) * s.lda + k0 + ka, a.K - k0 - ka, m0 + ra < q.M, va);
            } else {
                ka = tid >> 3, ra = (tid & 7) * 8;
                load8(A + (int64_t)(k0 + ka) * s.lda + m0 + ra, q.M - m0 - ra, k0 + ka < a.K, va);
            }
            // EPI_GATE: rows 0..31 of the tile come from Wg, 32..63 from Wu
            if (BKc) {
                rb = tid >> 2, kb = (tid & 3) * 8;
                const int half = EPI == EPI_GATE ? rb / NT : 0, n = n0 + rb - half * NT;
                const Product& t = EPI == EPI_GATE ? a.p[half] : s;
                load8((const E*)t.B + (int64_t)n * t.ldb + k0 + kb, a.K - k0 - kb, n < q.N, vb);
            } else {
                kb = tid >> 3, rb = (tid & 7) * 8;
                const int half = EPI == EPI_GATE ? rb / NT : 0, n = n0 + rb - half * NT;
                const Product& t = EPI == EPI_GATE ? a.p[half] : s;
                load8((const E*)t.B + (int64_t)(k0 + kb) * t.ldb + n, q.N - n, k0 + kb < a.K, vb);
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
                    constexpr int V = 16 / (int)sizeof(E);
#pragma unroll
                    for (int kk = 0; kk < KS; kk += 4 * V) acc[i][j] = T::mfma(*(const s8*)(pb + kk + g * V), *(const s8*)(pa + kk + g * V), acc[i][j]);
                }
        }
    }
    const int r = lane & 15, g = lane >> 4;
    if constexpr (EPI == EPI_GATE) {
        const int m[2] = {m0 + wm * 32 + r, m0 + wm * 32 + 16 + r}, n[2] = {n0 + wn * 16 + g * 4, n0 + wn * 16 + g * 4};
        const f4 c[2] = {acc[0][0], acc[1][0]}, v[2] = {acc[0][1], acc[1][1]};
        finish<T, EPI, 2>(a, q, m, n, c, v);
    } else {
        const int m[4] = {m0 + wm * 32 + r, m0 + wm * 32 + r, m0 + wm * 32 + 16 + r, m0 + wm * 32 + 16 + r};
        const int n[4] = {n0 + wn * 32 + g * 4, n0 + wn * 32 + 16 + g * 4, n0 + wn * 32 + g * 4, n0 + wn * 32 + 16 + g * 4};
        const f4 c[4] = {acc[0][0], acc[0][1], acc[1][0], acc[1][1]};
        finish<T, EPI, 4>(a, q, m, n, c, c);
    }
}

// ---- the tile kernel -------------------------------------------------------------------------------------------------------------------
// A BM x BN tile of C by NWM x NWN wavefronts; K in steps of 128 bytes (64 k of the 16-bit kinds, 32 of Float32) through LDS buffers that buffer_load .. lds fills 16 bytes a lane,
// straight from memory: while step k is multiplied, the next ones are on their way.  What a descriptor's record count does not cover is
// filled with zeros, so that edges cost no branches; a lane outside asks for OUTSIDE.
//
// LDS layouts (a 1 KB piece is one instruction of one wavefront, lane l at 16 l):
//   "K" operand [row][128 B of k]: the 16-byte chunk c of row r lies at chunk c ^ (r & 7) -- 16 lanes that read chunk c of 16 consecutive
//       rows touch every bank once.
//   "R" operand [k][W rows] (W = 128 or 64): a k-row's groups of 16 rows lie at group ^ spread(k), which spreads what is read together over
//       the banks.  16-bit kinds are read through ds_read_b64_tr_b16, which hands each lane four consecutive k of one row (8 k-rows read
//       together), Float32 one by one (4 k-rows).
constexpr unsigned OUTSIDE = 0x80000000u;
typedef int i4 __attribute__((ext_vector_type(4)));

static __device__ inline i4 records(const char* base, int64_t bytes) {
    const uint64_t p = (uint64_t)base;
    const int64_t n = bytes < 0 ? 0 : bytes > 0x7ffffffc ? 0x7ffffffc : (bytes + 3) & ~(int64_t)3;
    i4 r;
    r[0] = __builtin_amdgcn_readfirstlane((int)p);
    r[1] = __builtin_amdgcn_readfirstlane((int)(p >> 32) & 0xffff);
    r[2] = __builtin_amdgcn_readfirstlane((int)n);
    r[3] = 0x00020000;
    return r;
}
static __device__ inline void to_lds(unsigned at, unsigned off, i4 r, unsigned from) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(at), "v"(off), "s"(r), "s"(from) : "m0");
}
static __device__ inline unsigned lds_address(const void* p) { return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const char*)p; }

template <int ES, int W>
static __device__ constexpr int spread(int k) {
    return ES == 4 ? (k >> 2) & 3 : W == 128 ? (k & 3) | ((k >> 3) & 1) << 2 : ((k >> 1) & 1) | ((k >> 3) & 1) << 1;
}

// One operand of a tile: ROWS rows (of HALVES matrices, ROWS / HALVES each) by 128 bytes of k
template <class T, bool KC, int ROWS, int NW, int HALVES>
struct Operand {
    typedef typename T::E E;
    static constexpr int ES = sizeof(E), V = 16 / ES, KS = 128 / ES;   // elements of 16 bytes; k of a step
    static constexpr int N = ROWS / 8 / NW;                            // 1 KB pieces of a wavefront
    static constexpr int W = KC ? 0 : (ROWS / HALVES >= 128 ? 128 : 64);  // width of a sub-tile of an "R" operand
    static constexpr int BYTES = ROWS * 128;
    static_assert(N * 8 * NW == ROWS && N % HALVES == 0, "pieces");
    const char* base[HALVES];
    i4 rec[HALVES];
    unsigned step[HALVES];  // bytes of a step
    unsigned off[N];
    int koff;           // "K": first k of this lane's chunks; "R": not used
    int short_at, kleft;  // the step that has only kleft < KS k, or -1

    // columns k0.. of rows row0.. of matrices with `rows` rows and K columns
    __device__ inline void init(const void* const* p, const int64_t* ld, int row0, int rows, int k0, int K, int wave, int lane) {
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
            base[h] = (const char*)p[h] + (KC ? (int64_t)row0 * ld[h] + k0 : (int64_t)k0 * ld[h] + row0) * ES;
            rec[h] = records(base[h], (KC ? (int64_t)(rows - 1 - row0) * ld[h] + K - k0 : (int64_t)(K - 1 - k0) * ld[h] + rows - row0) * ES);
            step[h] = KC ? 128 : 128 * (unsigned)ld[h];
        }
        koff = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int h = i / (N / HALVES), piece = (i % (N / HALVES)) * NW + wave;
            if constexpr (KC) {
                const int r = piece * 8 + (lane >> 3);
                koff = ((lane & 7) ^ (lane >> 3)) * V;
                off[i] = row0 + r < rows ? (unsigned)(r * (int)ld[h] * ES + koff * ES) : OUTSIDE;
            } else {
                constexpr int PP = W / 8, UR = W / V, RP = 64 / UR, UG = 16 / V;  // pieces of a sub-tile; 16-byte units of a k-row; k-rows of a piece; units of 16 rows
                const int sub = piece / PP, k = (piece % PP) * RP + lane / UR, u = lane % UR;
                const int r = sub * W + ((u / UG) ^ spread<ES, W>(k)) * 16 + (u % UG) * V;
                off[i] = row0 + r < rows ? (unsigned)(k * (int)ld[h] * ES + r * ES) : OUTSIDE;
            }
        }
    }
    // the pieces of step n.  END: it may be the short one or lie behind the last (zeros, without a trip to memory)
    unsigned from[HALVES];
    int size[HALVES];
    template <bool END>
    __device__ inline void aim(int n, int last) {
        const bool on = !END || n <= last;
#pragma unroll
        for (int h = 0; h < HALVES; ++h) from[h] = on ? n * step[h] : 0, size[h] = on ? rec[h][2] : 0;
        if constexpr (END && KC)
            if (n == short_at) {  // (chunks behind a row's end.  The rows of an "R" operand behind the last k are behind its records)
#pragma unroll
                for (int i = 0; i < N; ++i) off[i] = koff < kleft ? off[i] : OUTSIDE;
            }
    }
    __device__ inline void piece(int i, unsigned at, int wave) {
        const int h = i / (N / HALVES);
        i4 r = rec[h];
        r[2] = size[h];
        to_lds(at + (i * NW + wave) * 1024, off[i], r, from[h]);
    }
    // where a row ends inside 16 bytes: zeros behind its end, in the buffer of that step
    static __device__ inline void clear(char* lds, int kleft, int tid) {
        if constexpr (KC) {
            const int c = kleft / V, e0 = kleft % V;
            for (int r = tid; r < ROWS; r += 64 * NW) {
                E* p = (E*)(lds + r * 128 + ((c ^ (r & 7)) << 4));
#pragma unroll
                for (int e = 1; e < V; ++e)
                    if (e >= e0) p[e] = 0;
            }
        }
    }
    // the 16 bytes of k of row `row` (a multiple of 16, plus lane & 15) that a lane feeds to the matrix instructions of k-half kk
    static __device__ inline s8 fragment(const char* lds, int row, int kk, int lane) {
        const int g = lane >> 4;
        if constexpr (KC) {
            return *(const s8*)(lds + (row + (lane & 15)) * 128 + (((kk * 4 + g) ^ (lane & 7)) << 4));
        } else if constexpr (ES == 4) {
            const int kr = kk * 16 + g * 4;
            const float* p = (const float*)(lds + (row / W) * (W * 128)) + kr * W + (((row % W) >> 4) ^ spread<ES, W>(kr)) * 16 + (lane & 15);
            const f4 x = {p[0], p[W], p[2 * W], p[3 * W]};
            return __builtin_bit_cast(s8, x);
        } else {
            const int kr = g * 8 + ((lane & 15) >> 2);
            const char* p = lds + (row / W) * (W * 128) + kr * (W * 2) + ((((row % W) >> 4) ^ spread<ES, W>(kr)) << 5) + (lane & 3) * 8 + kk * 32 * (W * 2);
            typedef __attribute__((address_space(3))) s4* P;
            const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)p), y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(p + 4 * (W * 2)));
            return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
};

// Workgroup b runs on XCD b % 8: each XCD takes a contiguous run of tiles, in groups of 8 rows of tiles, so that its L2 holds the rows of A
// of a group and a few columns of B
static __device__ inline int on_its_xcd(int b, int n) {
    const int each = n / 8, more = n % 8, x = b % 8, l = b / 8;
    return (x < more ? x * (each + 1) : more * (each + 1) + (x - more) * each) + l;
}
struct Place {
    int z, m0, n0;
};
template <int BM, int BN, int HALVES>
static __device__ inline Place place(const Args& a, int t) {
    constexpr int GM = 8, NT = BN / HALVES;
    int tm = BM, tn = NT, down = 1, piece = 0;
    if (a.tm) {
        tm = a.tm, tn = a.tn, down = tm / BM;
        const int pieces = down * (tn / NT);
        piece = t % pieces;
        t = t / pieces + a.first;
    }
    int z = 0, nm = (a.p[0].M + tm - 1) / tm, nn = (a.p[0].N + tn - 1) / tn;
    while (z + 1 < a.nprod && t >= nm * nn) {
        t -= nm * nn;
        ++z;
        nm = (a.p[z].M + tm - 1) / tm, nn = (a.p[z].N + tn - 1) / tn;
    }
    const int group = t / (GM * nn), gm0 = group * GM, gsize = nm - gm0 < GM ? nm - gm0 : GM;
    return {z, (gm0 + (t - group * GM * nn) % gsize) * tm + (a.tm ? piece % down * BM : 0), (t - group * GM * nn) / gsize * tn + (a.tm ? piece / down * NT : 0)};
}

// STAGES: so many buffers of both operands, each step loaded that many steps ahead; 0: three of A and two of B, which is what 256 x 256 and two
// workgroups of 128 x 128 leave room for.
template <class T, int EPI, bool AK, bool BKc, int BM, int BN, int NWM, int NWN, int OCC, int STAGES>
__global__ __launch_bounds__(64 * NWM * NWN) __attribute__((amdgpu_waves_per_eu(OCC, OCC))) void gemm_tile(const Args a) {
    constexpr int NW = NWM * NWN, FM = BM / NWM / 16, FN = BN / NWN / 16, HALVES = EPI == EPI_GATE ? 2 : 1;
    constexpr int NT = BN / HALVES;  // output columns of a tile
    typedef Operand<T, AK, BM, NW, 1> OA;
    typedef Operand<T, BKc, BN, NW, HALVES> OB;
    constexpr int KS = OA::KS;
    constexpr bool DEEP = STAGES > 0;
    constexpr int STAGE = OA::BYTES + OB::BYTES;  // DEEP: a step's A, then its B; otherwise two of B, then three of A
    constexpr int BUFFERS = DEEP ? STAGES * STAGE : 2 * OB::BYTES + 3 * OA::BYTES;
    __shared__ __attribute__((aligned(1024))) char lds[BUFFERS];
    touch(a);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave % NWM, wn = wave / NWM;
    int t = on_its_xcd((int)blockIdx.x, a.tiles * a.split);
    const int tiles = a.tiles, part = a.split > 1 ? t / tiles : 0;
    const Place at_tile = place<BM, BN, HALVES>(a, a.split > 1 ? t % tiles : t);
    const Product& q = a.p[at_tile.z];
    const int z = at_tile.z, m0 = at_tile.m0, n0 = at_tile.n0;
    if (m0 >= q.M || n0 >= q.N) return;

    f4 acc[FM][FN] = {};
    s8 fa[2][FM], fb[2][FN];
    OA oa;
    OB ob;
    const unsigned at = __builtin_amdgcn_readfirstlane(lds_address(lds));
    auto read_a = [&](int i, int kk, int stage) { return OA::fragment(lds + stage, wm * (BM / NWM) + i * 16, kk, lane); };
    auto read_b = [&](int j, int kk, int stage) {
        return OB::fragment(lds + stage, HALVES == 2 ? (j / (FN / 2)) * NT + wn * (NT / NWN) + (j % (FN / 2)) * 16 : wn * (BN / NWN) + j * 16, kk, lane);
    };
    // (behind the last step: zeros, into buffers that are not read, so that the number of loads on their way is always the same)
    auto load_a = [&](int stage, int n, int last) {
        oa.template aim<true>(n, last);
#pragma unroll
        for (int i = 0; i < OA::N; ++i) oa.piece(i, at + stage, wave);
    };
    auto load_b = [&](int stage, int n, int last) {
        ob.template aim<true>(n, last);
#pragma unroll
        for (int i = 0; i < OB::N; ++i) ob.piece(i, at + stage, wave);
    };
    // rows of products are the grain that reads and loads are dealt out over; the compiler keeps the order of the grains
    auto reads = [&](int i, int half, int sa, int sb) {
#pragma unroll
        for (int r = 0; r < FM + FN; ++r) {
            if (r * 3 * FM / (4 * (FM + FN)) != i) continue;  // all of them in the first three quarters
            if (r < FN)
                fb[half][r] = read_b(r, half, sb);
            else
                fa[half][r - FN] = read_a(r - FN, half, sa);
        }
    };
    // Step n, whose first half is in registers, out of the buffers sa and sb; leaves the first half of step n + 1 (in sa1, sb1) there, starts
    // the loads of the steps that come to lie in sa and sb.  A load has one step less than it is ahead to arrive: about 0.4 microseconds out
    // of L2, which is what a step of a small tile took with two buffers.  (Without DEEP the loads of a step take about as long to issue as
    // half a step's products: A's third buffer lets the later half of them arrive a step later.)
    constexpr int AHEAD_A = DEEP ? STAGES : 3, AHEAD_B = DEEP ? STAGES : 2, OUT = DEEP ? (STAGES - 2) * (OA::N + OB::N) : OA::N;
    // A last step that is not whole is loaded and multiplied like the others, with zeros behind its end; where that is inside 16 bytes they are
    // written into LDS once it has arrived.  (As a step of its own behind the loop it cost a trip to memory: 142 instead of 136 us for forward
    // and pullback of 1000 x 1000 x 2730 in Float16.)  The steps whose loads ahead are whole have a body without those questions: 1 % of
    // the largest products.
    int ragged = -1;  // the step that ends inside 16 bytes, or -1
    auto clear = [&](int sa, int sb) {
        OA::clear(lds + sa, oa.kleft, tid);
        OB::clear(lds + sb, oa.kleft, tid);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };
    // (END: one of the last steps, whose loads ahead may be short or none)
    auto body = [&](auto end, int sa, int sa1, int sb, int sb1, int n, int last) {
        constexpr bool END = decltype(end)::value;
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            reads(i, 1, sa, sb);
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = T::mfma(fb[0][j], fa[0][i], acc[i][j]);
            __builtin_amdgcn_sched_barrier(0);
        }
        oa.template aim<END>(n + AHEAD_A, last), ob.template aim<END>(n + AHEAD_B, last);
        __builtin_amdgcn_sched_barrier(0);
        // step n + 1 has arrived (the loads behind it need not have), and nobody reads this step's buffers any more
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(OUT) : "memory");
        if constexpr (END)
            if (n + 1 == ragged) clear(sa1, sb1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < FM; ++i) {
#pragma unroll
            for (int p = i * (OA::N + OB::N) / FM; p < (i + 1) * (OA::N + OB::N) / FM; ++p)
                if (p < OB::N)
                    ob.piece(p, at + sb, wave);
                else
                    oa.piece(p - OB::N, at + sa, wave);
            reads(i, 0, sa1, sb1);
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = T::mfma(fb[1][j], fa[1][i], acc[i][j]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    constexpr int A0 = DEEP ? 0 : 2 * OB::BYTES, A1 = A0 + OA::BYTES, A2 = A1 + OA::BYTES, B0 = DEEP ? OA::BYTES : 0;
    // Offsets within a run of steps stay below 2^31: a run of an "R" operand with long rows is shorter than K
    int64_t most = 1 << 22;
    if (!AK && (1 << 30) / (128 * q.lda) < most) most = (1 << 30) / (128 * q.lda);
#pragma unroll
    for (int h = 0; h < 2; ++h)
        if (!BKc && (h ? HALVES == 2 || a.nseg == 2 : true) && (1 << 30) / (128 * a.p[z + h].ldb) < most) most = (1 << 30) / (128 * a.p[z + h].ldb);
    const int run = (int)most;
    // this part's steps out of the nseg * ksteps ones
    const int ksteps = (a.K + KS - 1) / KS, each = (a.nseg * ksteps + a.split - 1) / a.split;
    for (int seg = 0; seg < a.nseg; ++seg) {
        const int lo = part * each - seg * ksteps, hi = lo + each;
        const int64_t kend = hi >= ksteps ? a.K : (int64_t)hi * KS;
        for (int64_t k0 = lo > 0 ? (int64_t)lo * KS : 0; k0 < kend; k0 += (int64_t)run * KS) {
            {
                const Product& s = a.p[a.nseg > 1 ? seg : z];
                const void* pa[1] = {s.A};
                const int64_t la[1] = {s.lda};
                oa.init(pa, la, m0, q.M, (int)k0, a.K, wave, lane);
                const void* pb[2] = {s.B, a.p[1].B};
                const int64_t lb[2] = {s.ldb, a.p[1].ldb};
                ob.init(pb, lb, n0, q.N, (int)k0, a.K, wave, lane);
            }
            const int left = (int)((kend - k0) / KS), full = left < run ? left : run, rest = left < run ? (int)((kend - k0) % KS) : 0;
            const int steps = full + (rest != 0), last = steps - 1;
            oa.short_at = ob.short_at = rest ? full : -1, oa.kleft = ob.kleft = rest;
            ragged = rest % OA::V && (AK || BKc) ? full : -1;
            if constexpr (DEEP) {
#pragma unroll
                for (int k = 0; k < STAGES; ++k) load_a(k * STAGE, k, last), load_b(k * STAGE + B0, k, last);
                asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((STAGES - 1) * (OA::N + OB::N)) : "memory");
            } else {
                load_a(A0, 0, last), load_b(0, 0, last);
                load_a(A1, 1, last), load_b(OB::BYTES, 1, last);
                load_a(A2, 2, last);
                asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(2 * OA::N + OB::N) : "memory");
            }
            if (ragged == 0) clear(A0, B0);
#pragma unroll
            for (int j = 0; j < FN; ++j) fb[0][j] = read_b(j, 0, B0);
#pragma unroll
            for (int i = 0; i < FM; ++i) fa[0][i] = read_a(i, 0, A0);
            // (two "R" operands need nothing special at the end; their transposed reads take more registers, which two bodies do not have)
            constexpr bool APART = AK || BKc;
            int n = 0;
            if constexpr (DEEP) {
                int here = 0;
                auto step = [&](auto end) {
                    const int next = here + STAGE < STAGES * STAGE ? here + STAGE : 0;
                    body(end, here, next, here + B0, next + B0, n, last);
                    here = next;
                };
                if constexpr (APART)
                    for (; n + AHEAD_A < last; ++n) step(std::false_type());
                for (; n < steps; ++n) step(std::true_type());
            } else {
                int s0 = A0, s1 = A1, s2 = A2;
                auto turn = [&] {
                    const int s = s0;
                    s0 = s2, s2 = s1, s1 = s;
                };
                if constexpr (APART)
                    for (; n + 1 + AHEAD_A < last; n += 2, turn()) {
                        body(std::false_type(), s0, s1, 0, OB::BYTES, n, last);
                        body(std::false_type(), s1, s2, OB::BYTES, 0, n + 1, last);
                    }
                for (; n < steps; n += 2, turn()) {
                    body(std::true_type(), s0, s1, 0, OB::BYTES, n, last);
                    if (n + 1 < steps) body(std::true_type(), s1, s2, OB::BYTES, 0, n + 1, last);
                }
            }
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
    }
    if (a.split > 1) {
        f4* to = (f4*)a.part + (((int64_t)(t % tiles) * a.split + part) * NW + wave) * FM * FN * 64 + lane;
#pragma unroll
        for (int i = 0; i < FM; ++i)
            if (m0 + wm * (BM / NWM) + i * 16 + (lane & 15) < q.M)
#pragma unroll
                for (int j = 0; j < FN; ++j) to[(i * FN + j) * 64] = acc[i][j];
        return;
    }
    // epilogue: 32 rows of a wavefront at a time through LDS, so that the code of finish() stands in a loop and a row's lanes store side by
    // side, up to four stores a turn.  (The rows are four floats longer than they need to be: 8 lanes that write 16 bytes of 8 rows touch every
    // bank once.)
    constexpr int COLS = BN / NWN, LDC = COLS + 4, CT = COLS / HALVES, MOST = EPI == EPI_PULL && BM == 256 ? 8 : 4, TURN = 32 * CT / 4 < 64 * MOST ? 32 * CT / 4 / 64 : MOST;
    static_assert(NW * 32 * LDC * 4 <= BUFFERS && 32 * CT / 4 % (64 * TURN) == 0, "epilogue");
    float* mine = (float*)lds + wave * 32 * LDC;
#pragma unroll 1
    for (int p = 0; p < FM / 2; ++p) {
        if (m0 + wm * (BM / NWM) + p * 32 >= q.M) break;
#pragma unroll
        for (int i = 0; i < FM; ++i)
            if (i / 2 == p)
#pragma unroll
                for (int j = 0; j < FN; ++j) *(f4*)(mine + (i % 2 * 16 + (lane & 15)) * LDC + j * 16 + (lane >> 4) * 4) = acc[i][j];
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll 1
        for (int e0 = lane; e0 < 32 * CT / 4; e0 += 64 * TURN) {
            int m[TURN], n[TURN];
            f4 c[TURN], v[TURN];
#pragma unroll
            for (int i = 0; i < TURN; ++i) {
                const int row = (e0 + 64 * i) / (CT / 4), col = (e0 + 64 * i) % (CT / 4) * 4;
                m[i] = m0 + wm * (BM / NWM) + p * 32 + row;
                n[i] = n0 + wn * CT + col;
                c[i] = *(const f4*)(mine + row * LDC + col);
                v[i] = EPI == EPI_GATE ? *(const f4*)(mine + row * LDC + CT + col) : f4{};
            }
            finish<T, EPI, TURN>(a, q, m, n, c, v);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

// Adds up the parts of K of a tile, in their order, and does what the tile kernel would have done with the sums.  One wavefront per 16 x 16 of
// a wavefront's tile (EPI_GATE: two of them, of gate and of up); the parts lie as the lanes held them, so that every access is one contiguous
// 1 KB.  Bound by the way to memory and back: 8 parts at once.
template <class T, int EPI, int BM, int BN, int NWM, int NWN>
__global__ __launch_bounds__(64 * NWM * NWN) void join_parts(const Args a) {
    constexpr int NW = NWM * NWN, FM = BM / NWM / 16, FN = BN / NWN / 16, HALVES = EPI == EPI_GATE ? 2 : 1, NT = BN / HALVES;
    touch(a);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave % NWM, wn = wave / NWM, i = blockIdx.y, j = blockIdx.z;
    const Place at = place<BM, BN, HALVES>(a, (int)blockIdx.x);
    const Product& q = a.p[at.z];
    const int m[1] = {at.m0 + wm * (BM / NWM) + i * 16 + (lane & 15)}, n[1] = {at.n0 + wn * (NT / NWN) + j * 16 + (lane >> 4) * 4};
    if (m[0] >= q.M) return;  // (rows outside have no parts)
    const f4* from = (const f4*)a.part + (((int64_t)blockIdx.x * a.split) * NW + wave) * FM * FN * 64 + (i * FN + j) * 64 + lane;
    f4 c[1] = {}, v[1] = {};
    constexpr int U = 8;
    for (int s = 0; s < a.split; s += U) {
        f4 x[U], y[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {  // (behind the last one: that again, not added)
            const f4* p = from + (int64_t)(s + u < a.split ? s + u : a.split - 1) * (NW * FM * FN * 64);
            x[u] = p[0];
            if constexpr (HALVES == 2) y[u] = p[FN / 2 * 64];
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s + u < a.split) {
                c[0] += x[u];
                if constexpr (HALVES == 2) v[0] += y[u];
            }
    }
    finish<T, EPI, 1>(a, q, m, n, c, v);
}

// ---- a few rows ------------------------------------------------------------------------------------------------------------------------
// C[m, n] = sum_k A(m, k) B(n, k) for at most ROWS rows of A where B's k are adjacent: a wavefront for NB rows of B (EPI_GATE: half of them of Wg, half
// of Wu), 16 bytes of k a lane, sums in Float32 over the lanes at the end.  Bound by reading B, once and in full lines: a tile of matrix instructions
// does that too, but has to cut K to fill the card and join the parts in launches of their own.  One row through a block of 4096 x 11264 in
// BFloat16 takes 44 us = 6.3 TB/s (32 x 128 tiles: 67 to 75), four rows 64 to 66 (67 to 75), one row in Float32 84 = 6.6 TB/s (118); through 2048 x 5632 15 to 17 us
// (27 to 32) and 25 (27 to 32): the same weights again, and six sets of them in turn.  With more
// rows the loads of A and the conversions outweigh those of B (eight rows: 150 us): four rows of B a wavefront instead of two took two
// rows from 64 to 57 us and four from 89 to 68.
template <int EPI, int ROWS>
struct Few {
    static constexpr int NB = ROWS == 1 ? 2 : 4, HALVES = EPI == EPI_GATE ? 2 : 1, NT = NB / HALVES;  // rows of B; output columns
};
template <class T, int EPI, int ROWS>
__global__ __launch_bounds__(256) void few_rows(const Args a) {
    typedef typename T::E E;
    constexpr int V = 16 / (int)sizeof(E), NB = Few<EPI, ROWS>::NB, HALVES = Few<EPI, ROWS>::HALVES, NT = Few<EPI, ROWS>::NT;
    typedef E EV __attribute__((ext_vector_type(V)));
    touch(a);
    const Product& q = a.p[0];
    const int lane = threadIdx.x & 63, n0 = ((int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * NT;
    if (n0 >= q.N) return;
    const E *b[NB], *x[ROWS];
#pragma unroll
    for (int j = 0; j < NB; ++j) {  // (columns outside: the first one again, not stored)
        const Product& p = a.p[j / NT];
        b[j] = (const E*)p.B + (int64_t)(n0 + j % NT < q.N ? n0 + j % NT : n0) * p.ldb;
    }
#pragma unroll
    for (int m = 0; m < ROWS; ++m) x[m] = (const E*)q.A + (m < q.M ? m : 0) * q.lda;
    float s[ROWS][NB] = {};
#pragma unroll (ROWS == 1 ? 4 : 2)
    for (int k = lane * V; k <= a.K - V; k += 64 * V) {
        EV w[NB], y[ROWS];
#pragma unroll
        for (int j = 0; j < NB; ++j) w[j] = __builtin_nontemporal_load((const EV*)(b[j] + k));
#pragma unroll
        for (int m = 0; m < ROWS; ++m) y[m] = *(const EV*)(x[m] + k);
#pragma unroll
        for (int m = 0; m < ROWS; ++m)
#pragma unroll
            for (int e = 0; e < V; ++e)
#pragma unroll
                for (int j = 0; j < NB; ++j) s[m][j] = fmaf(T::to(y[m][e]), T::to(w[j][e]), s[m][j]);
    }
    if (const int k = a.K / V * V + lane; k < a.K) {
#pragma unroll
        for (int m = 0; m < ROWS; ++m)
#pragma unroll
            for (int j = 0; j < NB; ++j) s[m][j] = fmaf(T::to(x[m][k]), T::to(b[j][k]), s[m][j]);
    }
    float c[NB];
#pragma unroll
    for (int m = 0; m < ROWS; ++m)
#pragma unroll
        for (int j = 0; j < NB; ++j) {
#pragma unroll
            for (int d = 32; d; d >>= 1) s[m][j] += __shfl_xor(s[m][j], d);
            c[j] = lane == m ? s[m][j] : m ? c[j] : 0.f;
        }
    if (lane >= q.M) return;  // lane m stores row m
    E* to = (E*)q.C + lane * q.ldc + n0;
    float act[NT], slope[NT];
    if constexpr (EPI == EPI_GATE) gate_acts<sizeof(E) == 2, NT>(a.act, c, act, slope);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        if (n0 + j >= q.N) return;
        if constexpr (EPI == EPI_GATE) {
            to[j] = T::from(act[j] * c[j + NT]);
            if (a.gate) a.gate[(int64_t)lane * q.N + n0 + j] = c[j], a.up[(int64_t)lane * q.N + n0 + j] = c[j + NT];
        } else {
            to[j] = T::from(c[j]);
        }
    }
}

}  // namespace gated
