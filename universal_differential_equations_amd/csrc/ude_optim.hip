// ude_optim.hip -- optimiser operators over many tensors (include/udecore.h): the AdamW step with moments in 32 (64) or 8 bits, and the
// global gradient norm.  A launch takes the descriptors of up to ADAM_NT / NORM_NT tensors by value (kernel arguments: nothing is copied
// to the device, a captured call needs no host memory) and cuts the tensors into chunks, one workgroup per chunk.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "ude_ctx.h"

namespace {

struct OnDevice {  // the caller's current device is left as it was
    int old = -1, now;
    bool ok;
    explicit OnDevice(int d) : now(d) { ok = hipGetDevice(&old) == hipSuccess && (old == d || hipSetDevice(d) == hipSuccess); }
    ~OnDevice() {
        if (ok && old != now) (void)hipSetDevice(old);
    }
};

struct DF64 {
    typedef double E;
    typedef double W;  // arithmetic of the step
};
struct DF32 {
    typedef float E;
    typedef float W;
};
struct DF16 {
    typedef _Float16 E;
    typedef float W;
};
struct DBF16 {
    typedef __bf16 E;
    typedef float W;
};

constexpr int ADAM_NT = 44, NORM_NT = 160;
constexpr int64_t ADAM_CHUNK = 4096;    // elements of one workgroup that writes out 8-bit moments' values: 16 a thread
constexpr int64_t ADAM8_CHUNK = 4096;   // with 8-bit moments: 16 a thread
constexpr int64_t ADAM32_CHUNK = 1024;  // with 32-bit moments: 4 a thread
constexpr int64_t NORM_CHUNK = 4096;
constexpr int NORM_BLOCKS = 2048, NORM_ONE = 64;
constexpr int64_t MOST_CHUNKS = (int64_t)1 << 23;                   // of one launch: 256 threads each, fewer than 2^32
constexpr int64_t MOST_ELEMENTS = MOST_CHUNKS * ADAM32_CHUNK;       // of one tensor

struct AdamTensor {
    void* p;
    const void* g;
    float* master;
    void *m, *v;
    float *ms, *vs;
    int64_t n;
    double wd;
};
struct AdamArgs {
    double eta, b1, b2, eps, c1, c2;  // c1, c2: 1 - b^t for the step number of the host
    const int64_t* step_dev;
    const double* clip;
    int32_t skip, nt;
    int32_t first[ADAM_NT + 1];  // first chunk of each tensor
    AdamTensor t[ADAM_NT];
};
static_assert(sizeof(AdamArgs) <= 4096, "kernel arguments");

template <class A>
__device__ int tensor_of(const A& a, int chunk) {
    int lo = 0, hi = a.nt - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (a.first[mid] <= chunk)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

// the factors of one step, from the device's step number where there is one
template <class W>
__device__ bool step_factors(const AdamArgs& a, W& s, W& rate, W& rc2) {
    __shared__ double c[2];
    s = 1;
    if (a.clip) {
        if (a.skip && !(fabs(a.clip[0]) < __builtin_inf())) return false;
        s = (W)a.clip[1];
    }
    double c1 = a.c1, c2 = a.c2;
    if (a.step_dev) {
        if (threadIdx.x == 0) {
            const double t = (double)*a.step_dev;
            c[0] = 1 - pow(a.b1, t);
            c[1] = 1 - pow(a.b2, t);
        }
        __syncthreads();
        c1 = c[0], c2 = c[1];
    }
    rate = (W)(a.eta / c1);
    rc2 = (W)(1 / c2);
    return true;
}

template <class W>
__device__ inline W root(W x);
template <>
__device__ inline float root(float x) { return sqrtf(x); }
template <>
__device__ inline double root(double x) { return sqrt(x); }

// N consecutive elements as one or a few 16-byte (or one shorter) accesses; p is aligned to them
template <int N, class E>
__device__ inline void get(const E* p, E* o) {
    constexpr int V = 16 / sizeof(E) < N ? 16 / sizeof(E) : N;
    typedef E T __attribute__((ext_vector_type(V)));
#pragma unroll
    for (int i = 0; i < N / V; ++i) {
        const T x = ((const T*)p)[i];
#pragma unroll
        for (int j = 0; j < V; ++j) o[i * V + j] = x[j];
    }
}
template <int N, class E>
__device__ inline void put(E* p, const E* o) {
    constexpr int V = 16 / sizeof(E) < N ? 16 / sizeof(E) : N;
    typedef E T __attribute__((ext_vector_type(V)));
#pragma unroll
    for (int i = 0; i < N / V; ++i) {
        T x;
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = o[i * V + j];
        ((T*)p)[i] = x;
    }
}
template <int N, class E>
__host__ __device__ inline bool fits(const E* p) {
    return (uintptr_t)p % (N * sizeof(E) < 16 ? N * sizeof(E) : 16) == 0;
}

// Bound by memory: 28 bytes an element with 16-bit parameters and 32-bit copies, 138.4 M of them in 713 us = 5.4 TB/s (a large copy: 4.7).  A thread
// has 4 elements, side by side where the tensor's pointers allow it, and asks for all of them before it uses the first.
template <class P, class G>
__global__ __launch_bounds__(256) void adamw32_kernel(const AdamArgs a) {
    typedef typename P::W W;
    typedef typename P::E PE;
    typedef typename G::E GE;
    const int k = tensor_of(a, (int)blockIdx.x);
    const AdamTensor& t = a.t[k];
    const int64_t at = (int64_t)((int)blockIdx.x - a.first[k]) * ADAM32_CHUNK;
    PE* const p = (PE*)t.p;
    const GE* const g = (const GE*)t.g;
    W *const m = (W*)t.m, *const v = (W*)t.v;
    float* const master = t.master;
    PE pp[4];
    GE gg[4];
    W mm[4], vv[4];
    float ww[4];
    const bool four = at + ADAM32_CHUNK <= t.n && fits<4>(p) && fits<4>(g) && fits<4>(m) && fits<4>(v) && fits<4>(master);
    const int64_t i4 = at + threadIdx.x * 4;
    if (four) {
        get<4>(g + i4, gg);
        get<4>(m + i4, mm);
        get<4>(v + i4, vv);
        if (master)
            get<4>(master + i4, ww);
        else
            get<4>(p + i4, pp);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t i = at + j * 256 + threadIdx.x;
            const bool in = i < t.n;
            gg[j] = in ? g[i] : (GE)0;
            mm[j] = in ? m[i] : (W)0;
            vv[j] = in ? v[i] : (W)0;
            if (master)
                ww[j] = in ? master[i] : 0.f;
            else
                pp[j] = in ? p[i] : (PE)0;
        }
    }
    W s, rate, rc2;
    if (!step_factors<W>(a, s, rate, rc2)) return;
    const W keep = (W)(1 - a.eta * t.wd), b1 = (W)a.b1, d1 = (W)(1 - a.b1), b2 = (W)a.b2, d2 = (W)(1 - a.b2), eps = (W)a.eps;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const W gr = (W)gg[j] * s;
        mm[j] = b1 * mm[j] + d1 * gr;
        vv[j] = b2 * vv[j] + d2 * gr * gr;
        W w = master ? (W)ww[j] : (W)pp[j];
        w = w * keep - rate * mm[j] / (root<W>(vv[j] * rc2) + eps);
        ww[j] = (float)w;
        pp[j] = (PE)w;
    }
    if (four) {
        put<4>(m + i4, mm);
        put<4>(v + i4, vv);
        put<4>(p + i4, pp);
        if (master) put<4>(master + i4, ww);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t i = at + j * 256 + threadIdx.x;
            if (i < t.n) {
                m[i] = mm[j];
                v[i] = vv[j];
                p[i] = pp[j];
                if (master) master[i] = ww[j];
            }
        }
    }
}

// Codes of the 8-bit moments, decided in Float64.  With y = 127^2 |m| / a (255^4 v / c) the code is the q with (q - 1/2)^2 <= y < (q + 1/2)^2
// (the same squared).  A Float32 root, less what it may be too large by, gives q or q - 1; the border between the two is a whole number
// plus 1/4 below 2^17 (exact in Float32; its square has at most 38 bits) and is compared with y in Float64.
__device__ inline int code_m(double y) {
    const float q = truncf(__builtin_amdgcn_sqrtf((float)y) + 0.4999f);  // roots up to 127, a few 2^-24 of them off
    const int r = (int)q + (y >= (double)(fmaf(q, q, q) + 0.25f));
    return r > 127 ? 127 : r;
}
__device__ inline int code_v(double y) {
    const float q = truncf(__builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf((float)y)) + 0.499f);
    const double border = (double)(fmaf(q, q, q) + 0.25f);
    const int r = (int)q + (y >= border * border);
    return r > 255 ? 255 : r == 0 && y > 0 ? 1 : r;
}
// what a code stands for, over the scale: signed squares of up to 14 bits, fourth powers of up to 32
__device__ inline double m_part(int q) { return (double)(q * (q < 0 ? -q : q)); }
__device__ inline double v_part(int r) { return (double)((unsigned)(r * r) * (unsigned)(r * r)); }
constexpr double M_UNIT = 1.0 / 16129.0, V_UNIT = 1.0 / 4228250625.0;

// root of x >= 0 and 1 / x by the hardware's instructions, 2^-23 of the value off (measured over every float: 1.56 and 1.54 2^-24); what they take
// for zero is scaled first.  A step has a dozen roundings of 2^-24 besides.
__device__ inline float quick_root(float x) {
    const bool tiny = x < 0x1p-96f;
    const float r = __builtin_amdgcn_sqrtf(tiny ? x * 0x1p64f : x);
    return tiny ? r * 0x1p-32f : r;
}

// the largest of 16 lanes' values, as whole numbers (that is the order of floats >= 0, and above them infinity and NaN), by rotations in a row of 16
__device__ inline int row_max(int x) {
    x = max(x, __builtin_amdgcn_mov_dpp(x, 0x128, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_mov_dpp(x, 0x124, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_mov_dpp(x, 0x122, 0xf, 0xf, false));
    return max(x, __builtin_amdgcn_mov_dpp(x, 0x121, 0xf, 0xf, false));
}

// 16 lanes hold one block of 256 elements, 8 consecutive ones of each half, so that the 16-byte accesses of 16-bit parameters lie side by
// side.  Bound by its arithmetic: 88 vector instructions an element, 30 of them Float64, five roots and reciprocals at a quarter of the rate.  138.4 M
// elements in BFloat16 take 353 us (launches in a row; 377 to 509 alone, where the clock rises first) where their 10 bytes each would take 245 at the rate of the Float32 moments' step (with correctly rounded
// root and quotient, 108 instructions: 430).  Deciding the codes in Float32 where they are clear took longer: the branches cost more.
template <class P, class G>
__global__ __launch_bounds__(256) void adamw8_kernel(const AdamArgs a) {
    typedef typename P::E PE;
    typedef typename G::E GE;
    const int k = tensor_of(a, (int)blockIdx.x);
    const AdamTensor& t = a.t[k];
    const int64_t block = (int64_t)((int)blockIdx.x - a.first[k]) * (ADAM8_CHUNK / UDE_ADAMW_BLOCK) + threadIdx.x / 16;
    const int64_t at = block * UDE_ADAMW_BLOCK + (threadIdx.x & 15) * 8;
    const bool any = block * UDE_ADAMW_BLOCK < t.n;
    PE* const p = (PE*)t.p + at;
    const GE* const g = (const GE*)t.g + at;
    int8_t* const mq = (int8_t*)t.m + at;
    uint8_t* const vq = (uint8_t*)t.v + at;
    float* const master = t.master ? t.master + at : nullptr;
    PE pp[16];
    GE gg[16];
    int8_t mm[16];
    uint8_t vv[16];
    float ww[16];
    // (the same for a whole block: its elements lie behind one another)
    const bool eight = (block + 1) * UDE_ADAMW_BLOCK <= t.n && fits<8>(p) && fits<8>(g) && fits<8>(mq) && fits<8>(vq) && fits<8>(master);
    if (eight) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            get<8>(g + 128 * h, gg + 8 * h);
            get<8>(mq + 128 * h, mm + 8 * h);
            get<8>(vq + 128 * h, vv + 8 * h);
            if (master)
                get<8>(master + 128 * h, ww + 8 * h);
            else
                get<8>(p + 128 * h, pp + 8 * h);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int e = i / 8 * 128 + i % 8;
            const bool in = at + e < t.n;
            gg[i] = in ? g[e] : (GE)0;
            mm[i] = in ? mq[e] : (int8_t)0;
            vv[i] = in ? vq[e] : (uint8_t)0;
            if (master)
                ww[i] = in ? master[e] : 0.f;
            else
                pp[i] = in ? p[e] : (PE)0;
        }
    }
    const double sa = any ? (double)t.ms[block] : 0, sc = any ? (double)t.vs[block] : 0;
    float s, rate, rc2;
    if (!step_factors<float>(a, s, rate, rc2)) return;
    const double factor = a.clip ? a.clip[1] : 1.0;
    const double d1 = 1 - a.b1, d2 = 1 - a.b2;
    double m[16], v[16];
    int am = 0, av = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {  // (elements behind the end: codes and gradients of zero)
        // (in the order of the formula: constants multiplied beforehand would round otherwise, and a largest element whose gradient comes
        // again lies half way between two scales more often than chance has it)
        const double x = (double)(float)gg[i] * factor;
        m[i] = a.b1 * (m_part(mm[i]) * M_UNIT * sa) + d1 * x;
        v[i] = a.b2 * (v_part(vv[i]) * V_UNIT * sc) + d2 * (x * x);
        am = max(am, __float_as_int(fabsf((float)m[i])));
        av = max(av, __float_as_int(fabsf((float)v[i])));
    }
    am = row_max(am);
    av = row_max(av);
    // (a gradient that is not finite makes the moments of its block NaN)
    const bool bad = am >= 0x7f800000 || av >= 0x7f800000;
    const float fa = bad ? __builtin_nanf("") : __int_as_float(am), fc = bad ? __builtin_nanf("") : __int_as_float(av);
    const double ia = fa > 0 ? 16129.0 / (double)fa : 0, ic = fc > 0 ? 4228250625.0 / (double)fc : 0;
    const float keep = (float)(1 - a.eta * t.wd), eps = (float)a.eps;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int q = code_m(fabs(m[i]) * ia);
        mm[i] = (int8_t)(m[i] < 0 ? -q : q);
        vv[i] = (uint8_t)code_v(v[i] * ic);
        float w = master ? ww[i] : (float)pp[i];
        w = w * keep - rate * (float)m[i] * __builtin_amdgcn_rcpf(quick_root((float)v[i] * rc2) + eps);
        ww[i] = w;
        pp[i] = (PE)w;
    }
    if (any && (threadIdx.x & 15) == 0) {
        t.ms[block] = fa;
        t.vs[block] = fc;
    }
    if (eight) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            put<8>(mq + 128 * h, mm + 8 * h);
            put<8>(vq + 128 * h, vv + 8 * h);
            put<8>(p + 128 * h, pp + 8 * h);
            if (master) put<8>(master + 128 * h, ww + 8 * h);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int e = i / 8 * 128 + i % 8;
            if (at + e < t.n) {
                mq[e] = mm[i];
                vq[e] = vv[i];
                p[e] = pp[i];
                if (master) master[e] = ww[i];
            }
        }
    }
}

struct MomentTensor {
    const int8_t* m;
    const uint8_t* v;
    const float *ms, *vs;
    float *mo, *vo;
    int64_t n;
};
struct MomentArgs {
    int32_t nt;
    int32_t first[ADAM_NT + 1];
    MomentTensor t[ADAM_NT];
};
static_assert(sizeof(MomentArgs) <= 4096, "kernel arguments");

// What the codes stand for.  Bound by memory: 10 bytes an element, eight of them written; 138.4 M elements in 230 us = 6.0 TB/s with 4 elements
// side by side a thread and store (8, whose two stores leave gaps that the other one fills: 310).
__global__ __launch_bounds__(256) void moments_kernel(const MomentArgs a) {
    const int k = tensor_of(a, (int)blockIdx.x);
    const MomentTensor& t = a.t[k];
    const int64_t at = (int64_t)((int)blockIdx.x - a.first[k]) * ADAM_CHUNK;
    const int64_t end = t.n < at + ADAM_CHUNK ? t.n : at + ADAM_CHUNK;
    if (end == at + ADAM_CHUNK && fits<4>(t.m) && fits<4>(t.v) && fits<4>(t.mo) && fits<4>(t.vo)) {
        int8_t m[16];
        uint8_t v[16];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            get<4>(t.m + at + h * 1024 + threadIdx.x * 4, m + 4 * h);
            get<4>(t.v + at + h * 1024 + threadIdx.x * 4, v + 4 * h);
        }
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            const int64_t i = at + h * 1024 + threadIdx.x * 4;
            const double sa = (double)t.ms[i / UDE_ADAMW_BLOCK], sc = (double)t.vs[i / UDE_ADAMW_BLOCK];
            float mo[4], vo[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) mo[j] = (float)(m_part(m[4 * h + j]) * M_UNIT * sa), vo[j] = (float)(v_part(v[4 * h + j]) * V_UNIT * sc);
            put<4>(t.mo + i, mo);
            put<4>(t.vo + i, vo);
        }
    } else {
        for (int64_t i = at + threadIdx.x; i < end; i += 256) {
            t.mo[i] = (float)(m_part(t.m[i]) * M_UNIT * (double)t.ms[i / UDE_ADAMW_BLOCK]);
            t.vo[i] = (float)(v_part(t.v[i]) * V_UNIT * (double)t.vs[i / UDE_ADAMW_BLOCK]);
        }
    }
}

struct NormArgs {
    int32_t nt, chunks;
    double* part;  // one sum per workgroup
    int32_t first[NORM_NT + 1];
    const void* g[NORM_NT];
    int64_t n[NORM_NT];
};
static_assert(sizeof(NormArgs) <= 4096, "kernel arguments");

// sum over the workgroup (up to 16 wavefronts) in a fixed order; valid in thread 0
__device__ inline double block_sum(double x) {
    __shared__ double s[16];
#pragma unroll
    for (int d = 32; d; d /= 2) x += __shfl_down(x, d, 64);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
    __syncthreads();
    double all = 0;
    for (unsigned i = 0; i < blockDim.x / 64; ++i) all += s[i];
    return all;
}

// the 16 elements of chunk c, of tensor k, that thread t of 256 adds: 16-byte loads side by side where the tensor allows it
template <class E>
__device__ inline void get_chunk(const NormArgs& a, int k, int c, int t, E* x) {
    constexpr int V = 16 / sizeof(E);
    const int64_t at = (int64_t)(c - a.first[k]) * NORM_CHUNK;
    const int64_t end = a.n[k] < at + NORM_CHUNK ? a.n[k] : at + NORM_CHUNK;
    const E* g = (const E*)a.g[k];
    if (end == at + NORM_CHUNK && fits<V>(g)) {
#pragma unroll
        for (int j = 0; j < 16 / V; ++j) get<V>(g + at + j * 256 * V + t * V, x + j * V);
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int64_t i = at + j * 256 + t;
            x[j] = i < end ? g[i] : (E)0;
        }
    }
}
template <class G>
__device__ inline void add_squares(const typename G::E* x, double* sum) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const double y = (double)(typename G::W)x[j];
        sum[j % 4] = fma(y, y, sum[j % 4]);
    }
}
__device__ inline void write_norm(double sum, double max_norm, double* out) {
    const double norm = sqrt(sum);
    out[0] = norm;
    out[1] = !(max_norm > 0) ? (norm != norm ? norm : 1) : norm <= max_norm ? 1 : max_norm / norm;
}

// Bound by reading: 277 MB of BFloat16 in 42 us = 6.6 TB/s, the sum of the workgroups' sums 4 us more.  Squares and sums in Float64, where those
// of smaller types neither overflow nor vanish.
template <class G>
__global__ __launch_bounds__(256) void norm_part_kernel(const NormArgs a) {
    double sum[4] = {};
    for (int c = (int)blockIdx.x; c < a.chunks; c += (int)gridDim.x) {
        typename G::E x[16];
        get_chunk(a, tensor_of(a, c), c, threadIdx.x, x);
        add_squares<G>(x, sum);
    }
    const double all = block_sum((sum[0] + sum[1]) + (sum[2] + sum[3]));
    if (threadIdx.x == 0) a.part[blockIdx.x] = all;
}

__global__ __launch_bounds__(256) void norm_join_kernel(const double* part, int n, double max_norm, double* out) {
    double sum = 0;
    for (int i = threadIdx.x; i < n; i += 256) sum += part[i];
    sum = block_sum(sum);
    if (threadIdx.x == 0) write_norm(sum, max_norm, out);
}

// few chunks: one workgroup, four chunks side by side, four (Float64: two) such rounds in flight, and no second launch (which costs more than what one compute unit takes for them).  The tensor of
// a chunk is counted out of all that begin before it: looked up in the arguments step by step, it took longer than the sums.
template <class G>
__global__ __launch_bounds__(1024) void norm_one_kernel(const NormArgs a, double max_norm, double* out) {
    constexpr int L = (NORM_NT + 63) / 64;
    int first[L];  // lane l: where the tensors l, l + 64, .. begin
#pragma unroll
    for (int i = 0; i < L; ++i) {
        const int k = i * 64 + (threadIdx.x & 63);
        first[i] = k < a.nt ? a.first[k] : INT32_MAX;
    }
    double sum[4] = {};
    constexpr int U = sizeof(typename G::E) == 8 ? 2 : 4;
    for (int c0 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8); c0 < a.chunks; c0 += 4 * U) {
        typename G::E x[U][16];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = c0 + 4 * u;
            int k = -1;
#pragma unroll
            for (int i = 0; i < L; ++i) k += __popcll(__ballot(first[i] <= c));
            if (c < a.chunks) get_chunk(a, k, c, threadIdx.x & 255, x[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (c0 + 4 * u < a.chunks) add_squares<G>(x[u], sum);
    }
    const double all = block_sum((sum[0] + sum[1]) + (sum[2] + sum[3]));
    if (threadIdx.x == 0) write_norm(all, max_norm, out);
}

int esize(int dt) { return dt == UDE_DT_F64 ? 8 : dt == UDE_DT_F32 ? 4 : 2; }
bool off(const void* p, int e) { return (uintptr_t)p % e != 0; }

int check_state(ude_ctx* c, const ude_adamw_tensor& t, int64_t i, int bits, int we) {
    if (t.n < 0) return fail(c, UDE_ERR_INVALID, "adamw: tensor %lld has %lld elements", (long long)i, (long long)t.n);
    if (t.n == 0) return UDE_OK;
    if (!t.m || !t.v || (bits == 8 && (!t.m_scale || !t.v_scale))) return fail(c, UDE_ERR_INVALID, "adamw: tensor %lld: NULL state", (long long)i);
    if (bits == 8 ? off(t.m_scale, 4) || off(t.v_scale, 4) : off(t.m, we) || off(t.v, we))
        return fail(c, UDE_ERR_INVALID, "adamw: tensor %lld: a pointer is not aligned to its element type", (long long)i);
    return UDE_OK;
}

template <class P, class G>
void adam_launch(ude_ctx* c, const AdamArgs& a, int bits, unsigned chunks) {
    if (bits == 8) {
        if constexpr (sizeof(typename P::W) == 4) hipLaunchKernelGGL((adamw8_kernel<P, G>), dim3(chunks), dim3(256), 0, c->operators(), a);
    } else {
        hipLaunchKernelGGL((adamw32_kernel<P, G>), dim3(chunks), dim3(256), 0, c->operators(), a);
    }
}

// tensors[i..] with elements, as many as a launch takes: calls put(slot, tensor index) and go(chunks)
template <class N, class Put, class Go>
int in_launches(int64_t ntensors, int most, int64_t chunk, int32_t* first, N n, Put put, Go go) {
    int used = 0;
    int64_t chunks = 0;
    for (int64_t i = 0; i < ntensors; ++i) {
        const int64_t of = (n(i) + chunk - 1) / chunk;
        if (of == 0) continue;
        if (used == most || (used && chunks + of > MOST_CHUNKS)) {
            first[used] = (int32_t)chunks;
            if (int rc = go(used, chunks)) return rc;
            used = 0;
            chunks = 0;
        }
        first[used] = (int32_t)chunks;
        put(used, i);
        ++used;
        chunks += of;
    }
    if (used) {
        first[used] = (int32_t)chunks;
        return go(used, chunks);
    }
    return UDE_OK;
}

}  // namespace

extern "C" int ude_adamw_step_dev(ude_ctx* c, const ude_adamw_opts* o, int64_t nt, const ude_adamw_tensor* ts) {
    if (!c) return UDE_ERR_INVALID;
    if (!o || nt < 0 || (nt && !ts)) return fail(c, UDE_ERR_INVALID, "adamw: NULL argument");
    const int pd = o->param_dtype, gd = o->grad_dtype;
    const bool half = pd == UDE_DT_F16 || pd == UDE_DT_BF16;
    if (pd < UDE_DT_F64 || pd > UDE_DT_BF16 || !(gd == pd || (half && gd == UDE_DT_F32)))
        return fail(c, UDE_ERR_UNSUPPORTED, "adamw: param_dtype %d with grad_dtype %d", pd, gd);
    if ((o->state_bits != 32 && o->state_bits != 8) || (o->state_bits == 8 && pd == UDE_DT_F64))
        return fail(c, UDE_ERR_UNSUPPORTED, "adamw: state_bits %d with param_dtype %d", o->state_bits, pd);
    if (!(o->beta1 >= 0 && o->beta1 < 1 && o->beta2 >= 0 && o->beta2 < 1 && o->eps >= 0 && o->eta == o->eta) || (!o->step_dev && o->step < 1))
        return fail(c, UDE_ERR_INVALID, "adamw: eta %g, beta (%g, %g), eps %g, step %lld", o->eta, o->beta1, o->beta2, o->eps, (long long)o->step);
    if (o->skip_nonfinite && !o->clip) return fail(c, UDE_ERR_INVALID, "adamw: skip_nonfinite needs the norm that clip points to");
    if (off(o->step_dev, 8) || off(o->clip, 8)) return fail(c, UDE_ERR_INVALID, "adamw: step_dev and clip are 8-byte aligned");
    for (int64_t i = 0; i < nt; ++i) {
        const ude_adamw_tensor& t = ts[i];
        if (int rc = check_state(c, t, i, o->state_bits, pd == UDE_DT_F64 ? 8 : 4)) return rc;
        if (t.n > MOST_ELEMENTS) return fail(c, UDE_ERR_UNSUPPORTED, "adamw: tensor %lld has %lld elements", (long long)i, (long long)t.n);
        if (t.n && (!t.param || !t.grad)) return fail(c, UDE_ERR_INVALID, "adamw: tensor %lld: NULL param or grad", (long long)i);
        if (t.master && !half) return fail(c, UDE_ERR_INVALID, "adamw: tensor %lld: master copies go with 16-bit parameters", (long long)i);
        if (off(t.param, esize(pd)) || off(t.grad, esize(gd)) || off(t.master, 4))
            return fail(c, UDE_ERR_INVALID, "adamw: tensor %lld: a pointer is not aligned to its element type", (long long)i);
        if (!(t.weight_decay == t.weight_decay)) return fail(c, UDE_ERR_INVALID, "adamw: tensor %lld: weight_decay", (long long)i);
    }
    OnDevice dev(c->device);
    if (!dev.ok) return fail(c, UDE_ERR_HIP, "adamw: device %d", c->device);
    AdamArgs a{};
    a.eta = o->eta, a.b1 = o->beta1, a.b2 = o->beta2, a.eps = o->eps;
    a.c1 = 1 - pow(o->beta1, (double)o->step), a.c2 = 1 - pow(o->beta2, (double)o->step);
    a.step_dev = o->step_dev, a.clip = o->clip, a.skip = o->skip_nonfinite;
    return in_launches(
        nt, ADAM_NT, o->state_bits == 8 ? ADAM8_CHUNK : ADAM32_CHUNK, a.first, [&](int64_t i) { return ts[i].n; },
        [&](int slot, int64_t i) {
            const ude_adamw_tensor& t = ts[i];
            a.t[slot] = {t.param, t.grad, t.master, t.m, t.v, t.m_scale, t.v_scale, t.n, t.weight_decay};
        },
        [&](int used, int64_t chunks) {
            a.nt = used;
            const unsigned g = (unsigned)chunks;
            if (pd == UDE_DT_F64)
                adam_launch<DF64, DF64>(c, a, 32, g);
            else if (pd == UDE_DT_F32)
                adam_launch<DF32, DF32>(c, a, o->state_bits, g);
            else if (pd == UDE_DT_F16)
                gd == pd ? adam_launch<DF16, DF16>(c, a, o->state_bits, g) : adam_launch<DF16, DF32>(c, a, o->state_bits, g);
            else
                gd == pd ? adam_launch<DBF16, DBF16>(c, a, o->state_bits, g) : adam_launch<DBF16, DF32>(c, a, o->state_bits, g);
            HIPCHK(c, hipGetLastError());
            return (int)UDE_OK;
        });
}

extern "C" int ude_adamw_moments_dev(ude_ctx* c, int64_t nt, const ude_adamw_tensor* ts, float* const* m_out, float* const* v_out) {
    if (!c) return UDE_ERR_INVALID;
    if (nt < 0 || (nt && (!ts || !m_out || !v_out))) return fail(c, UDE_ERR_INVALID, "adamw_moments: NULL argument");
    for (int64_t i = 0; i < nt; ++i) {
        if (int rc = check_state(c, ts[i], i, 8, 4)) return rc;
        if (ts[i].n > MOST_ELEMENTS) return fail(c, UDE_ERR_UNSUPPORTED, "adamw_moments: tensor %lld has %lld elements", (long long)i, (long long)ts[i].n);
        if (ts[i].n && (!m_out[i] || !v_out[i] || off(m_out[i], 4) || off(v_out[i], 4))) return fail(c, UDE_ERR_INVALID, "adamw_moments: output %lld", (long long)i);
    }
    OnDevice dev(c->device);
    if (!dev.ok) return fail(c, UDE_ERR_HIP, "adamw_moments: device %d", c->device);
    MomentArgs a{};
    return in_launches(
        nt, ADAM_NT, ADAM_CHUNK, a.first, [&](int64_t i) { return ts[i].n; },
        [&](int slot, int64_t i) { a.t[slot] = {(const int8_t*)ts[i].m, (const uint8_t*)ts[i].v, ts[i].m_scale, ts[i].v_scale, m_out[i], v_out[i], ts[i].n}; },
        [&](int used, int64_t chunks) {
            a.nt = used;
            hipLaunchKernelGGL(moments_kernel, dim3((unsigned)chunks), dim3(256), 0, c->operators(), a);
            HIPCHK(c, hipGetLastError());
            return (int)UDE_OK;
        });
}

extern "C" int ude_grad_norm_workspace(int64_t nt, const int64_t* n, int64_t* bytes) {
    if (!bytes || nt < 0 || (nt && !n)) return UDE_ERR_INVALID;
    int64_t sums = 0;
    int32_t first[NORM_NT + 1];
    for (int64_t i = 0; i < nt; ++i)
        if (n[i] < 0 || n[i] > MOST_ELEMENTS) return UDE_ERR_INVALID;
    (void)in_launches(
        nt, NORM_NT, NORM_CHUNK, first, [&](int64_t i) { return n[i]; }, [](int, int64_t) {},
        [&](int, int64_t chunks) {
            sums += chunks < NORM_BLOCKS ? chunks : NORM_BLOCKS;
            return 0;
        });
    *bytes = 8 * (sums ? sums : 1);
    return UDE_OK;
}

extern "C" int ude_grad_norm_dev(ude_ctx* c, int32_t dtype, int64_t nt, const void* const* grads, const int64_t* n, double max_norm,
                                 double* out, void* ws, int64_t ws_bytes) {
    if (!c) return UDE_ERR_INVALID;
    if (dtype < UDE_DT_F64 || dtype > UDE_DT_BF16) return fail(c, UDE_ERR_UNSUPPORTED, "grad_norm: dtype %d", dtype);
    if (nt < 0 || (nt && (!grads || !n)) || !out || !ws || off(out, 8) || off(ws, 8)) return fail(c, UDE_ERR_INVALID, "grad_norm: NULL or misaligned argument");
    int64_t need = 0;
    if (int rc = ude_grad_norm_workspace(nt, n, &need)) return fail(c, rc, "grad_norm: a tensor's number of elements");
    if (ws_bytes < need) return fail(c, UDE_ERR_INVALID, "grad_norm: workspace of %lld bytes, got %lld", (long long)need, (long long)ws_bytes);
    for (int64_t i = 0; i < nt; ++i)
        if (n[i] && (!grads[i] || off(grads[i], esize(dtype)))) return fail(c, UDE_ERR_INVALID, "grad_norm: tensor %lld: NULL or misaligned", (long long)i);
    OnDevice dev(c->device);
    if (!dev.ok) return fail(c, UDE_ERR_HIP, "grad_norm: device %d", c->device);
    NormArgs a{};
    int64_t sums = 0;
    bool done = false;
    auto run = [&](auto g, int64_t chunks) {
        typedef decltype(g) G;
        if (sums == 0 && chunks <= NORM_ONE && need <= 8 * chunks) {  // (they are all there are)
            hipLaunchKernelGGL((norm_one_kernel<G>), dim3(1), dim3(1024), 0, c->operators(), a, max_norm, out);
            done = true;
            return;
        }
        const unsigned blocks = (unsigned)(chunks < NORM_BLOCKS ? chunks : NORM_BLOCKS);
        hipLaunchKernelGGL((norm_part_kernel<G>), dim3(blocks), dim3(256), 0, c->operators(), a);
        sums += blocks;
    };
    const int rc = in_launches(
        nt, NORM_NT, NORM_CHUNK, a.first, [&](int64_t i) { return n[i]; },
        [&](int slot, int64_t i) { a.g[slot] = grads[i], a.n[slot] = n[i]; },
        [&](int used, int64_t chunks) {
            a.nt = used;
            a.chunks = (int32_t)chunks;
            a.part = (double*)ws + sums;
            if (dtype == UDE_DT_F64)
                run(DF64(), chunks);
            else if (dtype == UDE_DT_F32)
                run(DF32(), chunks);
            else if (dtype == UDE_DT_F16)
                run(DF16(), chunks);
            else
                run(DBF16(), chunks);
            HIPCHK(c, hipGetLastError());
            return (int)UDE_OK;
        });
    if (rc || done) return rc;
    hipLaunchKernelGGL(norm_join_kernel, dim3(1), dim3(256), 0, c->operators(), (const double*)ws, (int)sums, max_norm, out);
    HIPCHK(c, hipGetLastError());
    return UDE_OK;
}
