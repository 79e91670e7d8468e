// ude_optim.hip -- optimiser operators over many tensors (include/udecore.h): the AdamW step with moments in 32 (64) or 8 bits, and the
// global gradient norm.  A launch takes the descriptors of up to ADAM_NT / NORM_NT tensors by value (kernel arguments: nothing is copied
// to the device, a captured call needs no host memory) and cuts the tensors into chunks, one workgroup per chunk.
#include <hip/hip_runtime.h>

#include <cstdint>

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
constexpr int64_t ADAM_CHUNK = 4096;   // elements of one workgroup (a multiple of UDE_ADAMW_BLOCK)
constexpr int64_t NORM_CHUNK = 16384;
constexpr int NORM_BLOCKS = 2048;
constexpr int64_t MOST_CHUNKS = (int64_t)1 << 23;                   // of one launch: 256 threads each, fewer than 2^32
constexpr int64_t MOST_ELEMENTS = MOST_CHUNKS * ADAM_CHUNK;         // of one tensor

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

template <class P, class G>
__global__ __launch_bounds__(256) void adamw32_kernel(const AdamArgs a) {
    typedef typename P::W W;
    W s, rate, rc2;
    if (!step_factors<W>(a, s, rate, rc2)) return;
    const int k = tensor_of(a, (int)blockIdx.x);
    const AdamTensor& t = a.t[k];
    const int64_t at = (int64_t)((int)blockIdx.x - a.first[k]) * ADAM_CHUNK;
    const W keep = (W)(1 - a.eta * t.wd), b1 = (W)a.b1, d1 = (W)(1 - a.b1), b2 = (W)a.b2, d2 = (W)(1 - a.b2), eps = (W)a.eps;
    const int64_t end = t.n < at + ADAM_CHUNK ? t.n : at + ADAM_CHUNK;
    typename P::E* p = (typename P::E*)t.p;
    const typename G::E* g = (const typename G::E*)t.g;
    W *m = (W*)t.m, *v = (W*)t.v;
    for (int64_t i = at + threadIdx.x; i < end; i += 256) {
        const W gr = (W)g[i] * s;
        const W mi = b1 * m[i] + d1 * gr, vi = b2 * v[i] + d2 * gr * gr;
        m[i] = mi;
        v[i] = vi;
        W w = t.master ? (W)t.master[i] : (W)p[i];
        w = w * keep - rate * mi / (root<W>(vi * rc2) + eps);
        if (t.master) t.master[i] = (float)w;
        p[i] = (typename P::E)w;
    }
}

// Codes of the 8-bit moments.  A code is decided in Float64: a Float32 root gives the candidate, the borders (q - 1/2)^2, (q + 1/2)^2 (and
// their squares) are whole numbers plus a power of two, exact in Float64, and move it by one where the root was on the wrong side.
__device__ inline int code_m(double y) {  // y = 127^2 |m| / a
    int q = (int)rintf(sqrtf((float)y));
    const double lo = (double)(q * q - q) + 0.25, hi = (double)(q * q + q) + 0.25;
    if (q > 0 && y < lo) --q;
    if (y >= hi) ++q;
    return q > 127 ? 127 : q;
}
__device__ inline int code_v(double y) {  // y = 255^4 v / c
    int q = (int)rintf(sqrtf(sqrtf((float)y)));
    const double lo = (double)(q * q - q) + 0.25, hi = (double)(q * q + q) + 0.25;
    if (q > 0 && y < lo * lo) --q;
    if (y >= hi * hi) ++q;
    q = q > 255 ? 255 : q;
    return q == 0 && y > 0 ? 1 : q;
}
__device__ inline double value_m(int q, double a) { return a * ((double)(q * (q < 0 ? -q : q)) * (1.0 / 16129.0)); }
__device__ inline double value_v(int r, double c) { return c * ((double)(unsigned)(r * r) * (double)(unsigned)(r * r) * (1.0 / 4228250625.0)); }

// 16 lanes hold one block of 256 elements, 16 consecutive ones each: a code row is one 16-byte load, the two maxima are four exchanges
template <class P, class G>
__global__ __launch_bounds__(256) void adamw8_kernel(const AdamArgs a) {
    float s, rate, rc2;
    if (!step_factors<float>(a, s, rate, rc2)) return;
    const double factor = a.clip ? a.clip[1] : 1.0;
    const int k = tensor_of(a, (int)blockIdx.x);
    const AdamTensor& t = a.t[k];
    const int64_t at = (int64_t)((int)blockIdx.x - a.first[k]) * ADAM_CHUNK + threadIdx.x * 16;
    const float keep = (float)(1 - a.eta * t.wd), eps = (float)a.eps;
    const int64_t left = t.n - at;
    const int n = left < 0 ? 0 : left > 16 ? 16 : (int)left;
    const int64_t block = at / UDE_ADAMW_BLOCK;
    typename P::E* p = (typename P::E*)t.p + at;
    const typename G::E* g = (const typename G::E*)t.g + at;
    int8_t* mq = (int8_t*)t.m + at;
    uint8_t* vq = (uint8_t*)t.v + at;
    float* master = t.master ? t.master + at : nullptr;
    double am = 0, av = 0;
    float bad = 0;
    double m[16], v[16];
    const bool any = block * UDE_ADAMW_BLOCK < t.n;
    const double sa = any ? (double)t.ms[block] : 0, sc = any ? (double)t.vs[block] : 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        m[i] = v[i] = 0;
        if (i < n) {
            const double gr = (double)(float)g[i] * factor;
            m[i] = a.b1 * value_m(mq[i], sa) + (1 - a.b1) * gr;
            v[i] = a.b2 * value_v(vq[i], sc) + (1 - a.b2) * gr * gr;
            bad += (float)(m[i] - m[i]) + (float)(v[i] - v[i]);
            am = fmax(am, fabs(m[i]));
            av = fmax(av, v[i]);
        }
    }
#pragma unroll
    for (int d = 1; d < 16; d *= 2) {
        am = fmax(am, __shfl_xor(am, d, 64));
        av = fmax(av, __shfl_xor(av, d, 64));
        bad += __shfl_xor(bad, d, 64);
    }
    // (a gradient that is not finite makes the moments of its block NaN: they are then read as such)
    const float fa = (float)am + bad, fc = (float)av + bad;
    if (any && (threadIdx.x & 15) == 0) {
        t.ms[block] = fa;
        t.vs[block] = fc;
    }
    const double ia = fa > 0 ? 16129.0 / (double)fa : 0, ic = fc > 0 ? 4228250625.0 / (double)fc : 0;
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (i < n) {
            const int q = code_m(fabs(m[i]) * ia);
            mq[i] = (int8_t)(m[i] < 0 ? -q : q);
            vq[i] = (uint8_t)code_v(v[i] * ic);
            float w = master ? master[i] : (float)p[i];
            w = w * keep - rate * (float)m[i] / (sqrtf((float)v[i] * rc2) + eps);
            if (master) master[i] = w;
            p[i] = (typename P::E)w;
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

__global__ __launch_bounds__(256) void moments_kernel(const MomentArgs a) {
    const int k = tensor_of(a, (int)blockIdx.x);
    const MomentTensor& t = a.t[k];
    const int64_t at = (int64_t)((int)blockIdx.x - a.first[k]) * ADAM_CHUNK;
    const int64_t end = t.n < at + ADAM_CHUNK ? t.n : at + ADAM_CHUNK;
    for (int64_t i = at + threadIdx.x; i < end; i += 256) {
        t.mo[i] = (float)value_m(t.m[i], (double)t.ms[i / UDE_ADAMW_BLOCK]);
        t.vo[i] = (float)value_v(t.v[i], (double)t.vs[i / UDE_ADAMW_BLOCK]);
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

// sum over the workgroup in a fixed order; valid in thread 0
__device__ inline double block_sum(double x) {
    __shared__ double s[4];
#pragma unroll
    for (int d = 32; d; d /= 2) x += __shfl_down(x, d, 64);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
    __syncthreads();
    return s[0] + s[1] + s[2] + s[3];
}

template <class G>
__global__ __launch_bounds__(256) void norm_part_kernel(const NormArgs a) {
    double sum = 0;
    for (int c = (int)blockIdx.x; c < a.chunks; c += (int)gridDim.x) {
        const int k = tensor_of(a, c);
        const int64_t at = (int64_t)(c - a.first[k]) * NORM_CHUNK;
        const int64_t end = a.n[k] < at + NORM_CHUNK ? a.n[k] : at + NORM_CHUNK;
        const typename G::E* g = (const typename G::E*)a.g[k];
        for (int64_t i = at + threadIdx.x; i < end; i += 256) {
            const double x = (double)(typename G::W)g[i];
            sum += x * x;
        }
    }
    sum = block_sum(sum);
    if (threadIdx.x == 0) a.part[blockIdx.x] = sum;
}

__global__ __launch_bounds__(256) void norm_join_kernel(const double* part, int n, double max_norm, double* out) {
    double sum = 0;
    for (int i = threadIdx.x; i < n; i += 256) sum += part[i];
    sum = block_sum(sum);
    if (threadIdx.x == 0) {
        const double norm = sqrt(sum);
        out[0] = norm;
        out[1] = !(max_norm > 0) ? (norm != norm ? norm : 1) : norm <= max_norm ? 1 : max_norm / norm;
    }
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
        if constexpr (sizeof(typename P::W) == 4) hipLaunchKernelGGL((adamw8_kernel<P, G>), dim3(chunks), dim3(256), 0, c->stream, a);
    } else {
        hipLaunchKernelGGL((adamw32_kernel<P, G>), dim3(chunks), dim3(256), 0, c->stream, a);
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
        nt, ADAM_NT, ADAM_CHUNK, a.first, [&](int64_t i) { return ts[i].n; },
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
            hipLaunchKernelGGL(moments_kernel, dim3((unsigned)chunks), dim3(256), 0, c->stream, a);
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
    const int rc = in_launches(
        nt, NORM_NT, NORM_CHUNK, a.first, [&](int64_t i) { return n[i]; },
        [&](int slot, int64_t i) { a.g[slot] = grads[i], a.n[slot] = n[i]; },
        [&](int used, int64_t chunks) {
            a.nt = used;
            a.chunks = (int32_t)chunks;
            a.part = (double*)ws + sums;
            const unsigned g = (unsigned)(chunks < NORM_BLOCKS ? chunks : NORM_BLOCKS);
            sums += g;
            if (dtype == UDE_DT_F64)
                hipLaunchKernelGGL((norm_part_kernel<DF64>), dim3(g), dim3(256), 0, c->stream, a);
            else if (dtype == UDE_DT_F32)
                hipLaunchKernelGGL((norm_part_kernel<DF32>), dim3(g), dim3(256), 0, c->stream, a);
            else if (dtype == UDE_DT_F16)
                hipLaunchKernelGGL((norm_part_kernel<DF16>), dim3(g), dim3(256), 0, c->stream, a);
            else
                hipLaunchKernelGGL((norm_part_kernel<DBF16>), dim3(g), dim3(256), 0, c->stream, a);
            HIPCHK(c, hipGetLastError());
            return (int)UDE_OK;
        });
    if (rc) return rc;
    hipLaunchKernelGGL(norm_join_kernel, dim3(1), dim3(256), 0, c->stream, (const double*)ws, (int)sums, max_norm, out);
    HIPCHK(c, hipGetLastError());
    return UDE_OK;
}
