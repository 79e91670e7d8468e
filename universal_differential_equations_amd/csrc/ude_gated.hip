// ude_gated.hip -- C entries of the gated feed-forward block (include/udecore.h); kernels: ude_gated.h
#include "ude_gated.h"

#include "ude_ctx.h"

using namespace gated;

namespace {

// the caller's current device is left as it was
struct OnDevice {
    int old = -1, now;
    bool ok;
    explicit OnDevice(int d) : now(d) { ok = hipGetDevice(&old) == hipSuccess && (old == d || hipSetDevice(d) == hipSuccess); }
    ~OnDevice() {
        if (ok && old != now) (void)hipSetDevice(old);
    }
};

int esize(int dt) { return dt == UDE_DT_F32 ? 4 : 2; }
int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }
// leading dimension of a workspace matrix with n columns: rows 16-byte aligned
int64_t wld(int64_t n) { return (n + 7) / 8 * 8; }

int check(ude_ctx* c, const ude_gated_ffn_desc* d) {
    if (!d) return fail(c, UDE_ERR_INVALID, "gated_ffn: no descriptor");
    if (d->dtype != UDE_DT_F32 && d->dtype != UDE_DT_F16 && d->dtype != UDE_DT_BF16)
        return fail(c, UDE_ERR_UNSUPPORTED, "gated_ffn: dtype %d (Float32, Float16, BFloat16 are supported)", d->dtype);
    if (d->act < UDE_GATE_IDENTITY || d->act > UDE_GATE_GELU_ERF) return fail(c, UDE_ERR_INVALID, "gated_ffn: activation %d", d->act);
    if ((d->w_order != 0 && d->w_order != 1) || d->reserved) return fail(c, UDE_ERR_INVALID, "gated_ffn: w_order %d, reserved %d", d->w_order, d->reserved);
    const int64_t most = INT32_MAX - 1024;
    if (d->T < 0 || d->D < 1 || d->F < 1 || d->O < 1 || d->T > most || d->D > most || d->F > most / 2 || d->O > most)
        return fail(c, UDE_ERR_INVALID, "gated_ffn: sizes T = %lld, D = %lld, F = %lld, O = %lld", (long long)d->T, (long long)d->D, (long long)d->F, (long long)d->O);
    const int64_t gcols = d->w_order ? d->D : d->F, dcols = d->w_order ? d->F : d->O;
    if (d->ldx < d->D || d->ldy < d->O || d->ldg < gcols || d->ldu < gcols || d->ldd < dcols || d->ldx > most || d->ldy > most || d->ldg > most || d->ldu > most || d->ldd > most)
        return fail(c, UDE_ERR_INVALID, "gated_ffn: a leading dimension is smaller than what it spans, or over 2^31");
    return UDE_OK;
}

int misaligned(const void* p, int e) { return (uintptr_t)p % e != 0; }

int vec(const void* p, int64_t ld, int e) { return (uintptr_t)p % 16 == 0 && ld * e % 16 == 0; }

// a row of 16-bit elements starts on a 4-byte boundary, and a tile's offsets fit 31 bits
bool tileable(const void* p, int64_t ld) { return (uintptr_t)p % 4 == 0 && ld % 2 == 0 && ld < (1 << 22); }

template <class T, int EPI, bool AK, bool BKc>
int launch3(ude_ctx* c, const Args& a, int batch, bool tile) {
    constexpr int H = EPI == EPI_GATE ? 2 : 1;
    auto tiles = [&](int bm, int bn) { return (int64_t)((a.M + bm - 1) / bm) * ((a.N + bn / H - 1) / (bn / H)); };
    if constexpr (sizeof(typename T::E) == 2) {
        if (tile && tiles(128, 128) < 1 << 22) {
            if (tiles(256, 256) * batch >= 128)
                hipLaunchKernelGGL((gemm_tile<T, EPI, AK, BKc, 256, 256, 2, 2, 1>), dim3((unsigned)tiles(256, 256), 1, batch), dim3(256), 0, c->stream, a);
            else
                hipLaunchKernelGGL((gemm_tile<T, EPI, AK, BKc, 128, 128, 2, 2, 2>), dim3((unsigned)tiles(128, 128), 1, batch), dim3(256), 0, c->stream, a);
            HIPCHK(c, hipGetLastError());
            return UDE_OK;
        }
    }
    const int64_t n = tiles(64, 64);
    if (n >= 1 << 24) return fail(c, UDE_ERR_UNSUPPORTED, "gated_ffn: %lld tiles", (long long)n);
    hipLaunchKernelGGL((gemm_any<T, EPI, AK, BKc>), dim3((unsigned)n, 1, batch), dim3(256), 0, c->stream, a);
    HIPCHK(c, hipGetLastError());
    return UDE_OK;
}
template <class T, int EPI>
int launch2(ude_ctx* c, const Args& a, bool ak, bool bk, int batch, bool tile) {
    if constexpr (EPI == EPI_STORE)
        if (!ak) return bk ? fail(c, UDE_ERR_INVALID, "gated_ffn: operand orders") : launch3<T, EPI, false, false>(c, a, batch, tile);
    return bk ? launch3<T, EPI, true, true>(c, a, batch, tile) : launch3<T, EPI, true, false>(c, a, batch, tile);
}
template <int EPI>
int launch(ude_ctx* c, int dtype, Args a, bool ak, bool bk, int batch = 1) {
    const int e = esize(dtype);
    a.vecA = a.vecB = a.vecC = 1;
    bool tile = true;
    for (int i = 0; i < 2; ++i) {
        if (a.A[i] && !vec(a.A[i], a.lda, e)) a.vecA = 0;
        if (a.B[i] && !vec(a.B[i], a.ldb[i], e)) a.vecB = 0;
        if (a.C[i] && ((uintptr_t)a.C[i] % (4 * e) || a.ldc[i] % 4)) a.vecC = 0;
        tile = tile && (!a.A[i] || tileable(a.A[i], a.lda)) && (!a.B[i] || tileable(a.B[i], a.ldb[i]));
    }
    // gate and up are rows of N floats; dg, du, h lie in the workspace, rows of a multiple of 8
    if (EPI != EPI_STORE && a.gate && (a.N % 4 || (uintptr_t)a.gate % 16 || (uintptr_t)a.up % 16)) a.vecC = 0;
    if (dtype == UDE_DT_F32) return launch2<F32, EPI>(c, a, ak, bk, batch, false);
    if (dtype == UDE_DT_F16) return launch2<F16, EPI>(c, a, ak, bk, batch, tile);
    return launch2<BF16, EPI>(c, a, ak, bk, batch, tile);
}

}  // namespace

extern "C" int ude_gated_ffn_workspace(const ude_gated_ffn_desc* d, int32_t pullback, int64_t* bytes) {
    if (!bytes) return UDE_ERR_INVALID;
    if (int rc = check(nullptr, d)) return rc;
    const int e = esize(d->dtype);
    // forward: h; pullback: dg and du side by side, h
    *bytes = pullback ? up256(d->T * wld(2 * wld(d->F)) * e) + up256(d->T * wld(d->F) * e) : up256(d->T * wld(d->F) * e);
    return UDE_OK;
}

extern "C" int ude_gated_ffn_forward_dev(ude_ctx* c, const ude_gated_ffn_desc* d, const void* x, const void* wg, const void* wu, const void* wd,
                                         void* y, float* gate, float* up, void* ws, int64_t ws_bytes) {
    if (!c) return UDE_ERR_INVALID;
    if (int rc = check(c, d)) return rc;
    if (d->T == 0) return UDE_OK;
    int64_t need = 0;
    if (int rc = ude_gated_ffn_workspace(d, 0, &need)) return rc;
    const int e = esize(d->dtype);
    if (!x || !wg || !wu || !wd || !y || !ws) return fail(c, UDE_ERR_INVALID, "gated_ffn: NULL argument");
    if (!gate != !up) return fail(c, UDE_ERR_INVALID, "gated_ffn: gate and up: both or neither");
    if (ws_bytes < need || misaligned(ws, 256)) return fail(c, UDE_ERR_INVALID, "gated_ffn: workspace of %lld bytes (256-byte aligned), got %lld", (long long)need, (long long)ws_bytes);
    if (misaligned(x, e) || misaligned(wg, e) || misaligned(wu, e) || misaligned(wd, e) || misaligned(y, e) || misaligned(gate, 4) || misaligned(up, 4))
        return fail(c, UDE_ERR_INVALID, "gated_ffn: a pointer is not aligned to its element type");
    OnDevice dev(c->device);
    if (!dev.ok) return fail(c, UDE_ERR_HIP, "gated_ffn: device %d", c->device);
    const bool rows = d->w_order == 1;
    Args a{};
    a.A[0] = x, a.lda = d->ldx;
    a.B[0] = wg, a.B[1] = wu, a.ldb[0] = d->ldg, a.ldb[1] = d->ldu;
    a.C[0] = ws, a.ldc[0] = wld(d->F);
    a.M = (int)d->T, a.N = (int)d->F, a.K = (int)d->D, a.nseg = 1, a.act = d->act;
    a.gate = gate, a.up = up;
    if (int rc = launch<EPI_GATE>(c, d->dtype, a, true, rows)) return rc;
    Args b{};
    b.A[0] = ws, b.lda = wld(d->F);
    b.B[0] = wd, b.ldb[0] = d->ldd;
    b.C[0] = y, b.ldc[0] = d->ldy;
    b.M = (int)d->T, b.N = (int)d->O, b.K = (int)d->F, b.nseg = 1;
    return launch<EPI_STORE>(c, d->dtype, b, true, rows);
}

extern "C" int ude_gated_ffn_backward_dev(ude_ctx* c, const ude_gated_ffn_desc* d, const void* x, const void* wg, const void* wu, const void* wd,
                                          const float* gate, const float* up, const void* dy, void* dx, void* dwg, void* dwu, void* dwd,
                                          void* ws, int64_t ws_bytes) {
    if (!c) return UDE_ERR_INVALID;
    if (int rc = check(c, d)) return rc;
    int64_t need = 0;
    if (int rc = ude_gated_ffn_workspace(d, 1, &need)) return rc;
    const int e = esize(d->dtype);
    if (d->T && (!x || !wg || !wu || !wd || !gate || !up || !dy || !ws)) return fail(c, UDE_ERR_INVALID, "gated_ffn: NULL argument");
    if (d->T && (ws_bytes < need || misaligned(ws, 256))) return fail(c, UDE_ERR_INVALID, "gated_ffn: workspace of %lld bytes (256-byte aligned), got %lld", (long long)need, (long long)ws_bytes);
    if (misaligned(x, e) || misaligned(wg, e) || misaligned(wu, e) || misaligned(wd, e) || misaligned(dy, e) || misaligned(dx, e) || misaligned(dwg, e) ||
        misaligned(dwu, e) || misaligned(dwd, e) || misaligned(gate, 4) || misaligned(up, 4))
        return fail(c, UDE_ERR_INVALID, "gated_ffn: a pointer is not aligned to its element type");
    OnDevice dev(c->device);
    if (!dev.ok) return fail(c, UDE_ERR_HIP, "gated_ffn: device %d", c->device);
    const bool rows = d->w_order == 1;
    const int T = (int)d->T, D = (int)d->D, F = (int)d->F, O = (int)d->O;
    const int64_t ldg = wld(2 * wld(F)), ldh = wld(F);
    char* dg = (char*)ws;
    char* du = dg + wld(F) * e;
    char* h = (char*)ws + up256(d->T * ldg * e);
    if (T) {
        Args a{};
        a.A[0] = dy, a.lda = d->ldy;
        a.B[0] = wd, a.ldb[0] = d->ldd;
        a.M = T, a.N = F, a.K = O, a.nseg = 1, a.act = d->act;
        a.gate = (float*)gate, a.up = (float*)up, a.dg = dg, a.du = du, a.h = h, a.ldc[0] = ldg, a.ldc[1] = ldh;
        if (int rc = launch<EPI_PULL>(c, d->dtype, a, true, !rows)) return rc;
    }
    if (dx && T) {
        Args a{};
        a.A[0] = dg, a.A[1] = du, a.lda = ldg;
        a.B[0] = wg, a.B[1] = wu, a.ldb[0] = d->ldg, a.ldb[1] = d->ldu;
        a.C[0] = dx, a.ldc[0] = D;
        a.M = T, a.N = D, a.K = F, a.nseg = 2;
        if (int rc = launch<EPI_STORE>(c, d->dtype, a, true, !rows)) return rc;
    }
    // gradients of the weights in the order of the weights: the axis whose elements are adjacent is n.  (T = 0: an empty sum, zeros.)
    if (dwg || dwu) {
        Args a{};
        int nb = 0;
        for (int i = 0; i < 2; ++i) {
            void* out = i ? dwu : dwg;
            if (!out) continue;
            const char* s = i ? du : dg;
            a.A[nb] = rows ? (const void*)s : x;
            a.B[nb] = rows ? x : (const void*)s;
            a.ldb[nb] = rows ? d->ldx : ldg;
            a.C[nb] = out;
            a.ldc[nb] = rows ? D : F;
            ++nb;
        }
        a.lda = rows ? ldg : d->ldx;
        a.M = rows ? F : D, a.N = rows ? D : F, a.K = T, a.nseg = 1;
        if (int rc = launch<EPI_STORE>(c, d->dtype, a, false, false, nb)) return rc;
    }
    if (dwd) {
        Args a{};
        a.A[0] = rows ? dy : (const void*)h, a.lda = rows ? d->ldy : ldh;
        a.B[0] = rows ? (const void*)h : dy, a.ldb[0] = rows ? ldh : d->ldy;
        a.C[0] = dwd, a.ldc[0] = rows ? F : O;
        a.M = rows ? O : F, a.N = rows ? F : O, a.K = T, a.nseg = 1;
        if (int rc = launch<EPI_STORE>(c, d->dtype, a, false, false)) return rc;
    }
    return UDE_OK;
}
