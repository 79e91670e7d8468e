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

// Tiles of the 16-bit kinds on the 256 compute units of an MI355X.  Costs in microseconds, measured at long K:
//   256 x 256, one per compute unit:    1.55 a step of 64 k, then the epilogue  (4096 x 4096 x 11264: 271 us = 1395 TFLOP/s)
//   256 x 128, one per compute unit:    0.885                                   (two rounds of the same product: 311 us)
//   128 x 128, two per compute unit:    1.04 for both, about 0.62 where one has the unit alone   (365 us)
//   32 x 128, three per compute unit:   for few rows
// Float32 is bound by its matrix instructions (1/16 of the 16-bit rate) whatever the tile: 128 x 128, 7.4 a step of 32 k.
// The larger the tile, the less is read again; the smaller, the less of the last round stands idle.  EPI_PULL reads two floats and writes
// three values per element between the products: 53, 33 and 20 us a round, hidden by the other workgroup's products where two share a unit.
// Where tiles are few and K is long, K is cut into parts whose sums go through memory (3 TB/s) and one more launch.
constexpr int CUS = 256, MOST_PARTS = 2 * CUS, MOST_PARTS_32 = 3 * CUS;
struct Plan {
    int which;         // 0: 256 x 256, 1: 256 x 128, 2: 128 x 128, 3: whole rounds of 256 x 256, the rest as quarters, 4: 32 x 128
    int64_t big, all;  // tiles of the first launch; of all
    int split;         // 2, 4: parts of K
};
Plan plan(const Args& a, int epi, bool ak, int es) {
    const int H = epi == EPI_GATE ? 2 : 1;
    bool few = ak;  // (32 x 128 reads A by rows)
    for (int i = 0; i < a.nprod; ++i) few = few && a.p[i].M <= 32;
    auto tiles = [&](int bm, int bn) {
        int64_t n = 0;
        for (int i = 0; i < a.nprod; ++i) n += (int64_t)((a.p[i].M + bm - 1) / bm) * ((a.p[i].N + bn / H - 1) / (bn / H));
        return n;
    };
    const int total = a.nseg * ((a.K + 128 / es - 1) / (128 / es));
    const bool pull = epi == EPI_PULL;
    const double steps = total + 3, e2 = pull ? 20 : 8, c2 = es == 4 ? 7.4 : 1.04;
    const double r0 = steps * 1.55 + (pull ? 53 : 10), r1 = steps * 0.885 + (pull ? 33 : 8), r2 = steps * c2 + e2;
    auto small = [&](int64_t n, double r) {
        const int64_t whole = n / (2 * CUS), rest = n % (2 * CUS);
        return whole * r + (rest == 0 ? 0 : rest <= CUS ? 0.62 * r : r);
    };
    const int64_t n0 = tiles(256, 256), n1 = tiles(256, 128), n2 = tiles(few ? 32 : 128, 128), rest = n0 % CUS;
    Plan best = {few ? 4 : 2, n2, n2, 1};
    if (few) {  // bound by reading B: parts until every compute unit has three workgroups, each of 4 steps at least
        const int64_t most = MOST_PARTS_32 / n2 < total / 4 ? MOST_PARTS_32 / n2 : total / 4;
        if (most > 1) best.split = (int)most;
        return best;
    }
    double least = small(n2, r2);
    for (int s = 2; s * n2 <= MOST_PARTS && s * 2 <= total; ++s) {
        const double cost = small(n2 * s, ((total + s - 1) / s + 3) * c2) + n2 * s * (2 * 65536 / 3e6) + e2 + 4;
        if (cost < least) least = cost, best.split = s;
    }
    const double cost[3] = {(n0 + CUS - 1) / CUS * r0, (n1 + CUS - 1) / CUS * r1, n0 > CUS && rest ? n0 / CUS * r0 + small(4 * rest, r2) + 4 : 1e30};
    if (es == 4) return best;
    if (cost[0] < least) least = cost[0], best = {0, n0, n0, 1};
    if (cost[1] < least) least = cost[1], best = {1, n1, n1, 1};
    if (cost[2] < least) least = cost[2], best = {3, n0 - rest, n0, 1};
    return best;
}
// no product of these sizes, nor some of `n` such products side by side, leaves more bytes of parts than this
int64_t part_bytes(int64_t M, int64_t N, int64_t steps, int n) {
    const int64_t all = n * ((M + 127) / 128) * ((N + 63) / 64) * (steps / 2);
    return (all < MOST_PARTS ? all : MOST_PARTS) * 65536;
}
static_assert(MOST_PARTS * 65536 / 2 >= MOST_PARTS_32 * 16384, "parts of 32 rows need less");

// a row starts on a 4-byte boundary, and a tile's offsets fit 31 bits
bool tileable(const void* p, int64_t ld, int e) { return (uintptr_t)p % 4 == 0 && ld * e % 4 == 0 && ld * e < (1 << 23); }

template <class T, int EPI, bool AK, bool BKc>
int launch3(ude_ctx* c, Args a, bool tile) {
    a.split = 1;
    constexpr bool WIDE = sizeof(typename T::E) == 2;  // (the tiles of 256 rows)
    {
        const Plan p = plan(a, EPI, AK, sizeof(typename T::E));
        if (tile && p.big < 1 << 22 && p.all < 1 << 22) {
            a.split = p.split;
            const dim3 grid((unsigned)(p.big * p.split)), block(256);
            if (WIDE && (p.which == 0 || p.which == 3)) {
                if constexpr (WIDE) hipLaunchKernelGGL((gemm_tile<T, EPI, AK, BKc, 256, 256, 2, 2, 1>), grid, block, 0, c->stream, a);
            } else if (WIDE && p.which == 1) {
                if constexpr (WIDE) hipLaunchKernelGGL((gemm_tile<T, EPI, AK, BKc, 256, 128, 2, 2, 1>), grid, block, 0, c->stream, a);
            } else if (p.which == 2)
                hipLaunchKernelGGL((gemm_tile<T, EPI, AK, BKc, 128, 128, 2, 2, 2>), grid, block, 0, c->stream, a);
            else if constexpr (AK)
                hipLaunchKernelGGL((gemm_tile<T, EPI, AK, BKc, 32, 128, 1, 4, 3>), grid, block, 0, c->stream, a);
            HIPCHK(c, hipGetLastError());
            if (p.which == 3) {
                a.first = (int)p.big, a.quarters = 1;
                hipLaunchKernelGGL((gemm_tile<T, EPI, AK, BKc, 128, 128, 2, 2, 2>), dim3((unsigned)(4 * (p.all - p.big))), block, 0, c->stream, a);
                HIPCHK(c, hipGetLastError());
            }
            if (p.split > 1) {
                if (p.which == 2)
                    hipLaunchKernelGGL((join_parts<T, EPI, 128, 128, 2, 2>), dim3((unsigned)p.big, 4), block, 0, c->stream, a);
                else
                    hipLaunchKernelGGL((join_parts<T, EPI, 32, 128, 1, 4>), dim3((unsigned)p.big, 2), block, 0, c->stream, a);
                HIPCHK(c, hipGetLastError());
            }
            return UDE_OK;
        }
    }
    constexpr int NT = EPI == EPI_GATE ? 32 : 64;
    int64_t n = 0;
    for (int i = 0; i < a.nprod; ++i) {
        const int64_t t = (int64_t)((a.p[i].M + 63) / 64) * ((a.p[i].N + NT - 1) / NT);
        n = t > n ? t : n;
    }
    if (n >= 1 << 24) return fail(c, UDE_ERR_UNSUPPORTED, "gated_ffn: %lld tiles", (long long)n);
    hipLaunchKernelGGL((gemm_any<T, EPI, AK, BKc>), dim3((unsigned)n, 1, a.nprod), dim3(256), 0, c->stream, a);
    HIPCHK(c, hipGetLastError());
    return UDE_OK;
}
template <class T, int EPI>
int launch2(ude_ctx* c, const Args& a, bool ak, bool bk, bool tile) {
    if constexpr (EPI == EPI_STORE)
        if (!ak) return bk ? fail(c, UDE_ERR_INVALID, "gated_ffn: operand orders") : launch3<T, EPI, false, false>(c, a, tile);
    return bk ? launch3<T, EPI, true, true>(c, a, tile) : launch3<T, EPI, true, false>(c, a, tile);
}
// ak, bk: consecutive k are adjacent
template <int EPI>
int launch(ude_ctx* c, int dtype, Args a, bool ak, bool bk) {
    const int e = esize(dtype);
    bool tile = true;
    const int used = EPI == EPI_GATE || a.nseg > 1 ? 2 : a.nprod;
    for (int i = 0; i < used; ++i) {
        Product& p = a.p[i];
        p.vecA = vec(p.A, p.lda, e), p.vecB = vec(p.B, p.ldb, e);
        p.vecC = (uintptr_t)p.C % (4 * e) == 0 && p.ldc % 4 == 0;
        // gate and up are rows of N floats; dg, du, h lie in the workspace, rows of a multiple of 8
        if (EPI != EPI_STORE && a.gate && (p.N % 4 || (uintptr_t)a.gate % 16 || (uintptr_t)a.up % 16)) p.vecC = 0;
        tile = tile && tileable(p.A, p.lda, e) && tileable(p.B, p.ldb, e);
    }
    if (dtype == UDE_DT_F32) return launch2<F32, EPI>(c, a, ak, bk, tile);
    if (dtype == UDE_DT_F16) return launch2<F16, EPI>(c, a, ak, bk, tile);
    return launch2<BF16, EPI>(c, a, ak, bk, tile);
}

}  // namespace

namespace {
// workspace: forward: h; pullback: dg and du side by side, h; then the parts of the products that are cut along K (one product at a time)
struct Space {
    int64_t ldg, ldh, h, part, all;
};
Space space(const ude_gated_ffn_desc* d, bool pullback) {
    const int e = esize(d->dtype);
    Space s;
    s.ldh = wld(d->F), s.ldg = 2 * s.ldh;
    s.h = pullback ? up256(d->T * s.ldg * e) : 0;
    s.part = s.h + up256(d->T * s.ldh * e);
    s.all = s.part;
    if (d->T) {
        auto steps = [e](int64_t k) { return (k + 128 / e - 1) / (128 / e); };
        const int64_t wide = d->D > d->O ? d->D : d->O;
        const int64_t a = pullback ? part_bytes(d->T, d->F, steps(d->O), 1) : part_bytes(d->T, d->F, steps(d->D), 1);
        const int64_t b = pullback ? part_bytes(d->T, d->D, 2 * steps(d->F), 1) : part_bytes(d->T, d->O, steps(d->F), 1);
        const int64_t g = pullback ? part_bytes(wide, d->F, steps(d->T), 3) : 0, h = pullback ? part_bytes(d->F, wide, steps(d->T), 3) : 0;
        const int64_t most = a > b ? a : b, mostw = g > h ? g : h;
        s.all += most > mostw ? most : mostw;
    }
    return s;
}
}  // namespace

extern "C" int ude_gated_ffn_workspace(const ude_gated_ffn_desc* d, int32_t pullback, int64_t* bytes) {
    if (!bytes) return UDE_ERR_INVALID;
    if (int rc = check(nullptr, d)) return rc;
    *bytes = space(d, pullback != 0).all;
    return UDE_OK;
}

extern "C" int ude_gated_ffn_forward_dev(ude_ctx* c, const ude_gated_ffn_desc* d, const void* x, const void* wg, const void* wu, const void* wd,
                                         void* y, float* gate, float* up, void* ws, int64_t ws_bytes) {
    if (!c) return UDE_ERR_INVALID;
    if (int rc = check(c, d)) return rc;
    if (d->T == 0) return UDE_OK;
    const Space sp = space(d, false);
    const int e = esize(d->dtype);
    if (!x || !wg || !wu || !wd || !y || !ws) return fail(c, UDE_ERR_INVALID, "gated_ffn: NULL argument");
    if (!gate != !up) return fail(c, UDE_ERR_INVALID, "gated_ffn: gate and up: both or neither");
    if (ws_bytes < sp.all || misaligned(ws, 256)) return fail(c, UDE_ERR_INVALID, "gated_ffn: workspace of %lld bytes (256-byte aligned), got %lld", (long long)sp.all, (long long)ws_bytes);
    if (misaligned(x, e) || misaligned(wg, e) || misaligned(wu, e) || misaligned(wd, e) || misaligned(y, e) || misaligned(gate, 4) || misaligned(up, 4))
        return fail(c, UDE_ERR_INVALID, "gated_ffn: a pointer is not aligned to its element type");
    OnDevice dev(c->device);
    if (!dev.ok) return fail(c, UDE_ERR_HIP, "gated_ffn: device %d", c->device);
    const bool rows = d->w_order == 1;
    const int T = (int)d->T, D = (int)d->D, F = (int)d->F, O = (int)d->O;
    Args a{};
    a.nprod = a.nseg = 1, a.K = D, a.act = d->act, a.gate = gate, a.up = up, a.part = (float*)((char*)ws + sp.part);
    a.p[0] = {x, wg, ws, d->ldx, d->ldg, wld(F), T, F};
    a.p[1] = {x, wu, ws, d->ldx, d->ldu, wld(F), T, F};
    if (int rc = launch<EPI_GATE>(c, d->dtype, a, true, rows)) return rc;
    Args b{};
    b.nprod = b.nseg = 1, b.K = F, b.part = a.part;
    b.p[0] = {ws, wd, y, wld(F), d->ldd, d->ldy, T, O};
    return launch<EPI_STORE>(c, d->dtype, b, true, rows);
}

extern "C" int ude_gated_ffn_backward_dev(ude_ctx* c, const ude_gated_ffn_desc* d, const void* x, const void* wg, const void* wu, const void* wd,
                                          const float* gate, const float* up, const void* dy, void* dx, void* dwg, void* dwu, void* dwd,
                                          void* ws, int64_t ws_bytes) {
    if (!c) return UDE_ERR_INVALID;
    if (int rc = check(c, d)) return rc;
    const Space sp = space(d, true);
    const int e = esize(d->dtype);
    if (d->T && (!x || !wg || !wu || !wd || !gate || !up || !dy || !ws)) return fail(c, UDE_ERR_INVALID, "gated_ffn: NULL argument");
    if (d->T && (ws_bytes < sp.all || misaligned(ws, 256))) return fail(c, UDE_ERR_INVALID, "gated_ffn: workspace of %lld bytes (256-byte aligned), got %lld", (long long)sp.all, (long long)ws_bytes);
    if (misaligned(x, e) || misaligned(wg, e) || misaligned(wu, e) || misaligned(wd, e) || misaligned(dy, e) || misaligned(dx, e) || misaligned(dwg, e) ||
        misaligned(dwu, e) || misaligned(dwd, e) || misaligned(gate, 4) || misaligned(up, 4))
        return fail(c, UDE_ERR_INVALID, "gated_ffn: a pointer is not aligned to its element type");
    OnDevice dev(c->device);
    if (!dev.ok) return fail(c, UDE_ERR_HIP, "gated_ffn: device %d", c->device);
    const bool rows = d->w_order == 1;
    const int T = (int)d->T, D = (int)d->D, F = (int)d->F, O = (int)d->O;
    const int64_t ldg = sp.ldg, ldh = sp.ldh;
    char* dg = (char*)ws;
    char* du = dg + ldh * e;
    char* h = (char*)ws + sp.h;
    float* part = (float*)((char*)ws + sp.part);
    if (T) {
        Args a{};
        a.nprod = a.nseg = 1, a.K = O, a.act = d->act;
        a.p[0] = {dy, wd, dg, d->ldy, d->ldd, ldg, T, F};
        a.gate = (float*)gate, a.up = (float*)up, a.dg = dg, a.du = du, a.h = h, a.ldh = ldh, a.part = part;
        if (int rc = launch<EPI_PULL>(c, d->dtype, a, true, !rows)) return rc;
    }
    if (dx && T) {
        Args a{};
        a.nprod = 1, a.nseg = 2, a.K = F, a.part = part;
        a.p[0] = {dg, wg, dx, ldg, d->ldg, D, T, D};
        a.p[1] = {du, wu, dx, ldg, d->ldu, D, T, D};
        if (int rc = launch<EPI_STORE>(c, d->dtype, a, true, !rows)) return rc;
    }
    // gradients of the weights in the order of the weights, side by side in one launch: the axis whose elements are adjacent is n.
    // (T = 0: an empty sum, zeros.)
    Args a{};
    a.nseg = 1, a.K = T, a.part = part;
    auto add = [&](const void* out, const void* in, int64_t ldout, int64_t ldin, void* grad, int no, int ni) {
        if (!grad) return;
        if (rows)
            a.p[a.nprod++] = {out, in, grad, ldout, ldin, ni, no, ni};
        else
            a.p[a.nprod++] = {in, out, grad, ldin, ldout, no, ni, no};
    };
    add(dg, x, ldg, d->ldx, dwg, F, D);
    add(du, x, ldg, d->ldx, dwu, F, D);
    add(dy, h, d->ldy, ldh, dwd, O, F);
    return a.nprod ? launch<EPI_STORE>(c, d->dtype, a, false, false) : (int)UDE_OK;
}
