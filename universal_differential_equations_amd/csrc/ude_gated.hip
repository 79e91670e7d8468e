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
    if (d->T * d->F > (int64_t)1 << 58)  // (three such matrices of four bytes an element: the workspace's size has to fit 64 bits)
        return fail(c, UDE_ERR_UNSUPPORTED, "gated_ffn: a hidden layer of T x F = %lld x %lld", (long long)d->T, (long long)d->F);
    const int64_t gcols = d->w_order ? d->D : d->F, dcols = d->w_order ? d->F : d->O;
    if (d->ldx < d->D || d->ldy < d->O || d->ldg < gcols || d->ldu < gcols || d->ldd < dcols || d->ldx > most || d->ldy > most || d->ldg > most || d->ldu > most || d->ldd > most)
        return fail(c, UDE_ERR_INVALID, "gated_ffn: a leading dimension is smaller than what it spans, or over 2^31");
    return UDE_OK;
}

int misaligned(const void* p, int e) { return (uintptr_t)p % e != 0; }

int vec(const void* p, int64_t ld, int e) { return (uintptr_t)p % 16 == 0 && ld * e % 16 == 0; }

// Tiles on the 256 compute units of an MI355X: microseconds that a step of 128 bytes of k takes with 1, 2, 3 workgroups on a compute unit, and
// the start and epilogue of a round, as measured (kernel times over products of 64 x 512 x 1408 to 4096 x 4096 x 11264).
//   256 x 256: the least that is read again: 4096 x 4096 x 11264 in 279 us at best and 298 in the median of a profiled run (1355 and 1268 TFLOP/s: the
//   card's clock); in the run that these times were fitted to 271, with 256 x 128 311 and with 128 x 128 365.
//   The smaller ones leave less of the last round idle, but a step costs them 0.25 to 0.5 however little there is in it (LDS, barrier, the
//   loads' way: 64 x 64 takes 0.28 with its loads four steps ahead, 0.41 with two), so that they are for small products, and for Float32, whose matrix instructions (1/16 of the 16-bit rate) bound it with
//   any tile.
// EPI_GATE writes ten bytes an element at the end, EPI_PULL reads eight and writes six: with one workgroup on a compute unit nothing is
// multiplied meanwhile, so that a pull of 4096 x 5632 x 2048 is done in 159 us by 128 x 128 tiles, 171 by 256 x 256 and pieces, 185 by 256 x 128.  Where tiles are few and K is long, K is cut into
// parts whose sums go through caches and memory (there and back: 5 TB/s, 2.2 past 16 MB) and one more launch (5 us).
constexpr int CUS = 256;
constexpr int64_t MOST_PART_BYTES = (int64_t)2 * CUS * 128 * 128 * 4;
enum { T256 = 0, T256x128 = 1, T128 = 2, T64 = 3, T32 = 4, TILES = 5 };
struct Tile {
    int bm, bn, bn_gate;             // EPI_GATE: of which half are output columns
    int slots, slots32;              // workgroups of a compute unit, 16-bit kinds and Float32
    double step[3], gate[3];         // 16-bit kinds; EPI_GATE's where its tile is another
    double step32[3], gate32[3];     // Float32 (0: there is none)
    double end[3];                   // EPI_STORE, EPI_GATE, EPI_PULL
};
constexpr Tile TILE[TILES] = {
    {256, 256, 256, 1, 1, {1.46}, {1.46}, {}, {}, {12, 20, 60}},
    {256, 128, 128, 1, 1, {0.85}, {0.85}, {}, {}, {9, 13, 34}},
    {128, 128, 128, 2, 2, {0.48, 1.02}, {0.48, 1.02}, {1.95, 3.8}, {1.95, 3.8}, {7, 9, 20}},
    {64, 64, 128, 2, 3, {0.28, 0.46}, {0.40, 0.64}, {0.54, 1.08, 1.6}, {1.08, 2.1, 3.2}, {5, 6, 7}},
    {32, 128, 128, 3, 3, {0.46, 0.50, 0.65}, {0.46, 0.50, 0.65}, {0.55, 1.1, 1.65}, {0.55, 1.1, 1.65}, {5, 6, 7}}};
struct Plan {
    int which, split;  // tile; parts of K
    int rest;          // not 0: a second launch does the tiles that do not fill a round, as pieces with so many parts of K
    int64_t big, all;  // tiles of the first launch; of all
};
int64_t tiles_of(const Args& a, int epi, int which) {
    const int bm = TILE[which].bm, bn = epi == EPI_GATE ? TILE[which].bn_gate / 2 : TILE[which].bn;
    int64_t n = 0;
    for (int i = 0; i < a.nprod; ++i) n += (int64_t)((a.p[i].M + bm - 1) / bm) * ((a.p[i].N + bn - 1) / bn);
    return n;
}
int slots_of(int which, int es) { return es == 4 ? TILE[which].slots32 : TILE[which].slots; }
double tiles_cost(int which, int epi, int es, int64_t n, double steps) {
    const Tile& t = TILE[which];
    const double* c = epi == EPI_GATE ? (es == 4 ? t.gate32 : t.gate) : (es == 4 ? t.step32 : t.step);
    const int slots = slots_of(which, es);
    const int64_t whole = n / (slots * CUS), rest = (n % (slots * CUS) + CUS - 1) / CUS;
    return whole * (steps * c[slots - 1] + t.end[epi]) + (rest ? steps * c[rest - 1] + t.end[epi] : 0);
}
int64_t part_size(int which, int epi) { return (int64_t)TILE[which].bm * (epi == EPI_GATE ? TILE[which].bn_gate : TILE[which].bn) * 4; }
// what the rest of a product is done with, and how many of them make a tile
int piece_of(int which) { return which == T128 ? T64 : T128; }
int cols_of(int which, int epi) { return epi == EPI_GATE ? TILE[which].bn_gate / 2 : TILE[which].bn; }
int pieces_of(int which, int epi) { return TILE[which].bm / TILE[piece_of(which)].bm * (cols_of(which, epi) / cols_of(piece_of(which), epi)); }
// the least that n tiles cost with K whole or cut into parts; room: bytes of workspace for them
double cut(int which, int epi, int es, int64_t n, int total, int64_t room, int* parts) {
    double least = tiles_cost(which, epi, es, n, total);
    *parts = 1;
    for (int s = 2; s * n <= slots_of(which, es) * CUS && s * n * part_size(which, epi) <= room && s * 2 <= total; ++s) {
        const double bytes = (double)(n * s * part_size(which, epi)), far = bytes > 16e6 ? bytes - 16e6 : 0;
        const double c = tiles_cost(which, epi, es, n * s, (total + s - 1) / s) + bytes / 2.5e6 + far / 2e6 + 5;
        if (c < least) least = c, *parts = s;
    }
    return least;
}
Plan plan(const Args& a, int epi, bool ak, int es, int64_t room) {
    const int total = a.nseg * ((a.K + 128 / es - 1) / (128 / es));
    bool few = ak;
    for (int i = 0; i < a.nprod; ++i) few = few && a.p[i].M <= 32;
    if (few) {  // bound by reading B: parts until every compute unit has three workgroups, each of 4 steps at least
        const int64_t n = tiles_of(a, epi, T32), fit = room / (n * part_size(T32, epi));
        int64_t most = 3 * CUS / n < total / 4 ? 3 * CUS / n : total / 4;
        most = most < fit ? most : fit;
        return {T32, most > 1 ? (int)most : 1, 0, n, n};
    }
    Plan best{};
    double least = 1e30;
    for (int which = 0; which < TILES; ++which) {
        if ((es == 4 && TILE[which].step32[0] == 0) || (which == T32 && !ak)) continue;
        const int64_t n = tiles_of(a, epi, which);
        const double cost = tiles_cost(which, epi, es, n, total);
        if (cost < least) least = cost, best = {which, 1, 0, n, n};
        if (which <= T128 && n > CUS && n % CUS) {
            int parts;
            const double c = tiles_cost(which, epi, es, n - n % CUS, total) + cut(piece_of(which), epi, es, pieces_of(which, epi) * (n % CUS), total, room, &parts) + 2;
            if (c < least) least = c, best = {which, 1, parts, n - n % CUS, n};
        }
        if (which < T128) continue;
        int parts;
        const double c = cut(which, epi, es, n, total, room, &parts);
        if (c < least) least = c, best = {which, parts, 0, n, n};
    }
    return best;
}
// Whether few_rows takes a product of up to four rows, and the tiles the others.  A wavefront has its rows of B to itself, so that few and long ones
// take as long as their steps do one after the other, and many short ones as long as their starts and sums over the lanes: microseconds of a
// step, and of 1024 wavefronts, as measured for one, two and four rows (128 x 2048 x 64 to 128 x 65536 x 2048).  The tiles cut K where it is
// long, for 8 us of joining.  One row of BFloat16, K x N: 8192 x 64 in 10 us (tiles: 15), 32768 x 64 in 30 (24), 16384 x 2048 in 24 (31), 65536 x 2048
// in 85 (72), 128 x 32768 in 14 (6); four rows: 2048 x 64 in 11 (12), 8192 x 64 in 23 (15).
constexpr double FEW_STEP[3] = {0.5, 0.6, 1.0}, FEW_STEP32[3] = {0.25, 0.43, 0.84}, FEW_WAVES[3] = {0.44, 0.75, 1.1};
bool few(const Args& a, int epi, int es, bool tile) {
    const Product& p = a.p[0];
    if (p.M > 4 || a.nprod > 1 || a.nseg > 1 || !p.vecA || !p.vecB || (epi == EPI_GATE && !a.p[1].vecB)) return false;
    if (p.N >= 1 << 25) return false;  // (a launch has fewer than 2^32 threads, 64 for a column at most)
    const int rows = p.M == 1 ? 0 : p.M == 2 ? 1 : 2;
    const double steps = a.K * (es / 1024.0), waves = (double)p.N * (epi == EPI_GATE ? 2 : 1) / (rows ? 4 : 2);
    const double one = steps * (es == 4 ? FEW_STEP32 : FEW_STEP)[rows], all = waves / 1024 * FEW_WAVES[rows];
    const double read = (double)p.N * a.K * es * (epi == EPI_GATE ? 2 : 1) / 5.7e6, tiles = (0.2 * steps > read ? 0.2 * steps : read) + (steps < 1 ? 3 : 8);
    return !tile || (one > all ? one : all) <= tiles;
}
// no product of these sizes, nor some of `n` such products side by side, leaves more bytes of parts than this
int64_t part_bytes(int64_t M, int64_t N, int64_t steps, int n) {
    const double all = (double)n * ((M + 127) / 128) * ((N + 63) / 64) * (steps / 2);  // (exact where it counts; part bytes of a tile go with its area: the largest tile's)
    return all < MOST_PART_BYTES / 65536 ? (int64_t)all * 65536 : MOST_PART_BYTES;
}

// a row starts on a 4-byte boundary, and a tile's offsets fit 31 bits
bool tileable(const void* p, int64_t ld, int e) { return (uintptr_t)p % 4 == 0 && ld * e % 4 == 0 && ld * e < (1 << 23); }

template <class T, int EPI, bool AK, bool BKc>
int launch3(ude_ctx* c, Args a, bool tile) {
    if constexpr (EPI != EPI_PULL && AK && BKc) {
        if (few(a, EPI, sizeof(typename T::E), tile)) {
            const int M = a.p[0].M;
            auto go = [&](auto kernel, int columns) { hipLaunchKernelGGL(kernel, dim3((unsigned)((a.p[0].N + 4 * columns - 1) / (4 * columns))), dim3(256), 0, c->operators(), a); };
            if (M == 1) go(few_rows<T, EPI, 1>, Few<EPI, 1>::NT);
            else if (M == 2) go(few_rows<T, EPI, 2>, Few<EPI, 2>::NT);
            else go(few_rows<T, EPI, 4>, Few<EPI, 4>::NT);
            HIPCHK(c, hipGetLastError());
            return UDE_OK;
        }
    }
    const Plan p = plan(a, EPI, AK, sizeof(typename T::E), a.room);
    if (tile && p.big * p.split < 1 << 22 && p.all < 1 << 22) {
        constexpr bool GATE = EPI == EPI_GATE, HALF = sizeof(typename T::E) == 2;
        const dim3 block(256);
        auto go = [&](auto kernel, dim3 g) { hipLaunchKernelGGL(kernel, g, block, 0, c->operators(), a); };
        // `tiles` of a kind, each cut into `split` parts
        auto run = [&](int which, int64_t tiles, int split) {
            a.split = split, a.tiles = (int)tiles;
            const dim3 grid((unsigned)(tiles * split));
            if constexpr (HALF) {
                if (which == T256) go(gemm_tile<T, EPI, AK, BKc, 256, 256, 2, 2, 1, 0>, grid);
                if (which == T256x128) go(gemm_tile<T, EPI, AK, BKc, 256, 128, 2, 2, 1, 0>, grid);
            }
            if (which == T128) go(gemm_tile<T, EPI, AK, BKc, 128, 128, 2, 2, 2, 0>, grid);
            if (which == T64) go(gemm_tile<T, EPI, AK, BKc, 64, GATE ? 128 : 64, 2, 2, HALF || GATE ? 2 : 3, HALF ? (GATE ? 3 : 4) : 0>, grid);
            if constexpr (AK)
                if (which == T32) go(gemm_tile<T, EPI, AK, BKc, 32, 128, 1, 4, 3, 0>, grid);
            HIPCHK(c, hipGetLastError());
            if (split > 1) {
                if (which == T128) go(join_parts<T, EPI, 128, 128, 2, 2>, dim3((unsigned)tiles, 4, GATE ? 2 : 4));
                if (which == T64) go(join_parts<T, EPI, 64, GATE ? 128 : 64, 2, 2>, dim3((unsigned)tiles, 2, 2));
                if (which == T32) go(join_parts<T, EPI, 32, 128, 1, 4>, dim3((unsigned)tiles, 2, GATE ? 1 : 2));
                HIPCHK(c, hipGetLastError());
            }
            return (int)UDE_OK;
        };
        if (int rc = run(p.which, p.big, p.split)) return rc;
        if (p.rest) {
            a.first = (int)p.big, a.tm = TILE[p.which].bm, a.tn = cols_of(p.which, EPI);
            return run(piece_of(p.which), pieces_of(p.which, EPI) * (p.all - p.big), p.rest);
        }
        return UDE_OK;
    }
    a.split = 1;
    constexpr int NT = EPI == EPI_GATE ? 32 : 64;
    int64_t n = 0;
    for (int i = 0; i < a.nprod; ++i) {
        const int64_t t = (int64_t)((a.p[i].M + 63) / 64) * ((a.p[i].N + NT - 1) / NT);
        n = t > n ? t : n;
    }
    if (n >= 1 << 24) return fail(c, UDE_ERR_UNSUPPORTED, "gated_ffn: %lld tiles", (long long)n);
    hipLaunchKernelGGL((gemm_any<T, EPI, AK, BKc>), dim3((unsigned)n, 1, a.nprod), dim3(256), 0, c->operators(), a);
    HIPCHK(c, hipGetLastError());
    return UDE_OK;
}
template <class T, int EPI>
int launch2(ude_ctx* c, const Args& a, bool ak, bool bk, bool tile) {
    if constexpr (EPI == EPI_STORE)
        if (!ak) return bk ? fail(c, UDE_ERR_INVALID, "gated_ffn: operand orders") : launch3<T, EPI, false, false>(c, a, tile);
    return bk ? launch3<T, EPI, true, true>(c, a, tile) : launch3<T, EPI, true, false>(c, a, tile);
}
// rows begin on a multiple of so many elements
int begins(const void* p, int64_t ld, int e) {
    return (uintptr_t)p % (4 * e) == 0 && ld % 4 == 0 ? 4 : (uintptr_t)p % (2 * e) == 0 && ld % 2 == 0 ? 2 : 1;
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
        p.vecC = begins(p.C, p.ldc, e);
        tile = tile && tileable(p.A, p.lda, e) && tileable(p.B, p.ldb, e);
    }
    const int g = begins(a.gate, a.p[0].N, 4), u = begins(a.up, a.p[0].N, 4);
    a.vecG = g < u ? g : u;
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
    a.nprod = a.nseg = 1, a.K = D, a.act = d->act, a.gate = gate, a.up = up, a.part = (float*)((char*)ws + sp.part), a.room = sp.all - sp.part;
    a.p[0] = {x, wg, ws, d->ldx, d->ldg, wld(F), T, F};
    a.p[1] = {x, wu, ws, d->ldx, d->ldu, wld(F), T, F};
    if (int rc = launch<EPI_GATE>(c, d->dtype, a, true, rows)) return rc;
    Args b{};
    b.nprod = b.nseg = 1, b.K = F, b.part = a.part, b.room = a.room;
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
    const int64_t room = sp.all - sp.part;
    if (T) {
        Args a{};
        a.nprod = a.nseg = 1, a.K = O, a.act = d->act;
        a.p[0] = {dy, wd, dg, d->ldy, d->ldd, ldg, T, F};
        a.gate = (float*)gate, a.up = (float*)up, a.dg = dg, a.du = du, a.h = h, a.ldh = ldh, a.part = part, a.room = room;
        if (int rc = launch<EPI_PULL>(c, d->dtype, a, true, !rows)) return rc;
    }
    if (dx && T) {
        Args a{};
        a.nprod = 1, a.nseg = 2, a.K = F, a.part = part, a.room = room;
        a.p[0] = {dg, wg, dx, ldg, d->ldg, D, T, D};
        a.p[1] = {du, wu, dx, ldg, d->ldu, D, T, D};
        if (int rc = launch<EPI_STORE>(c, d->dtype, a, true, !rows)) return rc;
    }
    // gradients of the weights in the order of the weights, side by side in one launch: the axis whose elements are adjacent is n.
    // (T = 0: an empty sum, zeros.)
    Args a{};
    a.nseg = 1, a.K = T, a.part = part, a.room = room;
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
