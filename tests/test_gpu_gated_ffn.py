"""The gated feed-forward block against its Float64 statement, entry by entry within the rounding bounds of tests/_training_ops.py."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")
import _training_ops as R  # noqa: E402

pytestmark = pytest.mark.gpu
KINDS = [torch.bfloat16, torch.float16, torch.float32]
IDS = ["bf16", "fp16", "fp32"]
# (T, D, F, O): single elements, odd sizes, exact tiles, one over a tile, rows that are and are not 16-byte aligned, few and many samples
SIZES = [(1, 1, 1, 1), (1, 64, 64, 64), (2, 300, 500, 128), (3, 5, 7, 9), (16, 512, 200, 96), (17, 100, 110, 100), (33, 1000, 72, 40),
         (64, 64, 64, 64), (65, 96, 130, 33), (130, 257, 66, 129), (300, 128, 64, 256), (513, 136, 264, 520), (1500, 40, 48, 24)]


def made(T, D, F, O, kind, rows, seed=0, gap=0):
    """x, wg, wu, wd, dy on the GPU; gap > 0: every matrix is a view whose gaps hold NaN"""
    gen = torch.Generator().manual_seed(seed)

    def matrix(r, c, by, by_rows=True):
        if not by_rows:
            return matrix(c, r, by).T
        t = torch.full((r, c + gap), float("nan"), dtype=kind, device="cuda")
        t[:, :c] = (torch.randn((r, c), generator=gen) * by).to(kind).cuda()
        return t[:, :c]

    return (matrix(T, D, 1.0), matrix(F, D, D ** -0.5, rows), matrix(F, D, D ** -0.5, rows), matrix(O, F, F ** -0.5, rows), matrix(T, O, 1.0))


def check(x, wg, wu, wd, dy, act="swish"):
    import universal_differential_equations_amd as U
    want = R.gated(x, wg, wu, wd, act, dy)
    plain = U.gated_ffn(x, wg, wu, wd, act=act)
    y, saved = U.gated_ffn(x, wg, wu, wd, act=act, save=True)
    got = dict(zip(("dx", "dwg", "dwu", "dwd"), U.gated_ffn_pullback(saved, dy)), y=y, gate=saved.gate[0], up=saved.gate[1])
    for name, value in got.items():
        assert value.shape == want[name][0].shape and (name in ("gate", "up") or value.dtype == x.dtype)
        assert R.within(value, want[name]) <= 1, (name, R.within(value, want[name]))
    assert R.within(plain, want["y"]) <= 1
    for name, w in zip(("dwg", "dwu", "dwd"), (wg, wu, wd)):
        if min(w.shape) > 1:
            assert (got[name].stride(1) == 1) == (w.stride(1) == 1)
    return got


@pytest.mark.parametrize("rows", [True, False], ids=["rows", "cols"])
@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_forward_and_pullback(size, kind, rows):
    check(*made(*size, kind, rows))


@pytest.mark.parametrize("act", sorted(R.ACTS))
@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_activations(act, kind):
    check(*made(70, 64, 100, 40, kind, True, seed=1), act=act)


@pytest.mark.parametrize("rows", [True, False], ids=["rows", "cols"])
@pytest.mark.parametrize("gap", [1, 8, 24])
@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_views_with_gaps(kind, gap, rows):
    """leading dimensions larger than the rows, NaN in the gaps: nothing outside the matrices is used"""
    check(*made(37, 72, 88, 56, kind, rows, seed=2, gap=gap))
    check(*made(140, 264, 136, 72, kind, rows, seed=3, gap=gap))


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_views_that_start_off_alignment(kind):
    """one element behind an aligned address; gate and up weights as halves of one matrix; x with more than two axes"""
    x, wg, wu, wd, dy = made(40, 65, 80, 33, kind, True, seed=4)
    check(x[:, 1:], wg[:, 1:], wu[:, 1:], wd, dy)
    both = torch.cat((wg, wu))
    check(x, both[:80], both[80:], wd, dy)
    import universal_differential_equations_amd as U
    y, saved = U.gated_ffn(x.view(5, 8, 65), wg, wu, wd, save=True)
    dx = U.gated_ffn_pullback(saved, dy.view(5, 8, 33))[0]
    flat, saved2 = U.gated_ffn(x, wg, wu, wd, save=True)
    assert y.shape == (5, 8, 33) and dx.shape == (5, 8, 65)
    assert torch.equal(y.view(40, 33), flat) and torch.equal(dx.view(40, 65), U.gated_ffn_pullback(saved2, dy)[0])


@pytest.mark.parametrize("size", [(1, 2048, 1100, 640), (7, 640, 2048, 1100), (300, 1100, 640, 2048), (1030, 512, 776, 512), (2100, 64, 520, 72), (4000, 200, 72, 136)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_larger(size, kind):
    for rows in (True, False):
        check(*made(*size, kind, rows, seed=5))


@pytest.mark.parametrize("size", [(72, 2052, 4100, 264), (2100, 328, 2310, 2050), (4100, 2052, 136, 72), (4100, 72, 2056, 136), (4096, 256, 2048, 2048)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("kind", KINDS[:2], ids=IDS[:2])
def test_many_large_tiles(size, kind):
    """enough output for the largest tiles in each of the products, inner sizes that end inside a step of 64 among them"""
    for rows in (True, False):
        check(*made(*size, kind, rows, seed=15))


@pytest.mark.parametrize("size", [(1, 4096, 1408, 512), (24, 1000, 2730, 264), (32, 2048, 512, 4100), (33, 72, 5000, 136), (200, 136, 3000, 80), (3000, 72, 136, 264), (600, 2056, 72, 1032)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("kind", KINDS[:2], ids=IDS[:2])
def test_products_cut_along_k(size, kind):
    """few tiles and a long inner axis: parts of K, some of them across the two halves of dx's product, some empty; the same bits twice"""
    import universal_differential_equations_amd as U
    for rows in (True, False):
        s = made(*size, kind, rows, seed=16)
        got = check(*s)
        y, saved = U.gated_ffn(*s[:4], save=True)
        again = dict(zip(("dx", "dwg", "dwu", "dwd"), U.gated_ffn_pullback(saved, s[4])), y=y)
        assert all(torch.equal(got[k], again[k]) for k in again)


@pytest.mark.parametrize("T", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_few_rows(T, kind):
    """at most a handful of samples: aligned rows whose last k do not fill 16 bytes, output columns that no wavefront's share divides, NaN in the
    gaps; more k than the lanes take at once; the same bits for a sample alone and next to others of its number of rows"""
    import universal_differential_equations_amd as U
    for size, gap in (((T, 1021, 525, 131), 3), ((T, 3, 11, 5), 5), ((T, 2304, 1029, 64), 3), ((T, 4096, 520, 257), 0)):
        s = made(*size, kind, True, seed=17, gap=gap)
        check(*s)
        x, *w = s[:4]
        y = U.gated_ffn(x, *w)
        assert torch.equal(y, U.gated_ffn(x, *w, save=True)[0])
        x[1:] = 1  # (in place: a copy would have no gaps, and what is aligned is summed in another order)
        assert torch.equal(U.gated_ffn(x, *w)[0], y[0])


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_broadcast_samples_and_cotangents(kind):
    """x and dy as views whose rows are one row, one column among them: what sums and means hand back"""
    for size in ((40, 24, 30, 1), (40, 1, 30, 7)):
        x, wg, wu, wd, dy = made(*size, kind, True, seed=18)
        check(x[:1].expand(40, -1), wg, wu, wd, dy[:1].expand(40, -1))
        check(x, wg, wu, wd, dy[:1, :1].expand(40, size[3]))


@pytest.mark.parametrize("rows", [True, False], ids=["rows", "cols"])
@pytest.mark.parametrize("size", [(6, 29, 45, 13), (70, 61, 45, 93), (300, 1021, 525, 1029), (2061, 1021, 525, 2061), (1101, 93, 4101, 61)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_rows_that_end_inside_16_bytes(size, kind, rows):
    """aligned rows with NaN right behind an end that 16 bytes reach over, in every operand, for small and large tiles: the last step, the only
    one, the last of a part"""
    check(*made(*size, kind, rows, seed=19, gap=3))


def test_very_many_columns():
    """one sample through more hidden columns than a launch of one wavefront per column could have, and a product as long as that: the columns
    at both ends and the one that the output is made of"""
    import universal_differential_equations_amd as U
    D, F = 8, (1 << 26) + 24
    x, dt = torch.linspace(-1, 1, D, device="cuda").view(1, D).bfloat16(), torch.bfloat16
    wg, wu = torch.empty((F, D), dtype=dt, device="cuda").normal_(), torch.empty((F, D), dtype=dt, device="cuda").normal_()
    wd = torch.zeros((1, F), dtype=dt, device="cuda")
    wd[0, F - 3] = 1
    y, saved = U.gated_ffn(x, wg, wu, wd, act="identity", save=True)
    for at in (0, F // 2, 1 << 25, F - 64):
        for got, w in zip(saved.gate, (wg, wu)):
            p = w[at:at + 64].double() * x.double()
            # eight products, each exact in Float32, and at most eight sums
            assert bool(((got[0, at:at + 64].double() - p.sum(1)).abs() <= 8 * 2.0 ** -24 * p.abs().sum(1)).all()), at
    h = (saved.gate[0, 0, F - 3] * saved.gate[1, 0, F - 3]).to(dt)
    assert torch.equal(y[0, 0], h)


def test_against_differences():
    """directional derivatives of sum(y * c) by central differences of the Float64 statement"""
    import universal_differential_equations_amd as U
    T, D, F, O = 9, 20, 30, 12
    x, wg, wu, wd, c = made(T, D, F, O, torch.float32, True, seed=6)
    _, saved = U.gated_ffn(x, wg, wu, wd, act="gelu_tanh", save=True)
    grads = U.gated_ffn_pullback(saved, c)
    gen = torch.Generator(device="cuda").manual_seed(7)
    args = [t.double() for t in (x, wg, wu, wd)]

    def loss(*a):
        return float((R.ACTS["gelu_tanh"][0](a[0] @ a[1].T) * (a[0] @ a[2].T) @ a[3].T * c.double()).sum())

    for i, g in enumerate(grads):
        d = torch.randn(args[i].shape, generator=gen, device="cuda", dtype=torch.float64)
        at = [[a + (s * 1e-5 * d if j == i else 0) for j, a in enumerate(args)] for s in (1, -1)]
        slope = (loss(*at[0]) - loss(*at[1])) / 2e-5
        # truncation (1e-5)^2 and Float64 rounding / 1e-5 are below 1e-8 of the terms; Float32 sums of up to 30 terms: 1e-5
        assert abs(slope - float((g.double() * d).sum())) <= 1e-5 * float((g.double() * d).abs().sum())


def test_rows_are_independent_and_non_finite_rows_stay_alone():
    import universal_differential_equations_amd as U
    x, wg, wu, wd, _ = made(70, 96, 64, 48, torch.bfloat16, True, seed=8)
    y = U.gated_ffn(x, wg, wu, wd)
    bad = x.clone()
    bad[3, 5], bad[69, 0] = float("nan"), float("inf")
    z = U.gated_ffn(bad, wg, wu, wd)
    keep = [i for i in range(70) if i not in (3, 69)]
    assert torch.equal(z[keep], y[keep]) and not torch.isfinite(z[3]).any() and not torch.isfinite(z[69]).all()


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("act", sorted(R.ACTS))
def test_far_gates(act, kind):
    """gates of any size: act and its derivative are finite (0 or 1 or g), so that u = 0 gives dg = 0"""
    import universal_differential_equations_amd as U
    most = 6e4 if kind == torch.float16 else 1e30
    x = torch.tensor([[most], [-most], [200.0], [-200.0], [0.0], [1e-4]], dtype=kind, device="cuda")
    one, zero = torch.ones(1, 1, dtype=kind, device="cuda"), torch.zeros(1, 1, dtype=kind, device="cuda")
    y, saved = U.gated_ffn(x, one, zero, one, act=act, save=True)
    dx, dwg, dwu, dwd = U.gated_ffn_pullback(saved, torch.ones_like(x))
    assert not y.any() and not dwg.any() and not dwd.any() and not dx.any()
    act64 = R.ACTS[act][0](x.double())
    assert torch.isfinite(saved.gate).all() and torch.isfinite(act64).all()
    y, saved = U.gated_ffn(x[2:], one, one, one, act=act, save=True)
    assert torch.isfinite(y).all() and all(torch.isfinite(t).all() for t in U.gated_ffn_pullback(saved, torch.ones_like(y))) or kind == torch.float16


def test_no_samples_and_partial_pullbacks():
    import universal_differential_equations_amd as U
    x, wg, wu, wd, dy = made(0, 24, 16, 40, torch.float16, False)
    y, saved = U.gated_ffn(x, wg, wu, wd, save=True)
    dx, dwg, dwu, dwd = U.gated_ffn_pullback(saved, dy)
    assert y.shape == (0, 40) and dx.shape == (0, 24)
    assert not dwg.any() and not dwu.any() and not dwd.any() and dwg.shape == (16, 24) and dwd.shape == (40, 16)
    x, wg, wu, wd, dy = made(21, 24, 16, 40, torch.float16, False)
    _, saved = U.gated_ffn(x, wg, wu, wd, save=True)
    every = U.gated_ffn_pullback(saved, dy)
    for names in (("x",), ("w_up",), ("w_gate", "w_down"), ()):
        some = U.gated_ffn_pullback(saved, dy, need=names)  # (and a second, third, ... pullback of one forward)
        for name, a, b in zip(("x", "w_gate", "w_up", "w_down"), some, every):
            assert (a is None) == (name not in names) and (a is None or torch.equal(a, b))


def test_output_rows_with_gaps_are_left_alone():
    """ldy > O through the C entry: what lies between the rows of y, and behind its last row, keeps its bits"""
    from universal_differential_equations_amd import _lib
    from universal_differential_equations_amd.layers import _Block
    for T, D, F, O in ((5, 40, 24, 20), (70, 72, 136, 90)):
        x, wg, wu, wd, _ = made(T, D, F, O, torch.bfloat16, True, seed=9)
        b = _Block(x, wg, wu, wd, "swish")
        b.D.ldy = O + 6
        y = torch.full((T + 1, O + 6), 7.0, dtype=torch.bfloat16, device="cuda")
        ws, size = b.workspace(0)
        b.bind()
        b.eng.check(b.eng.L.ude_gated_ffn_forward_dev(b.eng.h, C.byref(b.D), *(t.data_ptr() for t in (x, wg, wu, wd, y)), None, None, ws.data_ptr(), size))
        assert bool((y[:, O:] == 7).all()) and bool((y[T] == 7).all())
        assert R.within(y[:T, :O], R.gated(x, wg, wu, wd, "swish")["y"]) <= 1
        assert _lib.GATE["swish"] == b.D.act


def test_refusals():
    import universal_differential_equations_amd as U
    x, wg, wu, wd, dy = made(8, 24, 16, 40, torch.float16, True)
    for bad in ((x.double(), wg, wu, wd), (x.float(), wg, wu, wd), (x, wg.cpu(), wu, wd), (x, wg[:8], wu, wd), (x, wg, wu[:, :8], wd), (x, wg, wu, wd.T.contiguous()),
                (x[:, :23], wg, wu, wd), (x, wg, wu, wd[:, ::2]), (x, wg.T.contiguous().T, wu, wd), (x, wg[0], wu, wd), (x[:, :0], wg[:, :0], wu[:, :0], wd)):
        with pytest.raises(ValueError):
            U.gated_ffn(*bad)
    with pytest.raises(ValueError):
        U.gated_ffn(x, wg, wu, wd, act="softmax")
    _, saved = U.gated_ffn(x, wg, wu, wd, save=True)
    for bad in (dy.float(), dy[:4], dy[:, :39], dy.cpu()):
        with pytest.raises(ValueError):
            U.gated_ffn_pullback(saved, bad)
    with pytest.raises(ValueError):
        U.gated_ffn_pullback(saved, dy, need=("w",))


def test_workspace_is_checked():
    """too small a workspace, or one off its alignment, is refused before anything is launched"""
    from universal_differential_equations_amd.layers import _Block
    x, wg, wu, wd, _ = made(64, 512, 1408, 512, torch.bfloat16, True)
    b = _Block(x, wg, wu, wd, "swish")
    ws, size = b.workspace(0)
    y = torch.full((64, 512), 7.0, dtype=torch.bfloat16, device="cuda")
    b.bind()
    for at, n in ((ws.data_ptr(), size - 1), (ws.data_ptr() + 16, size), (None, size)):
        assert b.eng.L.ude_gated_ffn_forward_dev(b.eng.h, C.byref(b.D), *(t.data_ptr() for t in (x, wg, wu, wd, y)), None, None, at, n) == -1
    assert bool((y == 7).all())


def test_streams_and_graphs():
    """the same bits on a side stream, and from two captured graphs that are replayed in turn with other inputs and eager work between"""
    import universal_differential_equations_amd as U
    sets = [made(150, 136, 200, 72, torch.bfloat16, True, seed=s) for s in (10, 11)]

    def work(s):
        y, saved = U.gated_ffn(*s[:4], save=True)
        return (y,) + U.gated_ffn_pullback(saved, s[4])

    want = [work(s) for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work(sets[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    torch.cuda.synchronize()
    held = [[t.clone() for t in s] for s in sets]
    graphs, outs = [], []
    for s in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(work(s))
        graphs.append(g)
    for turn in range(3):
        for i in (0, 1):
            src = sets[(i + turn) % 2]
            for a, b in zip(held[i], src):
                a.copy_(b)
            graphs[i].replay()
        eager = work(sets[turn % 2])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, want[turn % 2]))
        for i in (0, 1):
            assert all(torch.equal(a, b) for a, b in zip(outs[i], want[(i + turn) % 2])), (turn, i)


def test_two_threads():
    import threading
    import universal_differential_equations_amd as U
    sets = [made(90, 72, 104, 40, torch.float32, False, seed=s) for s in (12, 13)]
    want = [U.gated_ffn(*s[:4]) for s in sets]
    torch.cuda.synchronize()
    bad = []

    def go(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                if not torch.equal(U.gated_ffn(*sets[i][:4]), want[i]):
                    bad.append(i)

    ts = [threading.Thread(target=go, args=(i,)) for i in (0, 1)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad


def test_pullback_in_another_thread_and_stream():
    """what is saved in one thread and stream is pulled back in others, two at a time, while the first goes on: each thread has a context of its
    own, and the saved activations' memory is not reused before the other stream has read them"""
    import threading
    import universal_differential_equations_amd as U
    sets = [made(90, 72, 104, 40, torch.float32, True, seed=s) for s in (12, 13)]
    want = [U.gated_ffn_pullback(U.gated_ffn(*s[:4], save=True)[1], s[4]) for s in sets]
    torch.cuda.synchronize()
    bad = []

    def go(i, saved, ready):
        stream = torch.cuda.Stream()
        stream.wait_event(ready)
        with torch.cuda.stream(stream):
            got = U.gated_ffn_pullback(saved, sets[i][4])
            del saved
            stream.synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                bad.append(i)

    for _ in range(10):
        ts = []
        for i in (0, 1):
            y, saved = U.gated_ffn(*sets[i][:4], save=True)
            ready = torch.cuda.Event()
            ready.record()
            ts.append(threading.Thread(target=go, args=(i, saved, ready)))
            del y, saved
        [t.start() for t in ts]
        for _ in range(5):
            torch.full((2, 90, 104), float("nan"), device="cuda")  # (the size of what was saved)
        [t.join() for t in ts]
    assert not bad
