"""The training operators on more than one stream and thread: what they keep, what they wait for."""
import threading

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def made(T, D, F, O, kind, seed):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=gen) * by).to(kind).cuda()
            for s, by in (((D, T), 1.0), ((F, D), D ** -0.5), ((F, D), D ** -0.5), ((O, F), F ** -0.5), ((T, O), 1.0))]


def occupy(n=24):
    """some milliseconds of work on the current stream"""
    a = torch.ones((4096, 4096), device="cuda")
    for _ in range(n):
        a = (a @ a).mul_(2.0 ** -12)
    return a


def fill_with_nan(shapes, kind):
    """what the allocator hands out next on the current stream, in the sizes of what a call holds"""
    return [torch.full(s, float("nan"), dtype=k, device="cuda") for s in shapes for k in (kind, torch.float32) for _ in range(4)]


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("view", [lambda x: x.T, lambda x: x.T.reshape(30, 20, 72), lambda x: x.T[:1].expand(600, -1)], ids=["transposed", "three axes", "broadcast"])
def test_pullback_on_another_stream_after_saved_is_dropped(view, kind):
    """x is copied by the forward call, and `saved` is dropped while the other stream has not reached the pullback: the copy's memory, and that
    of gate and up, is not given to new work of the forward's stream before"""
    import universal_differential_equations_amd as U
    T, D, F, O = 600, 72, 104, 40
    xt, wg, wu, wd, dy = made(T, D, F, O, kind, 21)
    x = view(xt)
    dy = dy.view(*x.shape[:-1], O)
    want = U.gated_ffn_pullback(U.gated_ffn(x, wg, wu, wd, save=True)[1], dy)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(5):
        saved = U.gated_ffn(x, wg, wu, wd, save=True)[1]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            occupy()
            got = U.gated_ffn_pullback(saved, dy)
        del saved
        held = fill_with_nan([(T, D), (2, T, F)], kind)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        del held, got


def test_pullbacks_in_threads_that_hold_the_last_reference():
    """each thread takes its `saved` out of a list, so that its own reference is the last one; every comparison is counted, every error kept"""
    import universal_differential_equations_amd as U
    T, D, F, O = 90, 72, 104, 40
    sets = [made(T, D, F, O, torch.float32, s) for s in (22, 23)]
    want = [U.gated_ffn_pullback(U.gated_ffn(s[0].T, *s[1:4], save=True)[1], s[4]) for s in sets]
    torch.cuda.synchronize()
    good, bad = [], []

    def go(i, box, ready):
        try:
            stream = torch.cuda.Stream()
            stream.wait_event(ready)
            with torch.cuda.stream(stream):
                occupy(4)
                got = U.gated_ffn_pullback(box.pop(), sets[i][4])
                stream.synchronize()
            (good if all(torch.equal(a, b) for a, b in zip(got, want[i])) else bad).append(i)
        except Exception as e:  # (an error in a thread would otherwise be lost)
            bad.append(e)

    for _ in range(5):
        ts = []
        for i in (0, 1):
            box = [U.gated_ffn(sets[i][0].T, *sets[i][1:4], save=True)[1]]
            ready = torch.cuda.Event()
            ready.record()
            ts.append(threading.Thread(target=go, args=(i, box, ready)))
            del box
        [t.start() for t in ts]
        for _ in range(5):
            fill_with_nan([(T, D), (2, T, F)], torch.float32)
        [t.join() for t in ts]
    assert not bad and len(good) == 10


def test_forward_calls_of_two_threads_are_all_compared():
    import universal_differential_equations_amd as U
    sets = [made(90, 72, 104, 40, torch.float32, s) for s in (24, 25)]
    want = [U.gated_ffn(s[0].T, *s[1:4]) for s in sets]
    torch.cuda.synchronize()
    good, bad = [], []

    def go(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    (good if torch.equal(U.gated_ffn(sets[i][0].T, *sets[i][1:4]), want[i]) else bad).append(i)
        except Exception as e:
            bad.append(e)

    ts = [threading.Thread(target=go, args=(i,)) for i in (0, 1)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad and len(good) == 40


@pytest.mark.parametrize("kw", [dict(bits=32), dict(bits=8, capturable=True), dict(bits=32, master=True)], ids=["32", "8", "copies"])
def test_adamw_dropped_while_its_step_is_pending_on_another_stream(kw):
    """its states' memory is not given to new work of the stream that made them: the step would write into that"""
    from universal_differential_equations_amd import training
    kind = torch.bfloat16 if kw.get("master") else torch.float32
    n = 30000
    start, g = torch.linspace(-1, 1, n, device="cuda").to(kind), torch.ones(n, dtype=kind, device="cuda")
    p = start.clone()
    training.AdamW([p], **kw).step([g])
    want = p.clone()
    side = torch.cuda.Stream()
    for _ in range(3):
        p.copy_(start)
        opt = training.AdamW([p], **kw)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            occupy()
            opt.step([g])
        del opt
        held = [torch.full((k,), 3, dtype=dt, device="cuda") for dt, k in ((torch.float32, n), (torch.int8, n), (torch.uint8, n), (torch.float32, -(-n // 256)), (torch.int64, 1))
                for _ in range(6)]
        torch.cuda.synchronize()
        assert torch.equal(p, want) and all(bool((t == 3).all()) for t in held)
        del held


def test_captured_pullback_of_an_eager_forward():
    """the forward call on the main stream, its pullback captured on another and replayed three times with other cotangents and eager work between; what
    was saved is dropped in the end, and the memory is used again"""
    import universal_differential_equations_amd as U
    T, D, F, O = 150, 72, 104, 40
    xt, wg, wu, wd, dy = made(T, D, F, O, torch.bfloat16, 26)
    dys = [dy * k for k in (1.0, -2.0, 0.5)]
    want = [U.gated_ffn_pullback(U.gated_ffn(xt.T, wg, wu, wd, save=True)[1], d) for d in dys]
    saved = U.gated_ffn(xt.T, wg, wu, wd, save=True)[1]
    held = dy.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = U.gated_ffn_pullback(saved, held)
    for d, w in zip(dys, want):
        held.copy_(d)
        graph.replay()
        again = U.gated_ffn_pullback(saved, d)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(got, w, again))
    del graph, got, saved
    held = fill_with_nan([(T, D), (2, T, F)], torch.bfloat16)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want[0], U.gated_ffn_pullback(U.gated_ffn(xt.T, wg, wu, wd, save=True)[1], dys[0])))
