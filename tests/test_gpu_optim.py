"""The AdamW step over many tensors, the gradient norm, and both behind a gated feed-forward block, against Float64 statements."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import _training_ops as R  # noqa: E402

pytestmark = pytest.mark.gpu
SIZES = [1, 3, 255, 256, 257, 4095, 4096, 4097, 5000, 16383, 16385, 40000]
HYPER = dict(eta=0.01, beta=(0.9, 0.99), eps=1e-8)
U24 = 2.0 ** -24


def tensors(sizes, dtype, seed, by=1.0, odd=False):
    """views of one storage of NaN: with `odd`, each starts one element behind an aligned address"""
    gen = torch.Generator().manual_seed(seed)
    out = []
    for n in sizes:
        t = torch.full((n + 2,), float("nan"), dtype=dtype, device="cuda")
        v = t[1:n + 1] if odd else t[:n]
        v.copy_((torch.randn(n, generator=gen) * by).to(dtype))
        out.append((t, v))
    return out


def gaps_kept(pairs, odd):
    return all(bool(torch.isnan(t.float()[-2:] if not odd else t.float()[[0, -1]]).all()) for t, _ in pairs)


def close(got, want, bound):
    d = (got.double().reshape(-1) - want.reshape(-1)).abs()
    return bool((d <= bound.reshape(-1)).all())


@pytest.mark.parametrize("odd", [False, True], ids=["aligned", "odd"])
@pytest.mark.parametrize("pd,gd,master", [("float32", "float32", False), ("float64", "float64", False), ("bfloat16", "bfloat16", True), ("bfloat16", "float32", True),
                                          ("float16", "float16", False), ("float16", "float32", False), ("bfloat16", "bfloat16", False)])
def test_adamw_32(pd, gd, master, odd):
    from universal_differential_equations_amd import training
    pd, gd = getattr(torch, pd), getattr(torch, gd)
    u = 2.0 ** -53 if pd == torch.float64 else U24
    ps = tensors(SIZES, pd, 1, 0.5, odd)
    decay = [0.1 * (i % 3) for i in range(len(SIZES))]
    opt = training.AdamW([v for _, v in ps], weight_decay=decay, master=master, **HYPER)
    clip = torch.tensor([2.0, 0.5], dtype=torch.float64, device="cuda")
    ws = [(s["master"] if master else v).double().clone() for s, (_, v) in zip(opt.state, ps)]   # (double() of a float64 tensor is that tensor)
    ms, vs = [torch.zeros_like(w) for w in ws], [torch.zeros_like(w) for w in ws]
    for t in (1, 2, 3):
        gs = tensors(SIZES, gd, 10 + t, 0.1, odd)
        opt.step([v for _, v in gs], clip=clip)
        for i, s in enumerate(opt.state):
            w, m, v, step = R.adamw(ws[i], gs[i][1], ms[i], vs[i], t, HYPER["eta"], HYPER["beta"], HYPER["eps"], decay[i], 0.5)
            g = gs[i][1].double() * 0.5
            # three roundings of each term and of each sum; both moments start from the values that the device holds
            assert close(s["m"], m, 4 * u * (ms[i].abs() + g.abs()))
            assert close(s["v"], v, 6 * u * (vs[i] + g * g) + 2.0 ** -140)
            # a step of about 12 roundings, among them those of m where its two terms cancel (4 u of them)
            size = HYPER["eta"] * ((ms[i].abs() * 0.9 + g.abs() * 0.1) / (1 - 0.9 ** t)) / ((v / (1 - 0.99 ** t)).sqrt() + 1e-8)
            e = 20 * u * size + 3 * u * ws[i].abs()
            held = s["master"] if master else ps[i][1]
            k = UNITS[held.dtype]
            assert close(held, w, e + (k * (w.abs() + e) + (2.0 ** -24 if held.dtype == torch.float16 else 0) if k > u else 0))
            if master:
                assert torch.equal(ps[i][1], s["master"].to(pd))
            ws[i], ms[i], vs[i] = held.double().clone(), s["m"].double().clone(), s["v"].double().clone()
    assert gaps_kept(ps, odd) and opt.steps == 3


UNITS = {torch.float64: 2.0 ** -53, torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def codes_of(m, v):
    """codes and scales of Float64 moments, and how near each code is to its border (relative)"""
    mb, vb = R.blocks(m), R.blocks(v)
    a, c = mb.abs().amax(1).float(), vb.amax(1).float()
    x = 127 * (mb.abs() / a.double().clamp_min(1e-300)[:, None]).sqrt()
    y = 255 * (vb / c.double().clamp_min(1e-300)[:, None]) ** 0.25
    q, r = torch.round(x).clamp_max(127), torch.round(y).clamp_max(255)
    r = torch.where((vb > 0) & (r == 0), 1.0, r)
    near = torch.minimum((x - torch.floor(x) - 0.5).abs(), (y - torch.floor(y) - 0.5).abs())
    n = m.numel()
    return (q * mb.sign()).reshape(-1)[:n], r.reshape(-1)[:n], a, c, near.reshape(-1)[:n]


@pytest.mark.parametrize("odd", [False, True], ids=["aligned", "odd"])
@pytest.mark.parametrize("pd,gd,master", [("float32", "float32", False), ("bfloat16", "bfloat16", False), ("bfloat16", "float32", True), ("float16", "float16", True)])
def test_adamw_8(pd, gd, master, odd):
    """codes and scales are those of Float64 arithmetic (borders nearer than 1e-9 aside), over steps of which each starts from the
    device's own codes; blocks of zeros, of one nonzero element and of elements 1e10 apart are among them"""
    from universal_differential_equations_amd import training
    pd, gd = getattr(torch, pd), getattr(torch, gd)
    ps = tensors(SIZES, pd, 1, 0.5, odd)
    opt = training.AdamW([v for _, v in ps], weight_decay=0.1, bits=8, master=master, **HYPER)
    clip = torch.tensor([2.0, 0.75], dtype=torch.float64, device="cuda")
    for t in (1, 2, 3):
        gs = tensors(SIZES, gd, 20 + t, 0.1, odd)
        big = gs[-1][1]
        big[:256] = 0
        big[256:512] = 0
        big[300] = 3
        big[512:768] *= torch.logspace(-5, 5, 256, device="cuda").to(gd) if gd != torch.float16 else 1
        before = [{k: x.clone() for k, x in s.items()} for s in opt.state]
        held = [(b["master"] if master else v.clone()).double() for b, (_, v) in zip(before, ps)]
        opt.step([v for _, v in gs], clip=clip)
        values = opt.moments()
        for i, s in enumerate(opt.state):
            n, b = SIZES[i], before[i]
            m0, v0 = R.value_m(b["m"], b["m_scale"]).reshape(-1)[:n], R.value_v(b["v"], b["v_scale"]).reshape(-1)[:n]
            w, m, v, step = R.adamw(held[i], gs[i][1], m0, v0, t, HYPER["eta"], HYPER["beta"], HYPER["eps"], 0.1, 0.75)
            q, r, a, c, near = codes_of(m, v)
            assert torch.equal(s["m_scale"], a) and torch.equal(s["v_scale"], c)
            clear = near > 1e-9
            assert torch.equal(s["m"].double()[clear], q[clear]) and torch.equal(s["v"].double()[clear], r[clear])
            assert not (s["v"][v > 0] == 0).any()
            vm, vv = R.value_m(s["m"], a).reshape(-1)[:n], R.value_v(s["v"], c).reshape(-1)[:n]
            assert close(values[i][0], vm, U24 * vm.abs() + 2.0 ** -149) and close(values[i][1], vv, U24 * vv + 2.0 ** -149)
            e = 16 * U24 * step.abs() + 3 * U24 * held[i].abs()
            now = s["master"] if master else ps[i][1]
            k = UNITS[now.dtype]
            assert close(now, w, e + (k * (w.abs() + e) + (2.0 ** -24 if now.dtype == torch.float16 else 0) if k > U24 else 0))
            if master:
                assert torch.equal(ps[i][1], s["master"].to(pd))
    assert gaps_kept(ps, odd)


def test_many_tensors_none_gradients_and_empty_ones():
    """more tensors than one launch takes; a tensor without a gradient keeps its bits and its moments"""
    from universal_differential_equations_amd import training
    sizes = [(i * 37) % 700 for i in range(130)]
    ps, gs = tensors(sizes, torch.float32, 1), tensors(sizes, torch.float32, 2)
    before = [v.clone() for _, v in ps]
    for bits in (32, 8):
        opt = training.AdamW([v for _, v in ps], bits=bits, **HYPER)
        opt.step([None if i % 5 == 0 else g for i, (_, g) in enumerate(gs)])
        for i, (_, p) in enumerate(ps):
            if i % 5 == 0:
                assert torch.equal(p, before[i]) and not any(x.any() for x in opt.state[i].values())
            elif sizes[i]:
                w = R.adamw(before[i], gs[i][1], torch.zeros_like(p), torch.zeros_like(p), 1, 0.01, (0.9, 0.99), 1e-8, 0.01)
                assert close(p, w[0], 16 * U24 * w[3].abs() + 3 * U24 * before[i].double().abs())
        for p, b in zip(ps, before):
            p[1].copy_(b)
    assert gaps_kept(ps, False)


def test_skip_nonfinite_and_nan_blocks():
    from universal_differential_equations_amd import training
    for bits in (32, 8):
        p = torch.ones(600, device="cuda")
        g = torch.ones(600, device="cuda")
        opt = training.AdamW([p], bits=bits, skip_nonfinite=True, **HYPER)
        opt.step([g], clip=training.grad_norm([g], 1.0))
        kept = [x.clone() for x in (p, *opt.state[0].values())]
        for worst in (float("nan"), float("inf")):
            g[300] = worst
            opt.step([g], clip=training.grad_norm([g], 1.0))
            assert all(torch.equal(a, b) for a, b in zip(kept, (p, *opt.state[0].values())))
        g[300] = 1
        opt.step([g], clip=training.grad_norm([g], 1.0))
        assert not torch.equal(p, kept[0]) and opt.steps == 4
    # without it, the moments of the block are NaN, the others not
    g[300] = float("nan")
    opt = training.AdamW([p], bits=8, **HYPER)
    opt.step([g])
    m, v = opt.moments()[0]
    bad = torch.isnan(m)
    assert bool(bad[256:512].all()) and not bad[:256].any() and not bad[512:].any() and torch.equal(bad, torch.isnan(v)) and bool(torch.isnan(p[300]))


def test_state_of_another_instance_continues_it():
    from universal_differential_equations_amd import training
    for bits in (32, 8):
        p = [torch.linspace(-1, 1, 900, device="cuda").bfloat16()]
        g = [torch.linspace(1, -2, 900, device="cuda").bfloat16()]
        one = training.AdamW(p, bits=bits, master=True, **HYPER)
        one.step(g)
        q, state = [p[0].clone()], [{k: x.clone() for k, x in one.state[0].items()}]
        two = training.AdamW(q, bits=bits, master=True, state=state, step=one.steps, **HYPER)
        one.step(g), two.step(g)
        assert torch.equal(p[0], q[0]) and all(torch.equal(one.state[0][k], two.state[0][k]) for k in state[0])


def test_refusals():
    from universal_differential_equations_amd import UdeError, training
    p, q = torch.zeros(300, device="cuda"), torch.zeros(300, device="cuda")
    for bad in (dict(bits=4), dict(master=True), dict(weight_decay=[0.1, 0.2]), dict(state=[{}, {}])):
        with pytest.raises(ValueError):
            training.AdamW([p], **bad)
    for params in ([p, p], [p, p[100:200]], [p[::2]], [p, q.double()], [p, q.cpu()], [p.int()]):
        with pytest.raises(ValueError):
            training.AdamW(params)
    with pytest.raises(ValueError):
        training.AdamW([p.double()], bits=8)
    s = {"m": torch.zeros(300, device="cuda"), "v": torch.zeros(300, device="cuda")}
    with pytest.raises(ValueError, match="share"):
        training.AdamW([p, q], state=[s, s])
    opt = training.AdamW([p])
    for grads in ([], [q, q], [q[:10]], [q.cpu()], [q.double()], [q.half()]):
        with pytest.raises((ValueError, UdeError)):
            opt.step(grads)
    with pytest.raises(ValueError):
        opt.step([q], clip=torch.zeros(2, device="cuda"))
    with pytest.raises(UdeError):
        training.AdamW([p], skip_nonfinite=True).step([q])
    with pytest.raises(UdeError):
        training.AdamW([p], beta=(1.0, 0.9)).step([q])
    with pytest.raises(ValueError):
        training.grad_norm([p, q.double()])
    with pytest.raises(ValueError):
        opt.moments and training.AdamW([p], bits=8).moments(out=[(q, q[:5])])
    assert opt.steps == 0 and not p.any()


def test_a_parameter_given_other_storage():
    from universal_differential_equations_amd import training
    p, g = torch.ones(500, device="cuda"), torch.ones(500, device="cuda")
    opt = training.AdamW([p], eta=0.1)
    opt.step([g])
    after = p.clone()
    p.data = torch.full((500,), 5.0, device="cuda")
    opt.step([g])
    assert bool((p < 5).all()) and bool((p > 4).all()) and bool((after < 1).all())
    p.data = torch.zeros(400, device="cuda")
    with pytest.raises(ValueError):
        opt.step([g])


@pytest.mark.parametrize("dtype", ["float64", "float32", "float16", "bfloat16"])
@pytest.mark.parametrize("sizes", [[1], [7, 0, 300], [16384], [16385, 1, 16383], [250001] + [3] * 20, [(i * 101) % 900 for i in range(400)]], ids=lambda s: "%d" % len(s))
@pytest.mark.parametrize("odd", [False, True], ids=["aligned", "odd"])
def test_grad_norm(dtype, sizes, odd):
    from universal_differential_equations_amd import training
    gs = tensors(sizes, getattr(torch, dtype), 3, 1.0, odd)
    exact = math.sqrt(math.fsum(math.fsum(x * x for x in v.double().cpu().tolist()) for _, v in gs))
    for most in (exact / 3, exact * 3, 0.0):
        norm, factor = training.grad_norm([v for _, v in gs], max_norm=most).tolist()
        # squares and sums in Float64: at most one rounding of 2^-53 per element and level, halved by the root
        assert abs(norm - exact) <= 2.0 ** -53 * (sum(sizes) / 2 + 4) * exact
        assert factor == (1.0 if most <= 0 or norm <= most else most / norm)
    assert torch.equal(training.grad_norm([v for _, v in gs], 1.0), training.grad_norm([v for _, v in gs], 1.0))


def test_grad_norm_extremes():
    from universal_differential_equations_amd import training
    big = torch.full((1000,), 3e38, device="cuda")
    norm, factor = training.grad_norm([big], 1.0).tolist()
    assert abs(norm / (float(big[0]) * math.sqrt(1000)) - 1) < 1e-12 and factor == 1 / norm
    assert training.grad_norm([torch.zeros(10, device="cuda"), torch.zeros(0, device="cuda")], 1.0).tolist() == [0.0, 1.0]
    assert training.grad_norm([torch.zeros(0, device="cuda")], 1.0).tolist() == [0.0, 1.0]
    big[7] = float("inf")
    assert training.grad_norm([big], 1.0).tolist() == [math.inf, 0.0]
    big[8] = float("nan")
    assert all(math.isnan(x) for x in training.grad_norm([big], 1.0).tolist()) and math.isnan(training.grad_norm([big])[1])


def block_step(sets, params, opt):
    """one training step of a gated block: forward, pullback of mean square error, norm, update"""
    import universal_differential_equations_amd as U
    from universal_differential_equations_amd import training
    x, target = sets
    y, saved = U.gated_ffn(x, *params, save=True)
    grads = U.gated_ffn_pullback(saved, (y - target) * (2 / y.numel()), need=("w_gate", "w_up", "w_down"))[1:]
    norm = training.grad_norm(grads, 0.05)
    opt.step(grads, clip=norm)
    return y, norm


def block(seed, dtype, T=64, D=40, F=72, O=24):
    gen = torch.Generator().manual_seed(seed)
    made = [(torch.randn(s, generator=gen) * by).to(dtype).cuda() for s, by in (((T, D), 1), ((T, O), 1), ((F, D), D ** -0.5), ((F, D), D ** -0.5), ((O, F), F ** -0.5))]
    return made[:2], made[2:]


def test_training_step_of_a_block_against_float64():
    from universal_differential_equations_amd import training
    (x, target), params = block(1, torch.float32)
    old = [p.double() for p in params]
    opt = training.AdamW(params, weight_decay=0.1, eta=0.01, beta=(0.9, 0.99), eps=1e-3)
    y, norm = block_step((x, target), params, opt)
    g, u = x.double() @ old[0].T, x.double() @ old[1].T
    a = g * torch.sigmoid(g)
    want = (a * u) @ old[2].T
    dy = (want - target.double()) * (2 / want.numel())
    dh = dy @ old[2]
    grads = [(dh * u * R.ACTS["swish"][1](g)).T @ x.double(), (dh * a).T @ x.double(), dy.T @ (a * u)]
    size = math.sqrt(sum(float((t ** 2).sum()) for t in grads))
    # Float32 products of up to 72 terms, three deep: relative 1e-5 of the largest element; the update divides by sqrt(v) + 1e-3
    assert float((y.double() - want).abs().max()) <= 1e-5 * float(want.abs().max())
    assert abs(float(norm[0]) / size - 1) <= 1e-5 and abs(float(norm[1]) / min(1, 0.05 / size) - 1) <= 1e-5
    for p, o, t in zip(params, old, grads):
        w, m, v, step = R.adamw(o, t, torch.zeros_like(t), torch.zeros_like(t), 1, 0.01, (0.9, 0.99), 1e-3, 0.1, float(norm[1]))
        # |d step / d g| <= eta / eps * factor; gradients are off by 1e-5 of the largest
        bound = 0.01 / 1e-3 * float(norm[1]) * 1e-5 * float(t.abs().max()) + 16 * U24 * (step.abs() + o.abs())
        assert close(p, w, bound)


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_training_steps_are_the_eager_ones(bits):
    """a whole step in a graph, replayed with new data and eager work between: the bits of eager steps"""
    from universal_differential_equations_amd import training
    hyper = dict(weight_decay=0.1, bits=bits, master=True, **HYPER)
    data = [block(s, torch.bfloat16)[0] for s in range(5)]
    params = block(9, torch.bfloat16)[1]
    eager = [p.clone() for p in params]
    opt = training.AdamW(eager, **hyper)
    for d in data:
        block_step(d, eager, opt)
    held = [t.clone() for t in data[0]]
    opt2 = training.AdamW(params, capturable=True, **hyper)
    start = [[x.clone() for x in s.values()] for s in opt2.state]
    first = [p.clone() for p in params]
    block_step(held, params, opt2)            # (outside the capture: loads what is loaded on first use)
    for p, f in zip(params, first):
        p.copy_(f)
    for s, b in zip(opt2.state, start):
        for x, y in zip(s.values(), b):
            x.copy_(y)
    opt2.count.zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block_step(held, params, opt2)
    opt2.count.zero_()
    for d in data:
        for a, b in zip(held, d):
            a.copy_(b)
        graph.replay()
        assert math.isfinite(float(training.grad_norm([params[0]])[0]))
        torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(params, eager))
    assert all(torch.equal(x, y) for s, r in zip(opt.state, opt2.state) for x, y in zip(s.values(), r.values()))
    # (the bias corrections of the device are pow()'s of the device's library: at most one unit in the last place off the host's)


def test_adamw_loop_and_host_loop_agree():
    """training.adamw on a CUDA tensor against the same loop on numpy in Float64"""
    from universal_differential_equations_amd import training
    start = np.linspace(-2, 2, 301)
    target = np.cos(start)

    def host(th):
        return float(((th - target) ** 2).sum()), 2 * (th - target)

    t = torch.tensor(target, device="cuda")

    def dev(th):
        return ((th - t) ** 2).sum(), 2 * (th - t)

    kw = dict(eta=0.05, decay=0.02, maxiters=30, max_norm=3.0)
    for result in ("updated", "evaluated"):
        a, la = training.adamw(host, start, result=result, **kw)
        b, lb = training.adamw(dev, torch.tensor(start, device="cuda"), result=result, **kw)
        assert np.allclose(la, lb, rtol=1e-10) and np.allclose(a, b.cpu().numpy(), rtol=1e-10, atol=1e-12)


def test_deep_bsde_trains_with_adamw():
    """pde.solve with Flux.ADAMW: decay 0 without clipping is ADAM's trajectory up to Float32 rounding; decay and ClipNorm change it as the formula says"""
    from universal_differential_equations_amd import pde
    prob = pde.TerminalPDEProblem(pde.hjb(1.0), np.zeros(100, dtype=np.float32), (0.0, 1.0))
    rng = np.random.default_rng(0)
    th0 = pde.NNPDENS(100, 110).init_params(rng)
    kw = dict(maxiters=3, trajectories=32, alg=pde.LambaEM(), pabstol=1e-9, abstol=0.1, reltol=0.1)

    def run(opt):
        return pde.solve(prob, pde.NNPDENS(100, 110, opt=opt), th0, **kw)

    _, a, la = run(pde.ADAM(0.01))
    _, b, lb = run(pde.ADAMW(0.01))
    assert la[0] == lb[0] and np.allclose(la, lb, rtol=1e-4) and float((a - b).abs().max()) <= 1e-4
    seen = []
    _, c, lc = pde.solve(prob, pde.NNPDENS(100, 110, opt=pde.ADAMW(0.01, decay=0.001, max_norm=0.5)), th0, callback=lambda it, l, u: seen.append(l), **kw)
    assert lc[0] == la[0] and seen == lc and bool(torch.isfinite(c).all()) and not torch.equal(b, c)
