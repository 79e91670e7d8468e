"""The training operators as workloads: the gated feed-forward block with its pullback, the AdamW step over many tensors, and the global
gradient norm with its clipping factor.  `run` computes them as elementary torch operations, or, where `own` is set, through the package's
entry points.

    y = (swish(x Wg^T) * (x Wu^T)) Wd^T          x: T x D, Wg, Wu: F x D, Wd: D x F
    m' = b1 m + (1 - b1) s g,  v' = b2 v + (1 - b2) (s g)^2,  p' = p (1 - eta wd) - eta / (1 - b1^t) m' / (sqrt(v' / (1 - b2^t)) + eps)
    (sqrt(sum g^2), min(1, max_norm / that))

Moments in 8 bits: 256 consecutive elements of a tensor share two scales, a = max |m| and c = max v, and hold the codes
q = sign(m) round(127 sqrt(|m| / a)) and r = round(255 (v / c)^(1/4)), r >= 1 where v > 0; they stand for a sign(q) (q / 127)^2 and c (r / 255)^4.
"""
import math

import torch

own = False

BLOCK = 256
ETA, B1, B2, EPS, WD, STEP0, MAX_NORM = 1e-3, 0.9, 0.999, 1e-8, 0.01, 100, 1.0
KINDS = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
# the two networks of the deep-BSDE solver at d = 100, hls = 110: 100-110-110-1 and 101-110-110-110-100, weights and biases
HJB = "11000,110,12100,110,110,1,11110,110,12100,110,12100,110,11000,100"
# four gated blocks of 2048 x 5632 with a scale vector each
BLOCKS = "11534336*12,2048*4"


def listed():
    return [
        # one token through a block: the step of a program that samples one sequence, bound by reading the weights
        {"name": "ffn token", "op": "ffn", "kind": "bfloat16", "train": False, "rows": True, "T": 1, "D": 4096, "F": 11264},
        # a step of two dozen sequences at once, weights as vec(W) of out x in matrices hold them
        {"name": "ffn few tokens", "op": "ffn", "kind": "float16", "train": False, "rows": False, "T": 24, "D": 2048, "F": 5632},
        # a long prompt: bound by the matrix units
        {"name": "ffn prompt", "op": "ffn", "kind": "bfloat16", "train": False, "rows": True, "T": 4096, "D": 4096, "F": 11264},
        # a training step's share of one block, forward and pullback
        {"name": "ffn training", "op": "ffn", "kind": "bfloat16", "train": True, "rows": True, "T": 4096, "D": 2048, "F": 5632},
        # sizes that no tile divides, rows of F elements that are not 16-byte aligned
        {"name": "ffn training ragged", "op": "ffn", "kind": "float16", "train": True, "rows": False, "T": 1000, "D": 1000, "F": 2730},
        # single precision, the type of this package's deep-BSDE networks
        {"name": "ffn training single", "op": "ffn", "kind": "float32", "train": True, "rows": True, "T": 2048, "D": 1024, "F": 2816},
        # the smallest: 100 trajectories through a hidden layer of width 110, where the launches count
        {"name": "ffn training small", "op": "ffn", "kind": "float32", "train": True, "rows": False, "T": 100, "D": 110, "F": 220},
        # the update of the deep-BSDE networks, views into one flat vector: where the launch counts
        {"name": "adamw networks", "op": "adamw", "kind": "float32", "master": False, "bits": 32, "pad": 1, "sizes": HJB},
        # mixed precision: 16-bit weights with 32-bit copies and moments
        {"name": "adamw blocks", "op": "adamw", "kind": "bfloat16", "master": True, "bits": 32, "pad": 256, "sizes": BLOCKS},
        # the same weights where memory is short: moments in 8 bits, no copies
        {"name": "adamw blocks 8 bits", "op": "adamw", "kind": "bfloat16", "master": False, "bits": 8, "pad": 256, "sizes": BLOCKS},
        # the norm of the gradients of either
        {"name": "norm networks", "op": "norm", "kind": "float32", "pad": 1, "sizes": HJB},
        {"name": "norm blocks", "op": "norm", "kind": "bfloat16", "pad": 256, "sizes": BLOCKS},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("ffn", "ffn", "ffn", "adamw", "adamw", "norm"))
    kind = rng.choice(sorted(KINDS))
    if op == "ffn":
        T, D, F = _log(rng, 1, 8192), _log(rng, 64, 4096), _log(rng, 64, 11264)
        if rng.random() < 0.6:  # most widths are multiples of 64, the rest anything
            D, F = 64 * max(1, round(D / 64)), 64 * max(1, round(F / 64))
        train = rng.random() < 0.5
        most = 4096 * 2048 * 5632 // (4 if kind == "float32" else 1)
        T = max(1, min(T, most // (D * F)))
        return {"op": op, "kind": kind, "train": train, "rows": rng.random() < 0.5, "T": T, "D": D, "F": F}
    n = _log(rng, 1, 60)
    sizes = [_log(rng, 1, 4000000) for _ in range(n)]
    case = {"op": op, "kind": kind, "pad": rng.choice((1, 256)), "sizes": ",".join(map(str, sizes))}
    if op == "adamw":
        case["bits"] = rng.choice((32, 8))
        case["master"] = kind != "float32" and rng.random() < 0.5
        case["pad"] = 256 if case["bits"] == 8 else case["pad"]
    return case


def _sizes(case):
    found = []
    for s in case["sizes"].split(","):
        n, _, times = s.partition("*")
        found += [int(n)] * int(times or 1)
    return found


def _places(case):
    """where each tensor starts in the flat storage, and its length"""
    at, places = 0, []
    for n in _sizes(case):
        places.append((at, n))
        at += -(-n // case["pad"]) * case["pad"]
    return places, at


def _split(flat, places, per=1):
    return [flat[at // per: at // per + -(-n // per)] for at, n in places]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = KINDS[case["kind"]]

    def normal(*shape, by=1.0, dtype=kind):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(by).to(dtype)

    if case["op"] == "ffn":
        T, D, F = case["T"], case["D"], case["F"]
        # weights of the usual start; out x in matrices, held by rows or by columns
        s = {"x": normal(T, D)}
        for name, o, i in (("wg", F, D), ("wu", F, D), ("wd", D, F)):
            s[name] = normal(o, i, by=i ** -0.5) if case["rows"] else normal(i, o, by=i ** -0.5).T
        if case["train"]:
            s["dy"] = normal(T, D)
        return s | {"op": "ffn"}

    places, total = _places(case)
    # gradients whose sizes differ from tensor to tensor, as they do from layer to layer; nothing between the tensors
    g = torch.zeros(total, device="cuda", dtype=kind)
    for k, (at, n) in enumerate(places):
        g[at:at + n] = normal(n, by=1e-3 * 2.0 ** -(k % 5))
    s = {"op": case["op"], "g": g, "grads": _split(g, places)}
    if case["op"] == "norm":
        return s
    p = torch.where(g == 0, 0, normal(total, by=0.02, dtype=torch.float32))
    m = torch.where(g == 0, 0, normal(total, by=5e-4, dtype=torch.float32))
    v = torch.where(g == 0, 0, normal(total, by=1e-3, dtype=torch.float32).square_())
    s |= {"bits": case["bits"], "step": STEP0, "p": p.to(kind), "master": p if case["master"] else None, "factor": torch.full((2,), 0.5, device="cuda", dtype=torch.float64)}
    if case["bits"] == 8:
        ms, vs = m.view(-1, BLOCK).abs().amax(1), v.view(-1, BLOCK).amax(1)
        s |= {"ms": ms, "vs": vs, "m": _m_code(m, ms), "v": _v_code(v, vs)}
    else:
        s |= {"m": m, "v": v}
    if own:
        from universal_differential_equations_amd import training
        state = [{"m": a, "v": b} for a, b in zip(_split(s["m"], places), _split(s["v"], places))]
        for name in ("ms", "vs") if case["bits"] == 8 else ():
            for d, x in zip(state, _split(s[name], places, BLOCK)):
                d["m_scale" if name == "ms" else "v_scale"] = x
        if case["master"]:
            for d, x in zip(state, _split(p, places)):
                d["master"] = x
        s["opt"] = training.AdamW(_split(s["p"], places), eta=ETA, beta=(B1, B2), eps=EPS, weight_decay=WD, bits=case["bits"], master=case["master"], state=state, step=STEP0)
        s["values"] = (torch.zeros(total, device="cuda"), torch.zeros(total, device="cuda"))
        s["views"] = list(zip(_split(s["values"][0], places), _split(s["values"][1], places)))
    return s


def _m_code(m, a):
    x = (m.view(-1, BLOCK).double() / a.double().clamp_min(1e-300)[:, None]).view(-1)
    return torch.floor(x.abs().sqrt().mul(127).add(0.5)).clamp_max(127).mul(x.sign()).to(torch.int8)


def _v_code(v, c):
    x = (v.view(-1, BLOCK).double() / c.double().clamp_min(1e-300)[:, None]).view(-1)
    return torch.floor(x.sqrt().sqrt().mul(255).add(0.5)).clamp(max=255).maximum((x > 0).double()).to(torch.uint8)


def _m_value(q, a):
    q = q.double()
    return ((q * q.abs() / 127 ** 2).view(-1, BLOCK) * a.double()[:, None]).view(-1)


def _v_value(r, c):
    return ((r.double() / 255).pow(4).view(-1, BLOCK) * c.double()[:, None]).view(-1)


def run(state):
    return {"ffn": _ffn, "adamw": _adamw, "norm": _norm}[state["op"]](state)


def _ffn(s):
    x, wg, wu, wd, dy = s["x"], s["wg"], s["wu"], s["wd"], s.get("dy")
    if own:
        from universal_differential_equations_amd import gated_ffn, gated_ffn_pullback
        if dy is None:
            return gated_ffn(x, wg, wu, wd, act="swish")
        y, saved = gated_ffn(x, wg, wu, wd, act="swish", save=True)
        return (y,) + tuple(gated_ffn_pullback(saved, dy))
    kind = x.dtype
    x, wg, wu, wd = x.float(), wg.float(), wu.float(), wd.float()
    g, u = x @ wg.T, x @ wu.T
    sig = 1 / (1 + torch.exp(-g))
    a = g * sig
    h = a * u
    y = (h @ wd.T).to(kind)
    if dy is None:
        return y
    dy = dy.float()
    dh = dy @ wd
    dg = dh * u * (sig * (1 + g * (1 - sig)))
    du = dh * a
    return tuple(t.to(kind) for t in (y, dg @ wg + du @ wu, dg.T @ x, du.T @ x, dy.T @ h))


def _adamw(s):
    if own:
        s["opt"].step(s["grads"], clip=s["factor"])
        if s["bits"] == 32:
            return tuple(x for x in (s["p"], s["master"], s["m"], s["v"]) if x is not None)
        s["opt"].moments(out=s["views"])
        return tuple(x for x in (s["p"], s["master"], *s["values"]) if x is not None)
    s["step"] += 1
    c1, c2 = 1 - B1 ** s["step"], 1 - B2 ** s["step"]
    p, master = s["p"], s["master"]
    if s["bits"] == 32:
        g = s["g"].float() * s["factor"][1].float()
        m, v = s["m"], s["v"]
        m.mul_(B1).add_(g * (1 - B1))
        v.mul_(B2).add_(g * g * (1 - B2))
        values = m, v
    else:  # which code a value next to a border takes is decided in 64 bits
        g = s["g"].double() * s["factor"][1]
        m = _m_value(s["m"], s["ms"]) * B1 + g * (1 - B1)
        v = _v_value(s["v"], s["vs"]) * B2 + g * g * (1 - B2)
        s["ms"].copy_(m.view(-1, BLOCK).abs().amax(1))
        s["vs"].copy_(v.view(-1, BLOCK).amax(1))
        s["m"].copy_(_m_code(m, s["ms"]))
        s["v"].copy_(_v_code(v, s["vs"]))
        values = _m_value(s["m"], s["ms"]).float(), _v_value(s["v"], s["vs"]).float()
    w = p.float() if master is None else master
    w = w * (1 - ETA * WD) - (m / c1 * ETA / ((v / c2).sqrt() + EPS)).float()
    p.copy_(w)
    if master is not None:
        master.copy_(w)
    return tuple(x for x in (p, master, *values) if x is not None)


def _norm(s):
    if own:
        from universal_differential_equations_amd import training
        return training.grad_norm(s["grads"], max_norm=MAX_NORM)
    norm = s["g"].double().square().sum().sqrt()
    return torch.stack((norm, (MAX_NORM / norm).clamp_max(1)))


def work(case):
    e = 4 if case["kind"] == "float32" else 2
    if case["op"] == "ffn":
        T, D, F = case["T"], case["D"], case["F"]
        io = 2 * T * D + 3 * D * F
        return {"bytes": e * io * (2 if case["train"] else 1), "flops": 6.0 * T * D * F * (3 if case["train"] else 1)}
    n = sum(_sizes(case))
    if case["op"] == "norm":
        return {"bytes": e * n, "flops": 2.0 * n}
    # gradient and weight in, weight out; copies and moments in and out, 8-bit ones as values too
    each = 3 * e + (8 if case["master"] else 0) + (16 if case["bits"] == 32 else 4 + 16 / BLOCK + 8)
    return {"bytes": each * n, "flops": 14.0 * n}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "ffn":
        T = case["T"]
        x, wg, wu, wd = (s[k].double() for k in ("x", "wg", "wu", "wd"))
        g, u = torch.mm(x, wg.t()), torch.mm(x, wu.t())
        y = torch.mm(torch.sigmoid(g) * g * u, wd.t())
        if not case["train"]:
            return y
        dy = s["dy"].double()
        dh = torch.mm(dy, wd)
        t = torch.sigmoid(g)
        slope = t + g * t * torch.sigmoid(-g)
        dg, du = slope * (u * dh), (g * t) * dh
        cat = torch.cat((dg, du), 1)
        dw = torch.mm(cat.t().contiguous(), x)
        assert cat.shape[0] == T
        return y, torch.mm(cat, torch.cat((wg, wu), 0)), dw[:case["F"]], dw[case["F"]:], torch.mm(dy.t().contiguous(), g * t * u)
    if case["op"] == "norm":
        total = sum(float((t.double() ** 2).sum()) for t in s["grads"])
        return torch.tensor([math.sqrt(total), min(1.0, MAX_NORM / math.sqrt(total))], dtype=torch.float64)
    outs = []
    places, total = _places(case)
    t = STEP0 + 1
    many = max(BLOCK, (1 << 24))
    for at in range(0, total, many):
        part = slice(at, min(total, at + many))
        rows = slice(at // BLOCK, -(-part.stop // BLOCK))
        g = s["g"][part].double() * 0.5
        w = (s["p"] if s["master"] is None else s["master"])[part].double()
        m, v = s["m"][part].double(), s["v"][part].double()
        if case["bits"] == 8:
            m = torch.sign(m) * (m / 127) ** 2 * s["ms"][rows].double().repeat_interleave(BLOCK)
            v = (v / 255) ** 2 * (v / 255) ** 2 * s["vs"][rows].double().repeat_interleave(BLOCK)
        m, v = B1 * m + (1 - B1) * g, B2 * v + (1 - B2) * g ** 2
        w = w - ETA * WD * w - ETA * (m / (1 - B1 ** t)) / (torch.sqrt(v / (1 - B2 ** t)) + EPS)
        if case["bits"] == 8:
            a = m.abs().view(-1, BLOCK).max(1).values.float().double().repeat_interleave(BLOCK)
            c = v.view(-1, BLOCK).max(1).values.float().double().repeat_interleave(BLOCK)
            q = torch.round(127 * torch.sqrt(m.abs() / torch.where(a > 0, a, 1))).clamp_max(127)
            r = torch.round(255 * (v / torch.where(c > 0, c, 1)) ** 0.25).clamp_max(255)
            r = torch.where((v > 0) & (r == 0), 1.0, r)
            m, v = torch.sign(m) * a * q ** 2 / 127 ** 2, c * r ** 4 / 255 ** 4
        outs.append([x for x in (w, w if case["master"] else None, m, v) if x is not None])
    return tuple(torch.cat(x) for x in zip(*outs))
