"""What an AdamW step takes, refuses and counts, on the device, against Float64 statements."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import _training_ops as R  # noqa: E402

pytestmark = pytest.mark.gpu
U24 = 2.0 ** -24
HYPER = dict(eta=0.01, beta=(0.9, 0.99), eps=1e-8, weight_decay=0.01)


def near(got, start, g, t=1, m=None, v=None, factor=1.0):
    """got: a Float32 parameter after the step from `start` with gradient g; dozen roundings of the step, three of the parameter"""
    zero = torch.zeros_like(g, dtype=torch.float64)
    w, m, v, step = R.adamw(start, g, zero if m is None else m, zero if v is None else v, t, HYPER["eta"], HYPER["beta"], HYPER["eps"], HYPER["weight_decay"], factor)
    assert bool(((got.double() - w).abs() <= 16 * U24 * step.abs() + 3 * U24 * start.double().abs()).all())
    return w, m, v


def test_weights_by_columns_through_block_and_step():
    """weights that a block holds by columns are stepped as their storage: each element by its own gradient"""
    import universal_differential_equations_amd as U
    from universal_differential_equations_amd import training
    gen = torch.Generator().manual_seed(31)
    T, D, F, O = 20, 12, 18, 10
    x, dy = (torch.randn(s, generator=gen).cuda() for s in ((T, D), (T, O)))
    stores = [(torch.randn(s, generator=gen) * 0.3).cuda() for s in ((D, F), (D, F), (F, O))]
    weights = [s.T for s in stores]
    opt = training.AdamW(stores, **HYPER)
    before = [s.clone() for s in stores]
    _, saved = U.gated_ffn(x, *weights, save=True)
    grads = U.gated_ffn_pullback(saved, dy)[1:]
    for wrong in (grads, [grads[0].T, grads[1].T, grads[2]]):
        with pytest.raises(ValueError, match="gradient"):
            opt.step(wrong)
    assert opt.steps == 0 and all(torch.equal(a, b) for a, b in zip(stores, before))
    opt.step([g.T for g in grads])
    for s, b, g in zip(stores, before, grads):
        near(s, b, g.T.contiguous())
    # and a gradient of the right shape in the other order of strides: the same bits
    again = [b.clone() for b in before]
    training.AdamW(again, **HYPER).step([g.contiguous().T for g in grads])
    assert all(torch.equal(a, s) for a, s in zip(again, stores))


@pytest.mark.parametrize("bits", [32, 8])
def test_resumed_after_replays(bits):
    """a checkpoint (state, steps) taken after a graph was replayed goes on like the instance that was never captured"""
    from universal_differential_equations_amd import training
    gen = torch.Generator().manual_seed(32)
    start, g = (torch.randn(700, generator=gen).cuda() for _ in range(2))
    eager, held = start.clone(), start.clone()
    one = training.AdamW([eager], bits=bits, **HYPER)
    two = training.AdamW([held], bits=bits, capturable=True, **HYPER)
    one.step([g]), two.step([g])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        two.step([g])
        with pytest.raises(ValueError, match="captur"):
            two.steps
    assert two.steps == 1   # (captured, not run)
    for i in range(40):
        graph.replay()
        one.step([g])
        assert i % 13 or two.steps == i + 2
    assert one.steps == two.steps == 41
    copies = [held.clone()]
    three = training.AdamW(copies, bits=bits, state=[{k: x.clone() for k, x in two.state[0].items()}], step=two.steps, **HYPER)
    three.step([g]), one.step([g])
    # bias corrections of the device's pow() are at most one unit in the last place of Float64 off the host's: the same Float32 factors but for a
    # value next to a border.  Then each of 42 steps, of at most 2 eta with 8-bit moments, is two places off, and the parameter rounded otherwise
    assert three.steps == one.steps == 42
    assert float((copies[0] - eager).abs().max()) <= 42 * 2.0 ** -23 * (4 * 0.01 + float(eager.abs().max()))
