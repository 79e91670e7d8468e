"""What an AdamW step takes, refuses and counts: the host's part of it, on CPU tensors with the launch replaced by a record; no GPU."""
import ctypes as C
import types

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture
def training(monkeypatch):
    """the module, whose device checks take CPU tensors and whose launches append what they are given to `training.launched`: one dict of
    (grad as floats in the parameter's order, n) per tensor, and the step number"""
    from universal_differential_equations_amd import _lib, training
    launched, recorded = [], []

    def launch(handle, o, n, table):
        grads = []
        for i in range(n):
            t = table[i]
            grads.append(list((C.c_float * t.n).from_address(t.grad)) if t.n else None)
        launched.append(types.SimpleNamespace(step=o._obj.step, step_dev=o._obj.step_dev, grads=grads))
        return 0

    def check(rc):
        assert rc == 0

    eng = types.SimpleNamespace(h=None, check=check, operator_stream=7, L=types.SimpleNamespace(ude_adamw_step_dev=launch))
    monkeypatch.setattr(training, "_device_list", lambda what, ts: (ts[0].device, str(ts[0].dtype)[6:]))
    monkeypatch.setattr(training, "_bound_engine", lambda dev: eng)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: "stream %d" % eng.operator_stream)
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, stream: recorded.append((t.data_ptr(), stream)))
    monkeypatch.setattr(training, "launched", launched, raising=False)
    monkeypatch.setattr(training, "recorded", recorded, raising=False)
    assert _lib.ADAMW_BLOCK == 256
    return training


def test_a_gradient_of_another_shape_is_refused(training):
    """as many elements in another order: (D, F) parameters and the (F, D) gradient of their transpose"""
    p, q = torch.zeros(3, 5), torch.zeros(4)
    opt = training.AdamW([p, q])
    for bad in ((5, 3), (15,), (15, 1), (1, 3, 5)):
        with pytest.raises(ValueError, match="gradient 0"):
            opt.step([torch.ones(bad), torch.ones(4)])
        with pytest.raises(ValueError, match="gradient 0"):
            opt.step([torch.ones(bad), None])
    with pytest.raises(ValueError, match="gradient 1"):
        opt.step([None, torch.ones(2, 2)])
    assert opt.steps == 0 and not training.launched


def test_a_gradient_of_another_stride_order_is_taken_element_by_element(training):
    p = torch.zeros(3, 5)
    opt = training.AdamW([p])
    g = torch.arange(15.0).reshape(5, 3).T    # (3, 5), columns adjacent: what a pullback by columns hands back
    opt.step([g])
    opt.step([g.contiguous()])
    opt.step([None])
    assert [x.grads[0] for x in training.launched] == [g.reshape(-1).tolist()] * 2 + [None]
    assert [x.step for x in training.launched] == [1, 2, 3] and opt.steps == 3


def test_a_reshaped_or_transposed_parameter(training):
    """other views of the same storage, which starts where it did"""
    p = torch.zeros(3, 5)
    opt = training.AdamW([p])
    p.data = p.data.view(5, 3)
    opt.step([torch.ones(5, 3)])
    opt.step([torch.ones(5, 3)])
    with pytest.raises(ValueError, match="gradient 0"):
        opt.step([torch.ones(3, 5)])
    p.data = torch.zeros(4, 4)
    with pytest.raises(ValueError, match="parameter 0"):
        opt.step([torch.ones(4, 4)])
    p = torch.zeros(12)
    opt = training.AdamW([p])
    p.data = p.data[:4]   # (starts where it did, and is shorter than the moments)
    with pytest.raises(ValueError, match="parameter 0"):
        opt.step([torch.ones(4)])
    q = torch.zeros(4, 4)
    opt = training.AdamW([q])
    q.data = q.data.T
    with pytest.raises(ValueError, match="parameter 0"):
        opt.step([torch.ones(4, 4)])
    assert opt.steps == 0


def test_steps_counted_on_the_device_are_the_steps(training, monkeypatch):
    """capturable=True: a replayed graph counts in `count` alone, and `steps` is what another instance continues from"""
    p = torch.zeros(6)
    opt = training.AdamW([p], capturable=True, step=4)
    assert opt.steps == 4
    opt.step([torch.ones(6)])
    assert opt.steps == 5 and int(opt.count) == 5 and training.launched[-1].step_dev == opt.count.data_ptr()
    opt.count.add_(1000)   # (what replays do)
    assert opt.steps == 1005
    two = training.AdamW([torch.zeros(6)], step=opt.steps)
    two.step([torch.ones(6)])
    assert training.launched[-1].step == 1006 and two.steps == 1006
    opt.steps = 7
    assert opt.steps == 7 and int(opt.count) == 7
    two.steps = 7
    two.step([torch.ones(6)])
    assert training.launched[-1].step == 8 and two.steps == 8 and two.count is None
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(ValueError, match="captur"):
        opt.steps


def test_a_refused_launch_is_not_counted(training):
    from universal_differential_equations_amd import UdeError

    def check(rc):
        if rc:
            raise UdeError(rc, "refused")

    eng = training._bound_engine(None)
    eng.check, eng.L.ude_adamw_step_dev = check, lambda *a: -1
    for capturable in (True, False):
        opt = training.AdamW([torch.zeros(6)], capturable=capturable)
        with pytest.raises(UdeError):
            opt.step([torch.ones(6)])
        assert opt.steps == 0


def test_parameter_arrays_of_the_deep_bsde_networks():
    """their lengths, in the order of the flat vector: a glorot-uniform weight (no zero but by chance) and a zero bias in turn"""
    import numpy as np
    from universal_differential_equations_amd import pde
    for d, hls in ((100, 110), (3, 7), (1, 1)):
        nets = pde.NNPDENS(d, hls)
        sizes, theta = nets.array_sizes(), nets.init_params(np.random.default_rng(0))
        assert len(sizes) == 14 and sum(sizes) == theta.size == sum(nets.num_params()) and sum(sizes[:6]) == nets.num_params()[0]
        for i, part in enumerate(np.split(theta, np.cumsum(sizes)[:-1])):
            assert part.any() == (i % 2 == 0)


def test_states_are_kept_for_every_stream_that_steps(training):
    """moments, scales, copies and the count are the instance's own: where it is dropped while a step is pending on another stream than they were
    made on, their memory is not given away before"""
    for kw in (dict(bits=32), dict(bits=8, capturable=True), dict(bits=32, master=True)):
        p, q = (torch.zeros(600, dtype=torch.bfloat16 if "master" in kw else torch.float32) for _ in range(2))
        opt = training.AdamW([p, q], **kw)
        own = sorted(t.data_ptr() for t in [x for s in opt.state for x in s.values()] + ([opt.count] if kw.get("capturable") else []))
        eng = training._bound_engine(None)
        del training.recorded[:]
        for eng.operator_stream in (7, 9, 9, 7):
            opt.step([None, None])
        assert sorted(x for x, stream in training.recorded if stream == "stream 9") == own
        assert len(training.recorded) == 2 * len(own)    # (once a stream)
        if opt.bits == 8:
            eng.L.ude_adamw_moments_dev = lambda *a: 0
            eng.operator_stream = 11
            opt.moments()
            assert sorted(x for x, stream in training.recorded if stream == "stream 11") == own
        eng.operator_stream = 7


def test_parameters_that_were_given_shared_storage_are_refused(training):
    """two chunks of a launch would update the same element at once"""
    store = torch.zeros(20)
    p, q = torch.zeros(8), torch.zeros(8)
    opt = training.AdamW([p, q])
    for first, second in ((p.data, p.data), (store[:8], store[4:12])):
        p.data, q.data = first, second
        with pytest.raises(ValueError, match="share"):
            opt.step([torch.ones(8)] * 2)
    q.data = opt.state[0]["m"]
    with pytest.raises(ValueError, match="share"):
        opt.step([torch.ones(8)] * 2)
    q.data = store[8:16]
    opt.step([torch.ones(8)] * 2)
    assert opt.steps == 1 and len(training.launched) == 1


@pytest.mark.parametrize("most", [0, 0.0, -1.0, float("nan")])
def test_a_norm_to_scale_to_is_positive(most):
    """0 would scale to nothing on the host and not at all on the device (where grad_norm takes it for `no limit`)"""
    import numpy as np
    from universal_differential_equations_amd import pde, training as T
    with pytest.raises(ValueError, match="max_norm"):
        T.adamw(lambda th: (float(th @ th), 2 * th), np.ones(3), maxiters=2, max_norm=most)
    with pytest.raises(ValueError, match="max_norm"):
        pde.ADAMW(0.01, max_norm=most)


def test_steps_with_and_without_some_gradients_in_turn(training):
    """the table that is kept between steps: which tensors a launch leaves out is decided by that step's gradients alone"""
    ps = [torch.zeros(4), torch.zeros(5), torch.zeros(6)]
    opt = training.AdamW(ps, bits=8)
    training._bound_engine(None).L.ude_adamw_moments_dev = lambda *a: 0
    gs = [torch.full((k,), float(k)) for k in (4, 5, 6)]
    want = []
    for keep in ((1, 1, 1), (1, 0, 1), (0, 0, 0), (1, 1, 1), (0, 1, 0), (0, 1, 1), (1, 1, 1), (1, 1, 1)):
        given = [g if k else None for g, k in zip(gs, keep)]
        opt.step(given)
        want.append([None if g is None else g.tolist() for g in given])
        opt.moments()
        with pytest.raises(ValueError):
            opt.step([None, gs[0], gs[2]])
    assert [x.grads for x in training.launched] == want
