"""Refusals and host logic of the training operators; no GPU."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")


def lib():
    from universal_differential_equations_amd import _lib
    return _lib, _lib.load()


def desc(**kw):
    _lib, _ = lib()
    d = dict(dtype=3, act=5, w_order=1, T=4, D=8, F=16, O=8, ldx=8, ldy=8, ldg=8, ldu=8, ldd=16)
    d.update(kw)
    return _lib.GatedFfnDesc(**d)


def test_struct_sizes_match_header():
    _lib, _ = lib()
    assert C.sizeof(_lib.GatedFfnDesc) == 16 + 9 * 8
    assert C.sizeof(_lib.AdamwTensor) == 7 * 8 + 16
    assert C.sizeof(_lib.AdamwOpts) == 16 + 8 + 4 * 8 + 16


@pytest.mark.parametrize("kw,rc", [({}, 0), (dict(T=0), 0), (dict(dtype=0), -2), (dict(dtype=4), -2), (dict(act=8), -1), (dict(act=-1), -1), (dict(w_order=2), -1),
                                   (dict(reserved=1), -1), (dict(T=-1), -1), (dict(D=0), -1), (dict(F=0), -1), (dict(O=0), -1), (dict(T=2 ** 31), -1), (dict(F=2 ** 31), -1),
                                   (dict(ldx=7), -1), (dict(ldy=7), -1), (dict(ldg=7), -1), (dict(ldu=7), -1), (dict(ldd=15), -1), (dict(ldd=2 ** 32), -1),
                                   (dict(w_order=0), -1), (dict(w_order=0, ldg=16, ldu=16, ldd=8), 0)])
def test_gated_ffn_descriptor_refusals(kw, rc):
    _, L = lib()
    n = C.c_int64(-7)
    for pullback in (0, 1):
        assert L.ude_gated_ffn_workspace(C.byref(desc(**kw)), pullback, C.byref(n)) == rc
    assert L.ude_gated_ffn_workspace(C.byref(desc()), 0, None) == -1 and L.ude_gated_ffn_workspace(None, 0, C.byref(n)) == -1
    if rc == 0 and kw.get("T", 1):
        assert n.value >= 4 * 16 * 3 * 2


def test_no_context_is_refused():
    _lib, L = lib()
    assert L.ude_gated_ffn_forward_dev(None, C.byref(desc()), *[None] * 8, 0) == -1
    assert L.ude_gated_ffn_backward_dev(None, C.byref(desc()), *[None] * 12, 0) == -1
    assert L.ude_adamw_step_dev(None, C.byref(_lib.AdamwOpts()), 0, None) == -1
    assert L.ude_adamw_moments_dev(None, 0, None, None, None) == -1
    assert L.ude_grad_norm_dev(None, 1, 0, None, None, 1.0, None, None, 0) == -1


def test_grad_norm_workspace():
    _, L = lib()
    n = C.c_int64(0)
    for sizes in ([], [0], [1], [5, 0, 100000], [10] * 1000, [2 ** 33]):
        a = (C.c_int64 * len(sizes))(*sizes)
        assert L.ude_grad_norm_workspace(len(sizes), a, C.byref(n)) == 0 and 8 <= n.value <= 8 * 2048 * (1 + len(sizes) // 100)
    assert L.ude_grad_norm_workspace(1, (C.c_int64 * 1)(-1), C.byref(n)) == -1
    assert L.ude_grad_norm_workspace(-1, None, C.byref(n)) == -1


def test_cpu_tensors_are_refused():
    import universal_differential_equations_amd as U
    from universal_differential_equations_amd import training
    x, w = torch.zeros(2, 4), torch.zeros(4, 4)
    with pytest.raises(ValueError, match="CUDA"):
        U.gated_ffn(x, w, w, w)
    with pytest.raises(ValueError, match="CUDA"):
        training.AdamW([x])
    with pytest.raises(ValueError, match="CUDA"):
        training.grad_norm([x])
    with pytest.raises(ValueError, match="empty"):
        training.grad_norm([])
    with pytest.raises(ValueError, match="empty"):
        training.AdamW([])


def test_gated_ffn_shapes_and_orders():
    """the checks of the Python layer, on meta-free stand-ins: an object with the attributes of a CUDA tensor"""
    from universal_differential_equations_amd import layers
    a = torch.zeros(6, 4)
    assert layers._order("w", a) == 1 and layers._order("w", a.T) == 0 and layers._order("w", a[:1]) is None
    assert layers._order("w", a[:, :2]) == 1 and layers._order("w", a.T[:2]) == 0 and layers._order("w", a[:, :1]) == 1
    with pytest.raises(ValueError, match="contiguous"):
        layers._order("w", torch.zeros(6, 8)[::1, ::2])
    assert layers._ld(a, 1) == 4 and layers._ld(a.T, 0) == 4 and layers._ld(a[:, :2], 1) == 4 and layers._ld(torch.zeros(1, 4), 0) >= 1
    assert layers._rows(a.T).is_contiguous() and layers._rows(a[:, :3]).data_ptr() == a.data_ptr()


def test_adamw_host_loop():
    """training.adamw on numpy: the formula, written out for three steps; without decay and clipping, adam's trajectory"""
    from universal_differential_equations_amd import training
    th0 = np.array([1.0, -2.0, 0.5])

    def quad(th):
        return float(th @ th), 2 * th

    a, la = training.adam(quad, th0, eta=0.1, maxiters=5, eps=1e-8)
    b, lb = training.adamw(quad, th0, eta=0.1, maxiters=5, decay=0.0)
    assert np.allclose(a, b, rtol=1e-13) and np.allclose(la, lb, rtol=1e-13)
    th, m, v = th0.copy(), 0, 0
    for t in (1, 2, 3):
        g = 2 * th
        g = g * min(1, 0.5 / np.sqrt(g @ g))
        m, v = 0.9 * m + 0.1 * g, 0.999 * v + 0.001 * g * g
        th = th * (1 - 0.1 * 0.3) - 0.1 * (m / (1 - 0.9 ** t)) / (np.sqrt(v / (1 - 0.999 ** t)) + 1e-8)
    c, _ = training.adamw(quad, th0, eta=0.1, decay=0.3, maxiters=3, max_norm=0.5)
    assert np.allclose(c, th, rtol=1e-12)
    d, _ = training.adamw(quad, torch.tensor(th0), eta=0.1, decay=0.3, maxiters=3, max_norm=0.5)
    assert np.allclose(d.numpy(), th, rtol=1e-12)
    e, losses = training.adamw(quad, th0, maxiters=4, result="evaluated")
    assert abs(losses[-1] - float(e @ e)) < 1e-14
    f, losses = training.adamw(quad, th0, maxiters=4, callback=lambda th, l: True)
    assert np.array_equal(f, th0) and len(losses) == 1


def test_flux_adamw_tag():
    from universal_differential_equations_amd import pde
    o = pde.ADAMW(0.03, decay=0.01, max_norm=1.0)
    assert (o.eta, o.beta, o.decay, o.max_norm, o.eps) == (0.03, (0.9, 0.999), 0.01, 1.0, 1e-8)
    with pytest.raises(ValueError):
        pde.ADAMW(0.0)


@pytest.mark.parametrize("make", [lambda t: t.ones(1, 1).expand(5, 1), lambda t: t.ones(1, 3).expand(5, 3), lambda t: t.ones(5, 1).expand(5, 3),
                                  lambda t: t.arange(9.).as_strided((5, 3), (1, 1)), lambda t: t.arange(15.).view(3, 5).T, lambda t: t.ones(9, 3)[::2],
                                  lambda t: t.ones(5, 4)[:, :1], lambda t: t.ones(7, 3)[2:3], lambda t: t.ones(1, 3).as_strided((1, 3), (2 ** 40, 1))],
                         ids=["broadcast column", "broadcast row", "broadcast columns", "overlapping", "transposed", "every other row", "a column", "a row",
                              "a row with a far next"])
def test_rows_of_any_view(make):
    """what the kernels read through (address, leading dimension) is the tensor, for every view that x or dy may be"""
    from universal_differential_equations_amd import layers
    x = make(torch)
    y = layers._rows(x)
    n, cols = y.shape
    ld = layers._row_ld(y)
    last = (n - 1) * ld + cols  # the last element that is read, in the storage
    assert ld >= cols and y.storage_offset() + last <= y.untyped_storage().nbytes() // y.element_size()
    assert torch.equal(y.as_strided((n, cols), (ld, 1)), x)
