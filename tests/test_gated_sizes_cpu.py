"""Workspaces of the gated block for sizes whose products pass 64 bits; no GPU."""
import ctypes as C

import pytest

MOST = 2 ** 31 - 1 - 1024
UNSUPPORTED = -2


def ask(pullback, **kw):
    from universal_differential_equations_amd import _lib
    d = dict(dtype=1, act=5, w_order=1, T=4, D=8, F=16, O=8)
    d.update(kw)
    d.update(ldx=d["D"], ldy=d["O"], ldg=d["D"], ldu=d["D"], ldd=d["F"])
    if d["w_order"] == 0:
        d.update(ldg=d["F"], ldu=d["F"], ldd=d["O"])
    n = C.c_int64(-7)
    return _lib.load().ude_gated_ffn_workspace(C.byref(_lib.GatedFfnDesc(**d)), pullback, C.byref(n)), n.value


@pytest.mark.parametrize("dtype,size", [(1, 4), (2, 2), (3, 2)])
@pytest.mark.parametrize("order", [0, 1])
def test_bytes_are_those_of_the_hidden_layer_or_refused(dtype, size, order):
    """h in a forward call, h and its two cotangents in a pullback, each T x F in the block's type, and at most 33.6 MB of parts: never fewer bytes
    than that, whatever the sizes are"""
    big = (1, 1000, 2 ** 20 + 3, 2 ** 27, MOST)
    for T in big:
        for F in (1, 5000, 2 ** 22 + 1, MOST // 2):
            for D in (1, 2 ** 22 + 5, MOST):
                for O in (1, MOST):
                    for pullback in (0, 1):
                        rc, n = ask(pullback, dtype=dtype, w_order=order, T=T, F=F, D=D, O=O)
                        need = T * F * size * (3 if pullback else 1)
                        if need < 2 ** 59:
                            assert rc == 0 and need <= n <= T * (F + 7) * size * (3 if pullback else 1) + 512 + 2 * 256 * 128 * 128 * 4, (T, D, F, O, pullback, n)
                        else:
                            assert rc == UNSUPPORTED or (rc == 0 and n >= need), (T, D, F, O, pullback, rc, n)


def test_parts_of_long_products_have_room():
    """a product with few tiles and a K beyond them, whose number of parts times their bytes passes 64 bits before it is cut to what is used"""
    for kw in (dict(T=32, F=MOST // 2, D=MOST), dict(T=2 ** 20, F=64, D=MOST, O=MOST), dict(T=MOST, F=128, D=128, O=128)):
        for pullback in (0, 1):
            rc, n = ask(pullback, **kw)
            assert rc == 0 and n >= kw["T"] * kw["F"] * 4 * (3 if pullback else 1) + 2 * 256 * 128 * 128 * 4 - 512, (kw, n)
