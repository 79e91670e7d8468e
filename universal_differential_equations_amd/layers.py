"""The gated feed-forward block as a network layer, next to the Dense chains of .models (scenario_1.jl:62-64, lambaem.jl:23-30):

    y = Wd (act(Wg x) .* (Wu x))

forward and pullback as single calls of libudecore's matrix-core kernels on torch CUDA tensors.  Rows of x are samples (the ABI's columns:
a row-major (T, D) tensor IS the column-major D x T matrix); a weight is an (out, in) tensor held by rows (torch.nn.Linear's order) or by
columns (`vec(W)` of Flux / Lux: W = torch.empty(n_in, n_out).T), all three in the same order.
"""
import ctypes as C

from . import _lib
from .sciml import Engine


def _order(name, w):
    """1: rows adjacent, 0: columns adjacent, None: either (a single row or column fits both)"""
    rows, cols = w.shape
    by_rows = w.stride(1) == 1 or cols == 1
    by_cols = w.stride(0) == 1 or rows == 1
    if by_rows and by_cols:
        return None
    if not by_rows and not by_cols:
        raise ValueError("%s: one of its axes has to be contiguous, strides are %s" % (name, w.stride()))
    return 1 if by_rows else 0


def _ld(w, order):
    """elements from one row (order 1) or column (order 0) to the next"""
    rows, cols = w.shape
    n, length, ld = (rows, cols, w.stride(0)) if order else (cols, rows, w.stride(1))
    return ld if n > 1 else max(ld, length)


class _Block:
    """what one call knows: the descriptor and the tensors behind it"""

    def __init__(self, x, w_gate, w_up, w_down, act):
        import torch
        ws = (("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down))
        if x.device.type != "cuda":
            raise ValueError("gated_ffn: x is on %s, a CUDA tensor is needed (there is no CPU fallback)" % x.device)
        if str(x.dtype)[6:] not in ("float32", "float16", "bfloat16"):
            raise ValueError("gated_ffn: x is %s: float32, float16 and bfloat16 are supported" % x.dtype)
        if x.dim() < 1:
            raise ValueError("gated_ffn: x has no axis of features")
        for name, w in ws:
            if w.device != x.device or w.dtype != x.dtype:
                raise ValueError("gated_ffn: %s is %s on %s, x is %s on %s" % (name, w.dtype, w.device, x.dtype, x.device))
            if w.dim() != 2:
                raise ValueError("gated_ffn: %s has %d axes, 2 are needed" % (name, w.dim()))
        d, f, o = x.shape[-1], w_gate.shape[0], w_down.shape[0]
        if tuple(w_gate.shape) != (f, d) or tuple(w_up.shape) != (f, d) or tuple(w_down.shape) != (o, f):
            raise ValueError("gated_ffn: x (..., %d) with w_gate %s, w_up %s, w_down %s: (F, D), (F, D), (O, F) are needed"
                             % (d, tuple(w_gate.shape), tuple(w_up.shape), tuple(w_down.shape)))
        if act not in _lib.GATE:
            raise ValueError("gated_ffn: act %r, one of %s is needed" % (act, sorted(_lib.GATE)))
        orders = {o_ for o_ in (_order(name, w) for name, w in ws) if o_ is not None}
        if len(orders) > 1:
            raise ValueError("gated_ffn: the weights are held in different orders (strides %s)" % ", ".join(str(w.stride()) for _, w in ws))
        order = orders.pop() if orders else 1
        self.torch, self.shape, self.act = torch, x.shape, act
        self.x = _rows(x.reshape(-1, d))
        self.w = (w_gate, w_up, w_down)
        D = _lib.GatedFfnDesc()
        D.dtype, D.act, D.w_order = _lib.DTYPE_CODE[str(x.dtype)[6:]], _lib.GATE[act], order
        D.T, D.D, D.F, D.O = self.x.shape[0], d, f, o
        D.ldx, D.ldy = max(self.x.stride(0), d), o
        D.ldg, D.ldu, D.ldd = _ld(w_gate, order), _ld(w_up, order), _ld(w_down, order)
        self.D = D
        self.eng = Engine.get(x.device.index)

    def workspace(self, pullback):
        n = C.c_int64(0)
        rc = self.eng.L.ude_gated_ffn_workspace(C.byref(self.D), pullback, C.byref(n))
        if rc:
            raise _lib.UdeError(rc, "gated_ffn: sizes T = %d, D = %d, F = %d, O = %d" % (self.D.T, self.D.D, self.D.F, self.D.O))
        # (from torch's allocator on the current stream: a captured call gets memory of its graph, two calls never share one)
        return self.torch.empty(max(n.value, 256), dtype=self.torch.uint8, device=self.x.device)

    def bind(self):
        self.eng.set_stream(self.torch.cuda.current_stream(self.x.device).cuda_stream)


def _rows(x):
    """x with contiguous rows (copied where it has not)"""
    return x if x.shape[1] == 1 or (x.stride(1) == 1 and (x.stride(0) >= x.shape[1] or x.shape[0] <= 1)) else x.contiguous()


def _p(t):
    return t.data_ptr() if t is not None else None


def gated_ffn(x, w_gate, w_up, w_down, act="swish", save=False):
    """y = Wd (act(Wg x) .* (Wu x)) for every row of x (..., D); w_gate, w_up: (F, D), w_down: (O, F).  act: identity, tanh, rbf, relu,
    sigmoid, swish, gelu_tanh or gelu_erf.  save=True returns (y, saved) for `gated_ffn_pullback`: `saved` holds references to x and the
    weights -- change them in place only after the pullback -- and Wg x, Wu x in Float32."""
    b = _Block(x, w_gate, w_up, w_down, act)
    torch = b.torch
    t, f, o = b.D.T, b.D.F, b.D.O
    y = torch.empty((t, o), dtype=x.dtype, device=x.device)
    b.gate = torch.empty((2, t, f), dtype=torch.float32, device=x.device) if save else None
    ws = b.workspace(0)
    b.bind()
    b.eng.check(b.eng.L.ude_gated_ffn_forward_dev(b.eng.h, C.byref(b.D), _p(b.x), _p(w_gate), _p(w_up), _p(w_down), _p(y),
                                                  _p(b.gate), b.gate.data_ptr() + 4 * t * f if save else None, _p(ws), ws.numel()))
    y = y.view(*b.shape[:-1], o)
    return (y, b) if save else y


def gated_ffn_pullback(saved, dy, need=("x", "w_gate", "w_up", "w_down")):
    """(dx, dw_gate, dw_up, dw_down) for the cotangent dy (..., O) of a `gated_ffn(..., save=True)` call; None for what `need` leaves out.
    The gradients of the weights are contiguous in the weights' order.  May be called again on the same `saved`."""
    b = saved
    torch = b.torch
    if dy.device != b.x.device or dy.dtype != b.x.dtype or tuple(dy.shape) != tuple(b.shape[:-1]) + (b.D.O,):
        raise ValueError("gated_ffn_pullback: dy is %s %s on %s, %s %s on %s is needed"
                         % (dy.dtype, tuple(dy.shape), dy.device, b.x.dtype, tuple(b.shape[:-1]) + (b.D.O,), b.x.device))
    unknown = set(need) - {"x", "w_gate", "w_up", "w_down"}
    if unknown:
        raise ValueError("gated_ffn_pullback: need has %s" % sorted(unknown))
    dy = _rows(dy.reshape(-1, b.D.O))
    D = _lib.GatedFfnDesc.from_buffer_copy(b.D)
    D.ldy = max(dy.stride(0), D.O)
    t, f = D.T, D.F
    dx = torch.empty((t, D.D), dtype=dy.dtype, device=dy.device) if "x" in need else None
    grads = []
    for name, w in zip(("w_gate", "w_up", "w_down"), b.w):
        rows, cols = w.shape
        g = torch.empty((rows, cols) if D.w_order else (cols, rows), dtype=dy.dtype, device=dy.device) if name in need else None
        grads.append(g if g is None or D.w_order else g.T)
    ws = torch.empty(0, device=dy.device) if t == 0 else b.workspace(1)
    b.bind()
    b.eng.check(b.eng.L.ude_gated_ffn_backward_dev(b.eng.h, C.byref(D), _p(b.x), _p(b.w[0]), _p(b.w[1]), _p(b.w[2]),
                                                   _p(b.gate), b.gate.data_ptr() + 4 * t * f, _p(dy), _p(dx), _p(grads[0]), _p(grads[1]), _p(grads[2]),
                                                   _p(ws) or None, ws.numel()))
    if dx is not None:
        dx = dx.view(b.shape)
    return (dx,) + tuple(grads)
