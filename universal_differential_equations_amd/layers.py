"""The gated feed-forward block as a network layer, next to the Dense chains of .models (scenario_1.jl:62-64, lambaem.jl:23-30):

    y = Wd (act(Wg x) .* (Wu x))

forward and pullback as single calls of libudecore's matrix-core kernels on torch CUDA tensors.  Rows of x are samples (the ABI's columns:
a row-major (T, D) tensor IS the column-major D x T matrix); a weight is an (out, in) tensor held by rows (torch.nn.Linear's order) or by
columns (`vec(W)` of Flux / Lux: W = torch.empty(n_in, n_out).T), all three in the same order.  Calls enqueue on torch's current stream and
wait for no other: what was made on another stream is waited for by the caller, as everywhere in torch.
"""
import ctypes as C

from . import _lib
from .sciml import Engine, current_raw_stream


def _order(name, w):
    """1: rows adjacent, 0: columns adjacent, None: either (a single row or column fits both)"""
    (rows, cols), (r, c) = w.shape, w.stride()
    by_rows = c == 1 or cols == 1
    by_cols = r == 1 or rows == 1
    if by_rows != by_cols:
        return 1 if by_rows else 0
    if not by_rows:
        raise ValueError("%s: one of its axes has to be contiguous, strides are %s" % (name, w.stride()))
    return None


def _ld(w, order):
    """elements from one row (order 1) or column (order 0) to the next"""
    (rows, cols), (r, c) = w.shape, w.stride()
    n, length, ld = (rows, cols, r) if order else (cols, rows, c)
    return ld if n > 1 else max(ld, length)


_KINDS = {}


def _kinds():
    """torch dtype -> UDE_DT_* (torch is not imported before the first call)"""
    if not _KINDS:
        import torch
        _KINDS.update({getattr(torch, k): _lib.DTYPE_CODE[k] for k in ("float32", "float16", "bfloat16")})
    return _KINDS


class _Block:
    """what one call knows: the descriptor and the tensors behind it"""

    def __init__(self, x, w_gate, w_up, w_down, act):
        import torch
        dev, dtype = x.device, x.dtype
        if dev.type != "cuda":
            raise ValueError("gated_ffn: x is on %s, a CUDA tensor is needed (there is no CPU fallback)" % dev)
        code = _kinds().get(dtype)
        if code is None:
            raise ValueError("gated_ffn: x is %s: float32, float16 and bfloat16 are supported" % dtype)
        if x.dim() < 1:
            raise ValueError("gated_ffn: x has no axis of features")
        for name, w in (("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down)):
            if w.dtype != dtype or w.device != dev:
                raise ValueError("gated_ffn: %s is %s on %s, x is %s on %s" % (name, w.dtype, w.device, dtype, dev))
            if w.dim() != 2:
                raise ValueError("gated_ffn: %s has %d axes, 2 are needed" % (name, w.dim()))
        d, f, o = x.shape[-1], w_gate.shape[0], w_down.shape[0]
        if w_gate.shape != (f, d) or w_up.shape != (f, d) or w_down.shape != (o, f):
            raise ValueError("gated_ffn: x (..., %d) with w_gate %s, w_up %s, w_down %s: (F, D), (F, D), (O, F) are needed"
                             % (d, tuple(w_gate.shape), tuple(w_up.shape), tuple(w_down.shape)))
        if min(d, f, o) < 1:
            raise ValueError("gated_ffn: D = %d, F = %d, O = %d" % (d, f, o))
        gate = _lib.GATE.get(act)
        if gate is None:
            raise ValueError("gated_ffn: act %r, one of %s is needed" % (act, sorted(_lib.GATE)))
        orders = {_order("gated_ffn: w_gate", w_gate), _order("gated_ffn: w_up", w_up), _order("gated_ffn: w_down", w_down)} - {None}
        if len(orders) > 1:
            raise ValueError("gated_ffn: the weights are held in different orders (strides %s)" % ", ".join(str(w.stride()) for w in (w_gate, w_up, w_down)))
        order = orders.pop() if orders else 1
        self.torch, self.shape, self.device, self.dtype = torch, x.shape, dev, dtype
        self.x = _rows(x if x.dim() == 2 else x.reshape(-1, d))
        self.w = (w_gate, w_up, w_down)
        self.D = _lib.GatedFfnDesc(code, gate, order, 0, self.x.shape[0], d, f, o, _row_ld(self.x), o,
                                   _ld(w_gate, order), _ld(w_up, order), _ld(w_down, order))
        self.gate, self.stream = None, current_raw_stream(dev.index)

    @property
    def eng(self):
        return Engine.get(self.device.index, keep_current=True)

    def workspace(self, pullback):
        n = C.c_int64(0)
        rc = _lib.load().ude_gated_ffn_workspace(C.byref(self.D), pullback, C.byref(n))
        if rc:
            raise _lib.UdeError(rc, "gated_ffn: sizes T = %d, D = %d, F = %d, O = %d" % (self.D.T, self.D.D, self.D.F, self.D.O))
        # (from torch's allocator on the current stream: a captured call gets memory of its graph, two calls never share one)
        return self.torch.empty(max(n.value, 256), dtype=self.torch.uint8, device=self.device), n.value

    def bind(self):
        """this thread's context, its operators on the current stream"""
        eng, stream = self.eng, current_raw_stream(self.device.index)
        eng.set_operator_stream(stream)
        if stream != self.stream:
            # held since the forward call, on its stream; of x's copy (see _rows) and of gate and up nobody else has a reference: the memory is not
            # given away before this stream is done with it
            now = self.torch.cuda.current_stream(self.device)
            for t in (self.x, *self.w, self.gate):
                if t is not None:
                    t.record_stream(now)
        return eng


def _rows(x):
    """x with contiguous rows that do not overlap (copied where it has not)"""
    (rows, cols), (r, c) = x.shape, x.stride()
    return x if (c == 1 or cols == 1) and (r >= cols or rows <= 1) else x.contiguous()


def _row_ld(x):
    """elements from one row of `_rows`' result to the next (of a single row: without gaps, whatever its stride says)"""
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _p(t):
    return t.data_ptr() if t is not None else None


def gated_ffn(x, w_gate, w_up, w_down, act="swish", save=False):
    """y = Wd (act(Wg x) .* (Wu x)) for every row of x (..., D); w_gate, w_up: (F, D), w_down: (O, F).  act: identity, tanh, rbf, relu,
    sigmoid, swish, gelu_tanh or gelu_erf.  save=True returns (y, saved) for `gated_ffn_pullback`: `saved` holds references to x and the
    weights -- change them in place only after the pullback -- and Wg x, Wu x in Float32.  No autograd graph is recorded: the pullback is the
    gradient.  Rounding: sums and act in Float32; act(..) .* (..) is rounded to x's dtype once, where it enters the last product, and so are its
    two cotangents in the pullback.  With float16 that is a matter of range too: a hidden value from 65520 on is infinite, also where y would not be, and
    a hidden cotangent under 3e-8 is zero, with its share of the gradients -- scale the loss (the pullback is linear in dy), or take bfloat16."""
    b = _Block(x, w_gate, w_up, w_down, act)
    torch, D = b.torch, b.D
    t, f, o = D.T, D.F, D.O
    y = torch.empty((t, o), dtype=b.dtype, device=b.device)
    b.gate = torch.empty((2, t, f), dtype=torch.float32, device=b.device) if save else None
    gate = b.gate.data_ptr() if save else None
    ws, size = b.workspace(0)
    eng = b.bind()
    eng.check(eng.L.ude_gated_ffn_forward_dev(eng.h, C.byref(D), b.x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr(),
                                              y.data_ptr(), gate, gate + 4 * t * f if save else None, ws.data_ptr(), size))
    if x.dim() != 2:
        y = y.view(*b.shape[:-1], o)
    return (y, b) if save else y


def gated_ffn_pullback(saved, dy, need=("x", "w_gate", "w_up", "w_down")):
    """(dx, dw_gate, dw_up, dw_down) for the cotangent dy (..., O) of a `gated_ffn(..., save=True)` call; None for what `need` leaves out.
    The gradients of the weights are contiguous in the weights' order.  May be called again on the same `saved`."""
    b = saved
    torch = b.torch
    if dy.dtype != b.dtype or dy.device != b.device or dy.shape[:-1] != b.shape[:-1] or dy.shape[-1] != b.D.O:
        raise ValueError("gated_ffn_pullback: dy is %s %s on %s, %s %s on %s is needed"
                         % (dy.dtype, tuple(dy.shape), dy.device, b.dtype, tuple(b.shape[:-1]) + (b.D.O,), b.device))
    unknown = set(need) - {"x", "w_gate", "w_up", "w_down"}
    if unknown:
        raise ValueError("gated_ffn_pullback: need has %s" % sorted(unknown))
    dy = _rows(dy if dy.dim() == 2 else dy.reshape(-1, b.D.O))
    D = _lib.GatedFfnDesc.from_buffer_copy(b.D)
    D.ldy = _row_ld(dy)
    t, f = D.T, D.F
    dx = torch.empty((t, D.D), dtype=b.dtype, device=b.device) if "x" in need else None
    grads = []
    for name, w in zip(("w_gate", "w_up", "w_down"), b.w):
        rows, cols = w.shape
        g = torch.empty((rows, cols) if D.w_order else (cols, rows), dtype=b.dtype, device=b.device) if name in need else None
        grads.append(g if g is None or D.w_order else g.T)
    ws, size = b.workspace(1)
    gate = b.gate.data_ptr()
    eng = b.bind()
    eng.check(eng.L.ude_gated_ffn_backward_dev(eng.h, C.byref(D), b.x.data_ptr(), *[w.data_ptr() for w in b.w], gate, gate + 4 * t * f, dy.data_ptr(),
                                               _p(dx), _p(grads[0]), _p(grads[1]), _p(grads[2]), ws.data_ptr(), size))
    if dx is not None and dx.shape != b.shape:
        dx = dx.view(b.shape)
    return (dx, *grads)
