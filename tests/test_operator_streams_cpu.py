"""The training operators beside a context's other calls: which stream they launch on, what waits for what, which device stays current.  In a
process of its own, with the HIP runtime replaced by tests/fake_hip.c; no GPU."""
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
A, B, S = 0x1000, 0x2000, 0x3000    # streams

SETUP = """
import ctypes as C, sys, types
sys.modules["torch"] = None          # (nothing here may load the real runtime's users)
fake = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
fake.fake_log.restype = C.c_char_p
fake.fake_capture.argtypes = [C.c_size_t]
sys.path.insert(0, sys.argv[2])
from universal_differential_equations_amd import _lib, layers, sciml, training
A, B, S = 0x1000, 0x2000, 0x3000
at = {"stream": A}
for module in (layers, training, sciml):
    module.current_raw_stream = lambda device: at["stream"]
class Kept:
    def __init__(self, p=1 << 20):
        self.p = p
    def record_stream(self, s):
        pass
    def data_ptr(self):
        return self.p
class Device:                        # torch.cuda.device
    def __init__(self, d):
        self.d = d
    def __enter__(self):
        self.old = fake.fake_device()
        fake.hipSetDevice(self.d)
    def __exit__(self, *a):
        fake.hipSetDevice(self.old)
cuda = types.SimpleNamespace(current_stream=lambda d: at["stream"], device=Device, is_current_stream_capturing=lambda: False)
sys.modules["torch"] = types.SimpleNamespace(cuda=cuda)
def block(device=0, stream=A):
    b = layers._Block.__new__(layers._Block)
    b.torch, b.device, b.stream = types.SimpleNamespace(cuda=cuda), types.SimpleNamespace(index=device), stream
    b.x, b.w, b.gate = Kept(), (Kept(),) * 3, None
    b.D = _lib.GatedFfnDesc(3, 5, 1, 0, 8, 64, 64, 64, 64, 64, 64, 64, 64)
    return b
def forward(b):
    n = C.c_int64(0)
    eng = b.bind()
    assert eng.L.ude_gated_ffn_workspace(C.byref(b.D), 0, C.byref(n)) == 0
    eng.check(eng.L.ude_gated_ffn_forward_dev(eng.h, C.byref(b.D), *[1 << 20] * 5, None, None, 1 << 24, n.value))
def log():
    lines = [l.split() for l in fake.fake_log().decode().splitlines()]
    fake.fake_clear()
    return [(l[0], int(l[1]), int(l[2])) for l in lines]
"""


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    lib = str(tmp_path_factory.mktemp("fake_hip") / "libfake_hip.so")
    subprocess.check_call(["gcc", "-shared", "-fPIC", "-O1", "-fno-builtin", "-o", lib, os.path.join(HERE, "fake_hip.c")])
    return lib


def run(fake, code):
    r = subprocess.run([sys.executable, "-c", SETUP + code, fake, os.path.dirname(HERE)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr


def test_operators_wait_for_nothing_on_another_stream(fake):
    """they use none of the context's memory: on a side stream they overlap with what is queued on the main one"""
    run(fake, """
forward(block()); assert {l[:2] for l in log()} == {("launch", A)}
at["stream"] = S
forward(block(stream=S)); got = log(); assert {l[:2] for l in got} == {("launch", S)}, got
eng = training._bound_engine(types.SimpleNamespace(index=0))
n = (C.c_int64 * 1)(100)
p = (C.c_void_p * 1)(1 << 20)
eng.check(eng.L.ude_grad_norm_dev(eng.h, 1, 1, p, n, 1.0, 1 << 21, 1 << 22, 4096))
t = (_lib.AdamwTensor * 1)(); t[0].param = t[0].grad = t[0].m = t[0].v = t[0].m_scale = t[0].v_scale = 1 << 20; t[0].n = 100
o = _lib.AdamwOpts(param_dtype=1, grad_dtype=1, state_bits=32, step=1, eta=.1, beta1=.9, beta2=.9, eps=.1)
eng.check(eng.L.ude_adamw_step_dev(eng.h, C.byref(o), 1, t))
eng.check(eng.L.ude_adamw_moments_dev(eng.h, 1, t, p, p))
got = log(); assert len(got) == 3 and {l[:2] for l in got} == {("launch", S)}, got
""")


@pytest.mark.parametrize("captured", [False, True])
def test_a_solve_on_another_stream_still_waits_for_the_one_before(fake, captured):
    """the context's workspaces pass from a solve on A to one on B by an event, whatever operators ran, or were captured, in between"""
    run(fake, """
eng = sciml.Engine.get(0)
eng.set_stream(A); log()
at["stream"] = S
if %r: fake.fake_capture(S)
forward(block(stream=S)); got = log(); assert {l[:2] for l in got} == {("launch", S)}, got
fake.fake_capture(0)
eng.set_stream(B)
assert [l[:2] for l in log()] == [("record", A), ("wait", B)]
""" % captured)


def test_a_stream_set_later_counts(fake):
    """for C callers: the context's stream, where no other is set for the operators after it"""
    run(fake, """
eng = sciml.Engine.get(0)
def go(b=block()):
    n = C.c_int64(0)
    eng.L.ude_gated_ffn_workspace(C.byref(b.D), 0, C.byref(n))
    eng.check(eng.L.ude_gated_ffn_forward_dev(eng.h, C.byref(b.D), *[1 << 20] * 5, None, None, 1 << 24, n.value))
    got = {l[1] for l in log() if l[0] == "launch"}
    assert len(got) == 1
    return got.pop()
assert go() == 0
eng.set_stream(A); assert go() == A
assert eng.L.ude_set_operator_stream(eng.h, C.c_void_p(S)) == 0; assert go() == S
eng.set_stream(A); assert go() == A
assert eng.L.ude_set_operator_stream(None, None) == -1
""")


def test_the_current_device_stays(fake):
    """operators on device 1, the first of which makes that device's context, while device 0 is the current one"""
    run(fake, """
assert fake.fake_device() == 0
forward(block(device=1)); got = log(); assert {l for l in got} == {("launch", A, 1)}, got
assert fake.fake_device() == 0
at["stream"] = S
forward(block(device=1, stream=S))
assert fake.fake_device() == 0
""")


def test_the_current_device_stays_in_the_optimiser(fake):
    run(fake, """
training._bound_engine(types.SimpleNamespace(index=1))
assert fake.fake_device() == 0
at["stream"] = S
training._bound_engine(types.SimpleNamespace(index=1))
assert fake.fake_device() == 0
""")


def test_the_first_call_of_a_thread_inside_a_capture_is_refused(fake):
    """it would make the thread's context, whose allocations end a capture; afterwards, and with a context there, captures are taken"""
    run(fake, """
cuda.is_current_stream_capturing = lambda: True
for go in (lambda: block().bind(), lambda: training._bound_engine(types.SimpleNamespace(index=0))):
    try:
        go()
        assert False, "not refused"
    except ValueError as e:
        assert "captured" in str(e)
assert not sciml.Engine._by_device and not log()
cuda.is_current_stream_capturing = lambda: False
block().bind()
cuda.is_current_stream_capturing = lambda: True
fake.fake_capture(A)
forward(block()); got = log(); assert {l[:2] for l in got} == {("launch", A)}, got
""")
