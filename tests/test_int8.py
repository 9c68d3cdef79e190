"""The 8-bit layers' refusals and their C-ABI, without a GPU: every check of arguments comes before the device is touched."""
import ctypes as C

import numpy as np
import pytest
import torch          # before the library: they share one HIP runtime then

from kaldi_amd import abi
from kaldi_amd._lib import lib
from kaldi_amd.nnet import Layer, Model

P = C.c_void_p(1 << 20)         # stands for a device pointer: nothing may read it
F32, BF16, F16, I8 = 0, 1, 2, 3
ERR_ARG = -1


def norm(x=P, ld_x=8, residual=None, ld_r=0, type=F32, gain=None, eps=1e-6, rows=4, dim=8, sum=None, ld_sum=0, out=P, ld_out=8, out_type=F32, scale=None):
    return lib().kamd_rms_norm_device(x, ld_x, residual, ld_r, type, gain, eps, rows, dim, sum, ld_sum, out, ld_out, out_type, scale, None)


def quantize(x=P, ld_x=8, type=F32, rows=4, dim=8, offsets=(0,), n=None, q=P, ld_q=None, scale=P):
    off = (C.c_int32 * max(1, len(offsets)))(*offsets)
    n = len(offsets) if n is None else n
    return lib().kamd_quantize_rows_device(x, ld_x, type, rows, dim, off, n, q, dim * len(offsets) if ld_q is None else ld_q, scale, None)


@pytest.mark.parametrize("bad, says", [
    (dict(type=3), "input type"), (dict(type=-1), "input type"), (dict(out_type=BF16), "8 bits"), (dict(rows=-1), "sizes"), (dict(dim=0), "sizes"),
    (dict(eps=0.0), "eps"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(eps=1e-40), "eps"),
    (dict(ld_x=7), "leading"), (dict(ld_out=7), "leading"), (dict(residual=P, ld_r=7), "leading"), (dict(sum=P, ld_sum=7), "leading"),
    (dict(x=None), "null"), (dict(out=None), "null"), (dict(out_type=I8), "d_out_scale"),
])
def test_rms_norm_refuses(bad, says):
    assert norm(**bad) == ERR_ARG
    assert says in lib().kamd_last_error().decode()


def test_calls_without_rows_do_nothing():
    assert norm(rows=0, x=None, out=None) == 0
    assert quantize(rows=0, x=None) == 0
    assert quantize(rows=2, offsets=(-1, 0, 1), x=None) == 0        # no row has its context
    assert quantize(rows=6, offsets=(-3, 3), x=None) == 0


@pytest.mark.parametrize("bad, says", [
    (dict(type=3), "input type"), (dict(rows=-1), "sizes"), (dict(dim=0), "sizes"), (dict(n=0), "sizes"), (dict(n=9), "sizes"),
    (dict(dim=1 << 30, ld_x=1 << 30, offsets=(0, 1, 2), ld_q=1 << 32), "too long"), (dict(offsets=(-2 ** 31, 2 ** 31 - 1)), "far apart"),
    (dict(ld_x=7), "leading"), (dict(ld_q=7), "leading"), (dict(offsets=(0, 1), ld_q=15), "leading"), (dict(x=None), "null"), (dict(q=None), "null"), (dict(scale=None), "null"),
])
def test_quantize_rows_refuses(bad, says):
    assert quantize(**bad) == ERR_ARG
    assert says in lib().kamd_last_error().decode()


def test_component_i8_refuses():
    L = lib()

    def made(ld=8, in_dim=8, out_dim=4, w=P, scale=P):
        return L.kamd_component_i8_create_quantized(w, ld, scale, in_dim, out_dim, None, 0, None, None, None)

    for kw, says in ((dict(in_dim=0), "sizes"), (dict(out_dim=0), "sizes"), (dict(in_dim=131072, ld=131072), "131071"), (dict(ld=7), "leading"),
                     (dict(w=None), "null"), (dict(scale=None), "null"), (dict(out_dim=2 ** 31 - 1), "too many")):
        assert not made(**kw)
        assert says in L.kamd_last_error().decode(), kw
    W = np.ones((4, 8), np.float32)
    for layer, says in ((Layer("a", 8, 4, [0], -1, W, log_softmax=True), "plain"), (Layer("a", 4, 4, [0], -1, W, ivector_dim=4), "plain"),
                        (Layer("a", 8, 4, [0, 0], -1, W, slice_layers=[0, 1], slice_dims=[4, 4]), "plain")):
        assert not L.kamd_component_i8_create(Model([layer], 8, 0, 1, 4).descs())
        assert says in L.kamd_last_error().decode()
    assert not L.kamd_component_i8_create(None)
    for v in (np.nan, np.inf):
        W2 = W.copy()
        W2[2, 3] = v
        assert not L.kamd_component_i8_create(Model([Layer("a", 8, 4, [0], -1, W2)], 8, 0, 1, 4).descs())
        assert "weight 19 is not finite" in L.kamd_last_error().decode()
    assert L.kamd_component_i8_propagate(None, P, 16, P, 1, P, 16, F32, None) == ERR_ARG
    L.kamd_component_i8_destroy(None)


def test_tensors_off_the_gpu_are_refused():
    from kaldi_amd import int8
    from kaldi_amd._lib import KamdError
    x = torch.zeros(3, 8)
    for call in (lambda: int8.rms_norm(x), lambda: int8.rms_norm_int8(x), lambda: int8.quantize_rows(x), lambda: int8.quantize_rows(np.zeros((3, 8))),
                 lambda: int8.AffineInt8(x.to(torch.int8), torch.ones(3))):
        with pytest.raises(KamdError, match="on the GPU"):
            call()


def test_widths_a_launch_cannot_take_are_refused():
    L = lib()
    for in_dim, out_dim in ((8, 2 ** 26 + 1), (131071, 2 ** 18 + 1), (100000, 2 ** 26)):
        assert not L.kamd_component_i8_create_quantized(P, in_dim, P, in_dim, out_dim, None, 0, None, None, None)
        assert "too many outputs" in L.kamd_last_error().decode()


def test_tensors_without_memory_are_refused():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from kaldi_amd import int8
    from kaldi_amd._lib import KamdError
    with FakeTensorMode():
        x, w, v = torch.empty(3, 8, device="cuda"), torch.empty(4, 8, dtype=torch.int8, device="cuda"), torch.empty(4, device="cuda")
    for call in (lambda: int8.rms_norm(x), lambda: int8.rms_norm_int8(x), lambda: int8.quantize_rows(x), lambda: int8.AffineInt8(w, v)):
        with pytest.raises(KamdError, match="plain tensor"):
            call()


def test_a_handle_is_not_copied():
    import copy
    import pickle

    from kaldi_amd import int8
    from kaldi_amd._lib import KamdError
    layer = int8.AffineInt8.__new__(int8.AffineInt8)
    for call in (lambda: copy.copy(layer), lambda: copy.deepcopy(layer), lambda: pickle.dumps(layer)):
        with pytest.raises(KamdError, match="neither copied nor pickled"):
            call()


def refused(t, says):
    """what the calls look at in each of their tensors before anything else, on a tensor of the CPU"""
    from kaldi_amd import int8
    from kaldi_amd._lib import KamdError
    with pytest.raises(KamdError, match=says):
        int8._extension().plain(t, "t")


def test_wrappers_of_functionalization_are_refused():
    """their data_ptr() is null, which the C entries read as an argument that is not given"""
    seen = []

    def look(t):
        seen.append(t.data_ptr())
        refused(t, "plain tensor")
        return t + 1

    assert torch.func.functionalize(look)(torch.ones(4)).tolist() == [2.0] * 4
    assert seen == [0]


@pytest.mark.parametrize("left", [0, 16, 4 * 33 - 1])
def test_tensors_on_too_short_a_storage_are_refused(left):
    """a storage that was resized under its tensors: without memory their pointer is null, with some of it the rest would be read"""
    from kaldi_amd import int8
    from kaldi_amd._lib import KamdError
    whole = torch.zeros(6, 8)
    t = whole[1:5, 1:5]                       # spans elements 9 .. 36
    int8._extension().plain(t, "t")
    whole.untyped_storage().resize_(4 * 37)
    int8._extension().plain(t, "t")
    whole.untyped_storage().resize_(left)
    with pytest.raises(KamdError, match="shorter than the tensor"):          # (here: a failure prints no values of t)
        int8._extension().plain(t, "t")
    int8._extension().plain(torch.empty(0, 8), "t")


def test_vectors_that_ask_for_a_gradient_are_refused():
    """a layer's bias, maps and scales are copied into the handle: what is learned of them would be lost"""
    from kaldi_amd import int8
    from kaldi_amd._lib import KamdError
    v = torch.ones(4, requires_grad=True)
    with pytest.raises(KamdError, match="bias: has a gradient"):
        int8._vector(v, 4, "bias", torch.device("cpu"))
    with torch.no_grad():
        assert int8._vector(v, 4, "bias", torch.device("cpu")) == v.data_ptr()
    assert int8._vector(v.detach(), 4, "bias", torch.device("cpu")) == v.data_ptr()


def test_tensors_with_a_tangent_are_refused():
    import torch.autograd.forward_ad as fw
    from kaldi_amd import int8
    with fw.dual_level():
        t = fw.make_dual(torch.ones(4), torch.ones(4))
        refused(t, "tangent")
        with torch.no_grad():                     # (which switches the other direction off only)
            refused(t, "tangent")
        int8._extension().plain(t.detach(), "t")
        int8._extension().plain(fw.unpack_dual(t).primal, "t")


def test_calls_are_refused_while_torch_records():
    """a trace would hold their results as constants"""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    from kaldi_amd import int8
    from kaldi_amd._lib import KamdError
    calls = []

    def look(t):
        for call in (lambda: int8.rms_norm(t), lambda: int8.rms_norm_int8(t), lambda: int8.quantize_rows(t), lambda: int8._vector(t, 4, "t", t.device),
                     lambda: int8._extension().propagate(0, 4, 4, 0, t, t, torch.float32, None)):
            with pytest.raises(KamdError, match="cannot be traced"):
                call()
            calls.append(t)
        return t + 1

    x = torch.ones(4)
    torch.jit.trace(look, x, check_trace=False)
    make_fx(look)(x)
    with FakeTensorMode(allow_non_fake_inputs=True):
        look(x)
    assert len(calls) == 15
    int8._extension().plain(x, "x")


@pytest.mark.parametrize("shape", [(1, 2 ** 32 + 8), (2 ** 32 + 3, 1), (2 ** 31, 1)])
def test_weights_of_more_than_an_int_are_refused(shape):
    """(1, 2^32 + 8) was a layer of 8 inputs"""
    from kaldi_amd import int8
    from kaldi_amd._lib import KamdError

    class OnGpu(torch.Tensor):                    # is asked where it lives before its size
        is_cuda = True
    w = torch.zeros(1, dtype=torch.int8).expand(shape).as_subclass(OnGpu)
    with pytest.raises(KamdError, match="weight: %d x %d is too large" % shape):
        int8.AffineInt8(w, torch.ones(1).expand(shape[0]))


def test_overlapping_memory_is_found():
    """kamd::RowsMeet against the bytes themselves"""
    class Rows(C.Structure):
        _fields_ = [("p", C.c_void_p), ("ld", C.c_int64), ("width", C.c_int64), ("rows", C.c_int64)]
    meet = lib()["_ZN4kamd8RowsMeetERKNS_10MemoryRowsES2_"]
    meet.restype, meet.argtypes = C.c_bool, [C.POINTER(Rows), C.POINTER(Rows)]
    rng = np.random.default_rng(7)

    def draw(same_ld):
        rows, ld = int(rng.integers(1, 7)), same_ld or int(rng.integers(1, 24))
        return int(rng.integers(1000, 1090)), ld, int(rng.integers(1, ld + 1)) if rows > 1 else int(rng.integers(1, 40)), rows

    def touched(p, ld, width, rows):
        return {p + i * ld + j for i in range(rows) for j in range(width)}
    seen = [0, 0]
    for i in range(20000):
        same = int(rng.integers(1, 24)) if i % 2 else 0
        a, b = draw(same), draw(same)
        want = bool(touched(*a) & touched(*b))
        seen[want] += 1
        assert bool(meet(Rows(*a), Rows(*b))) == want, (a, b)
    assert min(seen) > 4000
    far = 1 << 46                                     # distances past 32 bits, and 2^30 rows of the same matrix
    assert meet(Rows(far, 1 << 20, 64, 1 << 30), Rows(far + (1 << 50) - (1 << 20) + 63, 1 << 20, 4, 2))
    assert not meet(Rows(far, 1 << 20, 64, 1 << 30), Rows(far + 64, 1 << 20, 64, 1 << 30))
    assert not meet(Rows(None, 1, 1, 1), Rows(None, 1, 1, 1))


def at(offset):
    return C.c_void_p((1 << 20) + offset)


@pytest.mark.parametrize("bad", [
    dict(out=at(4)), dict(out=at(0), ld_out=9), dict(out=at(4 * 8 * 3)), dict(out_type=BF16, type=BF16, out=at(2)),
    dict(out=at(4096), sum=at(16), ld_sum=8), dict(out=at(4096), residual=at(8192), ld_r=8, sum=at(8192), ld_sum=10),
    dict(out=at(4096), residual=at(8192 - 4), ld_r=8, sum=at(8192), ld_sum=8), dict(out=at(4096), sum=at(4096 + 4), ld_sum=8),
    dict(out=at(4096), gain=at(4096 + 32)), dict(out=at(4096), gain=at(8192), sum=at(8192), ld_sum=8),
    dict(out=at(0), out_type=I8, scale=at(4096)), dict(out=at(4096), out_type=I8, scale=at(4096 + 31)), dict(out=at(4096), out_type=I8, scale=at(12)),
    dict(out=at(4096), out_type=I8, scale=at(8192), gain=at(8192 + 12)),
])
def test_rms_norm_refuses_overlaps(bad):
    """an output that lies over another argument, but not exactly on a matrix of its type (4 rows of 8 are 128 bytes)"""
    assert norm(**bad) == ERR_ARG
    assert "overlaps" in lib().kamd_last_error().decode()


@pytest.mark.parametrize("bad", [dict(q=at(0), scale=at(4096)), dict(q=at(127), scale=at(4096)), dict(q=at(4096), scale=at(124)), dict(q=at(4096), scale=at(4096 + 28)),
                                 dict(q=at(4096), scale=at(4096 + 16), offsets=(0, 1))])
def test_quantize_rows_refuses_overlaps(bad):
    assert quantize(**bad) == ERR_ARG
    assert "overlaps" in lib().kamd_last_error().decode()


FAKE_HIP = r"""
// stands in for the HIP runtime: a device on which the Nth allocation and everything after it fails
#include <stddef.h>
int last, left;
static int result(int e) { if (e) last = e; return e; }
int hipGetDeviceCount(int *n) { *n = 1; return result(0); }
int hipGetDevice(int *d) { *d = 0; return result(0); }
int hipStreamIsCapturing(void *s, int *status) { (void)s; *status = 0; return result(0); }
int hipThreadExchangeStreamCaptureMode(int *m) { (void)m; return result(0); }
int hipMalloc(void **p, size_t n) { (void)n; *p = left > 0 ? (void *)4096 : NULL; return result(left-- > 0 ? 0 : 2); }
int hipFree(void *p) { (void)p; return result(1); }
int hipHostMalloc(void **p, size_t n, unsigned f) { (void)n; (void)f; *p = NULL; return result(2); }
int hipMemcpy(void *d, const void *s, size_t n, int k) { (void)d; (void)s; (void)n; (void)k; return result(2); }
int hipMemcpyAsync(void *d, const void *s, size_t n, int k, void *st) { (void)d; (void)s; (void)n; (void)k; (void)st; return result(2); }
int hipGetLastError(void) { int e = last; last = 0; return e; }
int hipPeekAtLastError(void) { return last; }
const char *hipGetErrorString(int e) { (void)e; return "out of memory"; }
"""

FAILED_LAYERS = r"""
import ctypes as C, sys
import numpy as np
fake = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)          # before the library: its calls find these
L = C.CDLL(sys.argv[2])
from kaldi_amd import abi
from kaldi_amd.nnet import Layer, Model
L.kamd_component_i8_create_quantized.restype = L.kamd_component_i8_create.restype = C.c_void_p
L.kamd_last_error.restype = C.c_char_p
left, last, P = C.c_int.in_dll(fake, "left"), C.c_int.in_dll(fake, "last"), C.c_void_p(1 << 20)
L.kamd_malloc.restype, L.kamd_malloc.argtypes = C.c_void_p, [C.c_size_t]
assert L.kamd_malloc(64) is None and left.value == -1   # it is the stand-in that the library has
fake.hipGetLastError()
for n in (0, 1):
    left.value = n
    assert not L.kamd_component_i8_create_quantized(P, C.c_int64(8), P, 8, 4, None, 0, None, None, None)
    assert b"out of memory" in L.kamd_last_error() and left.value == -1, L.kamd_last_error()
    assert last.value == 0, (n, last.value)
model = Model([Layer("a", 8, 4, [0], -1, np.ones((4, 8), np.float32))], 8, 0, 1, 4)
for n in (0, 1):
    left.value = n
    assert not L.kamd_component_i8_create(model.descs())
    assert b"out of memory" in L.kamd_last_error(), L.kamd_last_error()
    assert last.value == 0, (n, last.value)
print("fine")
"""


def test_a_layer_that_fails_leaves_no_error_behind(tmp_path):
    """torch asks for the thread's last error after each of its launches: that of a call which has told it is not to be found there"""
    import os
    import subprocess
    import sys

    import kaldi_amd
    (tmp_path / "fake.c").write_text(FAKE_HIP)
    subprocess.check_call(["gcc", "-shared", "-fPIC", "-o", str(tmp_path / "fake.so"), str(tmp_path / "fake.c")])
    root = os.path.dirname(os.path.abspath(kaldi_amd.__file__))
    r = subprocess.run([sys.executable, "-c", FAILED_LAYERS, str(tmp_path / "fake.so"), os.path.join(root, "lib", "libkaldi_amd.so")], capture_output=True, text=True,
                       cwd=os.path.dirname(root))
    assert r.stdout == "fine\n", r.stderr
