"""8-bit layers on device tensors: rows normalised and / or coded in 8 bits, and the affine product of the codes.

The calls take torch tensors that live on the GPU and run on torch's current stream of their device; nothing synchronises, no
call keeps anything for the next.  A layer in a row:

    q, scale, h = int8.rms_norm_int8(x, gain, residual=h)        # NormalizeComponent, residual added, 8-bit output
    y = layer.propagate(q, scale, dtype=torch.bfloat16)          # AffineComponent (+ ReLU, BatchNorm) on the codes

8-bit rows are codes in [-127, 127] with one float scale per row: value ~ code * scale.  `kaldi_amd.int8` is the device-tensor
form of kamd_rms_norm_device, kamd_quantize_rows_device and kamd_component_i8_* (include/kaldi_amd.h), which a C or C++ host
calls on plain pointers.
"""
import ctypes as C

import torch

from . import abi
from ._lib import KamdError, lib

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_I8 = 3
_L = None


def _library():
    """The C-ABI library, on the same HIP runtime as torch: a process that loaded the library before torch has two of them, and
    streams of one mean nothing to the other."""
    global _L
    if _L is None:
        loaded = lib()
        with open("/proc/self/maps") as f:
            runtimes = {line.split()[-1] for line in f if "libamdhip64.so" in line}
        if len(runtimes) > 1:
            raise KamdError("kaldi_amd.int8: two HIP runtimes are loaded (%s): import torch before the library is used" % ", ".join(sorted(runtimes)))
        _L = loaded
    return _L


def _fail():
    raise KamdError(_L.kamd_last_error().decode())


def _matrix(t, what, dtype=None, like=None):
    """leading dimension of a matrix on the device; raises unless it is one"""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise KamdError("%s: a tensor on the GPU is expected" % what)
    if t.dim() != 2:
        raise KamdError("%s: a matrix is expected, got shape %s" % (what, tuple(t.shape)))
    if dtype is not None and t.dtype != dtype:
        raise KamdError("%s: %s expected, got %s" % (what, dtype, t.dtype))
    if like is not None and t.device != like.device:
        raise KamdError("%s: on %s, the other arguments on %s" % (what, t.device, like.device))
    rows, cols = t.shape
    ld, step = t.stride()
    if step != 1 and cols > 1:
        raise KamdError("%s: the values of a row have to be contiguous (strides %s)" % (what, (ld, step)))
    return ld if rows > 1 else max(ld, cols)


def _vector(t, n, what, like):
    if not isinstance(t, torch.Tensor) or t.device != like.device or t.dtype != torch.float32 or t.dim() != 1 or t.shape[0] != n:
        raise KamdError("%s: a float32 vector of %d on %s is expected" % (what, n, like.device))
    if not t.is_contiguous():
        raise KamdError("%s: has to be contiguous" % what)
    return t.data_ptr()


def _type(t, what):
    code = _TYPES.get(t.dtype)
    if code is None:
        raise KamdError("%s: float32, bfloat16 or float16 expected, got %s" % (what, t.dtype))
    return code


def _call(device, fn, *args):
    """fn(*args, stream) with `device` as the current one"""
    if device.index == torch.cuda.current_device():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(device.index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(device.index))
    if rc < 0:
        _fail()


def empty_codes(rows, dim, device):
    """[rows x dim] int8 in the layout the product takes: each row begins on a multiple of 16 bytes"""
    return torch.empty((rows, (dim + 15) // 16 * 16), dtype=torch.int8, device=device)[:, :dim]


def _norm(x, gain, eps, residual, sum_out, out, ld_out, out_type, scale):
    L = _library()
    ld_x = _matrix(x, "x")
    rows, dim = x.shape
    code = _type(x, "x")
    ld_r = ld_s = 0
    if residual is not None:
        ld_r = _matrix(residual, "residual", x.dtype, x)
        if sum_out is None:
            sum_out = torch.empty_like(x, memory_format=torch.contiguous_format)
    if sum_out is not None:
        ld_s = _matrix(sum_out, "sum_out", x.dtype, x)
    for t, what in ((residual, "residual"), (sum_out, "sum_out")):
        if t is not None and t.shape != x.shape:
            raise KamdError("%s: shape %s expected, got %s" % (what, tuple(x.shape), tuple(t.shape)))
    g = None if gain is None else _vector(gain, dim, "gain", x)
    if rows:
        _call(x.device, L.kamd_rms_norm_device, x.data_ptr(), ld_x, None if residual is None else residual.data_ptr(), ld_r, code, g, eps, rows, dim,
              None if sum_out is None else sum_out.data_ptr(), ld_s, out.data_ptr(), ld_out, code if out_type is None else out_type,
              None if scale is None else scale.data_ptr())
    return sum_out


def rms_norm(x, gain=None, eps=1e-6, residual=None, sum_out=None, out=None):
    """y = h / sqrt(mean(h^2) + eps) * gain per row, h = x + residual -> y, or (y, h) with a residual (kamd_rms_norm_device).

    x: [rows, dim] float32 / bfloat16 / float16, rows any stride apart; residual: the same shape and type; gain: float32 [dim].
    NormalizeComponent is gain = target_rms, eps = 2^-66.  sum_out (h) and out (y) may be given; sum_out may be x or residual,
    out any of the three."""
    ld_x = _matrix(x, "x")
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    ld_out = _matrix(out, "out", x.dtype, x)
    if out.shape != x.shape:
        raise KamdError("out: shape %s expected, got %s" % (tuple(x.shape), tuple(out.shape)))
    h = _norm(x, gain, eps, residual, sum_out, out, ld_out, None, None)
    return out if h is None else (out, h)


def rms_norm_int8(x, gain=None, eps=1e-6, residual=None, sum_out=None, out=None):
    """rms_norm with y as 8-bit rows -> (codes, scale), or (codes, scale, h) with a residual.  out = (codes, scale) may be given."""
    _matrix(x, "x")
    q, scale, ld_q = _codes_out(out, x.shape[0], x.shape[1], x)
    h = _norm(x, gain, eps, residual, sum_out, q, ld_q, _I8, scale)
    return (q, scale) if h is None else (q, scale, h)


def _codes_out(out, rows, dim, like):
    q, scale = out if out is not None else (empty_codes(rows, dim, like.device), torch.empty(rows, dtype=torch.float32, device=like.device))
    ld_q = _matrix(q, "codes", torch.int8, like)
    if tuple(q.shape) != (rows, dim):
        raise KamdError("codes: shape %s expected, got %s" % ((rows, dim), tuple(q.shape)))
    _vector(scale, rows, "scale", like)
    return q, scale, ld_q


def quantize_rows(x, offsets=(0,), out=None):
    """8-bit rows of a (spliced) matrix -> (codes, scale): row j codes Append_i x[j + offsets[i] - min(offsets)], so that
    x.rows - (max - min) rows come back (kamd_quantize_rows_device; the input of a layer with these time offsets)."""
    L = _library()
    ld_x = _matrix(x, "x")
    code = _type(x, "x")
    offsets = [int(o) for o in offsets]
    if not 1 <= len(offsets) <= abi.KAMD_MAX_OFFSETS:
        raise KamdError("offsets: between 1 and %d of them expected" % abi.KAMD_MAX_OFFSETS)
    rows = max(0, x.shape[0] - (max(offsets) - min(offsets)))
    q, scale, ld_q = _codes_out(out, rows, x.shape[1] * len(offsets), x)
    if rows:
        _call(x.device, L.kamd_quantize_rows_device, x.data_ptr(), ld_x, code, x.shape[0], x.shape[1], (C.c_int32 * len(offsets))(*offsets), len(offsets),
              q.data_ptr(), ld_q, scale.data_ptr())
    return q, scale


class AffineInt8:
    """The affine layer on 8-bit rows (kamd_component_i8): out = mul * relu(codes @ weight.T * scale * weight_scale + bias) + add.

    weight: int8 [out_dim, in_dim], weight_scale: float32 [out_dim], both on the device; bias, mul, add: float32 [out_dim] or
    None.  They are laid out for the matrix units once, here; the tensors are not kept."""

    def __init__(self, weight, weight_scale, bias=None, relu=False, mul=None, add=None):
        L = _library()
        ld = _matrix(weight, "weight", torch.int8)
        n, k = weight.shape
        vectors = [None if v is None else _vector(v, n, what, weight) for v, what in
                   ((weight_scale, "weight_scale"), (bias, "bias"), (mul, "mul"), (add, "add"))]
        self.device, self.offsets = weight.device, (0,)
        with torch.cuda.device(weight.device):
            self._take(L.kamd_component_i8_create_quantized(weight.data_ptr(), ld, vectors[0], k, n, vectors[1], int(bool(relu)), vectors[2], vectors[3],
                                                            torch.cuda.current_stream().cuda_stream))

    @classmethod
    def from_layer(cls, layer, device="cuda"):
        """From a `kaldi_amd.nnet.Layer` (float weights on the host, coded per output channel here), ReLU, BatchNorm and post
        maps included; `quantize_input` then splices with the layer's time offsets."""
        from .nnet import Model
        L = _library()
        self = cls.__new__(cls)
        self._h = None
        with torch.cuda.device(device):
            self.device, self.offsets = torch.device("cuda", torch.cuda.current_device()), tuple(layer.offsets)
            model = Model([layer], layer.in_dim, 0, 1, layer.out_dim)
            self._take(L.kamd_component_i8_create(model.descs()))
        return self

    def _take(self, handle):
        self._h = handle
        if not handle:
            _fail()
        self.in_dim, self.out_dim = _L.kamd_component_i8_input_dim(handle), _L.kamd_component_i8_output_dim(handle)

    def __del__(self):
        if getattr(self, "_h", None):
            _L.kamd_component_i8_destroy(self._h)
            self._h = None

    def quantize_input(self, x, out=None):
        """the codes and scales of the layer's spliced input"""
        return quantize_rows(x, self.offsets, out)

    def propagate(self, q, scale, dtype=torch.float32, out=None):
        """codes [rows, in_dim] and scales [rows] -> [rows, out_dim] of `dtype`"""
        ld_q = _matrix(q, "codes", torch.int8)
        rows, k = q.shape
        if k != self.in_dim or q.device != self.device:
            raise KamdError("codes: [rows, %d] on %s expected, got %s on %s" % (self.in_dim, self.device, tuple(q.shape), q.device))
        if rows <= 1:
            ld_q = (ld_q + 15) // 16 * 16
        if ld_q % 16 or q.data_ptr() % 16:
            raise KamdError("codes: rows begin on multiples of 16 bytes (int8.empty_codes has the layout)")
        if k % 16 and q.untyped_storage().nbytes() - q.storage_offset() < (rows - 1) * ld_q + (k + 15) // 16 * 16:
            raise KamdError("codes: the last row ends inside a block of 16 bytes that is not the tensor's own")
        s = _vector(scale, rows, "scale", q)
        if out is None:
            out = torch.empty((rows, self.out_dim), dtype=dtype, device=q.device)
        ld_out = _matrix(out, "out", dtype, q)
        if tuple(out.shape) != (rows, self.out_dim):
            raise KamdError("out: shape %s expected, got %s" % ((rows, self.out_dim), tuple(out.shape)))
        if rows:
            _call(q.device, _L.kamd_component_i8_propagate, self._h, q.data_ptr(), ld_q, s, rows, out.data_ptr(), ld_out, _type(out, "out"))
        return out

    def Propagate(self, x, dtype=None):
        """nnet3::Component::Propagate's shape (nnet3/nnet-component-itf.h:130-132): consecutive time steps in,
        x.rows - (max offset - min offset) rows out, in x's type unless `dtype` says otherwise"""
        q, scale = self.quantize_input(x)
        return self.propagate(q, scale, x.dtype if dtype is None else dtype)
