"""8-bit layers on device tensors: rows normalised and / or coded in 8 bits, and the affine product of the codes.

The calls take torch tensors that live on the GPU and run on torch's current stream of their device; nothing synchronises, no
call keeps anything for the next.  A layer in a row:

    q, scale, h = int8.rms_norm_int8(x, gain, residual=h)        # NormalizeComponent, residual added, 8-bit output
    y = layer.propagate(q, scale, dtype=torch.bfloat16)          # AffineComponent (+ ReLU, BatchNorm) on the codes

8-bit rows are codes in [-127, 127] with one float scale per row: value ~ code * scale.  `kaldi_amd.int8` is the device-tensor
form of kamd_rms_norm_device, kamd_quantize_rows_device and kamd_component_i8_* (include/kaldi_amd.h), which a C or C++ host
calls on plain pointers.  Inference only: there are no gradients.
"""
import ctypes as C

import torch

from . import abi
from ._lib import KamdError, lib

_OFFSETS = [C.c_int32 * n for n in range(abi.KAMD_MAX_OFFSETS + 1)]
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


# Small calls are bound by what happens here and at the launch.  So the common case -- a contiguous matrix of the right kind -- is
# recognised by a few attribute reads; everything else, and every message, is _check's.

def _matrix(t, what, dtype=None, shape=None, dev=-1):
    """leading dimension of a matrix on the device (of this type, shape and device, where given); raises unless it is one"""
    try:
        if t.is_contiguous() and not t.requires_grad and (dtype is None or t.dtype is dtype):
            if (t.shape == shape and t.get_device() == dev) if shape is not None else (t.is_cuda and t.dim() == 2):
                return t.shape[1]
    except (AttributeError, TypeError):
        pass
    return _check(t, what, dtype, shape, dev)


def _check(t, what, dtype, shape, dev):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise KamdError("%s: a tensor on the GPU is expected" % what)
    if t.dim() != 2:
        raise KamdError("%s: a matrix is expected, got shape %s" % (what, tuple(t.shape)))
    if dtype is not None and t.dtype is not dtype:
        raise KamdError("%s: %s expected, got %s" % (what, dtype, t.dtype))
    if shape is not None and t.shape != shape:
        raise KamdError("%s: shape %s expected, got %s" % (what, tuple(shape), tuple(t.shape)))
    if dev >= 0 and t.get_device() != dev:
        raise KamdError("%s: on %s, the other arguments on cuda:%d" % (what, t.device, dev))
    if t.requires_grad and torch.is_grad_enabled():
        raise KamdError("%s: has a gradient to keep track of, and these calls have none (torch.no_grad or detach)" % what)
    ld, step = t.stride()
    rows, cols = t.shape
    if step != 1 and cols > 1:
        raise KamdError("%s: the values of a row have to be contiguous (strides %s)" % (what, (ld, step)))
    return ld if rows > 1 or ld > cols else cols


def _empty(rows, cols, dtype, device):
    return torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=device)


def _empty_as(x):
    """[rows x dim] like x, without gaps between the rows"""
    return torch.empty_like(x) if x.is_contiguous() else _empty(x.shape[0], x.shape[1], x.dtype, x.device)


def _vector(t, n, what, dev):
    try:
        if t.dtype is torch.float32 and t.get_device() == dev and t.shape == (n,) and t.is_contiguous():
            return t.data_ptr()
    except AttributeError:
        pass
    raise KamdError("%s: a contiguous float32 vector of %d on cuda:%d is expected" % (what, n, dev))


def _type(dtype, what):
    code = _TYPES.get(dtype)
    if code is None:
        raise KamdError("%s: float32, bfloat16 or float16 expected, got %s" % (what, dtype))
    return code


_current_device, _stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _call(dev, fn, *args):
    """fn(*args, stream) with device `dev` as the current one"""
    if dev == _current_device():
        rc = fn(*args, _stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _stream(dev))
    if rc < 0:
        _fail()


def empty_codes(rows, dim, device):
    """[rows x dim] int8 in the layout the product takes: each row begins on a multiple of 16 bytes"""
    ld = (dim + 15) // 16 * 16
    q = _empty(rows, ld, torch.int8, device)
    return q if ld == dim else q[:, :dim]


def _norm(x, ld_x, gain, eps, residual, sum_out, y, ld_y, scale):
    """the call behind rms_norm (scale None) and rms_norm_int8; returns h"""
    shape, dtype, dev = x.shape, x.dtype, x.get_device()
    rows, dim = shape
    code = _type(dtype, "x")
    r = h = g = None
    ld_r = ld_h = 0
    if residual is not None:
        ld_r = _matrix(residual, "residual", dtype, shape, dev)
        r = residual.data_ptr()
        if sum_out is None:
            sum_out = _empty_as(x)
            ld_h = dim
    if sum_out is not None:
        if not ld_h:
            ld_h = _matrix(sum_out, "sum_out", dtype, shape, dev)
        h = sum_out.data_ptr()
    if gain is not None:
        g = _vector(gain, dim, "gain", dev)
    if rows:
        _call(dev, _L.kamd_rms_norm_device, x.data_ptr(), ld_x, r, ld_r, code, g, eps, rows, dim, h, ld_h, y.data_ptr(), ld_y,
              code if scale is None else _I8, None if scale is None else scale.data_ptr())
    return sum_out


def rms_norm(x, gain=None, eps=1e-6, residual=None, sum_out=None, out=None):
    """y = h / sqrt(mean(h^2) + eps) * gain per row, h = x + residual -> y, or (y, h) with a residual (kamd_rms_norm_device).

    x: [rows, dim] float32 / bfloat16 / float16, rows any stride apart; residual: the same shape and type; gain: float32 [dim].
    NormalizeComponent is gain = target_rms, eps = 2^-66.  sum_out (h) and out (y) may be given; sum_out may be x or residual,
    out any of the three."""
    _L or _library()
    ld_x = _matrix(x, "x")
    if out is None:
        y, ld_y = _empty_as(x), x.shape[1]
    else:
        y, ld_y = out, _matrix(out, "out", x.dtype, x.shape, x.get_device())
    h = _norm(x, ld_x, gain, eps, residual, sum_out, y, ld_y, None)
    return y if h is None else (y, h)


def _codes_out(out, rows, dim, x):
    if out is None:
        q = empty_codes(rows, dim, x.device)
        return q, torch.empty_strided((rows,), (1,), dtype=torch.float32, device=x.device), (dim + 15) // 16 * 16
    q, scale = out
    ld_q = _matrix(q, "codes", torch.int8, (rows, dim), x.get_device())
    _vector(scale, rows, "scale", x.get_device())
    return q, scale, ld_q


def rms_norm_int8(x, gain=None, eps=1e-6, residual=None, sum_out=None, out=None):
    """rms_norm with y as 8-bit rows -> (codes, scale), or (codes, scale, h) with a residual.  out = (codes, scale) may be given."""
    _L or _library()
    ld_x = _matrix(x, "x")
    q, scale, ld_q = _codes_out(out, x.shape[0], x.shape[1], x)
    h = _norm(x, ld_x, gain, eps, residual, sum_out, q, ld_q, scale)
    return (q, scale) if h is None else (q, scale, h)


def quantize_rows(x, offsets=(0,), out=None):
    """8-bit rows of a (spliced) matrix -> (codes, scale): row j codes Append_i x[j + offsets[i] - min(offsets)], so that
    x.rows - (max - min) rows come back (kamd_quantize_rows_device; the input of a layer with these time offsets)."""
    L = _L or _library()
    ld_x = _matrix(x, "x")
    in_rows, dim = x.shape
    code = _type(x.dtype, "x")
    n = len(offsets)
    if not 1 <= n <= abi.KAMD_MAX_OFFSETS:
        raise KamdError("offsets: between 1 and %d of them expected" % abi.KAMD_MAX_OFFSETS)
    rows = max(0, in_rows - (max(offsets) - min(offsets)))
    q, scale, ld_q = _codes_out(out, rows, dim * n, x)
    if rows:
        _call(x.get_device(), L.kamd_quantize_rows_device, x.data_ptr(), ld_x, code, in_rows, dim, _OFFSETS[n](*offsets), n, q.data_ptr(), ld_q,
              scale.data_ptr())
    return q, scale


class AffineInt8:
    """The affine layer on 8-bit rows (kamd_component_i8): out = mul * relu(codes @ weight.T * scale * weight_scale + bias) + add.

    weight: int8 [out_dim, in_dim], weight_scale: float32 [out_dim], both on the device; bias, mul, add: float32 [out_dim] or
    None.  They are laid out for the matrix units once, here; the tensors are not kept."""

    def __init__(self, weight, weight_scale, bias=None, relu=False, mul=None, add=None):
        L = _library()
        ld = _matrix(weight, "weight", torch.int8)
        n, k = weight.shape
        dev = weight.get_device()
        vectors = [None if v is None else _vector(v, n, what, dev) for v, what in
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
        if getattr(self, "_h", None) and _L is not None:
            _L.kamd_component_i8_destroy(self._h)
            self._h = None

    def quantize_input(self, x, out=None):
        """the codes and scales of the layer's spliced input"""
        return quantize_rows(x, self.offsets, out)

    def propagate(self, q, scale, dtype=torch.float32, out=None):
        """codes [rows, in_dim] and scales [rows] -> [rows, out_dim] of `dtype`"""
        ld_q = _matrix(q, "codes", torch.int8)
        rows, k = q.shape
        dev = q.get_device()
        if k != self.in_dim or dev != self.device.index:
            raise KamdError("codes: [rows, %d] on %s expected, got %s on %s" % (self.in_dim, self.device, tuple(q.shape), q.device))
        if rows <= 1:
            ld_q = (ld_q + 15) // 16 * 16
        at = q.data_ptr()
        if ld_q % 16 or at % 16:
            raise KamdError("codes: rows begin on multiples of 16 bytes (int8.empty_codes has the layout)")
        if k % 16 and q.untyped_storage().nbytes() - q.storage_offset() < (rows - 1) * ld_q + (k + 15) // 16 * 16:
            raise KamdError("codes: the last row ends inside a block of 16 bytes that is not the tensor's own")
        s = _vector(scale, rows, "scale", dev)
        code = _type(dtype, "dtype")
        if out is None:
            out, ld_out = _empty(rows, self.out_dim, dtype, self.device), self.out_dim
        else:
            ld_out = _matrix(out, "out", dtype, (rows, self.out_dim), dev)
        if rows:
            _call(dev, _L.kamd_component_i8_propagate, self._h, at, ld_q, s, rows, out.data_ptr(), ld_out, code)
        return out

    def Propagate(self, x, dtype=None):
        """nnet3::Component::Propagate's shape (nnet3/nnet-component-itf.h:130-132): consecutive time steps in,
        x.rows - (max offset - min offset) rows out, in x's type unless `dtype` says otherwise"""
        q, scale = self.quantize_input(x)
        return self.propagate(q, scale, x.dtype if dtype is None else dtype)
