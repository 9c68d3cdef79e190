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
import importlib.util
import os
import sys

import torch

from ._lib import KamdError, lib

_L = _X = None


def _extension_path():
    """the module that was built against this torch and this Python, whose tensors it reads (csrc/Makefile names it the same way)"""
    name = "_torch_int8.%s.torch-%s.so" % (sys.implementation.cache_tag, torch.__version__)
    return os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", name)


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


def _extension():
    """The calls themselves (csrc/torch_int8.cc): checks of the tensors and allocations, around the library's entry points."""
    global _X
    if _X is None:
        L = _library()
        path = _extension_path()
        if not os.path.exists(path):
            raise KamdError("%s is missing: run `python -c 'import __graft_entry__ as g; g.build()'`" % path)
        spec = importlib.util.spec_from_file_location("_torch_int8", path)
        x = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(x)
        x.init(KamdError, torch._C._cuda_getCurrentRawStream,
               *[C.cast(f, C.c_void_p).value for f in (L.kamd_rms_norm_device, L.kamd_quantize_rows_device, L.kamd_component_i8_propagate, L.kamd_last_error)])
        _X = x
    return _X


def empty_codes(rows, dim, device):
    """[rows x dim] int8 in the layout the product takes: each row begins on a multiple of 16 bytes"""
    return torch.empty((rows, (dim + 15) // 16 * 16), dtype=torch.int8, device=device)[:, :dim]


def rms_norm(x, gain=None, eps=1e-6, residual=None, sum_out=None, out=None):
    """y = h / sqrt(mean(h^2) + eps) * gain per row, h = x + residual -> y, or (y, h) with a residual or sum_out
    (kamd_rms_norm_device).

    x: [rows, dim] float32 / bfloat16 / float16, rows any stride apart; residual: the same shape and type; gain: float32 [dim].
    NormalizeComponent with --target-rms=t is gain = t, eps = 2^-66 t^2, up to its floor: it takes the larger of mean(h^2) and eps
    where this call adds them (the same far above and far below, by up to sqrt(2) smaller where they are alike).  sum_out (h) and out (y) may be given; sum_out may be x or residual,
    out any of the three.  Any other overlap of an output with another argument is refused, here and in the calls below."""
    return (_X or _extension()).rms_norm(x, gain, eps, residual, sum_out, out, False)


def rms_norm_int8(x, gain=None, eps=1e-6, residual=None, sum_out=None, out=None):
    """rms_norm with y as 8-bit rows -> (codes, scale), or (codes, scale, h) with a residual or sum_out.  out = (codes, scale)
    may be given.  A row in which an h * gain is not a finite 32-bit number has scale NaN and codes 0."""
    return (_X or _extension()).rms_norm(x, gain, eps, residual, sum_out, out, True)


def quantize_rows(x, offsets=(0,), out=None):
    """8-bit rows of a (spliced) matrix -> (codes, scale): row j codes Append_i x[j + offsets[i] - min(offsets)], so that
    x.rows - (max - min) rows come back (kamd_quantize_rows_device; the input of a layer with these time offsets)."""
    return (_X or _extension()).quantize_rows(x, tuple(offsets), out)


def _vector(t, n, what, device):
    if not isinstance(t, torch.Tensor) or t.device != device or t.dtype != torch.float32 or t.shape != (n,) or not t.is_contiguous():
        raise KamdError("%s: a contiguous float32 vector of %d on %s is expected" % (what, n, device))
    _extension().plain(t, what)
    return t.data_ptr()


class AffineInt8:
    """The affine layer on 8-bit rows (kamd_component_i8): out = mul * relu(codes @ weight.T * scale * weight_scale + bias) + add.

    weight: int8 [out_dim, in_dim], weight_scale: float32 [out_dim], both on the device; bias, mul, add: float32 [out_dim] or
    None.  They are laid out for the matrix units once, here (not while the stream is captured); the tensors are not kept.  A
    layer has to live as long as the graphs that captured its calls."""

    def __init__(self, weight, weight_scale, bias=None, relu=False, mul=None, add=None):
        L = _library()
        if not isinstance(weight, torch.Tensor) or not weight.is_cuda:
            raise KamdError("weight: a tensor on the GPU is expected")
        if weight.dtype != torch.int8 or weight.dim() != 2:
            raise KamdError("weight: a matrix of torch.int8 expected, got %s %s" % (weight.dtype, tuple(weight.shape)))
        _extension().plain(weight, "weight")
        n, k = weight.shape
        if max(n, k) > 2 ** 31 - 1:               # (the C entry takes ints, to which ctypes cuts what it is given)
            raise KamdError("weight: %d x %d is too large" % (n, k))
        weight = weight.contiguous()
        vectors = [None if v is None else _vector(v, n, what, weight.device) for v, what in
                   ((weight_scale, "weight_scale"), (bias, "bias"), (mul, "mul"), (add, "add"))]
        self.device, self.offsets = weight.device, (0,)
        with torch.cuda.device(weight.device):
            self._take(L.kamd_component_i8_create_quantized(weight.data_ptr(), k, vectors[0], k, n, vectors[1], int(bool(relu)), vectors[2], vectors[3],
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
            if torch.cuda.is_current_stream_capturing():
                raise KamdError("AffineInt8: the stream is being captured: layers are made before")
            self.device, self.offsets = torch.device("cuda", torch.cuda.current_device()), tuple(layer.offsets)
            model = Model([layer], layer.in_dim, 0, 1, layer.out_dim)
            self._take(L.kamd_component_i8_create(model.descs()))
        return self

    def _take(self, handle):
        self._h = handle
        if not handle:
            raise KamdError(_L.kamd_last_error().decode())
        self.in_dim, self.out_dim = _L.kamd_component_i8_input_dim(handle), _L.kamd_component_i8_output_dim(handle)

    def __del__(self):
        if getattr(self, "_h", None) and _L is not None:
            _L.kamd_component_i8_destroy(self._h)
            self._h = None

    def __reduce__(self):
        raise KamdError("AffineInt8: a handle to device memory; neither copied nor pickled")

    def quantize_input(self, x, out=None):
        """the codes and scales of the layer's spliced input"""
        return quantize_rows(x, self.offsets, out)

    def propagate(self, q, scale, dtype=torch.float32, out=None):
        """codes [rows, in_dim] and scales [rows] -> [rows, out_dim] of `dtype`"""
        return (_X or _extension()).propagate(self._h, self.in_dim, self.out_dim, self.device.index, q, scale, dtype, out)

    def Propagate(self, x, dtype=None):
        """nnet3::Component::Propagate's shape (nnet3/nnet-component-itf.h:130-132): consecutive time steps in,
        x.rows - (max offset - min offset) rows out, in x's type unless `dtype` says otherwise"""
        q, scale = self.quantize_input(x)
        return self.propagate(q, scale, x.dtype if dtype is None else dtype)
