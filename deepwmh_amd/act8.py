"""8-bit activation checkpoints and the block-scaled 8-bit product.

A checkpoint (`Act8`) holds a tensor [N, C, spatial...] as one byte per value and one exponent byte per 128 consecutive values of a channel:
a block's scale is 2^e, e the smallest integer (not below -126) with max |value| <= Q 2^e, Q = 127 ('int8': evenly spaced codes, an error of
at most half a step of 2^e) or 448 ('e4m3': floating-point codes, a relative error of at most 2^-4 above 2^(e-6)).  Codes are rounded to
nearest even.  A block that holds an infinity or a NaN reads NaN as a whole.

  pack / unpack                        a tensor to its checkpoint and back, optionally behind InstanceNorm + LeakyReLU
  pack_columns                         blocks along the other axis of a matrix: the operand of a product's gradient
  instnorm_lrelu_backward              backward pass of InstanceNorm + LeakyReLU (+ segmentation head) on a checkpoint of its input
  product                              a b^T of two e4m3 checkpoints: float32 results from the codes widened to bfloat16 (exact operands, float32
                                       sums), bfloat16 results from the scaled 8-bit matrix instruction
  convtranspose_weight_gradient        the float32 product as the weight gradient of a transposed convolution (kernel = stride)

Calls are asynchronous on torch's current stream of the tensors' device; outputs and workspaces come from torch's allocator unless given.
There is no CPU path, and nothing is recorded for autograd: a tensor that requires grad is refused while grad mode is on.
UNetTrainer(checkpoint8=..., tu_wgrad=...) is what uses them in training.
"""
from collections import namedtuple

import torch

from . import _lib
from .network import LRELU_SLOPE

FORMATS = {'int8': (0, torch.int8), 'e4m3': (1, torch.float8_e4m3fn)}
_FORMAT_OF = {torch.int8: 0, torch.float8_e4m3fn: 1}
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
BLOCK = 128

InstNormGrads = namedtuple('InstNormGrads', 'dy dgamma dbeta dbias dwseg')


def _pitches(length):
    nb = -(-length // BLOCK)
    return nb * BLOCK, -(-nb // 4) * 4


def _length(shape):
    n = 1
    for v in shape[2:]:
        n *= v
    return n


class Act8:
    """A packed tensor: `shape` of what it stands for ([N, C, ...]), `codes` [N, C, pitch] (torch.int8 or torch.float8_e4m3fn; zero behind a row's
    end) and exponent bytes `scales` [N, C, scale pitch] (uint8; 1 to 249, or 255 for a block that is not finite)."""
    __slots__ = ('codes', 'scales', 'shape', 'length')
    requires_grad = False                                       # (to autograd; _device)

    def __init__(self, codes, scales, shape):
        shape = tuple(map(int, shape))
        if len(shape) < 3 or min(shape) < 0:
            raise ValueError('Act8: shape [N, C, ...] expected, got %s' % (shape,))
        length = _length(shape)
        pitch, spitch = _pitches(length)
        if codes.dtype not in _FORMAT_OF or scales.dtype != torch.uint8:
            raise TypeError('Act8: codes are int8 or float8_e4m3fn and scales uint8, got %s and %s' % (codes.dtype, scales.dtype))
        if codes.shape != shape[:2] + (pitch,) or scales.shape != shape[:2] + (spitch,):
            raise ValueError('Act8: %s needs codes %s and scales %s, got %s and %s'
                             % (shape, shape[:2] + (pitch,), shape[:2] + (spitch,), tuple(codes.shape), tuple(scales.shape)))
        if not (codes.is_contiguous() and scales.is_contiguous()) or codes.device != scales.device:
            raise ValueError('Act8: codes and scales must be contiguous and on one device')
        self.codes, self.scales, self.shape, self.length = codes, scales, shape, length

    @classmethod
    def empty(cls, shape, fmt, device):
        if fmt not in FORMATS:
            raise ValueError('format must be int8 or e4m3, got %r' % (fmt,))
        shape = tuple(shape)
        if len(shape) < 3 or min(shape) < 0:
            raise ValueError('Act8: shape [N, C, ...] expected, got %s' % (shape,))
        length = _length(shape)
        pitch, spitch = _pitches(length)
        self = cls.__new__(cls)                                 # (parts made to fit need no checks)
        self.shape, self.length = shape, length
        self.codes = torch.empty((shape[0], shape[1], pitch), dtype=FORMATS[fmt][1], device=device)
        self.scales = torch.empty((shape[0], shape[1], spitch), dtype=torch.uint8, device=device)
        return self

    @property
    def fmt(self):
        return 'int8' if self.codes.dtype == torch.int8 else 'e4m3'

    @property
    def device(self):
        return self.codes.device

    @property
    def nbytes(self):
        return self.codes.numel() + self.scales.numel()


def _device(what, first, *tensors):
    """The HIP device all of these are on.  With grad mode on none of them may require grad: its gradient would silently be missing."""
    dev, grad = first.device, torch.is_grad_enabled()
    lost = grad and first.requires_grad
    for t in tensors:
        if t is not None:
            if t.device != dev:
                raise ValueError('%s: tensors on %s and %s' % (what, dev, t.device))
            if grad and t.requires_grad:
                lost = True
    if lost:
        raise RuntimeError('%s records nothing for autograd, and one of its tensors requires grad: detach() it or call under torch.no_grad()' % what)
    if dev.type != 'cuda':
        raise RuntimeError('%s needs a HIP device; there is no CPU path' % what)
    return dev


def _f32(what, name, t, shape):
    if t is None:
        return
    if t.dtype != torch.float32 or t.shape != shape or not t.is_contiguous():
        raise ValueError('%s: %s must be contiguous float32 %s, got %s %s' % (what, name, tuple(shape), t.dtype, tuple(t.shape)))


def _p(t):
    return None if t is None else t.data_ptr()


def _run(what, dev, fn, *args):
    """fn(*args, stream) with torch's current stream of `dev`, on that device."""
    stream = torch._C._cuda_getCurrentRawStream(dev.index)      # (torch.cuda.current_stream(dev).cuda_stream takes 4 us of a call's 16)
    if dev.index == torch.cuda.current_device():
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, stream)
    if rc < 0:
        _lib.check(rc, what)


def _rows(what, x):
    """(x, batch stride, channel stride) with the spatial axes of x [N, C, ...] dense; a copy is made of one that is strided there."""
    if x.dim() < 3:
        raise ValueError('%s: [N, C, ...] expected, got %s' % (what, tuple(x.shape)))
    if x.dtype not in _DTYPES:
        raise TypeError('%s: float32, bfloat16 or float16 expected, got %s' % (what, x.dtype))
    if not x.is_contiguous():
        n = 1
        for size, stride in zip(reversed(x.shape[2:]), reversed(x.stride()[2:])):
            if size > 1 and stride != n:
                x = x.contiguous()
                break
            n *= size
    strides = x.stride()
    return x, strides[0], strides[1]


def pack(x, fmt='int8', ss=None, slope=LRELU_SLOPE, out=None, keep_sign=False):
    """x [N, C, ...] (float32 / bfloat16 / float16) -> Act8.  With ss [N, C, 2] what is packed is the float32 activation
    lrelu(x scale + shift), or with keep_sign x itself, by codes that leave the sign of x scale + shift as it is (one step off instead of half of
    one where the nearest code would not): the checkpoint for instnorm_lrelu_backward.  `out`: an Act8 of this shape to write into."""
    if keep_sign and ss is None:
        raise ValueError('pack: keep_sign needs ss')
    x, sn, sc = _rows('pack', x)
    if out is not None and (out.shape != tuple(x.shape) or out.fmt != fmt):
        raise ValueError('pack: out is %s %s, needed %s %s' % (out.fmt, out.shape, fmt, tuple(x.shape)))
    dev = _device('pack', x, ss, out)
    if out is None:
        out = Act8.empty(x.shape, fmt, dev)
    N, Cc = out.shape[:2]
    _f32('pack', 'ss', ss, (N, Cc, 2))
    _run('wmh_act8_pack', dev, _lib.load().wmh_act8_pack, _p(x), _DTYPES[x.dtype], sn, sc, _p(ss), 0 if ss is None else 2 if keep_sign else 1, slope,
         _FORMAT_OF[out.codes.dtype], _p(out.codes), _p(out.scales), N, Cc, out.length)
    return out


def pack_columns(x, fmt='e4m3', out=None):
    """x [B, R, S] -> Act8 of its transpose [B, S, R]: blocks of 128 along R.  The last axis must be dense (a copy is made otherwise)."""
    if x.dim() != 3:
        raise ValueError('pack_columns: [B, R, S] expected, got %s' % (tuple(x.shape),))
    if x.dtype not in _DTYPES:
        raise TypeError('pack_columns: float32, bfloat16 or float16 expected, got %s' % x.dtype)
    if x.shape[2] > 1 and x.stride(2) != 1:
        x = x.contiguous()
    B, R, S = x.shape
    if out is not None and (out.shape != (B, S, R) or out.fmt != fmt):
        raise ValueError('pack_columns: out is %s %s, needed %s %s' % (out.fmt, out.shape, fmt, (B, S, R)))
    dev = _device('pack_columns', x, out)
    if out is None:
        out = Act8.empty((B, S, R), fmt, dev)
    _run('wmh_act8_pack_columns', dev, _lib.load().wmh_act8_pack_columns, _p(x), _DTYPES[x.dtype], x.stride(0), x.stride(1), _FORMAT_OF[out.codes.dtype],
         _p(out.codes), _p(out.scales), B, R, S)
    return out


def unpack(ck, dtype=torch.float32, ss=None, slope=LRELU_SLOPE, out=None):
    """The tensor an Act8 stands for, or with ss [N, C, 2] its activation lrelu(value scale + shift), rounded once to `dtype`."""
    if dtype not in _DTYPES:
        raise TypeError('unpack: float32, bfloat16 or float16 expected, got %s' % dtype)
    if out is not None and (out.dtype != dtype or out.shape != ck.shape or not out.is_contiguous()):
        raise ValueError('unpack: out must be contiguous %s %s, got %s %s' % (dtype, ck.shape, out.dtype, tuple(out.shape)))
    dev = _device('unpack', ck, ss, out)
    if out is None:
        out = torch.empty(ck.shape, dtype=dtype, device=dev)
    N, Cc = ck.shape[:2]
    _f32('unpack', 'ss', ss, (N, Cc, 2))
    _run('wmh_act8_unpack', dev, _lib.load().wmh_act8_unpack, _p(ck.codes), _p(ck.scales), _FORMAT_OF[ck.codes.dtype], _p(ss), slope, _p(out), _DTYPES[dtype],
         N, Cc, ck.length)
    return out


def instnorm_lrelu_backward(ck, ss, mean_rstd, gamma=None, g1=None, g2=None, dlogits=None, wseg=None, slope=LRELU_SLOPE, out=None):
    """Backward pass of a = lrelu(instnorm(y)) on the checkpoint of y: ss and mean_rstd [N, C, 2] of the forward pass, gamma [C]; the gradient of
    a is g1 + g2 + wseg^T dlogits (any of the three; g1, g2 of y's shape, dlogits [N, K, ...], wseg [K, C]).  Returns InstNormGrads: dy of y's
    shape, dgamma, dbeta, dbias (the sum of dy) [C], and dwseg [K, C] or None.  `out`: an InstNormGrads of tensors to write into; one that is
    None there is not formed (dy always is; it may be g1 or g2 itself).  N C is at most 65535 and K 4."""
    what = 'instnorm_lrelu_backward'
    N, Cc = ck.shape[:2]
    if min(N, Cc, ck.length) < 1:
        raise ValueError('%s: empty tensor %s' % (what, ck.shape))
    if g1 is None and g2 is None and dlogits is None:
        raise ValueError('%s: one of g1, g2 and dlogits is needed' % what)
    _f32(what, 'ss', ss, (N, Cc, 2))
    _f32(what, 'mean_rstd', mean_rstd, (N, Cc, 2))
    if ss is None or mean_rstd is None:
        raise ValueError('%s: ss and mean_rstd of the forward pass are needed' % what)
    _f32(what, 'gamma', gamma, (Cc,))
    _f32(what, 'g1', g1, ck.shape)
    _f32(what, 'g2', g2, ck.shape)
    K = 0
    if dlogits is not None:
        K = dlogits.shape[1] if dlogits.dim() > 1 else 0
        if not 1 <= K <= 4 or wseg is None:
            raise ValueError('%s: dlogits needs wseg and 1 to 4 classes, got %s' % (what, tuple(dlogits.shape)))
        _f32(what, 'dlogits', dlogits, (N, K) + ck.shape[2:])
        if wseg.dtype != torch.float32 or wseg.numel() != K * Cc or wseg.shape[:1] != (K,) or not wseg.is_contiguous():
            raise ValueError('%s: wseg must be contiguous float32 %s, got %s %s' % (what, (K, Cc), wseg.dtype, tuple(wseg.shape)))
    dev = _device(what, ck, ss, mean_rstd, gamma, g1, g2, dlogits, wseg)
    lib = _lib.load()
    if out is None:
        like = g1 if g1 is not None else g2                    # (empty_like takes half of empty's 2.2 us)
        dy = torch.empty(ck.shape, dtype=torch.float32, device=dev) if like is None else torch.empty_like(like)
        out = InstNormGrads(dy, *torch.empty((3, Cc), dtype=torch.float32, device=dev).unbind(0),
                            torch.empty((K, Cc), dtype=torch.float32, device=dev) if K else None)
    else:
        _device(what, ck, *out)
        if out.dy is None:
            raise ValueError('%s: out.dy is needed' % what)
        _f32(what, 'out.dy', out.dy, ck.shape)
        for name in ('dgamma', 'dbeta', 'dbias'):
            _f32(what, 'out.' + name, getattr(out, name), (Cc,))
        if out.dwseg is not None and (not K or out.dwseg.dtype != torch.float32 or out.dwseg.numel() != K * Cc or not out.dwseg.is_contiguous()):
            raise ValueError('%s: out.dwseg must be contiguous float32 of %d x %d values' % (what, K, Cc))
    n = lib.wmh_act8_in_lrelu_bwd_scratch_doubles(N, Cc, ck.length)
    scratch = torch.empty(n, dtype=torch.float64, device=dev) if n else None
    _run('wmh_act8_in_lrelu_bwd', dev, lib.wmh_act8_in_lrelu_bwd, _p(ck.codes), _p(ck.scales), _FORMAT_OF[ck.codes.dtype], _p(ss), _p(mean_rstd), _p(gamma),
         _p(g1), _p(g2), _p(dlogits), _p(wseg), K, _p(out.dy), _p(out.dgamma), _p(out.dbeta), _p(out.dwseg), _p(out.dbias), _p(scratch), N, Cc, ck.length, slope)
    return out


def product(a, b, dtype=torch.float32, sum_batches=False, out=None):
    """a [B, M, K] and b [B, N, K] packed to e4m3 -> a b^T: [B, M, N], or [M, N] summed over the batch.  A float32 result is a
    sum in float32 of codes widened exactly to bfloat16 (a value below 2^-126 may lose bits); a bfloat16 result comes from the scaled 8-bit matrix
    instruction, twice as fast, whose sums of eight neighbours keep 14 bits of the largest product: 1.5e-5 of a sum of random terms, against the
    result's rounding of 2^-8, and at most 2^-10 of the sum of |terms|, which is more than that rounding where terms cancel.  A product's gradients
    are products again, of operands packed along the other axis (pack_columns):
    da = product(pack(dc), pack_columns(b)), db = product(pack_columns(dc), pack_columns(a))."""
    if a.codes.dtype != torch.float8_e4m3fn or b.codes.dtype != torch.float8_e4m3fn:
        raise TypeError('product: e4m3 operands expected, got %s and %s' % (a.fmt, b.fmt))
    if a.length != b.length or a.shape[0] != b.shape[0]:
        raise ValueError('product: operands %s and %s do not match' % (a.shape, b.shape))
    if dtype not in (torch.float32, torch.bfloat16):
        raise TypeError('product: float32 or bfloat16 output, got %s' % dtype)
    B, M = a.shape[:2]
    N = b.shape[1]
    shape = (M, N) if sum_batches else (B, M, N)
    dev = _device('product', a, b, out)
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=dev)
    elif out.dtype != dtype or out.shape != shape or not out.is_contiguous():
        raise ValueError('product: out must be contiguous %s %s, got %s %s' % (dtype, shape, out.dtype, tuple(out.shape)))
    lib = _lib.load()
    n = lib.wmh_act8_product_workspace_floats(B, M, N, a.length, int(sum_batches))
    ws = torch.empty(n, dtype=torch.float32, device=dev) if n else None
    _run('wmh_act8_product', dev, lib.wmh_act8_product, _p(a.codes), _p(a.scales), _p(b.codes), _p(b.scales), _p(out), _DTYPES[dtype], _p(ws), B, M, N, a.length,
         int(sum_batches))
    return out


def convtranspose_weight_gradient(x, ss, dy, slope=LRELU_SLOPE, out=None):
    """Weight gradient [Cin, Cout, kt, 2, 2] of a transposed convolution with kernel = stride = (kt, 2, 2), kt 1 or 2, from its float32 input
    x [N, Cin, D, H, W] (behind InstanceNorm + LeakyReLU where ss [N, Cin, 2] is given) and dy [N, Cout, kt D, 2 H, 2 W]: both are packed to
    e4m3 in blocks of 128 low-resolution voxels, and the codes multiplied as in `product` with a float32 result: widened exactly to bfloat16 with
    their scale, sums in float32."""
    what = 'convtranspose_weight_gradient'
    if x.dim() != 5 or dy.dim() != 5 or x.shape[0] != dy.shape[0]:
        raise ValueError('%s: [N, C, D, H, W] expected, got %s and %s' % (what, tuple(x.shape), tuple(dy.shape)))
    N, Cin, D, H, W = x.shape
    Cout = dy.shape[1]
    kt = dy.shape[2] // D if D else 0
    if min(x.shape) < 1 or Cout < 1 or kt not in (1, 2) or tuple(dy.shape[2:]) != (kt * D, 2 * H, 2 * W):
        raise ValueError('%s: dy %s is not (1 or 2, 2, 2) times x %s' % (what, tuple(dy.shape), tuple(x.shape)))
    _f32(what, 'x', x, x.shape)
    _f32(what, 'dy', dy, dy.shape)
    _f32(what, 'ss', ss, (N, Cin, 2))
    dev = _device(what, x, ss, dy, out)
    shape = (Cin, Cout, kt, 2, 2)
    if out is None:
        out = torch.empty(shape, dtype=torch.float32, device=dev)
    _f32(what, 'out', out, shape)
    lib = _lib.load()
    ws = torch.empty(lib.wmh_act8_convtranspose3d_wgrad_workspace_bytes(N, Cin, Cout, D, H, W, kt), dtype=torch.uint8, device=dev)
    _run('wmh_act8_convtranspose3d_wgrad', dev, lib.wmh_act8_convtranspose3d_wgrad, _p(x), _p(ss), _p(dy), _p(out), _p(ws), N, Cin, Cout, D, H, W, kt, slope)
    return out
