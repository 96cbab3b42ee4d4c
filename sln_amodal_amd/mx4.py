"""Microscaled 4-bit row products: the fourth operand format (csrc/mx4.hip, csrc/mx4_grad.hip).

32 neighbouring values of a row share a power-of-two scale and are held as e2m1 numbers (0, 0.5, 1, 1.5, 2, 3, 4, 6 and
their negatives): 4.25 bits per value.  `mx4_quantize` rounds a matrix, `mx4_linear` multiplies rounded rows with a rounded
weight -- forward on the scaled 4-bit matrix instructions, backward straight through the rounding with the products in
float32 accuracy.  `ops` re-exports both; `MaskRCNN.set_mx4_layers` runs the classifier head's layers this way."""
import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
FEW_ROWS = 16          # rows that sln_mx4_rows_product takes: rounded inside the product, no launch in front of it
MAX_K = 1 << 22


def _ptr(t):
    return C.c_void_p(t.data_ptr()) if t is not None else C.c_void_p(0)


def _stream(t):
    return C.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _need_float(t, name):
    if not torch.is_tensor(t):
        raise TypeError("%s must be a tensor" % name)
    if not t.is_cuda:
        raise RuntimeError("%s must live on the GPU (no CPU fallback in sln_amodal_amd)" % name)
    if t.dtype not in _DTYPES:
        raise TypeError("%s must be float32, bfloat16 or float16, got %s" % (name, t.dtype))
    return t


def _rows(t, name):
    """t [..., K] -> [R, K] whose rows lie anywhere with values side by side (a copy only where they do not)."""
    if t.dim() < 1 or not 1 <= t.shape[-1] <= MAX_K:
        raise ValueError("%s must be [..., K] with 1 <= K <= 2^22, got %s" % (name, tuple(t.shape)))
    t = t.detach()
    t = t.reshape(-1, t.shape[-1]) if t.dim() != 2 else t
    if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
    return t


def _pitch(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


class Mx4Tensor(object):
    """A matrix held in 4 bits: codes uint8 [R, Kp / 2] (Kp = K rounded up to 256), scales uint8 [R, Kp / 32], the
    `shape` and `dtype` of what it was made from.  Its rows are the last axis' vectors."""
    __slots__ = ("codes", "scales", "shape", "dtype")

    def __init__(self, codes, scales, shape, dtype):
        self.codes, self.scales, self.shape, self.dtype = codes, scales, torch.Size(shape), dtype

    @property
    def device(self):
        return self.codes.device

    def dequantize(self, dtype=None):
        """The values that the codes stand for, in `dtype` (default: the source's; exact in float32 and bfloat16)."""
        dtype = self.dtype if dtype is None else dtype
        if dtype not in _DTYPES:
            raise TypeError("dtype must be float32, bfloat16 or float16, got %s" % dtype)
        out = torch.empty(self.shape, dtype=dtype, device=self.device)
        with torch.cuda.device(self.device):
            _lib.check(_lib.lib().sln_mx4_values(_ptr(self.codes), _ptr(self.scales), self.codes.shape[0],
                                                 self.shape[-1], _ptr(out), _DTYPES[dtype], _stream(out)),
                       "sln_mx4_values")
        return out

    def __repr__(self):
        return "Mx4Tensor(%s, %s, %s)" % (tuple(self.shape), self.dtype, self.device)


def mx4_quantize(x):
    """x [..., K] float32 / bfloat16 / float16 -> Mx4Tensor.  Nearest e2m1 value, ties to the even code, saturated at 6
    times the block's scale 2^(floor(log2 max|x|) - 2); a block with an infinity or a NaN becomes all NaN.  Rows may be
    strided.  No gradient (mx4_linear has one)."""
    _need_float(x, "x")
    rows = _rows(x, "x")
    R, K = rows.shape
    kp = -(-K // 256) * 256
    codes = torch.empty((R, kp // 2), dtype=torch.uint8, device=x.device)
    scales = torch.empty((R, kp // 32), dtype=torch.uint8, device=x.device)
    with torch.cuda.device(x.device):
        _lib.check(_lib.lib().sln_mx4_round(_ptr(rows), _DTYPES[x.dtype], R, K, _pitch(rows), _ptr(codes), _ptr(scales),
                                            _stream(x)), "sln_mx4_round")
    return Mx4Tensor(codes, scales, x.shape, x.dtype)


def _forward(rows, xq, wq, scale, bias, relu, dtype):
    """rows [M,K] (few rows, not rounded) or xq (their codes) times wq -> [M, N]."""
    M, K = rows.shape
    N = wq.codes.shape[0]
    dev = wq.device
    y = torch.empty((M, N), dtype=dtype, device=dev)
    if M == 0 or N == 0:
        return y
    L = _lib.lib()
    nbytes = L.sln_mx4_product_workspace_bytes(M, N, K, 0 if xq is None else 1)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    with torch.cuda.device(dev):
        if xq is None:
            _lib.check(L.sln_mx4_rows_product(_ptr(rows), _DTYPES[dtype], M, K, _pitch(rows), _ptr(wq.codes),
                                              _ptr(wq.scales), N, _ptr(scale), _ptr(bias), int(relu), _ptr(y), _ptr(ws),
                                              nbytes, _stream(y)), "sln_mx4_rows_product")
        else:
            _lib.check(L.sln_mx4_product(_ptr(xq.codes), _ptr(xq.scales), _ptr(wq.codes), _ptr(wq.scales), M, N, K,
                                         _ptr(scale), _ptr(bias), int(relu), _ptr(y), _DTYPES[dtype], _ptr(ws), nbytes,
                                         _stream(y)), "sln_mx4_product")
    return y


class _Mx4LinearFn(torch.autograd.Function):
    """Saved for backward: the CODES of x and of the weight (0.53 B per value), and y where a ReLU masks the gradient."""

    @staticmethod
    def forward(ctx, x, weight, bias, scale, relu, wq):
        rows = _rows(x, "x")
        if wq is None:
            wq = mx4_quantize(weight)
        need_w = weight is not None and ctx.needs_input_grad[1]
        xq = mx4_quantize(rows) if need_w or rows.shape[0] > FEW_ROWS else None
        y = _forward(rows, xq, wq, scale, bias, relu, x.dtype)
        ctx.cfg = (tuple(x.shape), tuple(rows.shape), wq.codes.shape[0], x.dtype)
        ctx.save_for_backward(xq.codes if need_w else None, xq.scales if need_w else None, wq.codes, wq.scales, scale,
                              y if relu else None)
        return y if x.dim() == 2 else y.view(x.shape[:-1] + (y.shape[1],))

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        xc, xs, wc, wsc, scale, y = ctx.saved_tensors
        shape, (M, K), N, dtype = ctx.cfg
        dev = wc.device
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        gx = torch.empty((M, K), dtype=dtype, device=dev) if want_x else None
        gw = torch.empty((N, K), dtype=torch.float32, device=dev) if want_w else None
        gb = torch.empty((N,), dtype=torch.float32, device=dev) if want_b else None
        if M == 0 or N == 0:
            for t in (gx, gw, gb):
                if t is not None:
                    t.zero_()
        elif want_x or want_w or want_b:
            g = gy.reshape(M, N)
            if (N > 1 and g.stride(1) != 1) or (M > 1 and g.stride(0) < N):
                g = g.contiguous()
            L = _lib.lib()
            nbytes = L.sln_mx4_linear_bwd_workspace_bytes(M, N, K, _DTYPES[dtype], want_x, want_w, want_b)
            ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=dev)
            with torch.cuda.device(dev):
                _lib.check(L.sln_mx4_linear_bwd(_ptr(g), _DTYPES[dtype], _pitch(g), _ptr(y), _ptr(scale), _ptr(xc),
                                                _ptr(xs), _ptr(wc), _ptr(wsc), M, N, K, _ptr(gx), _ptr(gw), _ptr(gb),
                                                _ptr(ws), nbytes, _stream(g)), "sln_mx4_linear_bwd")
        return gx.view(shape) if want_x else None, gw, gb, None, None, None


def mx4_linear(x, weight, bias=None, scale=None, relu=False):
    """act((x^ w^T) * scale + bias) with x [..., K] and weight [N, K] rounded to microscaled 4 bits -> [..., N] in x's dtype
    (float32, bfloat16 or float16; products exact, sums float32, one rounding at the end).

    weight: an Mx4Tensor (rounded once and kept: serving; it gets no gradient) or a float32 [N, K] tensor that is rounded
    in every call (training).  bias, scale: float32 [N] or None; scale (a frozen normalisation's) gets no gradient.
    Backward (straight through the rounding): x, a float32 weight and bias.  Up to 16 rows take one pass over the weight
    without a separate rounding of x.  Deterministic."""
    _need_float(x, "x")
    wq = weight if isinstance(weight, Mx4Tensor) else None
    if wq is None:
        _need_float(weight, "weight")
        if weight.dtype != torch.float32:
            raise TypeError("weight must be float32 or an Mx4Tensor, got %s" % weight.dtype)
    if len(weight.shape) != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or weight.shape[1] < 1:
        raise ValueError("mx4_linear: x %s does not fit a weight %s" % (tuple(x.shape), tuple(weight.shape)))
    N = weight.shape[0]
    for t, name in ((bias, "bias"), (scale, "scale")):
        if t is None:
            continue
        if not torch.is_tensor(t) or t.dtype != torch.float32:
            raise TypeError("%s must be a float32 tensor" % name)
        if tuple(t.shape) != (N,):
            raise ValueError("%s must be [%d], got %s" % (name, N, tuple(t.shape)))
    for t, name in ((weight, "weight"), (bias, "bias"), (scale, "scale")):
        if t is not None and t.device != x.device:
            raise ValueError("%s is on %s, x on %s" % (name, t.device, x.device))
    if scale is not None and scale.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("mx4_linear: scale gets no gradient (a frozen normalisation's factor); detach it")
    bias = bias.contiguous() if bias is not None else None
    scale = scale.detach().contiguous() if scale is not None else None
    return _Mx4LinearFn.apply(x, None if wq is not None else weight, bias, scale, bool(relu), wq)
