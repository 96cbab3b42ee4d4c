"""Microscaled 4-bit row products: the fourth operand format (csrc/mx4.hip, csrc/mx4_grad.hip).

32 neighbouring values of a row share a power-of-two scale and are held as e2m1 numbers (0, 0.5, 1, 1.5, 2, 3, 4, 6 and
their negatives): 4.25 bits per value.  `mx4_quantize` rounds a matrix, `mx4_linear` multiplies rounded rows with a rounded
weight -- forward on the scaled 4-bit matrix instructions, backward straight through the rounding with the products in
float32 accuracy.  `ops` re-exports both; `MaskRCNN.set_mx4_layers` runs the classifier head's layers this way."""
import torch
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
FEW_ROWS = 16          # rows that sln_mx4_rows_product takes: rounded inside the product, no launch in front of it
MAX_K = 1 << 22
MAX_GRAD = 1 << 21     # rows and outputs that sln_mx4_linear_bwd takes


def _need_float(t, name):
    if not torch.is_tensor(t):
        raise TypeError("%s must be a tensor" % name)
    if not t.is_cuda:
        raise RuntimeError("%s must live on the GPU (no CPU fallback in sln_amodal_amd)" % name)
    if t.dtype not in _DTYPES:
        raise TypeError("%s must be float32, bfloat16 or float16, got %s" % (name, t.dtype))
    return t


def _rows(t, name):
    """t [..., K] -> (a [R, K] whose rows lie anywhere with values side by side -- a copy only where they do not --, R, K,
    row stride)."""
    shape = t.shape
    if len(shape) < 1 or not 1 <= shape[-1] <= MAX_K:
        raise ValueError("%s must be [..., K] with 1 <= K <= 2^22, got %s" % (name, tuple(shape)))
    if len(shape) != 2:
        t = t.detach().reshape(-1, shape[-1])
        shape = t.shape
    R, K = shape
    s0, s1 = t.stride()
    if (K > 1 and s1 != 1) or (R > 1 and s0 < K):
        t = t.detach().contiguous()
        s0 = K
    return t, R, K, (s0 if R > 1 else K)


class Mx4Tensor(object):
    """A matrix held in 4 bits, in one buffer: `codes` uint8 [R, Kp / 2] (Kp = K rounded up to 256) and `scales` uint8
    [R, Kp / 32] (held step by step: [Kp / 256][R][8]); the `shape` and `dtype` of what it was made from.  Its rows are the
    last axis' vectors."""
    __slots__ = ("data", "rows", "shape", "dtype")

    def __init__(self, data, rows, shape, dtype):
        self.data, self.rows, self.shape, self.dtype = data, rows, torch.Size(shape), dtype

    @property
    def device(self):
        return self.data.device

    @property
    def codes(self):
        kp = _padded(self.shape[-1])
        return self.data[:self.rows * (kp // 2)].view(self.rows, kp // 2)

    @property
    def scales(self):
        kp = _padded(self.shape[-1])
        return self.data[self.rows * (kp // 2):].view(kp // 256, self.rows, 8).permute(1, 0, 2).reshape(self.rows, kp // 32)

    def dequantize(self, dtype=None):
        """The values that the codes stand for, in `dtype` (default: the source's; exact in float32 and bfloat16)."""
        dtype = self.dtype if dtype is None else dtype
        if dtype not in _DTYPES:
            raise TypeError("dtype must be float32, bfloat16 or float16, got %s" % dtype)
        dev = self.data.device
        out = torch.empty(self.shape, dtype=dtype, device=dev)
        codes, scales = _pointers(self.data, self.rows, self.shape[-1])
        with _lib.on_device(dev):
            _lib.check(_lib.lib().sln_mx4_values(codes, scales, self.rows, self.shape[-1], out.data_ptr(),
                                                 _DTYPES[dtype], _lib.stream_of(dev)), "sln_mx4_values")
        return out

    def __repr__(self):
        return "Mx4Tensor(%s, %s, %s)" % (tuple(self.shape), self.dtype, self.device)


def _padded(K):
    return -(-K // 256) * 256


def _buffer(R, K, dev):
    return torch.empty(R * (_padded(K) // 32) * 17, dtype=torch.uint8, device=dev)


def _pointers(data, R, K):
    p = data.data_ptr()
    return p, p + R * (_padded(K) // 2)


def mx4_quantize(x):
    """x [..., K] float32 / bfloat16 / float16 -> Mx4Tensor.  Nearest e2m1 value, ties to the even code, saturated at 6
    times the block's scale 2^(floor(log2 max|x|) - 2); a block with an infinity or a NaN becomes all NaN.  Rows may be
    strided.  No gradient (mx4_linear has one)."""
    _need_float(x, "x")
    src, R, K, pitch = _rows(x, "x")
    dev = x.device
    data = _buffer(R, K, dev)
    codes, scales = _pointers(data, R, K)
    with _lib.on_device(dev):
        _lib.check(_lib.lib().sln_mx4_round(src.data_ptr(), _DTYPES[x.dtype], R, K, pitch, codes, scales, _lib.stream_of(dev)),
                   "sln_mx4_round")
    return Mx4Tensor(data, R, x.shape, x.dtype)


def _forward(x, weight, wq, bias, scale, relu, keep):
    """-> y [M, N] and, where the backward needs them (`keep`) or the rows are many, the codes of x; the weight's codes."""
    src, M, K, pitch = _rows(x, "x")
    dev = x.device
    L = _lib.lib()
    w = w_pitch = 0
    if wq is None:
        wsrc, N, _, w_pitch = _rows(weight, "weight")
        w, wdata = wsrc.data_ptr(), _buffer(N, K, dev)
    else:
        wdata, N = wq.data, wq.rows
    y = torch.empty((M, N), dtype=x.dtype, device=dev)
    xdata = _buffer(M, K, dev) if keep or M > FEW_ROWS else None
    if M == 0 or N == 0:
        return y, M, K, N, xdata, wdata
    xc, xs = _pointers(xdata, M, K) if xdata is not None else (0, 0)
    wc, ws = _pointers(wdata, N, K)
    nbytes = L.sln_mx4_product_workspace_bytes(M, N, K, xdata is not None)
    work = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    with _lib.on_device(dev):
        _lib.check(L.sln_mx4_linear_fwd(src.data_ptr(), _DTYPES[x.dtype], M, K, pitch, xc, xs, w, w_pitch, wc, ws, N,
                                        scale.data_ptr() if scale is not None else 0,
                                        bias.data_ptr() if bias is not None else 0, relu, y.data_ptr(),
                                        work.data_ptr() if nbytes else 0, nbytes, _lib.stream_of(dev)), "sln_mx4_linear_fwd")
    return y, M, K, N, xdata, wdata


class _Mx4LinearFn(torch.autograd.Function):
    """Saved for backward: the CODES of x and of the weight (0.53 B per value), and y where a ReLU masks the gradient."""

    @staticmethod
    def forward(ctx, x, weight, bias, scale, relu, wq):
        need_w = weight is not None and ctx.needs_input_grad[1]
        y, M, K, N, xdata, wdata = _forward(x, weight, wq, bias, scale, relu, need_w)
        ctx.cfg = (x.shape, M, K, N, x.dtype)
        ctx.save_for_backward(xdata if need_w else None, wdata, scale, y if relu else None)
        return y if x.dim() == 2 else y.view(x.shape[:-1] + (N,))

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        xdata, wdata, scale, y = ctx.saved_tensors
        shape, M, K, N, dtype = ctx.cfg
        dev = wdata.device
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        gx = torch.empty(shape, dtype=dtype, device=dev) if want_x else None
        gw = torch.empty((N, K), dtype=torch.float32, device=dev) if want_w else None
        gb = torch.empty((N,), dtype=torch.float32, device=dev) if want_b else None
        if M == 0 or N == 0:
            for t in (gx, gw, gb):
                if t is not None:
                    t.zero_()
        elif want_x or want_w or want_b:
            g = gy if gy.dim() == 2 else gy.reshape(M, N)
            g, _, _, pitch = _rows(g, "gradient")
            L = _lib.lib()
            kind = _DTYPES[dtype]
            nbytes = L.sln_mx4_linear_bwd_workspace_bytes(M, N, K, kind, want_x, want_w, want_b)
            work = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            xc, xs = _pointers(xdata, M, K) if want_w else (0, 0)
            wc, ws = _pointers(wdata, N, K)
            at = lambda t: t.data_ptr() if t is not None else 0
            with _lib.on_device(dev):
                _lib.check(L.sln_mx4_linear_bwd(g.data_ptr(), kind, pitch, at(y), at(scale), xc, xs, wc, ws, M, N, K,
                                                at(gx), at(gw), at(gb), work.data_ptr(), nbytes, _lib.stream_of(dev)),
                           "sln_mx4_linear_bwd")
        return gx, gw, gb, None, None, None


def mx4_linear(x, weight, bias=None, scale=None, relu=False):
    """act((x^ w^T) * scale + bias) with x [..., K] and weight [N, K] rounded to microscaled 4 bits -> [..., N] in x's dtype
    (float32, bfloat16 or float16; products exact, sums float32, one rounding at the end).

    weight: an Mx4Tensor (rounded once and kept: serving; it gets no gradient) or a float32 [N, K] tensor that is rounded
    in every call (training).  bias, scale: float32 [N] or None; scale (a frozen normalisation's) gets no gradient.
    Backward (straight through the rounding): x, a float32 weight and bias; no second derivative, no forward mode; a ReLU lets
    the gradient through where the output is > 0, not where it is a NaN, like the framework's convolutions.  Up to 16 rows take
    one pass over the weight without a separate rounding of x.  Deterministic."""
    _need_float(x, "x")
    wq = weight if isinstance(weight, Mx4Tensor) else None
    if wq is None:
        _need_float(weight, "weight")
        if weight.dtype != torch.float32:
            raise TypeError("weight must be float32 or an Mx4Tensor, got %s" % weight.dtype)
    wshape, dev = weight.shape, x.device
    if len(wshape) != 2 or x.dim() < 1 or x.shape[-1] != wshape[1] or wshape[1] < 1:
        raise ValueError("mx4_linear: x %s does not fit a weight %s" % (tuple(x.shape), tuple(wshape)))
    N = wshape[0]
    if weight.device != dev:
        raise ValueError("weight is on %s, x on %s" % (weight.device, dev))
    for t, name in ((bias, "bias"), (scale, "scale")):
        if t is None:
            continue
        if not torch.is_tensor(t) or t.dtype != torch.float32:
            raise TypeError("%s must be a float32 tensor" % name)
        if t.dim() != 1 or t.shape[0] != N:
            raise ValueError("%s must be [%d], got %s" % (name, N, tuple(t.shape)))
        if t.device != dev:
            raise ValueError("%s is on %s, x on %s" % (name, t.device, dev))
    _lib.need_no_tangent("mx4_linear", x, weight if wq is None else None, bias, scale)
    grad = torch.is_grad_enabled()
    if scale is not None:
        if grad and scale.requires_grad:
            raise RuntimeError("mx4_linear: scale gets no gradient (a frozen normalisation's factor); detach it")
        scale = scale.detach().contiguous() if scale.requires_grad or not scale.is_contiguous() else scale
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    if grad and (x.requires_grad or (wq is None and weight.requires_grad) or (bias is not None and bias.requires_grad)):
        if max(x.numel() // wshape[1], N) > MAX_GRAD:
            raise ValueError("mx4_linear: at most 2^21 rows and outputs with gradients, got %s for a weight %s" %
                             (tuple(x.shape), tuple(wshape)))
        return _Mx4LinearFn.apply(x, None if wq is not None else weight, bias, scale, bool(relu), wq)
    y = _forward(x, weight, wq, bias, scale, bool(relu), False)[0]
    return y if x.dim() == 2 else y.view(x.shape[:-1] + (N,))
