"""Operators of the acoustic model's serving path on MI355X: products with weights and activations
in microscaled 4-bit floating point (MXFP4), and the norms at a block's end and start fused with
its gate, scale and residual.

The reference's acoustic model is a stack of products with fixed weights, each followed by a norm
(TTS/Fastspeech_1.py:12-56); these are the kernels `FastSpeechAcousticModel.use_mxfp4` runs it on.
All arithmetic runs in libglvoc.so; torch owns the memory and the stream.  The functions enqueue
work on torch's current stream of the inputs' device, allocate their outputs and workspace from
torch (so they can be captured into a graph) and return without synchronising.  They are for
inference: a tensor that asks for a gradient is refused while gradients are recorded.
"""
from __future__ import annotations

import torch

from . import _lib

__all__ = ["MXFP4Tensor", "Norm", "block_norm", "mxfp4_conv1d", "mxfp4_linear", "mxfp4_quantize"]

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_MXFP4 = 3
_ACTIVATIONS = {None: 0, "relu": 1}
_NORMS = {"layer": 1, "rms": 2}
_GROUP = 128  # columns that share one dword of scales


def _launch(device, entry, *args):
    """entry(*args, stream) with `device` current, on torch's current stream of it."""
    index = device.index
    if torch.cuda.current_device() == index:
        rc = entry(*args, torch.cuda.current_stream(index).cuda_stream)
    else:
        with torch.cuda.device(index):
            rc = entry(*args, torch.cuda.current_stream(index).cuda_stream)
    if rc:
        _lib.check(rc)


def _check(t, name, device=None):
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dtype not in _TYPES:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a ROCm GPU (there is no CPU fallback), got {t.device}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient: this operator is for inference (use torch.no_grad() or detach)")


def _vector(t, name, n, device):
    _check(t, name, device)
    if t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{name} must have shape ({n},), got {tuple(t.shape)}")
    return t if t.stride(0) == 1 or n == 1 else t.contiguous()


def _rows(x):
    """x as (batch, rows, cols) with a contiguous last dimension; a copy only where no view will do."""
    if x.dim() == 1:
        x = x[None, None]
    elif x.dim() == 2:
        x = x[None]
    elif x.dim() > 3:
        x = x.reshape(-1, x.shape[-2], x.shape[-1]) if x.numel() else x.new_empty((0, *x.shape[-2:]))
    if x.stride(2) != 1 and x.shape[2] > 1:
        x = x.contiguous()
    return x


class MXFP4Tensor:
    """A tensor in MXFP4: along the last dimension every 32 elements share one power of two (E8M0)
    and an element is a 4-bit code for 0, 0.5, 1, 1.5, 2, 3, 4 or 6 with a sign (E2M1).

    shape   of the tensor it stands for
    codes   (groups, rows, 64) uint8, a group being 128 columns, two to a byte, the even one low
    scales  (groups, rows, 4) uint8, biased exponents of the group's four blocks; 255 is a NaN block
    """

    __slots__ = ("shape", "codes", "scales")

    def __init__(self, shape, codes, scales):
        shape = torch.Size(shape)
        if len(shape) < 1 or shape[-1] < 1:
            raise ValueError(f"an MXFP4 tensor needs a last dimension of at least 1, got {tuple(shape)}")
        rows, groups = shape[:-1].numel(), -(-shape[-1] // _GROUP)
        for t, name, want in ((codes, "codes", (groups, rows, 64)), (scales, "scales", (groups, rows, 4))):
            if t.dtype != torch.uint8 or tuple(t.shape) != want or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous uint8 tensor of shape {want}, got {t.dtype} "
                                 f"{tuple(t.shape)}")
        if codes.device != scales.device:
            raise ValueError(f"codes on {codes.device} but scales on {scales.device}")
        self.shape, self.codes, self.scales = shape, codes, scales

    @property
    def device(self):
        return self.codes.device

    def to(self, device):
        return MXFP4Tensor(self.shape, self.codes.to(device), self.scales.to(device))

    def dequantize(self, dtype=torch.float32):
        """The values the codes stand for, exact in float32 and bfloat16 (float16: within its range)."""
        if dtype not in _TYPES:
            raise ValueError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
        if not self.codes.is_cuda:
            raise ValueError(f"the tensor must be on a ROCm GPU (there is no CPU fallback), got {self.device}")
        out = torch.empty(self.shape, dtype=dtype, device=self.device)
        _launch(self.device, _lib.load().glv_mxfp4_dequantize, self.codes.data_ptr(), self.scales.data_ptr(),
                self.codes.shape[1], self.shape[-1], _TYPES[dtype], out.data_ptr())
        return out

    def __repr__(self):
        return f"MXFP4Tensor(shape={tuple(self.shape)}, device={self.device})"


def mxfp4_quantize(x):
    """(..., K) float tensor -> `MXFP4Tensor`.  The scale of 32 elements is 2 ** (floor(log2 max|x|) - 2),
    at least 2 ** -127; an element goes to the nearest code, ties to the even one, beyond 6 to 6.  A block
    that holds an infinity or a NaN reads back as NaN.  Any strides; a last dimension that is not
    contiguous is copied first."""
    _check(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must have a last dimension of at least 1, got {tuple(x.shape)}")
    v = _rows(x)
    rows, groups = v.shape[0] * v.shape[1], -(-v.shape[2] // _GROUP)
    codes = torch.empty((groups, rows, 64), dtype=torch.uint8, device=x.device)
    scales = torch.empty((groups, rows, 4), dtype=torch.uint8, device=x.device)
    _launch(x.device, _lib.load().glv_mxfp4_quantize, v.data_ptr(), _TYPES[x.dtype], *v.shape, v.stride(0), v.stride(1),
            codes.data_ptr(), scales.data_ptr())
    return MXFP4Tensor(x.shape, codes, scales)


def _product(x, weight, bias, taps, dilation, activation, out_dtype):
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be None or 'relu', got {activation!r}")
    n, cols = weight.shape[0], weight.shape[-1]
    device = weight.device
    if isinstance(x, MXFP4Tensor):
        if not x.codes.is_cuda:
            raise ValueError(f"x must be on a ROCm GPU (there is no CPU fallback), got {x.device}")
        if x.device != device:
            raise ValueError(f"x is on {x.device}, not on {device}")
        kind, data, scales = _MXFP4, x.codes.data_ptr(), x.scales.data_ptr()
        rows = x.shape[-2] if len(x.shape) > 1 else 1
        batch = x.codes.shape[1] // rows if rows else 0
        strides = (0, 0)
    else:
        _check(x, "x", device)
        if x.dim() < 1:
            raise ValueError("x must have at least one dimension")
    if x.shape[-1] != cols:
        raise ValueError(f"x has {x.shape[-1]} columns but the weight {cols}")
    if not isinstance(x, MXFP4Tensor):
        v = _rows(x)
        kind, data, scales = _TYPES[x.dtype], v.data_ptr(), None
        batch, rows, strides = v.shape[0], v.shape[1], (v.stride(0), v.stride(1))
    if taps == 1:  # rows of a linear layer need no batch entries, and fewer entries are fewer edges
        if strides[0] == rows * strides[1] or batch == 1:
            batch, rows = 1, batch * rows
    if out_dtype is None:
        out_dtype = torch.float32 if kind == _MXFP4 else x.dtype
    if out_dtype not in _TYPES:
        raise ValueError(f"out_dtype must be float32, bfloat16 or float16, got {out_dtype}")
    if bias is not None:
        bias = _vector(bias, "bias", n, device)
    lib = _lib.load()
    y = torch.empty((*x.shape[:-1], n), dtype=out_dtype, device=device)
    need = lib.glv_mxfp4_product_workspace(kind, batch, rows, cols, n, taps)
    work = torch.empty(need, dtype=torch.uint8, device=device) if need > 0 else None
    _launch(device, lib.glv_mxfp4_product, data, scales, kind, batch, rows, cols, strides[0], strides[1],
            weight.codes.data_ptr(), weight.scales.data_ptr(), n, taps, dilation,
            None if bias is None else bias.data_ptr(), 0 if bias is None else _TYPES[bias.dtype],
            _ACTIVATIONS[activation], y.data_ptr(), _TYPES[out_dtype], None if work is None else work.data_ptr(),
            max(need, 0))
    return y


def _check_weight(weight, dims, shape):
    if not isinstance(weight, MXFP4Tensor) or len(weight.shape) != dims:
        raise ValueError(f"weight must be an MXFP4Tensor of shape {shape} (mxfp4_quantize), got {weight!r}")
    if not weight.codes.is_cuda:
        raise ValueError(f"weight must be on a ROCm GPU (there is no CPU fallback), got {weight.device}")


def mxfp4_linear(x, weight, bias=None, *, activation=None, out_dtype=None):
    """(..., K) @ weight(N, K)^T + bias -> (..., N) with both operands in MXFP4 and sums in 32 bits.

    x           float tensor (quantised by the call, exactly as `mxfp4_quantize` does) or `MXFP4Tensor`
    weight      `MXFP4Tensor` of shape (N, K)
    bias        (N,) float tensor or None
    activation  None or "relu"
    out_dtype   default: the type of x; float32 for an `MXFP4Tensor`
    """
    _check_weight(weight, 2, "(N, K)")
    return _product(x, weight, bias, 1, 1, activation, out_dtype)


def mxfp4_conv1d(x, weight, bias=None, *, dilation=1, activation=None, out_dtype=None):
    """1-D convolution with 'same' zero padding over a channels-last sequence, in MXFP4: (B, T, C) or
    (T, C) -> (B, T, N) or (T, N), y[t] = sum_j x[t + j * dilation - left] weight[:, j] + bias with
    left = dilation * (taps - 1) // 2 (Keras Conv1D(padding='same'), torch padding='same').

    weight is an `MXFP4Tensor` of shape (N, taps, C): a torch.nn.Conv1d weight is
    ``mxfp4_quantize(conv.weight.permute(0, 2, 1))``.  The other arguments are `mxfp4_linear`'s."""
    _check_weight(weight, 3, "(N, taps, C)")
    if len(x.shape) not in (2, 3):
        raise ValueError(f"x must be (B, T, C) or (T, C), got {tuple(x.shape)}")
    if weight.shape[1] < 1:
        raise ValueError("weight must have at least one tap")
    if int(dilation) != dilation or dilation < 1:
        raise ValueError(f"dilation must be a positive integer, got {dilation!r}")
    return _product(x, weight, bias, weight.shape[1], int(dilation), activation, out_dtype)


class Norm:
    """One norm of `block_norm`: kind "layer" (LayerNorm) or "rms" (RMSNorm), eps, and optional weight
    and bias vectors (float32, or the type of the rows)."""

    __slots__ = ("weight", "bias", "eps", "kind")

    def __init__(self, weight=None, bias=None, eps=1e-5, kind="layer"):
        if kind not in _NORMS:
            raise ValueError(f"kind must be 'layer' or 'rms', got {kind!r}")
        if not eps >= 0:
            raise ValueError(f"eps must be >= 0, got {eps}")
        self.weight, self.bias, self.eps, self.kind = weight, bias, float(eps), kind


def block_norm(u, *, post=None, gate=None, scale=None, residual=None, pre=None):
    """y = residual + scale * gate * post(u), and z = pre(y) where `pre` is given: the end of a block
    and the start of the next in one pass.  Returns y, or (y, z).

    u         (..., C) float tensor: the block's output
    post      `Norm` of the block's output, or None
    gate      tensor of u's type that broadcasts to u's shape, or None
    scale     number, (C,) tensor, or None
    residual  tensor of u's shape and type, or None
    pre       `Norm` the next block starts with, or None

    Statistics are 32 bits; y enters `pre` before it is rounded to u's type.  C is at most 32768."""
    _check(u, "u")
    if u.dim() < 1 or u.shape[-1] < 1:
        raise ValueError(f"u must have a last dimension of at least 1, got {tuple(u.shape)}")
    device, dtype, cols = u.device, u.dtype, u.shape[-1]
    v = _rows(u)
    batch, rows, _ = v.shape
    vector_type = None
    vectors = []
    for side, norm in (("post", post), ("pre", pre)):
        if norm is not None and not isinstance(norm, Norm):
            raise ValueError(f"{side} must be a Norm or None, got {type(norm).__name__}")
        for name in ("weight", "bias"):
            t = getattr(norm, name, None)
            vectors.append(None if t is None else _vector(t, f"{side}.{name}", cols, device))
    factor = 1.0
    if isinstance(scale, torch.Tensor):
        vectors.append(_vector(scale, "scale", cols, device))
    else:
        vectors.append(None)
        if scale is not None:
            factor = float(scale)
    for t in vectors:
        if t is not None:
            if t.dtype not in (torch.float32, dtype) or vector_type not in (None, t.dtype):
                raise ValueError(f"weights, biases and scale must all be float32 or all {dtype}, got {t.dtype}")
            vector_type = t.dtype
    post_w, post_b, pre_w, pre_b, scale_vec = (None if t is None else t.data_ptr() for t in vectors)
    g = r = None
    g_strides, r_strides = (0, 0, 1), (0, 0)
    if gate is not None:
        _check(gate, "gate", device)
        if gate.dtype != dtype:
            raise ValueError(f"gate must be {dtype} like u, got {gate.dtype}")
        try:
            g = gate.expand(u.shape)
        except RuntimeError:
            raise ValueError(f"gate of shape {tuple(gate.shape)} does not broadcast to {tuple(u.shape)}") from None
        g = g[None, None] if g.dim() == 1 else g[None] if g.dim() == 2 else g
        if g.dim() > 3:
            g = g.reshape(batch, rows, cols) if g.numel() else g.new_empty((batch, rows, cols))
        if g.stride(2) not in (0, 1) and cols > 1:
            g = g.contiguous()
        g_strides = (g.stride(0), g.stride(1), g.stride(2) if cols > 1 else 0)
    if residual is not None:
        _check(residual, "residual", device)
        if residual.dtype != dtype or residual.shape != u.shape:
            raise ValueError(f"residual must be {dtype} {tuple(u.shape)} like u, got {residual.dtype} "
                             f"{tuple(residual.shape)}")
        r = _rows(residual)
        r_strides = (r.stride(0), r.stride(1))
    y = torch.empty(u.shape, dtype=dtype, device=device)
    z = torch.empty(u.shape, dtype=dtype, device=device) if pre is not None else None
    _launch(device, _lib.load().glv_block_norm, v.data_ptr(), _TYPES[dtype], batch, rows, cols, v.stride(0), v.stride(1),
            _TYPES[torch.float32 if vector_type is None else vector_type],
            0 if post is None else _NORMS[post.kind], post_w, post_b, 0.0 if post is None else post.eps,
            None if g is None else g.data_ptr(), *g_strides, scale_vec, factor,
            None if r is None else r.data_ptr(), *r_strides,
            0 if pre is None else _NORMS[pre.kind], pre_w, pre_b, 0.0 if pre is None else pre.eps,
            y.data_ptr(), None if z is None else z.data_ptr())
    return y if z is None else (y, z)
