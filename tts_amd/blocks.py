"""Operators of the acoustic model's serving path on MI355X: products with weights and activations
in microscaled 4-bit floating point (MXFP4), and the norms at a block's end and start fused with
its gate, scale and residual.

The reference's acoustic model is a stack of products with fixed weights, each followed by a norm
(TTS/Fastspeech_1.py:12-56); these are the kernels `FastSpeechAcousticModel.use_mxfp4` runs it on.
All arithmetic runs in libglvoc.so; torch owns the memory and the stream.  The functions enqueue
work on torch's current stream of the inputs' device, allocate their outputs and workspace from
torch (so they can be captured into a graph) and return without synchronising.  They are for
inference: a tensor that asks for a gradient is refused while gradients are recorded, one that carries a
forward-mode derivative always, and so is every call under `torch.jit.trace`, which would keep the outputs'
allocation and lose the work.
"""
from __future__ import annotations

import torch
import torch.autograd.forward_ad as _forward_ad

from . import _lib

__all__ = ["MXFP4Tensor", "Norm", "block_norm", "mxfp4_conv1d", "mxfp4_linear", "mxfp4_quantize"]

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_MXFP4 = 3
_ACTIVATIONS = {None: 0, "relu": 1}
_NORMS = {"layer": 1, "rms": 2}
_GROUP = 128  # columns that share one dword of scales
_INT = (1 << 31) - 1  # the library counts in ints; its own limits, which it names, are lower
_LARGE = 1 << 27  # elements of an output from which on the library is asked whether it takes the call before allocating


# The calls below take a few microseconds on the host, as much as a small launch on the device, so
# the checks are written to cost little when nothing is wrong, and the library is called in place.
# A call for another device than the current one makes that device current and starts again.
_current_device = torch.cuda.current_device
# the handle alone, without a Stream object around it, where torch offers that
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)

_is_tracing = torch._C._is_tracing


def _no_trace():
    if _is_tracing():
        raise ValueError("this operator cannot be traced: torch.jit.trace records torch's own operators alone")


def _check(t, name, index=None):
    """The element type's number, after the checks that every float input passes; `index` is the device
    that the call runs on."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor, got {type(t).__name__}")
    kind = _TYPES.get(t.dtype)
    if kind is None:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    if _forward_ad._current_level >= 0 and _forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{name} carries a forward-mode derivative: this operator is for inference and would drop it")
    at = t.get_device()
    if at < 0:
        raise ValueError(f"{name} must be on a ROCm GPU (there is no CPU fallback), got {t.device}")
    if index is not None and at != index:
        raise ValueError(f"{name} is on {t.device}, not on cuda:{index}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient: this operator is for inference (use torch.no_grad() or detach)")
    return kind


def _pointer(t, name):
    """The address of an argument that the library takes for absent where it is null: a tensor whose storage was given
    back (as sharded parameters' are between their uses) must not pass for none."""
    at = t.data_ptr()
    if not at and t.numel():
        raise ValueError(f"{name} has no memory: its storage was freed")
    return at


def _vector(t, name, n, index):
    """(n,) vector as (contiguous tensor, number of its type)."""
    kind = _check(t, name, index)
    if t.shape != (n,):
        raise ValueError(f"{name} must have shape ({n},), got {tuple(t.shape)}")
    return (t if t.stride(0) == 1 and n != 1 else t.resolve_neg().contiguous()), kind


def _rows(x, shape):
    """(tensor, batch, rows, batch stride, row stride) of x as (batch, rows, cols) with a contiguous last
    dimension; a copy only where no view will do.  The imaginary part of a conjugated tensor is such a case: its
    memory holds the values before a negation.  Those are two elements apart, so that any copy for the last
    dimension's sake resolves them, and only a single column has to be looked at."""
    if max(shape) > _INT:
        raise ValueError(f"a dimension of {tuple(shape)} is larger than {_INT}")
    dims = len(shape)
    if dims > 3:
        if shape[:-2].numel() > _INT:
            raise ValueError(f"the leading dimensions of {tuple(shape)} hold more than {_INT} entries")
        x = x.reshape(-1, shape[-2], shape[-1]) if x.numel() else x.new_empty((0, shape[-2], shape[-1]))
        shape, dims = x.shape, 3
    strides = x.stride()
    if shape[-1] == 1:
        x = x.resolve_neg()
        strides = x.stride()
    elif strides[-1] != 1:
        x = x.contiguous()
        strides = x.stride()
    if dims == 2:
        return x, 1, shape[0], 0, strides[0]
    if dims == 3:
        return x, shape[0], shape[1], strides[0], strides[1]
    return x, 1, 1, 0, 0


class MXFP4Tensor:
    """A tensor in MXFP4: along the last dimension every 32 elements share one power of two (E8M0)
    and an element is a 4-bit code for 0, 0.5, 1, 1.5, 2, 3, 4 or 6 with a sign (E2M1).

    shape   of the tensor it stands for; with rows = the product of all dimensions but the last and
            groups of 128 columns, the last one padded with zeros,
    data    the storage, (groups * rows * 68,) uint8 on one device: all codes, then all scales
    codes   (groups, rows, 64) view of it, two codes to a byte, the even column low
    scales  (groups, rows, 4) view of it, biased exponents of a group's four blocks; 255 is a NaN block
    """

    __slots__ = ("shape", "data", "rows", "groups")

    def __init__(self, shape, data):
        shape = torch.Size(shape)
        if len(shape) < 1 or shape[-1] < 1:
            raise ValueError(f"an MXFP4 tensor needs a last dimension of at least 1, got {tuple(shape)}")
        rows, groups = shape[:-1].numel(), -(-shape[-1] // _GROUP)
        if max(shape) > _INT or rows > _INT:
            raise ValueError(f"an MXFP4 tensor of shape {tuple(shape)} is too large")
        size = groups * rows * 68
        if data.dtype != torch.uint8 or data.shape != (size,) or not data.is_contiguous():
            raise ValueError(f"data must be a contiguous uint8 tensor of shape ({size},), got {data.dtype} "
                             f"{tuple(data.shape)}")
        if data.data_ptr() % 16:
            raise ValueError("data must start at a multiple of 16 bytes")
        self.shape, self.data, self.rows, self.groups = shape, data, rows, groups

    @property
    def device(self):
        return self.data.device

    @property
    def codes(self):
        return self.data[: self.groups * self.rows * 64].view(self.groups, self.rows, 64)

    @property
    def scales(self):
        return self.data[self.groups * self.rows * 64:].view(self.groups, self.rows, 4)

    def _pointers(self):
        at = _pointer(self.data, "the MXFP4 tensor")
        return at, at + self.groups * self.rows * 64

    def to(self, device):
        return MXFP4Tensor(self.shape, self.data.to(device))

    def dequantize(self, dtype=torch.float32):
        """The values the codes stand for, exact in float32 and bfloat16 (float16: within its range)."""
        kind = _TYPES.get(dtype)
        if kind is None:
            raise ValueError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
        _no_trace()
        data, shape = self.data, self.shape
        index = data.get_device()
        if index < 0:
            raise ValueError(f"the tensor must be on a ROCm GPU (there is no CPU fallback), got {self.device}")
        if _current_device() != index:
            with torch.cuda.device(index):
                return self.dequantize(dtype)
        out = data.new_empty(shape, dtype=dtype)
        codes, scales = self._pointers()
        array = _lib.mxfp4_array(out.data_ptr(), codes, scales, 0, 0, kind, 1, self.rows, shape[-1])
        rc = _lib.load().glv_mxfp4_dequantize(array, _current_stream(index))
        if rc:
            _lib.check(rc)
        return out

    def __repr__(self):
        return f"MXFP4Tensor(shape={tuple(self.shape)}, device={self.device})"


def mxfp4_quantize(x):
    """(..., K) float tensor -> `MXFP4Tensor`.  The scale of 32 elements is 2 ** (floor(log2 max|x|) - 2),
    at least 2 ** -127; an element goes to the nearest code, ties to the even one, beyond 6 to 6.  A block
    that holds an infinity or a NaN reads back as NaN.  Any strides; a last dimension that is not
    contiguous is copied first.  At most 2 ** 24 rows (all dimensions but the last) and 2 ** 18 columns."""
    _no_trace()
    kind, shape = _check(x, "x"), x.shape
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError(f"x must have a last dimension of at least 1, got {tuple(shape)}")
    index = x.get_device()
    if _current_device() != index:
        with torch.cuda.device(index):
            return mxfp4_quantize(x)
    v, batch, rows, batch_stride, row_stride = _rows(x, shape)
    cols = shape[-1]
    q = object.__new__(MXFP4Tensor)
    q.shape, q.rows, q.groups = shape, batch * rows, -(-cols // _GROUP)
    q.data = x.new_empty(q.rows * q.groups * 68, dtype=torch.uint8)
    codes, scales = q._pointers()
    array = _lib.mxfp4_array(v.data_ptr(), codes, scales, batch_stride, row_stride, kind, batch, rows, cols)
    rc = _lib.load().glv_mxfp4_quantize(array, _current_stream(index))
    if rc:
        _lib.check(rc)
    return q


def _product(x, weight, bias, taps, dilation, activation, out_dtype):
    _no_trace()
    act = _ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be None or 'relu', got {activation!r}")
    wshape = weight.shape
    n, cols, index = wshape[0], wshape[-1], weight.data.get_device()
    if _current_device() != index:
        with torch.cuda.device(index):
            return _product(x, weight, bias, taps, dilation, activation, out_dtype)
    scales, batch_stride, row_stride = 0, 0, 0
    if isinstance(x, MXFP4Tensor):
        like, shape = x.data, x.shape
        if like.get_device() < 0:
            raise ValueError(f"x must be on a ROCm GPU (there is no CPU fallback), got {like.device}")
        if like.get_device() != index:
            raise ValueError(f"x is on {like.device}, not on cuda:{index}")
        kind, (data, scales) = _MXFP4, x._pointers()
        rows = shape[-2] if len(shape) > 1 else 1
        batch = x.rows // rows if rows else 0
    else:
        kind, shape = _check(x, "x", index), x.shape
        if len(shape) < 1:
            raise ValueError("x must have at least one dimension")
    if shape[-1] != cols:
        raise ValueError(f"x has {shape[-1]} columns but the weight {cols}")
    if kind != _MXFP4:
        like, batch, rows, batch_stride, row_stride = _rows(x, shape)
        data = like.data_ptr()
    if taps == 1 and batch != 1 and batch_stride == rows * row_stride and batch * rows <= _INT:
        batch, rows = 1, batch * rows  # rows of a linear layer need no entries
    if out_dtype is None:
        out_dtype, out_kind = (torch.float32, 0) if kind == _MXFP4 else (x.dtype, kind)
    else:
        out_kind = _TYPES.get(out_dtype)
        if out_kind is None:
            raise ValueError(f"out_dtype must be float32, bfloat16 or float16, got {out_dtype}")
    bias_ptr, bias_kind = 0, 0
    if bias is not None:
        bias, bias_kind = _vector(bias, "bias", n, index)
        bias_ptr = _pointer(bias, "bias")
    lib = _lib.load()
    shape = (*shape[:-1], n)
    if batch * rows * n > _LARGE and lib.glv_mxfp4_product_workspace(_lib.mxfp4_product_args(
            0, 0, 0, 0, 0, 0, 0, 0, kind, batch, rows, cols, n, taps, dilation, 0, 0, 0)) < 0:
        _lib.check(-1)
    y = like.new_empty(shape) if out_kind == kind else like.new_empty(shape, dtype=out_dtype)
    args = _lib.mxfp4_product_args(data, scales, *weight._pointers(), bias_ptr, y.data_ptr(), batch_stride, row_stride, kind,
                                   batch, rows, cols, n, taps, dilation, bias_kind, act, out_kind)
    need = lib.glv_mxfp4_product_workspace(args)
    work_ptr = None
    if need > 0:
        work = like.new_empty(need, dtype=torch.uint8)
        work_ptr = work.data_ptr()
    rc = lib.glv_mxfp4_product(args, work_ptr, need, _current_stream(index))
    if rc:
        _lib.check(rc)
    return y


def _check_weight(weight, dims, shape):
    if not isinstance(weight, MXFP4Tensor) or len(weight.shape) != dims:
        raise ValueError(f"weight must be an MXFP4Tensor of shape {shape} (mxfp4_quantize), got {weight!r}")
    if weight.data.get_device() < 0:
        raise ValueError(f"weight must be on a ROCm GPU (there is no CPU fallback), got {weight.device}")


def mxfp4_linear(x, weight, bias=None, *, activation=None, out_dtype=None):
    """(..., K) @ weight(N, K)^T + bias -> (..., N) with both operands in MXFP4 and sums in 32 bits.

    x           float tensor (quantised by the call, exactly as `mxfp4_quantize` does) or `MXFP4Tensor`
    weight      `MXFP4Tensor` of shape (N, K)
    bias        (N,) float tensor or None
    activation  None or "relu"
    out_dtype   default: the type of x; float32 for an `MXFP4Tensor`

    At most 2 ** 24 rows of x, and K and N at most 2 ** 18.
    """
    _check_weight(weight, 2, "(N, K)")
    return _product(x, weight, bias, 1, 1, activation, out_dtype)


def mxfp4_conv1d(x, weight, bias=None, *, dilation=1, activation=None, out_dtype=None):
    """1-D convolution with 'same' zero padding over a channels-last sequence, in MXFP4: (B, T, C) or
    (T, C) -> (B, T, N) or (T, N), y[t] = sum_j x[t + j * dilation - left] weight[:, j] + bias with
    left = dilation * (taps - 1) // 2 (Keras Conv1D(padding='same'), torch padding='same').

    weight is an `MXFP4Tensor` of shape (N, taps, C): a torch.nn.Conv1d weight is
    ``mxfp4_quantize(conv.weight.permute(0, 2, 1))``.  The other arguments are `mxfp4_linear`'s.
    taps * C and N are at most 2 ** 18, B * T, N * taps and (taps - 1) * dilation at most 2 ** 24."""
    _check_weight(weight, 3, "(N, taps, C)")
    if not isinstance(x, (torch.Tensor, MXFP4Tensor)):
        raise ValueError(f"x must be a tensor, got {type(x).__name__}")
    if len(x.shape) not in (2, 3):
        raise ValueError(f"x must be (B, T, C) or (T, C), got {tuple(x.shape)}")
    if weight.shape[1] < 1:
        raise ValueError("weight must have at least one tap")
    if int(dilation) != dilation or not 1 <= dilation <= _INT:
        raise ValueError(f"dilation must be a positive integer of at most {_INT}, got {dilation!r}")
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


def _norm_vector(t, name, cols, index, kind, seen, held):
    """(pointer, number of its type) of a weight, bias or scale; all of a call share one type."""
    k = _check(t, name, index)
    if t.shape != (cols,):
        raise ValueError(f"{name} must have shape ({cols},), got {tuple(t.shape)}")
    if k != seen and (seen is not None or (k != 0 and k != kind)):
        raise ValueError(f"weights, biases and scale must all be float32 or all of u's type, got {t.dtype}")
    if t.stride(0) != 1 or cols == 1:
        t = t.resolve_neg().contiguous()
        held.append(t)
    return _pointer(t, name), k


def _broadcast(gate, shape, batch, rows, cols):
    """(tensor, [batch, row and column stride]) of a gate that broadcasts to `shape`, u's, taken as (batch,
    rows, cols)."""
    g = gate
    if len(shape) > 3:  # leading dimensions that a broadcast gate need not collapse like u's
        try:
            g = g.expand(shape)
        except RuntimeError:
            raise ValueError(f"gate of shape {tuple(gate.shape)} does not broadcast to {tuple(shape)}") from None
        g = g.reshape(batch, rows, cols) if g.numel() else g.new_empty((batch, rows, cols))
    dims = g.dim()
    sizes = (1, 1, 1)[dims:] + g.shape
    if dims > len(shape) or dims > 3 or sizes[0] not in (1, batch) or sizes[1] not in (1, rows) or sizes[2] not in (1, cols):
        raise ValueError(f"gate of shape {tuple(gate.shape)} does not broadcast to {tuple(shape)}")
    if sizes[2] == 1:
        g = g.resolve_neg()
    elif g.stride(-1) != 1:
        g = g.contiguous()
    strides = [0 if size == 1 else stride for size, stride in zip(sizes, (0, 0, 0)[dims:] + g.stride())]
    return g, strides


def block_norm(u, *, post=None, gate=None, scale=None, residual=None, pre=None):
    """y = residual + scale * gate * post(u), and z = pre(y) where `pre` is given: the end of a block
    and the start of the next in one pass.  Returns y, or (y, z).

    u         (..., C) float tensor: the block's output
    post      `Norm` of the block's output, or None
    gate      tensor of u's type that broadcasts to u's shape, or None
    scale     number, (C,) tensor, or None
    residual  tensor of u's shape and type, or None
    pre       `Norm` the next block starts with, or None

    Statistics are 32 bits; y enters `pre` before it is rounded to u's type.  C is at most
    32768, and there are at most 2 ** 24 rows."""
    _no_trace()
    kind, shape, index = _check(u, "u"), u.shape, u.get_device()
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError(f"u must have a last dimension of at least 1, got {tuple(shape)}")
    if _current_device() != index:
        with torch.cuda.device(index):
            return block_norm(u, post=post, gate=gate, scale=scale, residual=residual, pre=pre)
    cols = shape[-1]
    v, batch, rows, u_batch, u_row = _rows(u, shape)
    held, sides, vector_kind = [], [], None  # contiguous copies live until the launch
    for norm, side, weight_name, bias_name in ((post, "post", "post.weight", "post.bias"),
                                               (pre, "pre", "pre.weight", "pre.bias")):
        if norm is None:
            sides.append((0, 0, 0, 0.0))
        elif isinstance(norm, Norm):
            weight = bias = 0
            if norm.weight is not None:
                weight, vector_kind = _norm_vector(norm.weight, weight_name, cols, index, kind, vector_kind, held)
            if norm.bias is not None:
                bias, vector_kind = _norm_vector(norm.bias, bias_name, cols, index, kind, vector_kind, held)
            sides.append((_NORMS[norm.kind], weight, bias, norm.eps))
        else:
            raise ValueError(f"{side} must be a Norm or None, got {type(norm).__name__}")
    scale_ptr, factor = 0, 1.0
    if isinstance(scale, torch.Tensor):
        scale_ptr, vector_kind = _norm_vector(scale, "scale", cols, index, kind, vector_kind, held)
    elif scale is not None:
        factor = float(scale)
    gate_ptr, gate_strides = 0, (0, 0, 1)
    if gate is not None:
        if _check(gate, "gate", index) != kind:
            raise ValueError(f"gate must be {u.dtype} like u, got {gate.dtype}")
        if gate.shape == shape:
            g, _, _, *gate_strides = _rows(gate, shape)
            gate_strides.append(1)
        else:
            g, gate_strides = _broadcast(gate, shape, batch, rows, cols)
        gate_ptr = _pointer(g, "gate")
        held.append(g)
    res_ptr, res_batch, res_row = 0, 0, 0
    if residual is not None:
        if _check(residual, "residual", index) != kind or residual.shape != shape:
            raise ValueError(f"residual must be {u.dtype} {tuple(shape)} like u, got {residual.dtype} "
                             f"{tuple(residual.shape)}")
        r, _, _, res_batch, res_row = _rows(residual, shape)
        res_ptr = _pointer(r, "residual")
        held.append(r)
    if u.is_contiguous():  # the shorter call, which would keep other strides
        y = torch.empty_like(u)
        z = torch.empty_like(u) if pre is not None else None
    else:
        y = u.new_empty(shape)
        z = u.new_empty(shape) if pre is not None else None
    post_kind, post_w, post_b, post_eps = sides[0]
    pre_kind, pre_w, pre_b, pre_eps = sides[1]
    args = _lib.block_norm_args(v.data_ptr(), gate_ptr, res_ptr, post_w, post_b, scale_ptr, pre_w, pre_b, y.data_ptr(),
                                0 if z is None else z.data_ptr(), u_batch, u_row, gate_strides[0], gate_strides[1],
                                res_batch, res_row, kind, batch, rows, cols, vector_kind or 0, post_kind, pre_kind,
                                gate_strides[2], post_eps, pre_eps, factor)
    rc = _lib.load().glv_block_norm(args, _current_stream(index))
    if rc:
        _lib.check(rc)
    return y if z is None else (y, z)
