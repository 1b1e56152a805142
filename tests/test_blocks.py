"""The MXFP4 and block operators (tts_amd/blocks.py) against the float64 oracle, their refusals, and
their use on other streams and in graphs."""
import itertools
import os
import struct
import subprocess

import numpy as np
import pytest
import torch

import tts_amd
from oracle import blocks_oracle as O
from tts_amd import MXFP4Tensor, Norm, block_norm, mxfp4_conv1d, mxfp4_linear, mxfp4_quantize

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(dtype):
    """Largest relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2


def draw(rng, *shape, dtype=torch.float32, scale=1.0):
    x = rng.normal(0, scale, shape) * np.exp(rng.normal(0, 1, (*shape[:-1], 1)))
    return torch.from_numpy(x).to(dtype).cuda()


def f64(t):
    return t.detach().cpu().double().numpy()


def blocks_of(q):
    """codes (rows, blocks, 32) and scale bytes (rows, blocks) of an MXFP4Tensor's storage."""
    codes = q.codes.cpu().numpy().transpose(1, 0, 2)
    both = np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1, 32)
    scales = q.scales.cpu().numpy().transpose(1, 0, 2).reshape(codes.shape[0], -1)
    return both, scales


# -- quantisation -------------------------------------------------------------------------
def hard_values(dtype):
    """Blocks at the borders: ties, saturation, subnormals, the largest values, zeros of both signs."""
    big = torch.finfo(dtype).max
    tiny = float(np.float64(torch.finfo(dtype).tiny))
    ties = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.5]
    rows = []
    for s in (1.0, 2.0 ** -8, 2.0 ** 10, -1.0):
        rows.append([s * v for v in ties + [4.0]] + [0.0] * 21)
    rows.append([0.0, -0.0] * 16)
    rows.append([big, -big, big / 2, 1.0] + [0.0] * 28)
    sub = float(torch.finfo(dtype).smallest_normal) * 2.0 ** -3
    rows.append([tiny, -tiny, tiny * 1.5, sub, -sub, 3 * sub] + [0.0] * 26)
    rows.append([sub, -sub, 0.0] + [sub / 2] * 29)
    return torch.tensor(rows, dtype=torch.float64).to(dtype)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_borders_bit_for_bit(dtype):
    x = hard_values(dtype)
    q = mxfp4_quantize(x.cuda())
    codes, scales = blocks_of(q)
    want_codes, want_scales = O.mxfp4_encode(f64(x))
    assert np.array_equal(scales[:, :1], want_scales)
    # a value that rounds to zero keeps or loses its sign: both are zero
    a, b = codes[:, :1], want_codes
    assert np.array_equal(np.where((a & 7) == 0, 0, a), np.where((b & 7) == 0, 0, b))
    assert not codes[:, 1:].any() and not scales[:, 1:].any()  # the columns beyond the last are zeros


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 32), (3, 31), (17, 33), (16, 128), (5, 129), (33, 640), (2, 1001)])
def test_quantize_and_back_exactly(dtype, rows, cols):
    rng = np.random.default_rng(rows * 1000 + cols)
    x = draw(rng, rows, cols, dtype=dtype)
    x[rows // 2] = 0
    q = mxfp4_quantize(x)
    assert q.shape == (rows, cols)
    want = O.mxfp4_round(f64(x))
    assert np.array_equal(f64(q.dequantize()), want)
    assert np.array_equal(f64(q.dequantize(torch.bfloat16)), want)
    assert np.array_equal(f64(q.dequantize(torch.float16)), want.astype(np.float16).astype(np.float64))


@gpu
def test_every_finite_half_alone_and_all_exponents_of_float():
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.float16)
    every = every[torch.isfinite(every)]
    got = f64(mxfp4_quantize(every[:, None].cuda()).dequantize())[:, 0]
    v = f64(every)
    # alone in its block a value is scaled into [4, 8), subnormal scales aside, which halves do not reach
    assert np.array_equal(got, O.mxfp4_round(v[:, None])[:, 0])
    e = torch.arange(1, 255, dtype=torch.int32)
    mant = torch.tensor([0, 0x200000, 0x200001, 0x400000, 0x600000, 0x7fffff], dtype=torch.int32)
    x = ((e[:, None] << 23) | mant[None]).view(torch.float32)
    assert np.array_equal(f64(mxfp4_quantize(x.cuda()).dequantize()), O.mxfp4_round(f64(x)))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_infinity_and_nan_spoil_their_block_only(dtype):
    x = torch.ones(3, 96, dtype=dtype)
    x[0, 5], x[1, 40], x[2, 95] = float("nan"), float("inf"), -float("inf")
    got = mxfp4_quantize(x.cuda()).dequantize().cpu()
    bad = torch.zeros(3, 96, dtype=torch.bool)
    bad[0, :32] = bad[1, 32:64] = bad[2, 64:] = True
    assert torch.isnan(got[bad]).all()
    assert (got[~bad] == 1).all()


@gpu
def test_quantize_takes_any_strides():
    rng = np.random.default_rng(3)
    base = draw(rng, 6, 7, 80, dtype=torch.bfloat16)
    for x in (base[:, 1:6, 3:71], base.transpose(0, 1), base.permute(2, 0, 1), base[2], base[1, 2], base[:, ::2],
              base[0, 0, 5:6].expand(4, 33), base[None, :, None]):
        q = mxfp4_quantize(x)
        assert q.shape == x.shape
        assert np.array_equal(f64(q.dequantize()), O.mxfp4_round(f64(x)))


@gpu
def test_empty_inputs():
    w = mxfp4_quantize(torch.ones(5, 40, device="cuda"))
    for shape in ((0, 40), (2, 0, 40), (0, 3, 2, 40)):
        x = torch.empty(shape, device="cuda")
        assert mxfp4_quantize(x).dequantize().shape == x.shape
        assert mxfp4_linear(x, w).shape == (*shape[:-1], 5)
        assert mxfp4_linear(mxfp4_quantize(x), w).shape == (*shape[:-1], 5)
        assert block_norm(x, post=Norm()).shape == x.shape
    wc = mxfp4_quantize(torch.ones(5, 3, 40, device="cuda"))
    assert mxfp4_conv1d(torch.empty(0, 4, 40, device="cuda"), wc).shape == (0, 4, 5)
    assert mxfp4_conv1d(torch.empty(2, 0, 40, device="cuda"), wc).shape == (2, 0, 5)
    none = mxfp4_quantize(torch.empty(0, 40, device="cuda"))
    assert mxfp4_linear(torch.ones(2, 40, device="cuda"), none).shape == (2, 0)


# -- products -----------------------------------------------------------------------------
def product_bound(want, size, k, dtype):
    """Both operands' values are exact, so are their products (at most 5 bits).  A float sum of k of them in
    any order, through an adder that may cut instead of rounding, is off by at most k * 2^-23 times the sum
    of magnitudes; one is added for the bias.  The result is rounded once."""
    slack = (k + 1) * 2.0 ** -23 * size
    return slack + half_step(dtype) * (np.abs(want) + slack) + (2.0 ** -25 if dtype == torch.float16 else 1e-38)


def check_product(got, want, size, k, dtype):
    assert got.dtype == dtype
    err = np.abs(f64(got) - want)
    bound = product_bound(want, size, k, dtype)
    assert (err <= bound).all(), f"worst {np.max(err / bound):.3g} of the bound"


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 80, 256), (2, 33, 31), (7, 32, 128), (31, 5, 129), (32, 64, 257), (33, 65, 96),
                                   (65, 200, 513), (129, 130, 1001), (300, 257, 384), (1, 1000, 2049), (40, 40, 4101)])
def test_linear(dtype, m, n, k):
    rng = np.random.default_rng(m + 10 * n + 100 * k)
    x, w = draw(rng, m, k, dtype=dtype), draw(rng, n, k, scale=k ** -0.5)
    if m > 2:
        x[1] = 0
    bias = torch.from_numpy(rng.normal(0, 1, n)).to(dtype).cuda()
    q = mxfp4_quantize(w)
    xv, wv = O.mxfp4_round(f64(x)), f64(q.dequantize())
    want, size = xv @ wv.T, np.abs(xv) @ np.abs(wv).T
    check_product(mxfp4_linear(x, q), want, size, k, dtype)
    check_product(mxfp4_linear(mxfp4_quantize(x), q), want, size, k, torch.float32)
    for bias in (bias, bias.float()):
        b = f64(bias)
        check_product(mxfp4_linear(x, q, bias), want + b, size + np.abs(b), k, dtype)
        y = mxfp4_linear(x, q, bias, activation="relu", out_dtype=torch.float32)
        assert (y >= 0).all()
        check_product(y, np.maximum(want + b, 0), size + np.abs(b), k, torch.float32)


@gpu
@pytest.mark.parametrize("batch,time,c,n,taps,dilation", [
    (1, 1, 1, 1, 1, 1), (1, 1, 32, 40, 5, 2), (2, 3, 80, 33, 7, 3), (1, 9, 256, 64, 5, 2), (3, 40, 40, 80, 3, 1),
    (2, 33, 129, 31, 4, 1), (1, 165, 256, 256, 5, 2), (5, 65, 128, 70, 2, 4), (2, 2, 33, 20, 3, 50)])
@pytest.mark.parametrize("dtype", TYPES)
def test_conv1d(dtype, batch, time, c, n, taps, dilation):
    rng = np.random.default_rng(batch + 7 * time + 31 * c + taps)
    x, w = draw(rng, batch, time, c, dtype=dtype), draw(rng, n, taps, c, scale=(taps * c) ** -0.5)
    bias = torch.from_numpy(rng.normal(0, 1, n)).float().cuda()
    q = mxfp4_quantize(w)
    xv, wv = O.mxfp4_round(f64(x)), f64(q.dequantize())
    want, size = O.conv1d(xv, wv, f64(bias), dilation)
    check_product(mxfp4_conv1d(x, q, bias, dilation=dilation), want, size, taps * c, dtype)
    check_product(mxfp4_conv1d(mxfp4_quantize(x), q, bias, dilation=dilation), want, size, taps * c, torch.float32)
    check_product(mxfp4_conv1d(x[0], q, bias, dilation=dilation, activation="relu"), np.maximum(want[0], 0), size[0],
                  taps * c, dtype)


def gathered(x, taps, dilation):
    """(B, T, C) -> (B * T, taps * C), zeros outside."""
    b, t, c = x.shape
    left = dilation * (taps - 1) // 2
    padded = x.new_zeros((b, t + dilation * (taps - 1), c))
    padded[:, left:left + t] = x
    return torch.cat([padded[:, j * dilation:j * dilation + t] for j in range(taps)], -1).reshape(b * t, -1)


def check_product_on_device(got, rows, weight, bias, relu):
    """check_product with the float64 product formed on the device: rows (M, K), weight (N, K) float64."""
    dtype, k = got.dtype, rows.shape[1]
    wt = weight.t().contiguous()
    want, size = torch.mm(rows, wt), torch.mm(rows.abs(), wt.abs())
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    if relu:
        want = want.clamp_min(0)
    slack = (k + 1) * 2.0 ** -23 * size
    bound = slack + half_step(dtype) * (want.abs() + slack) + (2.0 ** -25 if dtype == torch.float16 else 1e-38)
    err = (got.double().reshape(want.shape) - want).abs()
    assert (err <= bound).all(), f"worst {(err / bound).max().item():.3g} of the bound"


# odd edges of every tiling: small outputs; more than 2 M of them; many rows of up to 256; long sums
LARGE = [(512, 512, 1), (1000, 300, 129), (255, 2049, 385), (4100, 70, 640), (30000, 9, 200), (2000, 257, 2300),
         (513, 6200, 100), (3100, 1100, 385), (12300, 257, 1001), (16500, 1030, 1100), (700, 8200, 1500), (260000, 9, 300),
         (33000, 129, 1), (40000, 200, 385), (32769, 256, 600), (16500, 1030, 4100), (100000, 70, 4200),
         (33000, 129, 1100), (50000, 250, 130), (12900, 1000, 1025), (8500, 1001, 4100), (4100, 2300, 4200),
         (33000, 128, 384), (50001, 100, 131), (50001, 255, 257),
         (3100, 1100, 300), (1000, 2000, 2900), (1250, 1500, 140)]


@gpu
@pytest.mark.parametrize("m,n,k", LARGE)
@pytest.mark.parametrize("dtype", TYPES)
def test_linear_of_many_rows_and_columns(dtype, m, n, k):
    rng = np.random.default_rng(m + n + k)
    x, w, bias = draw(rng, m, k, dtype=dtype), draw(rng, n, k, scale=k ** -0.5), draw(rng, n)
    x[m // 2] = 0
    q, xq = mxfp4_quantize(w), mxfp4_quantize(x)
    xv, wv = xq.dequantize().double(), q.dequantize().double()
    check_product_on_device(mxfp4_linear(x, q), xv, wv, None, False)
    check_product_on_device(mxfp4_linear(xq, q, bias, activation="relu", out_dtype=dtype), xv, wv, bias, True)


@gpu
@pytest.mark.parametrize("batch,time,c,n,taps,dilation", [
    (4, 300, 256, 260, 3, 1), (1, 1100, 80, 256, 5, 2), (7, 129, 130, 300, 4, 3), (600, 1, 64, 512, 3, 1), (40, 31, 40, 256, 7, 40),
    (2, 600, 300, 250, 2, 1), (64, 200, 256, 256, 3, 1), (3, 4100, 80, 300, 5, 2), (5000, 3, 130, 257, 4, 1), (130, 130, 60, 1030, 17, 20), (64, 700, 130, 200, 3, 2),
    (11000, 3, 40, 250, 4, 1), (130, 130, 60, 1030, 33, 3), (5500, 3, 100, 1000, 33, 1),
    (72, 700, 130, 200, 3, 2), (330, 100, 8, 80, 5, 7), (65, 505, 300, 128, 3, 1), (70, 705, 256, 250, 4, 5), (50001, 1, 384, 256, 1, 1),
    (25001, 2, 40, 33, 7, 2), (8, 500, 130, 515, 3, 1), (3, 1300, 100, 600, 5, 2), (5, 801, 260, 300, 3, 7), (11000, 3, 40, 250, 9, 1), (130, 65, 60, 1001, 33, 3), (3000, 3, 100, 1000, 33, 1)])
def test_conv1d_of_many_rows(batch, time, c, n, taps, dilation):
    rng = np.random.default_rng(batch + time + c)
    x, w, bias = draw(rng, batch, time, c), draw(rng, n, taps, c, scale=(taps * c) ** -0.5), draw(rng, n)
    q, xq = mxfp4_quantize(w), mxfp4_quantize(x)
    rows, wv = gathered(xq.dequantize().double(), taps, dilation), q.dequantize().double().reshape(n, -1)
    for dtype in TYPES:
        check_product_on_device(mxfp4_conv1d(xq, q, bias, dilation=dilation, out_dtype=dtype), rows, wv, bias, False)
    check_product_on_device(mxfp4_conv1d(x, q, bias, dilation=dilation, activation="relu"), rows, wv, bias, True)


@gpu
def test_conv1d_agrees_with_torch_same_padding():
    """The padding convention, at values that MXFP4 holds exactly: the sums are exact integers."""
    rng = np.random.default_rng(8)
    for taps, dilation in itertools.product((1, 2, 3, 4, 5), (1, 2, 3)):
        conv = torch.nn.Conv1d(48, 20, taps, padding="same", dilation=dilation)
        with torch.no_grad():
            conv.weight.copy_(torch.from_numpy(rng.integers(-2, 3, conv.weight.shape)).float())
            conv.bias.copy_(torch.from_numpy(rng.integers(-9, 9, 20)).float())
            conv.weight[:, 0], conv.weight[:, 32] = 4, 4  # the scale of every block is 1
            x = torch.from_numpy(rng.integers(-3, 4, (2, 11, 48))).float()
            x[..., 0], x[..., 32] = 4, 4
            want = conv(x.transpose(1, 2)).transpose(1, 2)
        q = mxfp4_quantize(conv.weight.detach().permute(0, 2, 1).cuda())
        got = mxfp4_conv1d(x.cuda(), q, conv.bias.detach().cuda(), dilation=dilation)
        assert torch.equal(got.cpu(), want)


@gpu
@pytest.mark.parametrize("m", [1, 5, 40, 300, 50000])
def test_a_spoilt_row_of_either_side_stays_in_its_place(m):
    x, w = torch.ones(m, 200, device="cuda"), torch.ones(70, 200, device="cuda")
    x[m - 1, 150] = float("nan")
    w[3, 7] = float("inf")
    y = mxfp4_linear(x, mxfp4_quantize(w)).cpu()
    bad = torch.zeros(m, 70, dtype=torch.bool)
    bad[m - 1], bad[:, 3] = True, True
    assert torch.isnan(y[bad]).all() and (y[~bad] == 200).all()
    assert torch.isnan(mxfp4_linear(x, mxfp4_quantize(w), activation="relu").cpu()[bad]).all()


@gpu
def test_conv1d_entries_do_not_reach_into_each_other():
    x = torch.zeros(3, 9, 64, device="cuda")
    x[1] = float("nan")
    w = mxfp4_quantize(torch.ones(10, 5, 64, device="cuda"))
    y = mxfp4_conv1d(x, w, dilation=2)
    assert torch.isnan(y[1]).all() and (y[0] == 0).all() and (y[2] == 0).all()


@gpu
def test_products_take_any_strides_and_leave_their_inputs():
    rng = np.random.default_rng(4)
    base = draw(rng, 5, 12, 100, dtype=torch.float16)
    kept = base.clone()
    w = mxfp4_quantize(draw(rng, 24, 64))
    wv = f64(w.dequantize())
    for x in (base[..., 7:71], base[:, :, :64].transpose(0, 1), base[:, ::3, 36:], base[2, 3, :64], base[:, :1, :64].expand(5, 40, 64),
              base[None, :, :, 30:94]):
        xv = O.mxfp4_round(f64(x))
        check_product(mxfp4_linear(x, w), xv @ wv.T, np.abs(xv) @ np.abs(wv).T, 64, torch.float16)
    assert torch.equal(base, kept)


# -- norms --------------------------------------------------------------------------------
def check_block_norm(u, post, gate, scale, residual, pre, got):
    """Bounds from the arithmetic: a float sum of C values over at most 64 + 6 + 16 additions in a row, so means
    are off by 100 * 2^-24 of the mean magnitude; the remaining steps are some ten roundings."""
    dtype, ulp = u.dtype, 2.0 ** -24
    rnd = half_step(dtype)
    x = f64(u)
    err = np.zeros_like(x)

    def through(x, err, norm):
        w = np.ones(x.shape[-1]) if norm.weight is None else f64(norm.weight)
        b = np.zeros(x.shape[-1]) if norm.bias is None else f64(norm.bias)
        y = O.norm(x, norm.kind, w, b, norm.eps)
        centred = x - x.mean(-1, keepdims=True) if norm.kind == "layer" else x
        r = 1 / np.sqrt((centred ** 2).mean(-1, keepdims=True) + norm.eps)
        hat = np.abs(centred) * r
        worst = err.max(-1, keepdims=True)  # of the inputs, reaching the result directly and through the statistics
        if norm.kind == "layer":
            worst = worst + 100 * ulp * np.abs(x).mean(-1, keepdims=True)
        e = np.abs(w) * (r * worst * (2 + hat) + (110 * ulp) * hat + r * ulp * np.abs(x)) + 4 * ulp * (np.abs(y) + np.abs(b))
        return y, e

    if post is not None:
        x, err = through(x, err, post)
    k = np.ones(x.shape[-1])
    if gate is not None:
        k = k * f64(gate)
    if scale is not None:
        k = k * (f64(scale) if isinstance(scale, torch.Tensor) else scale)
    x, err = x * k, err * np.abs(k)
    err = err + 4 * ulp * np.abs(x)
    if residual is not None:
        x = x + f64(residual)
        err = err + ulp * np.abs(x)
    outs = [(x, err)]
    if pre is not None:
        outs.append(through(x, err, pre))
    got = (got,) if pre is None else got
    assert len(got) == len(outs)
    for g, (want, e) in zip(got, outs):
        assert g.dtype == dtype and g.shape == u.shape and g.is_contiguous()
        bound = e + rnd * (np.abs(want) + e) + (2.0 ** -25 if dtype == torch.float16 else 1e-38)
        ratio = np.abs(f64(g) - want) / bound
        assert (ratio <= 1).all(), f"worst {ratio.max():.3g} of the bound"


def norm_vectors(rng, kind, c, dtype, eps=1e-3):
    v = [torch.from_numpy(centre + 0.2 * rng.normal(size=c)).to(dtype).cuda() for centre in (1.0, 0.0)]
    return Norm(v[0], v[1] if kind == "layer" else None, eps=eps, kind=kind)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("b,t,c", [(1, 1, 1), (1, 5, 7), (3, 2, 8), (1, 9, 63), (2, 33, 256), (1, 3, 512), (2, 7, 520),
                                   (1, 3, 1024), (1, 5, 1025), (2, 2, 4097), (1, 2, 8191), (1, 2, 8200), (1, 1, 32768)])
def test_block_norm_whole(dtype, kind, b, t, c):
    rng = np.random.default_rng(c + t)
    u, residual, gate = (draw(rng, b, t, c, dtype=dtype) + 0.5 for _ in range(3))
    post, pre = norm_vectors(rng, kind, c, torch.float32), norm_vectors(rng, kind, c, torch.float32)
    scale = torch.from_numpy(rng.normal(0.5, 0.1, c)).float().cuda()
    got = block_norm(u, post=post, gate=gate, scale=scale, residual=residual, pre=pre)
    check_block_norm(u, post, gate, scale, residual, pre, got)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_block_norm_parts(dtype):
    rng = np.random.default_rng(11)
    b, t, c = 2, 5, 200
    u, residual = draw(rng, b, t, c, dtype=dtype), draw(rng, b, t, c, dtype=dtype)
    scale = torch.from_numpy(rng.normal(0.5, 0.1, c)).to(dtype).cuda()
    gates = [None] + [draw(rng, *s, dtype=dtype) for s in ((b, t, c), (b, 1, c), (t, c), (c,), (b, t, 1), (1,))]
    for post, pre, gate, s, r in itertools.product((None, norm_vectors(rng, "layer", c, dtype), Norm(kind="rms")),
                                                   (None, norm_vectors(rng, "rms", c, dtype), Norm(eps=1e-5)), gates,
                                                   (None, 0.25, scale), (None, residual)):
        got = block_norm(u, post=post, gate=gate, scale=s, residual=r, pre=pre)
        check_block_norm(u, post, gate, s, r, pre, got)


@gpu
@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 3), (17, 129), (33, 250), (9, 505), (5, 1001), (3, 4097), (2, 20001)])
@pytest.mark.parametrize("dtype", TYPES)
def test_block_norm_in_place_of_each_input(dtype, rows, cols):
    """From C, y may be u, gate or residual itself."""
    from tts_amd import _lib
    rng = np.random.default_rng(rows + cols)
    u, gate, residual = (draw(rng, rows, cols, dtype=dtype) for _ in range(3))
    want, wantz = block_norm(u, post=Norm(), gate=gate, residual=residual, pre=Norm(kind="rms"))
    for which in range(3):
        t = [u.clone(), gate.clone(), residual.clone()]
        z = torch.empty_like(u)
        args = _lib.block_norm_args(*(v.data_ptr() for v in t), 0, 0, 0, 0, 0, t[which].data_ptr(), z.data_ptr(), 0, cols, 0, cols,
                                    0, cols, TYPES.index(dtype), 1, rows, cols, 0, 1, 2, 1, 1e-5, 1e-5, 1.0)
        rc = _lib.load().glv_block_norm(args, torch.cuda.current_stream().cuda_stream)
        assert rc == 0 and torch.equal(t[which], want) and torch.equal(z, wantz)


@gpu
def test_block_norm_any_strides_and_leading_dimensions():
    rng = np.random.default_rng(12)
    base = draw(rng, 4, 6, 150)
    other = draw(rng, 4, 6, 150)
    gate = draw(rng, 6, 300)[:, ::2]
    for cut in (lambda v: v[..., 11:140], lambda v: v.transpose(0, 1), lambda v: v.permute(2, 1, 0), lambda v: v[1],
                lambda v: v[1, 2], lambda v: v[:, ::2, :64], lambda v: v[None, :, :, None]):
        u, r = cut(base), cut(other)
        check_block_norm(u, Norm(), None, None, r, Norm(kind="rms"), block_norm(u, post=Norm(), residual=r, pre=Norm(kind="rms")))
    check_block_norm(base, Norm(), gate, None, other, None, block_norm(base, post=Norm(), gate=gate, residual=other))
    wide = gate[None].expand(3, 4, 6, 150)
    u = draw(rng, 3, 4, 6, 150)
    check_block_norm(u, None, wide, 2.0, None, None, block_norm(u, gate=wide, scale=2.0))


@gpu
def test_block_norm_constant_zero_and_spoilt_rows():
    u = torch.randn(6, 300, device="cuda")
    u[1], u[2], u[3, 7], u[4, 299] = 0, 1e4, float("nan"), float("inf")
    for kind in ("layer", "rms"):
        y, z = block_norm(u, post=Norm(kind=kind, eps=1e-3), residual=torch.zeros_like(u), pre=Norm(kind=kind, eps=1e-3))
        assert torch.isnan(y[3]).all() and torch.isnan(z[3]).all() and torch.isnan(z[4]).any()
        assert torch.isfinite(y[[0, 1, 2, 5]]).all() and torch.isfinite(z[[0, 1, 2, 5]]).all()
        assert (y[1] == 0).all()
        assert kind == "rms" or y[2].abs().max() < 1e4 * 100 * 2.0 ** -24 / 1e-3 ** 0.5


# -- use ----------------------------------------------------------------------------------
def serve(x, w1, b1, w2, b2, post, pre):
    """Two blocks as a model runs them: convolution, norm and the next block's norm, linear layer, norm."""
    h = mxfp4_conv1d(x, w1, b1, dilation=2, activation="relu")
    y, z = block_norm(h, post=post, residual=x, pre=pre)
    return block_norm(mxfp4_linear(z, w2, b2), post=post, residual=y, scale=0.5)


@gpu
@pytest.mark.parametrize("batch,time", [(1, 9), (3, 70)])
def test_a_run_of_them_against_float64(batch, time):
    """The chain with its own roundings: each stage is compared with the oracle on the stage's actual input, so
    that a value which falls on the other side of a 4-bit rounding border upstream is not an error here."""
    rng = np.random.default_rng(21)
    c = 96
    x = draw(rng, batch, time, c)
    w1, w2 = mxfp4_quantize(draw(rng, c, 5, c, scale=0.05)), mxfp4_quantize(draw(rng, c, c, scale=0.1))
    b1, b2 = draw(rng, c), draw(rng, c)
    post, pre = norm_vectors(rng, "layer", c, torch.float32), norm_vectors(rng, "layer", c, torch.float32)
    h = mxfp4_conv1d(x, w1, b1, dilation=2, activation="relu")
    want, size = O.conv1d(O.mxfp4_round(f64(x)), f64(w1.dequantize()), f64(b1), 2)
    check_product(h, np.maximum(want, 0), size, 5 * c, torch.float32)
    y, z = block_norm(h, post=post, residual=x, pre=pre)
    check_block_norm(h, post, None, None, x, pre, (y, z))
    o = mxfp4_linear(z, w2, b2)
    zv, wv = O.mxfp4_round(f64(z)), f64(w2.dequantize())
    check_product(o, zv @ wv.T + f64(b2), np.abs(zv) @ np.abs(wv).T + np.abs(f64(b2)), c, torch.float32)
    out = block_norm(o, post=post, residual=y, scale=0.5)
    check_block_norm(o, post, None, 0.5, y, None, out)
    assert torch.equal(out, serve(x, w1, b1, w2, b2, post, pre))  # and the same bits again


@gpu
def test_two_graphs_and_eager_work_in_turn():
    rng = np.random.default_rng(22)
    c = 128
    w1, w2 = mxfp4_quantize(draw(rng, c, 3, c, scale=0.05)), mxfp4_quantize(draw(rng, c, c, scale=0.1))
    b1, b2 = draw(rng, c), draw(rng, c)
    post, pre = norm_vectors(rng, "layer", c, torch.float32), norm_vectors(rng, "rms", c, torch.float32)
    graphs = []
    for time in (1, 50, 300):
        x = draw(rng, 2, time, c)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            serve(x, w1, b1, w2, b2, post, pre)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = serve(x, w1, b1, w2, b2, post, pre)
        graphs.append((g, x, out))
    for turn in range(4):
        for g, x, out in graphs:
            fresh = draw(rng, *x.shape)
            x.copy_(fresh)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, serve(fresh, w1, b1, w2, b2, post, pre)), f"turn {turn}"


@gpu
def test_other_streams_at_once_give_the_same_bits():
    rng = np.random.default_rng(23)
    c = 256
    w = mxfp4_quantize(draw(rng, c, c, scale=0.05))
    xs = [draw(rng, m, c, dtype=torch.bfloat16) for m in (3, 40, 200, 500)]
    want = [block_norm(mxfp4_linear(x, w), post=Norm(), pre=Norm()) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        got = []
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(block_norm(mxfp4_linear(x, w), post=Norm(), pre=Norm()))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


@gpu
def test_calls_from_several_threads_at_once():
    import threading
    rng = np.random.default_rng(24)
    w, post = mxfp4_quantize(draw(rng, 96, 96, scale=0.1)), norm_vectors(rng, "layer", 96, torch.float32)
    xs = [draw(rng, m, 96) for m in (1, 33, 400, 2500)]
    want = [block_norm(mxfp4_linear(x, w), post=post) for x in xs]
    torch.cuda.synchronize()
    got, errors = [None] * len(xs), []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i] = block_norm(mxfp4_linear(xs[i], w), post=post)
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001 - reported below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(xs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    assert all(torch.equal(g, v) for g, v in zip(got, want))


@gpu
def test_arrays_beyond_32_bit_offsets():
    """Inputs and outputs of more than 2^31 elements: their last rows against the same rows alone."""
    rng = np.random.default_rng(25)
    rows, cols, tail = 530000, 4100, 70
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    assert x.numel() > 2 ** 31
    x[-tail:] = draw(rng, tail, cols, dtype=torch.bfloat16)
    part = x[-tail:].clone()
    q = mxfp4_quantize(x)
    alone = mxfp4_quantize(part)
    assert torch.equal(q.codes[:, -tail:], alone.codes) and torch.equal(q.scales[:, -tail:], alone.scales)
    assert not q.codes[:, :-tail].any()
    values = q.dequantize(torch.bfloat16)
    assert torch.equal(values[-tail:], alone.dequantize(torch.bfloat16))
    del values
    w = mxfp4_quantize(draw(rng, 9, cols, scale=cols ** -0.5))
    y = mxfp4_linear(q, w)
    check_product_on_device(y[-tail:], alone.dequantize().double(), w.dequantize().double(), None, False)
    assert not y[:-tail].any()
    post = norm_vectors(rng, "layer", cols, torch.float32)
    z = block_norm(x, post=post, residual=x)
    assert torch.equal(z[-tail:], block_norm(part, post=post, residual=part))
    del x, q, y, z
    # a product whose result is that long
    m, n, k = 300000, 7300, 64
    x, w = torch.zeros(m, k, dtype=torch.float16, device="cuda"), mxfp4_quantize(draw(rng, n, k))
    x[-tail:] = draw(rng, tail, k, dtype=torch.float16)
    y = mxfp4_linear(x, w)
    assert y.numel() > 2 ** 31
    check_product_on_device(y[-tail:], mxfp4_quantize(x[-tail:]).dequantize().double(), w.dequantize().double(), None, False)
    assert not y[:5].any() and not y[m // 2].any()


# -- refusals -----------------------------------------------------------------------------
def packed(shape, device="cpu"):
    rows, groups = int(np.prod(shape[:-1])), -(-shape[-1] // 128)
    return MXFP4Tensor(shape, torch.zeros(groups * rows * 68, dtype=torch.uint8, device=device))


def test_refusals_without_gpu():
    x, w = torch.zeros(3, 40), packed((5, 40))
    for call in (lambda: mxfp4_quantize(x), lambda: mxfp4_linear(x, w), lambda: mxfp4_conv1d(x, packed((5, 3, 40))),
                 lambda: block_norm(x, post=Norm()), lambda: w.dequantize()):
        with pytest.raises(ValueError, match="ROCm GPU"):
            call()
    with pytest.raises(ValueError, match="must be a tensor"):
        mxfp4_quantize([1.0])
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        mxfp4_quantize(torch.zeros(3, 4, dtype=torch.int32))
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        block_norm(torch.zeros(3, 4, dtype=torch.float64))
    with pytest.raises(ValueError, match="dtype"):
        w.dequantize(torch.float64)
    for weight in (x, packed((5, 3, 40)), None):
        with pytest.raises(ValueError, match="weight must be an MXFP4Tensor"):
            mxfp4_linear(x, weight)
    with pytest.raises(ValueError, match="weight must be an MXFP4Tensor"):
        mxfp4_conv1d(x, w)
    for bad in (dict(kind="batch"), dict(eps=-1.0), dict(eps=float("nan"))):
        with pytest.raises(ValueError):
            Norm(**bad)
    for data in (torch.zeros(5 * 68 - 1, dtype=torch.uint8), torch.zeros(5 * 68), torch.zeros(1, 5 * 68, dtype=torch.uint8),
                 torch.zeros(10 * 68, dtype=torch.uint8)[::2]):
        with pytest.raises(ValueError, match="data must be"):
            MXFP4Tensor((5, 40), data)
    with pytest.raises(ValueError, match="16 bytes"):
        MXFP4Tensor((5, 40), torch.zeros(5 * 68 + 1, dtype=torch.uint8)[1:])
    with pytest.raises(ValueError, match="last dimension"):
        MXFP4Tensor((5, 0), torch.zeros(0, dtype=torch.uint8))
    for shape in ((0, 1 << 32), (1 << 32, 0, 40)):
        with pytest.raises(ValueError, match="too large"):
            MXFP4Tensor(shape, torch.zeros(0, dtype=torch.uint8))
    assert w.codes.shape == (1, 5, 64) and w.scales.shape == (1, 5, 4) and w.to("cpu").shape == (5, 40)
    for name in ("MXFP4Tensor", "Norm", "block_norm", "mxfp4_conv1d", "mxfp4_linear", "mxfp4_quantize"):
        assert name in tts_amd.__all__


def test_packed_arguments_are_the_headers_structs(tmp_path):
    from tts_amd import _lib
    # (struct, last field, its size) and the packed form with that field alone set
    structs = [("glv_mxfp4_array", "cols", 4, _lib.mxfp4_array(*[0] * 8, 1)),
               ("glv_mxfp4_product_args", "y_type", 4, _lib.mxfp4_product_args(*[0] * 17, 1)),
               ("glv_block_norm_args", "scale", 4, _lib.block_norm_args(*[0] * 26, 1.0))]
    source = "#include <stddef.h>\n#include \"glvoc.h\"\n"
    for name, last, size, packed in structs:
        at = next(i for i in range(0, len(packed), 4) if any(packed[i:i + 4]))
        source += f"_Static_assert(sizeof({name}) == {len(packed)} && offsetof({name}, {last}) == {at}, \"{name}\");\n"
    (tmp_path / "structs.c").write_text(source)
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-std=c11", "-fsyntax-only", "-I", include, str(tmp_path / "structs.c")], check=True)
    with pytest.raises(struct.error):
        _lib.mxfp4_array(0, 0, 0, 0, 0, 0, 1, 1 << 32, 1)


def test_c_entries_validate_before_any_device_call():
    from tts_amd import _lib
    lib = _lib.load()
    a, odd = 4096, 4097  # never looked at: every call below is refused first

    def quantize(x=a, kind=0, batch=1, rows=4, cols=32, codes=a, scales=a):
        return lib.glv_mxfp4_quantize(_lib.mxfp4_array(x or 0, codes or 0, scales or 0, rows * cols, cols, kind, batch, rows, cols), None)

    for kw in (dict(x=None), dict(codes=None), dict(scales=None), dict(kind=3), dict(kind=-1), dict(cols=0), dict(rows=-1),
               dict(batch=-1), dict(cols=1 << 19), dict(rows=(1 << 24) + 1), dict(batch=1 << 12, rows=1 << 13),
               dict(codes=4104), dict(scales=4098), dict(x=odd)):
        assert quantize(**kw) == -1, kw
        assert b"glv_mxfp4_quantize" in lib.glv_last_error()
    assert quantize(rows=0) == 0 and quantize(batch=0, x=None, codes=None, scales=None) == 0

    def dequantize(codes, scales, rows, cols, kind, out):
        return lib.glv_mxfp4_dequantize(_lib.mxfp4_array(out or 0, codes or 0, scales or 0, 0, 0, kind, 1, rows, cols), None)

    for kw in ((None, a, 4, 32, 0, a), (a, None, 4, 32, 0, a), (a, a, 4, 32, 0, None), (a, a, 4, 32, 3, a), (a, a, -1, 32, 0, a),
               (a, a, 4, 0, 0, a), (a, a, 4, 32, 0, odd), (4104, a, 4, 32, 0, a)):
        assert dequantize(*kw) == -1
    assert dequantize(None, None, 0, 32, 0, None) == 0

    def product(x=a, xs=None, kind=0, batch=1, rows=4, cols=32, wc=a, ws=a, n=8, taps=1, dilation=1, bias=None, bias_kind=0,
                act=0, y=a, y_kind=0, work=a, size=1 << 20):
        args = _lib.mxfp4_product_args(x or 0, xs or 0, wc or 0, ws or 0, bias or 0, y or 0, rows * cols, cols, kind, batch, rows, cols,
                                       n, taps, dilation, bias_kind, act, y_kind)
        return lib.glv_mxfp4_product(args, work, size, None)

    for kw in (dict(x=None), dict(wc=None), dict(ws=None), dict(y=None), dict(rows=64, cols=4096, work=None), dict(rows=64, cols=4096, size=8),
               dict(kind=4),
               dict(kind=3), dict(y_kind=3), dict(act=2), dict(taps=0), dict(dilation=0), dict(n=-1), dict(cols=0), dict(rows=-1),
               dict(taps=1 << 14), dict(taps=2, dilation=(1 << 24) + 1), dict(n=(1 << 18) + 1), dict(y=odd), dict(bias=odd), dict(x=odd),
               dict(bias=a, bias_kind=3), dict(wc=4104),
               dict(rows=64, cols=4096, work=4104),
               dict(kind=3, xs=a, x=4104), dict(taps=128, n=1 << 18)):
        assert product(**kw) == -1, kw
        assert b"glv_mxfp4_product" in lib.glv_last_error()
    assert product(rows=0, x=None, y=None, work=None) == 0 and product(n=0, wc=None) == 0
    assert lib.glv_mxfp4_product(None, None, 0, None) == lib.glv_mxfp4_quantize(None, None) == lib.glv_block_norm(None, None) == -1

    def size(*shape):
        return lib.glv_mxfp4_product_workspace(_lib.mxfp4_product_args(0, 0, 0, 0, 0, 0, 0, 0, *shape, 0, 0, 0))

    assert size(0, 1, 64, 4096, 8, 1, 1) > 0 and size(3, 1, 64, 4096, 8, 1, 1) == 0
    assert size(9, 1, 4, 32, 8, 1, 1) == -1 and size(0, 1, 4, 0, 8, 1, 1) == -1 and size(0, 1 << 13, 1 << 13, 32, 8, 1, 1) == -1
    assert size(0, 1, 4, 32, 8, 1, 0) == -1 and size(0, 1, 4, 32, 8, 0, 1) == -1

    def norm(u=a, kind=0, batch=1, rows=4, cols=32, vkind=0, post=1, pw=None, eps=1e-5, gate=None, gate_col=1, scale=None, res=None,
             pre=0, y=a, z=None):
        return lib.glv_block_norm(_lib.block_norm_args(
            u or 0, gate or 0, res or 0, pw or 0, 0, scale or 0, 0, 0, y or 0, z or 0, rows * cols, cols, 0, 0, 0, 0, kind, batch, rows,
            cols, vkind, post, pre, gate_col, eps, eps, 1.0), None)

    for kw in (dict(u=None), dict(y=None), dict(pre=2), dict(kind=3), dict(vkind=1), dict(post=3), dict(pre=-1), dict(eps=-1.0),
               dict(eps=float("nan")), dict(gate_col=2), dict(cols=0), dict(cols=32769), dict(rows=-1), dict(batch=1 << 13, rows=1 << 13),
               dict(u=odd), dict(gate=odd), dict(res=odd), dict(pw=4098), dict(scale=odd)):
        assert norm(**kw) == -1, kw
        assert b"glv_block_norm" in lib.glv_last_error()
    assert norm(rows=0, u=None, y=None) == 0

    # more threads than one launch can hold
    kw = dict(rows=1 << 24, cols=32768)
    assert quantize(**kw) == norm(**kw) == dequantize(a, a, kw["rows"], kw["cols"], 0, a) == -1
    assert b"too large for one call" in lib.glv_last_error()
    for n in (1 << 16, 1 << 18):
        assert product(kind=3, xs=a, rows=1 << 24, n=n) == -1 and b"too large for one call" in lib.glv_last_error()


@gpu
def test_sizes_that_do_not_fit_the_librarys_ints_are_refused():
    """Nothing here is allocated at its size: the rows are one row, seen many times."""
    one = torch.ones(1, 1, 8, device="cuda", dtype=torch.float16)
    w, wc = mxfp4_quantize(one[0]), mxfp4_quantize(one.expand(1, 3, 8))
    long, deep = one[0].expand((1 << 32) + 3, 8), one[None].expand(1 << 17, 1 << 16, 3, 8)
    for call in (lambda: mxfp4_quantize(long), lambda: mxfp4_linear(long, w), lambda: mxfp4_conv1d(long, wc),
                 lambda: block_norm(long, post=Norm()), lambda: mxfp4_quantize(long[None]), lambda: mxfp4_linear(deep, w)):
        with pytest.raises(ValueError, match="larger than|hold more than"):
            call()
    with pytest.raises(ValueError, match="dilation"):
        mxfp4_conv1d(one, wc, dilation=(1 << 32) + 1)
    # 2^32 + 2^16 rows in all, which an int would take for 2^16
    with pytest.raises(tts_amd._lib.GlvError, match="4295032832 rows"):
        mxfp4_linear(one.expand(1 << 16, (1 << 16) + 1, 8), w)


@gpu
def test_refusals_on_the_device():
    x = torch.ones(3, 40, device="cuda")
    w, wc = mxfp4_quantize(torch.ones(5, 40, device="cuda")), mxfp4_quantize(torch.ones(5, 3, 40, device="cuda"))
    grad = torch.ones(3, 40, device="cuda", requires_grad=True)
    for call in (lambda: mxfp4_quantize(grad), lambda: mxfp4_linear(grad, w), lambda: block_norm(grad, post=Norm()),
                 lambda: block_norm(x, residual=grad), lambda: block_norm(x, gate=grad),
                 lambda: block_norm(x, post=Norm(torch.ones(40, device="cuda", requires_grad=True)))):
        with pytest.raises(ValueError, match="requires a gradient"):
            call()
    with torch.no_grad():
        assert mxfp4_linear(grad, w).shape == (3, 5)
    bad = [
        (lambda: mxfp4_linear([1.0], w), "x must be a tensor"),
        (lambda: mxfp4_conv1d([1.0], wc), "x must be a tensor"),
        (lambda: block_norm(x, gate=[1.0]), "gate must be a tensor"),
        (lambda: block_norm(x, residual=1.0), "residual must be a tensor"),
        (lambda: mxfp4_linear(x, w, 1.0), "bias must be a tensor"),
        (lambda: mxfp4_linear(x[:, :39], w), "39 columns"),
        (lambda: mxfp4_linear(mxfp4_quantize(x[:, :39]), w), "39 columns"),
        (lambda: mxfp4_linear(x, w, torch.ones(6, device="cuda")), "bias must have shape"),
        (lambda: mxfp4_linear(x, w, torch.ones(5)), "bias must be on a ROCm GPU"),
        (lambda: mxfp4_linear(x, w, activation="gelu"), "activation"),
        (lambda: mxfp4_linear(x, w, out_dtype=torch.float64), "out_dtype"),
        (lambda: mxfp4_linear(x, packed((5, 40))), "weight must be on a ROCm GPU"),
        (lambda: mxfp4_linear(packed((3, 40)), w), "x must be on a ROCm GPU"),
        (lambda: mxfp4_linear(torch.ones((), device="cuda"), w), "at least one dimension"),
        (lambda: mxfp4_conv1d(x[0], wc), r"\(B, T, C\)"),
        (lambda: mxfp4_conv1d(x[None, None], wc), r"\(B, T, C\)"),
        (lambda: mxfp4_conv1d(x, wc, dilation=0), "dilation"),
        (lambda: mxfp4_conv1d(x, wc, dilation=1.5), "dilation"),
        (lambda: mxfp4_quantize(torch.ones((), device="cuda")), "last dimension"),
        (lambda: mxfp4_quantize(torch.ones(3, 0, device="cuda")), "last dimension"),
        (lambda: block_norm(x, post=1), "post must be a Norm"),
        (lambda: block_norm(x, post=Norm(torch.ones(39, device="cuda"))), "post.weight must have shape"),
        (lambda: block_norm(x, post=Norm(torch.ones(40, device="cuda").half())), "must all be"),
        (lambda: block_norm(x.half(), post=Norm(torch.ones(40, device="cuda").half()), scale=torch.ones(40, device="cuda")), "must all be"),
        (lambda: block_norm(x, gate=torch.ones(4, 40, device="cuda")), "does not broadcast"),
        (lambda: block_norm(x, gate=torch.ones(2, 3, 40, device="cuda")), "does not broadcast"),
        (lambda: block_norm(x, gate=x.half()), "gate must be"),
        (lambda: block_norm(x, residual=x[:2]), "residual must be"),
        (lambda: block_norm(x, residual=x.half()), "residual must be"),
        (lambda: block_norm(x, scale=torch.ones(1, device="cuda")), "scale must have shape"),
    ]
    for call, message in bad:
        with pytest.raises(ValueError, match=message):
            call()
    with pytest.raises(tts_amd._lib.GlvError, match="cols 32769"):
        block_norm(torch.ones(1, 32769, device="cuda"), post=Norm())


def test_forward_mode_derivatives_are_refused():
    """A dual tensor has requires_grad False and memory of its own; the tangent would be lost without a word."""
    import torch.autograd.forward_ad as forward_ad
    calls = (lambda x: mxfp4_quantize(x), lambda x: block_norm(x, post=Norm()))
    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.ones(3, 40), torch.ones(3, 40))
        for call in calls:
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(ValueError, match="forward-mode derivative"):
                    call(x)
            with pytest.raises(ValueError, match="ROCm GPU"):  # one without a tangent gets as far as any other
                call(torch.ones(3, 40))
    for call in calls:
        with pytest.raises((ValueError, RuntimeError), match="forward-mode derivative"):
            torch.func.jvp(call, (torch.ones(3, 40),), (torch.ones(3, 40),))


def test_tracing_is_refused():
    for call in (lambda x: mxfp4_quantize(x).dequantize(), lambda x: packed((3, 40)).dequantize(), lambda x: block_norm(x, post=Norm())):
        with pytest.raises(ValueError, match="traced"):
            torch.jit.trace(call, torch.ones(3, 40), check_trace=False)


@gpu
def test_derivatives_and_traces_of_products_are_refused():
    import torch.autograd.forward_ad as forward_ad
    x, bias = torch.ones(3, 40, device="cuda"), torch.ones(5, device="cuda")
    w, wc = mxfp4_quantize(torch.ones(5, 40, device="cuda")), mxfp4_quantize(torch.ones(5, 3, 40, device="cuda"))
    xq = mxfp4_quantize(x)
    with forward_ad.dual_level():
        dual, dual_bias = forward_ad.make_dual(x, x), forward_ad.make_dual(bias, bias)
        for call in (lambda: mxfp4_linear(dual, w), lambda: mxfp4_conv1d(dual, wc), lambda: mxfp4_linear(x, w, dual_bias),
                     lambda: mxfp4_linear(xq, w, dual_bias), lambda: block_norm(x, gate=dual), lambda: block_norm(x, residual=dual),
                     lambda: block_norm(x, post=Norm(dual[0])), lambda: block_norm(x, scale=dual[0])):
            with pytest.raises(ValueError, match="forward-mode derivative"):
                call()
        assert mxfp4_linear(x, w).shape == (3, 5)
    for call in (lambda x: mxfp4_linear(x, w), lambda x: mxfp4_conv1d(x, wc), lambda x: mxfp4_linear(xq, w, x[0, :5])):
        with pytest.raises(ValueError, match="traced"):
            torch.jit.trace(call, x, check_trace=False)


def negated(*shape, device="cpu"):
    """Values whose memory holds their opposites: the imaginary part of a conjugated tensor."""
    v = torch.arange(1.0, 1 + int(np.prod(shape)), device=device).reshape(shape)
    x = torch.complex(torch.zeros_like(v), -v).conj().imag
    assert x.is_neg() and torch.equal(x, v)
    return x


@pytest.mark.parametrize("shape", [(5, 3), (5, 1), (1, 1), (2, 4, 1), (1,), (4,), (2, 2, 2, 1), (2, 2, 2, 3)])
def test_pending_negations_are_resolved_on_the_way(shape):
    from tts_amd import blocks
    x = negated(*shape)
    t, batch, rows, batch_stride, row_stride = blocks._rows(x, x.shape)
    assert not t.is_neg() and torch.equal(t.as_strided((batch, rows, shape[-1]), (batch_stride, row_stride, 1)), x.reshape(batch, rows, -1))
    g, strides = blocks._broadcast(negated(4, 1), torch.Size((2, 4, 3)), 2, 4, 3)
    assert not g.is_neg() and torch.equal(g.as_strided((2, 4, 3), strides)[0, :, 2], torch.arange(1.0, 5))


@gpu
def test_pending_negations_reach_the_kernels_resolved():
    for n in (1, 3):
        x, w = negated(4, n, device="cuda"), mxfp4_quantize(torch.ones(n, n, device="cuda"))
        v = negated(n, device="cuda")
        plain, pv = x.resolve_neg(), v.resolve_neg()
        for got, want in ((mxfp4_quantize(x).dequantize(), mxfp4_quantize(plain).dequantize()), (mxfp4_linear(x, w, v), mxfp4_linear(plain, w, pv)),
                          (block_norm(x, gate=x, residual=x, scale=v), block_norm(plain, gate=plain, residual=plain, scale=pv)),
                          (block_norm(x, post=Norm(v, v), gate=x[:, :1]), block_norm(plain, post=Norm(pv, pv), gate=plain[:, :1]))):
            assert torch.equal(got, want) and not got.is_neg()
        assert (mxfp4_linear(x, w) > 0).all()


def test_workspace_refuses_what_the_product_refuses():
    from tts_amd import _lib
    lib = _lib.load()
    a = 4096  # never looked at: every call below is refused first
    shapes = [  # (x_type, batch, rows, cols, n_out, taps, dilation)
        (0, 1, 64, 4096, (1 << 18) + 1, 1, 1), (0, 1, 64, 4096, 8, 1 << 14, 1), (0, 1, 4, 32, 8, 2, (1 << 24) + 1), (0, 1, 4, 32, 1 << 18, 128, 1),
        (1, 1, 64, 4096, -1, 1, 1), (4, 1, 4, 32, 8, 1, 1), (0, -1, 4, 32, 8, 1, 1), (0, 1, -4, 32, 8, 1, 1), (0, 1, 4, 1 << 19, 8, 1, 1),
        (0, 1 << 12, 1 << 13, 32, 8, 1, 1), (2, 1, 1 << 24, 1 << 18, 8, 1, 1), (3, 1, 1 << 24, 32, 1 << 18, 1, 1), (0, 1, 1 << 24, 32, 1 << 18, 1, 1)]
    for shape in shapes:
        args = _lib.mxfp4_product_args(a, a, a, a, 0, a, 0, shape[3], *shape, 0, 0, 0)
        assert lib.glv_mxfp4_product_workspace(args) == -1, shape
        assert b"glv_mxfp4_product_workspace" in lib.glv_last_error()
        assert lib.glv_mxfp4_product(args, a, 1 << 62, None) == -1, shape
    assert lib.glv_mxfp4_product_workspace(None) == -1
    for shape in ((0, 1, 0, 32, 8, 1, 1), (0, 1, 4, 32, 0, 1, 1), (3, 1, 1 << 24, 1 << 18, 1 << 7, 1, 1), (0, 1, 1 << 24, 32, 127 << 7, 1, 1),
                  (0, 1, 64, 1 << 17, 1 << 18, 2, 1 << 24), (0, 1, 4, 32, 8, 1, (1 << 31) - 1)):
        args = _lib.mxfp4_product_args(0, 0, 0, 0, 0, 0, 0, shape[3], *shape, 0, 0, 0)
        assert lib.glv_mxfp4_product_workspace(args) >= 0, shape


@gpu
def test_a_large_refused_product_allocates_nothing():
    one, w = torch.ones(1, 1, 8, device="cuda", dtype=torch.float16), mxfp4_quantize(torch.ones(64, 8, device="cuda"))
    wide = MXFP4Tensor(((1 << 18) + 1, 8), torch.zeros(((1 << 18) + 1) * 68, dtype=torch.uint8, device="cuda"))
    before, _ = torch.cuda.memory_allocated(), torch.cuda.reset_peak_memory_stats()
    for call in (lambda: mxfp4_linear(one.expand(1 << 13, (1 << 12) + 1, 8), w), lambda: mxfp4_linear(one[0].expand(1 << 13, 8), wide)):
        with pytest.raises(tts_amd._lib.GlvError, match="outside"):
            call()
        assert torch.cuda.max_memory_allocated() == before


@gpu
def test_an_earlier_error_of_another_call_is_not_this_ones():
    """An error that its caller has dealt with (here: a device that does not exist) waits in the runtime."""
    from tts_amd import _lib
    lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream
    x, w, out = torch.ones(40, 64, device="cuda"), torch.ones(8, 64, device="cuda"), torch.empty(40, 64, device="cuda")
    q, y = mxfp4_quantize(w), torch.empty(40, 8, device="cuda")
    again = MXFP4Tensor((8, 64), torch.zeros_like(q.data))
    calls = [
        lambda: lib.glv_mxfp4_quantize(_lib.mxfp4_array(w.data_ptr(), *again._pointers(), 0, 64, 0, 1, 8, 64), stream),
        lambda: lib.glv_mxfp4_dequantize(_lib.mxfp4_array(out.data_ptr(), *q._pointers(), 0, 0, 0, 1, 8, 64), stream),
        lambda: lib.glv_mxfp4_product(_lib.mxfp4_product_args(x.data_ptr(), 0, *q._pointers(), 0, y.data_ptr(), 0, 64, 0, 1, 40, 64, 8,
                                                              1, 1, 0, 0, 0), None, 0, stream),
        lambda: lib.glv_block_norm(_lib.block_norm_args(x.data_ptr(), 0, 0, 0, 0, 0, 0, 0, out.data_ptr(), 0, 0, 64, 0, 0, 0, 0, 0, 1, 40,
                                                        64, 0, 2, 0, 1, 0.0, 0.0, 1.0), stream)]
    torch.cuda.synchronize()
    rcs = []
    for call in calls:
        refused = lib.hipSetDevice(1000)
        rcs.append((refused != 0, call()))
        lib.hipGetLastError()
    torch.cuda.synchronize()
    assert rcs == [(True, 0)] * 4, lib.glv_last_error()
    assert torch.equal(again.data, q.data) and (y == 64).all() and (out == 1).all()


def test_inline_assembly_names_the_registers_that_it_writes():
    """Every statement that writes M0 lists it, so that the compiler keeps its own uses of it away."""
    import re
    here = os.path.join(os.path.dirname(os.path.abspath(tts_amd.__file__)), "csrc")
    found = 0
    for name in ("mxfp4.hip", "block_norm.hip", "lowp.h"):
        with open(os.path.join(here, name)) as f:
            statements = re.findall(r"asm volatile\((.*?)\);", f.read(), re.S)
        for statement in (s for s in statements if "s_mov_b32 m0" in s):
            found += 1
            assert '"m0"' in statement.rsplit(":", 1)[1], (name, statement)
    assert found == 4


# shapes whose activations the tiled convolutions quantise themselves: of up to 128 columns of y and of more, channels
# that end inside a block, entries of one row and of many
@gpu
@pytest.mark.parametrize("batch,time,c,n,taps,dilation", [
    (330, 100, 8, 80, 5, 7), (65, 505, 300, 128, 3, 1), (25001, 2, 40, 33, 7, 2), (72, 700, 130, 200, 3, 2), (70, 705, 256, 250, 4, 5),
    (50001, 1, 384, 256, 1, 1), (64, 865, 256, 256, 3, 1), (71, 700, 101, 140, 2, 9)])
@pytest.mark.parametrize("dtype", TYPES)
def test_conv1d_quantising_in_its_tiles(dtype, batch, time, c, n, taps, dilation):
    rng = np.random.default_rng(batch + time + c + n)
    x, w, bias = draw(rng, batch, time, c, dtype=dtype), draw(rng, n, taps, c, scale=(taps * c) ** -0.5), draw(rng, n)
    x[batch // 2] = 0
    q = mxfp4_quantize(w)
    rows, wv = gathered(mxfp4_quantize(x).dequantize().double(), taps, dilation), q.dequantize().double().reshape(n, -1)
    y = mxfp4_conv1d(x, q, bias, dilation=dilation, activation="relu")
    check_product_on_device(y, rows, wv, bias, True)
    # the same rows between others, and 2 bytes off any alignment
    wide = torch.full((batch, time + 3, c + 5), float("nan"), dtype=dtype, device="cuda")
    wide[:, 2:2 + time, 1:1 + c] = x
    assert torch.equal(mxfp4_conv1d(wide[:, 2:2 + time, 1:1 + c], q, bias, dilation=dilation, activation="relu"), y)


@gpu
@pytest.mark.parametrize("m,n,k", [(2100, 1000, 100), (4000, 1000, 1), (2100, 1000, 300), (1900, 1100, 500)])
@pytest.mark.parametrize("dtype", TYPES)
def test_two_teams_share_out_one_group_and_odd_ones(dtype, m, n, k):
    rng = np.random.default_rng(m + n + k)
    x, w, bias = draw(rng, m, k, dtype=dtype), draw(rng, n, k, scale=k ** -0.5), draw(rng, n)
    q, xq = mxfp4_quantize(w), mxfp4_quantize(x)
    xv, wv = xq.dequantize().double(), q.dequantize().double()
    check_product_on_device(mxfp4_linear(x, q, bias), xv, wv, bias, False)
    check_product_on_device(mxfp4_linear(xq, q, bias, activation="relu", out_dtype=dtype), xv, wv, bias, True)


@gpu
@pytest.mark.parametrize("c", [12280, 12289, 16385, 20001, 32761])
@pytest.mark.parametrize("dtype", TYPES)
def test_block_norm_of_wide_ragged_rows(dtype, c):
    rng = np.random.default_rng(c)
    u, gate, residual = (draw(rng, 1, 3, c, dtype=dtype) for _ in range(3))
    scale = torch.from_numpy(rng.normal(0.5, 0.1, c)).to(dtype).cuda()
    for kind in ("layer", "rms"):
        post, pre = norm_vectors(rng, kind, c, dtype), norm_vectors(rng, kind, c, dtype)
        check_block_norm(u, post, gate, scale, residual, pre, block_norm(u, post=post, gate=gate, scale=scale, residual=residual, pre=pre))


def freed(t):
    t.untyped_storage().resize_(0)
    return t


def test_a_tensor_without_memory_is_not_none():
    from tts_amd import blocks
    with pytest.raises(ValueError, match="gate has no memory"):
        blocks._pointer(freed(torch.ones(3, 4)), "gate")
    assert blocks._pointer(torch.ones(0, 4), "gate") == 0
    q = packed((5, 40))
    freed(q.data)
    with pytest.raises(ValueError, match="no memory"):
        q._pointers()
    assert packed((0, 40))._pointers() == (0, 0)


@gpu
def test_freed_arguments_are_refused_by_name():
    def one(*shape):
        return torch.ones(shape, device="cuda")

    x, w = one(3, 40), mxfp4_quantize(one(5, 40))
    for call, name in ((lambda: block_norm(x, gate=freed(one(3, 40))), "gate"), (lambda: block_norm(x, gate=freed(one(3, 1))), "gate"),
                       (lambda: block_norm(x, residual=freed(one(3, 40))), "residual"), (lambda: block_norm(x, scale=freed(one(40))), "scale"),
                       (lambda: block_norm(x, post=Norm(freed(one(40)))), "post.weight"), (lambda: block_norm(x, pre=Norm(None, freed(one(40)))), "pre.bias"),
                       (lambda: mxfp4_linear(x, w, freed(one(5))), "bias")):
        with pytest.raises(ValueError, match=f"{name} has no memory"):
            call()
    for call in (lambda: block_norm(freed(one(3, 40)), post=Norm()), lambda: mxfp4_linear(freed(one(3, 40)), w), lambda: mxfp4_quantize(freed(one(3, 40)))):
        with pytest.raises(tts_amd._lib.GlvError, match="null argument"):
            call()
    freed(w.data)
    for call in (lambda: mxfp4_linear(x, w), lambda: w.dequantize()):
        with pytest.raises(ValueError, match="MXFP4 tensor has no memory"):
            call()
