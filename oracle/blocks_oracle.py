"""CPU oracle of the MXFP4 and block operators, in float64 numpy from their definitions."""
import numpy as np

MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def mxfp4_encode(x):
    """(rows, cols) float64 -> codes (rows, blocks, 32) 0..15, scale bytes (rows, blocks): the nearest of
    the eight magnitudes by distance, the even code of two at the same distance."""
    x = np.asarray(x, dtype=np.float64)
    rows, cols = x.shape
    v = np.zeros((rows, -(-cols // 32) * 32))
    v[:, :cols] = x
    v = v.reshape(rows, -1, 32)
    codes = np.zeros(v.shape, dtype=np.uint8)
    scales = np.zeros(v.shape[:2], dtype=np.uint8)
    for r in range(v.shape[0]):
        for b in range(v.shape[1]):
            block = v[r, b]
            if not np.isfinite(block).all():
                scales[r, b] = 255
                continue
            top = np.abs(block).max()
            s = max(int(np.frexp(top)[1]) - 1 - 2, -127) if top > 0 else -127
            scales[r, b] = s + 127
            m = np.abs(block) / 2.0 ** s
            d = np.abs(m[:, None] - MAGNITUDES[None, :])
            best = d.min(1, keepdims=True)
            tie = d == best
            # of two codes at the same distance the even one: codes are neighbours, so one is even
            code = np.where(tie.sum(1) > 1, np.argmax(tie & (np.arange(8) % 2 == 0), 1), np.argmax(tie, 1))
            codes[r, b] = code + 8 * (np.signbit(block) & (m > 0))
    return codes, scales


def mxfp4_values(codes, scales, cols):
    v = np.where(codes & 8, -MAGNITUDES[codes & 7], MAGNITUDES[codes & 7])
    scale = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return (v * scale[..., None]).reshape(codes.shape[0], -1)[:, :cols]


def mxfp4_round(x):
    """What a float64 array becomes in MXFP4 along its last dimension."""
    x = np.asarray(x, dtype=np.float64)
    flat = x.reshape(-1, x.shape[-1])
    return mxfp4_values(*mxfp4_encode(flat), x.shape[-1]).reshape(x.shape)


def conv1d(x, w, bias, dilation):
    """(B, T, C) with (N, taps, C) and 'same' zero padding; also the sum of the products' magnitudes."""
    b, t, c = x.shape
    n, taps, _ = w.shape
    left = dilation * (taps - 1) // 2
    y, size = np.zeros((b, t, n)), np.zeros((b, t, n))
    for j in range(taps):
        for i in range(t):
            k = i + j * dilation - left
            if 0 <= k < t:
                y[:, i] += x[:, k] @ w[:, j].T
                size[:, i] += np.abs(x[:, k]) @ np.abs(w[:, j]).T
    if bias is not None:
        y, size = y + bias, size + np.abs(bias)
    return y, size


def norm(x, kind, weight, bias, eps):
    x = np.asarray(x, dtype=np.float64)
    if kind == "layer":
        x = x - x.mean(-1, keepdims=True)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    y = y * (1.0 if weight is None else weight)
    return y + (0.0 if bias is None else bias)
