"""Plain definitions, in 64 bits, of the operators around the grouped matmuls: routing, dispatch, combine, and the NVFP4
format.  Written from the definitions in include/catlass_b200.h; numpy only."""
import numpy as np

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)


def e4m3_values():
    """The 127 finite magnitudes of E4M3 by code 0x00 .. 0x7E."""
    c = np.arange(127)
    return np.where(c < 8, c / 512.0, (1 + (c & 7) / 8.0) * 2.0 ** ((c >> 3) - 7.0))


def nearest_even(x, grid):
    """Index of the value of `grid` (ascending) nearest to x >= 0, a tie to the even index, at most the last."""
    middle = (grid[1:] + grid[:-1]) / 2
    low = np.searchsorted(middle, x, side="left")    # a value on a middle stays below it
    high = np.searchsorted(middle, x, side="right")  # ... goes above it
    return np.where(low == high, low, np.where(low % 2 == 0, low, high))


def route(logits, top_k, sigmoid, bias=None, groups=1, kept=1, top2=False, renormalize=False, scaling=1.0):
    """ids [T, top_k] (-1: none left) and weights, float64."""
    x = np.array(logits, np.float64)
    x[np.isnan(x)] = -np.inf
    t, e = x.shape
    top = x.max(1, keepdims=True)
    with np.errstate(invalid="ignore", over="ignore"):
        if sigmoid:
            s = 1 / (1 + np.exp(-x))
        else:
            d = np.where(x == top, 0.0, x - top)
            s = np.where(np.isneginf(x), 0.0, np.exp(d))
            total = s.sum(1, keepdims=True)
            s = np.divide(s, total, out=np.zeros_like(s), where=total > 0)
    shut = np.isneginf(x)
    key = x if bias is None else s + np.asarray(bias, np.float64)
    key = np.where(shut, -np.inf, key)
    if groups > 1 and kept < groups:
        by = key if bias is not None or not top2 else np.where(shut, -np.inf, s)
        by = np.sort(by.reshape(t, groups, e // groups), 2)[:, :, ::-1]
        g = by[:, :, 0].copy()
        if top2 and by.shape[2] > 1:
            g = np.where(np.isneginf(by[:, :, 1]), g, g + np.where(np.isneginf(by[:, :, 1]), 0, by[:, :, 1]))
        best = np.argsort(-g, axis=1, kind="stable")[:, :kept]
        keep = np.zeros((t, groups), bool)
        np.put_along_axis(keep, best, True, 1)
        key = np.where(np.repeat(keep, e // groups, 1), key, -np.inf)
    ids = np.argsort(-key, axis=1, kind="stable")[:, :top_k]
    chosen = np.take_along_axis(key, ids, 1)
    w = np.where(np.isneginf(chosen), 0.0, np.take_along_axis(s, ids, 1))
    ids = np.where(np.isneginf(chosen), -1, ids)
    if renormalize:
        total = w.sum(1, keepdims=True)
        w = np.divide(w, total, out=np.zeros_like(w), where=total > 0)
    return ids.astype(np.int32), w * scaling


def dispatch(ids, experts, expert_begin=0):
    """(sizes [experts], position like ids, pair of each row)."""
    flat = ids.reshape(-1).astype(np.int64) - expert_begin
    kept = np.flatnonzero((flat >= 0) & (flat < experts))
    pair = kept[np.argsort(flat[kept], kind="stable")]
    position = np.full(flat.shape, -1, np.int32)
    position[pair] = np.arange(pair.size)
    return np.bincount(flat[kept], minlength=experts), position.reshape(ids.shape), pair


def nvfp4_quantize(x, tensor_scale):
    """The definition, step by step in fp32: codes [rows, k] (bit 3 = sign), scale bytes [rows, k/16]."""
    f = np.float32
    x = np.asarray(x, f)
    rows, k = x.shape
    b = x.reshape(rows, k // 16, 16)
    bad = ~np.isfinite(b).all(2)
    b = np.where(bad[:, :, None], f(0), b)
    amax = np.abs(b).max(2)
    ratio = (amax / f(f(6) * f(tensor_scale))).astype(f)
    scale = nearest_even(np.minimum(ratio, f(448)).astype(np.float64), e4m3_values()).astype(np.uint8)
    step = (e4m3_values()[scale].astype(f) * f(tensor_scale)).astype(f)
    with np.errstate(divide="ignore", over="ignore"):
        inverse = (f(1) / step).astype(f)
    dead = (scale == 0) | ~np.isfinite(inverse)
    inverse = np.where(dead, f(0), inverse)
    scale = np.where(dead, 0, scale).astype(np.uint8)
    with np.errstate(over="ignore"):
        y = (b * inverse[:, :, None]).astype(f)
    code = nearest_even(np.abs(y).astype(np.float64), E2M1) + 8 * np.signbit(b)
    code = np.where((dead | bad)[:, :, None], 0, code)
    scale = np.where(bad, 0x7F, scale)
    return code.reshape(rows, k).astype(np.uint8), scale.astype(np.uint8)


def pack(codes):
    return (codes[:, 0::2] | codes[:, 1::2] << 4).astype(np.uint8)


def unpack(q):
    out = np.empty(q.shape[:-1] + (q.shape[-1] * 2,), np.uint8)
    out[..., 0::2] = q & 15
    out[..., 1::2] = q >> 4
    return out


def code_values(codes):
    return np.where(codes & 8, -1.0, 1.0) * E2M1[codes & 7]


def scale_values(scale):
    return np.concatenate([e4m3_values(), [np.nan]])[scale]


def nvfp4_values(codes, scale):
    """What codes [rows, k] and scale bytes [rows, k/16] stand for, without the tensor scale."""
    with np.errstate(invalid="ignore"):
        return code_values(codes) * np.repeat(scale_values(scale), 16, 1)


def tile_scales(scale):
    """[rows, blocks] bytes -> the tiled layout, as a flat byte array; padding bytes 0."""
    rows, blocks = scale.shape
    full = np.zeros((-(-rows // 128) * 128, -(-blocks // 4) * 4), np.uint8)
    full[:rows, :blocks] = scale
    t = full.reshape(full.shape[0] // 128, 4, 32, full.shape[1] // 4, 4)
    return np.ascontiguousarray(t.transpose(0, 3, 2, 1, 4)).reshape(-1)


def untile_scales(tiled, rows, blocks):
    words = -(-blocks // 4)
    t = tiled.reshape(-1, words, 32, 4, 4).transpose(0, 3, 2, 1, 4)
    return t.reshape(-1, words * 4)[:rows, :blocks], t.reshape(-1, words * 4)[:rows, blocks:]
