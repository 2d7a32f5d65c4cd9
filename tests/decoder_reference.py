"""Plain implementations of the decoder-layer operators in 64 bits (CPU), written from their formulas."""
import math

import numpy as np
import torch

STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}   # most a rounding is off, relative


# ------------------------------------------------------------------------------------------------------------ product
def planes_of(levels: torch.Tensor, wbits: int) -> torch.Tensor:
    """Levels [N, K] -> int32 [wbits, N, PAD128(K)/32], element k in bit 31 - k % 32."""
    lv = levels.cpu().numpy().astype(np.uint32)
    N, K = lv.shape
    full = np.zeros((N, (K + 127) // 128 * 128), dtype=np.uint32)
    full[:, :K] = lv
    shift = (31 - np.arange(32)).astype(np.uint32)
    out = np.stack([(((full >> p) & 1).reshape(N, -1, 32) << shift).sum(-1, dtype=np.uint64).astype(np.uint32) for p in range(wbits)])
    return torch.from_numpy(out.view(np.int32))


def activate(y: torch.Tensor, act: str) -> torch.Tensor:
    if act == "relu":
        return torch.where(y > 0, y, torch.where(torch.isnan(y), y, torch.zeros_like(y)))
    if act == "silu":
        return y * torch.sigmoid(y)
    if act == "gelu":
        return 0.5 * y * torch.erfc(-y / math.sqrt(2.0))
    if act == "gelu_tanh":
        return y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
    return y


def linear(x, levels, scale, zero, bias=None, act="none", residual=None):
    """(result in 64 bits, how far fp32 sums may be off it).

    The sums are taken over x * level and over x * zero, or over x * (level - zero): 2 K + 8 additions and products of fp32,
    each off by at most 2^-23 of the magnitudes summed so far (a tensor core truncates where an adder rounds).  The activations'
    slope is below 1.13; their own evaluation is held to 2^-18 of |v| + 1, a few dozen roundings of fp32."""
    xd, w = x.double().cpu(), levels.double().cpu()
    K = xd.shape[1]
    s = scale.double().cpu()
    v = (xd @ (w - zero).t()) * s
    mag = (xd.abs() @ (w + zero).t()) * s.abs()
    if bias is not None:
        v = v + bias.double().cpu()
        mag = mag + bias.double().cpu().abs()
    y = activate(v, act)
    off = 1.13 * (2 * K + 8) * 2.0 ** -23 * mag + (0 if act in ("none", "relu") else 2.0 ** -18 * (v.abs() + 1))
    if residual is not None:
        y = y + residual.double().cpu()
        off = off + 2.0 ** -24 * y.abs()
    return y, off


# ------------------------------------------------------------------------------------------------------------ cache
def quantise(x: np.ndarray, dtype):
    """fp32 rows [..., D] -> levels, step, low as the header states it: every operation rounded to fp32."""
    x = x.astype(np.float32)
    with np.errstate(all="ignore"):
        lo, hi = x.min(-1, keepdims=True), x.max(-1, keepdims=True)
        c = np.float32(1) / np.float32(15)
        step = hi * c - lo * c
        step, low = (torch.from_numpy(np.ascontiguousarray(a)).to(dtype).float().numpy() for a in (step, lo))
        step = np.where(step < np.float32(2.0 ** -126), np.float32(0), step)
        bad = ~(np.isfinite(x).all(-1, keepdims=True) & np.isfinite(step) & np.isfinite(low))
        inverse = np.where(step > 0, np.float32(1) / np.where(step > 0, step, np.float32(1)), np.float32(0))
        level = np.clip(np.rint((x - low) * inverse), 0, 15)
    level = np.where(bad, 0, level).astype(np.uint8)
    nan = np.float32("nan")
    return level, np.where(bad, nan, step), np.where(bad, nan, low)


def normed(x, weight, eps):
    """x [..., D] of a 16-bit type -> fp32, every operation rounded on its own, the mean in 64 bits."""
    y = x.float().cpu().numpy()
    if weight is None:
        return y
    mean = (y.astype(np.float64) ** 2).mean(-1, keepdims=True) + eps
    with np.errstate(all="ignore"):
        r = np.float32(1) / np.sqrt(mean.astype(np.float32))
        return (y * r) * weight.float().cpu().numpy()


def rotated(y, table, pos, interleaved):
    """y [T, H, D] fp32, table [P, rot]; rows whose position lies outside the table become NaN."""
    if table is None:
        return y
    table = table.cpu().numpy()
    rot = table.shape[1]
    half = rot // 2
    known = (pos >= 0) & (pos < table.shape[0])
    row = table[np.where(known, pos, 0)][:, None]
    c, s = row[..., :half], row[..., half:]
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if interleaved else (y[..., :half], y[..., half:rot])
    out = y.copy()
    with np.errstate(all="ignore"):
        first, second = a * c - b * s, b * c + a * s
    if interleaved:
        out[..., 0:rot:2], out[..., 1:rot:2] = first, second
    else:
        out[..., :half], out[..., half:rot] = first, second
    out[~known] = np.float32("nan")
    return out


class Cache:
    """A cache in plain arrays: levels [pages, heads, 2, page, D], params [pages, heads, 2, page, 2] (fp32 values)."""

    def __init__(self, data: torch.Tensor, page: int, D: int, dtype):
        raw = data.cpu().contiguous().view(torch.uint8)
        pages, heads = raw.shape[:2]
        n = page * D // 2
        code = raw[..., :2 * n].reshape(pages, heads, 2, page, D // 2).numpy()
        self.levels = np.empty((pages, heads, 2, page, D), dtype=np.uint8)
        self.levels[..., 0::2], self.levels[..., 1::2] = code & 15, code >> 4
        self.params = raw[..., 2 * n:].contiguous().view(dtype).float().reshape(pages, heads, 2, page, 2).numpy()
        self.page, self.D, self.pages = page, D, pages

    def values(self):
        return self.params[..., :1].astype(np.float64) * self.levels + self.params[..., 1:]


def words_of(levels: np.ndarray, params: np.ndarray, dtype) -> torch.Tensor:
    """The words of a cache from its plain arrays."""
    pages, heads = levels.shape[:2]
    codes = (levels[..., 0::2] | (levels[..., 1::2] << 4)).reshape(pages, heads, -1)
    par = torch.from_numpy(np.ascontiguousarray(params)).to(dtype).reshape(pages, heads, -1).view(torch.uint8)
    return torch.cat((torch.from_numpy(np.ascontiguousarray(codes)), par), -1).contiguous().view(torch.int32)


def attention(q, cache: Cache, cu_q, kv_len, table, scale, causal, window, max_q=None):
    """(out, lse, how far each may be off) in 64 bits; rows behind cu_q[-1] are NaN in out.

    Off: the scores by the fp32 sums of D products (2^-23 of the magnitudes for each of D + 8 roundings), taken through the
    softmax; the weights by one fp16 rounding, 2^-11 of themselves, against levels centred at 8 (so at most 8 steps); and 2^-16
    of the magnitudes for the sums over the keys (pairwise over tiles and splits, the exponential's own 2^-21 included)."""
    T, Hq, D = q.shape
    heads = cache.levels.shape[1]
    G = Hq // heads
    qd = q.double().cpu().numpy()
    out, off = np.full((T, Hq, D), np.nan), np.zeros((T, Hq, D))
    lse, loff = np.full((T, Hq), np.nan), np.zeros((T, Hq))
    vals, step = cache.values(), np.abs(cache.params[..., 0].astype(np.float64))
    for b in range(len(kv_len)):
        n, L = cu_q[b + 1] - cu_q[b], min(kv_len[b], len(table[b]) * cache.page)
        j = np.arange(max(L, 0))
        page, slot = np.asarray(table[b], dtype=np.int64)[j // cache.page], j % cache.page
        real = (page >= 0) & (page < cache.pages)
        page = np.where(real, page, 0)
        for i in range(n if max_q is None else min(n, max_q)):
            t, pos = cu_q[b] + i, kv_len[b] - n + i
            seen = real & (j < kv_len[b])
            if causal:
                seen &= j <= pos
                if window:
                    seen &= j > pos - window
            js = np.nonzero(seen)[0]
            for h in range(Hq):
                if len(js) == 0:
                    out[t, h], lse[t, h] = 0.0, -np.inf
                    continue
                K, V = vals[page[js], h // G, 0, slot[js]], vals[page[js], h // G, 1, slot[js]]
                par = np.abs(cache.params[page[js], h // G, 0, slot[js]].astype(np.float64))
                mag = np.abs(qd[t, h]) @ (15 * par[:, :1] + par[:, 1:]).repeat(D, 1).T
                x = (K @ qd[t, h]) * scale
                m = x.max()
                p = np.exp(x - m)
                l = p.sum()
                p /= l
                out[t, h], lse[t, h] = p @ V, m + np.log(l)
                ds = (abs(scale) * mag * (D + 8) * 2.0 ** -23 + np.abs(x) * 2.0 ** -22).max() + 2.0 ** -21
                size = p @ (8 * step[page[js], h // G, 1, slot[js]][:, None] + np.abs(V))
                off[t, h] = 2 * ds * size + (2.0 ** -11 + 2.0 ** -16) * size
                loff[t, h] = ds + 2.0 ** -20 * (1 + abs(lse[t, h]))
    return out, lse, off, loff
