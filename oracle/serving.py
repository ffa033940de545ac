"""Plain 64-bit restatements of the 8-bit rows, their product, the quantised
key/value cache and the attention over it (numpy; test infrastructure only).
The reference has none of these: the definitions are those of
include/memboost_b200.h."""
import numpy as np


def round_half_even(x):
    return np.rint(x)  # numpy's rint: nearest, ties to even


def quantize_rows(x):
    """(codes int8, scales fp32) of the rows (last axis) of x."""
    x = np.asarray(x, np.float64)
    a = np.abs(x).max(-1)
    finite = np.isfinite(x).all(-1)
    with np.errstate(all="ignore"):
        s = (np.where(finite, a, 0.0) / 127.0).astype(np.float32)
        q = round_half_even(np.where(finite[..., None], x, 0.0) / s.astype(np.float64)[..., None])
        q = np.clip(np.where((s > 0)[..., None], q, 0.0), -127, 127)
    return q.astype(np.int8), np.where(finite, s, np.float32(np.nan)).astype(np.float32)


def dequantize_rows(codes, scales):
    """fp32: one rounding of the exact product."""
    return codes.astype(np.float32) * scales[..., None]


def matmul(a_codes, a_scales, b_codes, b_scales, bias=None):
    """(y, |scaled sums|) in 64 bits; the integer sums (below 2^31) are exact."""
    acc = a_codes.astype(np.float64) @ b_codes.astype(np.float64).T
    y = acc * a_scales.astype(np.float64)[:, None] * b_scales.astype(np.float64)[None, :]
    mag = np.abs(y)
    return (y if bias is None else y + np.asarray(bias, np.float64)), mag


def quantize_groups(x):
    """4-bit (codes uint8 [..., D / 2], fp16 [..., D / 32, 2]) of the last
    axis of x."""
    x = np.asarray(x, np.float64)
    g = x.reshape(x.shape[:-1] + (-1, 32))
    lo, hi = g.min(-1), g.max(-1)
    with np.errstate(all="ignore"):
        m = lo.astype(np.float32).astype(np.float16)
        s = ((hi - lo) / 15.0).astype(np.float32).astype(np.float16)
        bad = ~np.isfinite(g).all(-1) | ~np.isfinite(m) | ~np.isfinite(s)
        m, s = (np.where(bad, np.float16(np.nan), v) for v in (m, s))
        q = round_half_even((g - m.astype(np.float64)[..., None])
                            / s.astype(np.float64)[..., None])
        q = np.where((s > 0)[..., None], np.clip(q, 0, 15), 0.0)
    q = q.astype(np.uint8).reshape(x.shape)
    return q[..., 0::2] | (q[..., 1::2] << 4), np.stack((s, m), -1)


def dequantize_groups(codes, groups):
    """64-bit values of 4-bit codes."""
    q = np.stack((codes & 15, codes >> 4), -1).reshape(groups.shape[:-1] + (32,))
    g = groups.astype(np.float64)
    return (g[..., 1:] + g[..., :1] * q).reshape(codes.shape[:-1] + (2 * codes.shape[-1],))


def encode(x, bits):
    return quantize_rows(x) if bits == 8 else quantize_groups(x)


def values(codes, scales, bits):
    if bits == 8:
        return codes.astype(np.float64) * scales.astype(np.float64)[..., None]
    return dequantize_groups(codes, scales)


class Cache:
    """numpy mirror of a QuantizedCache."""

    def __init__(self, cache):
        self.bits, self.page_size, self.pages = cache.bits, cache.page_size, cache.pages
        self.codes = [t.cpu().numpy().copy() for t in (cache.k_codes, cache.v_codes)]
        self.scales = [t.cpu().numpy().copy() for t in (cache.k_scales, cache.v_scales)]

    def write(self, k, v, slots):
        for t, slot in enumerate(slots):  # in order: the last token of a slot stays
            if not 0 <= slot < self.pages * self.page_size:
                continue
            p, i = divmod(int(slot), self.page_size)
            for w, x in ((0, k), (1, v)):
                self.codes[w][p, :, i], self.scales[w][p, :, i] = encode(x[t], self.bits)

    def read(self, which, slots):
        """64-bit [tokens, heads, dim]; 0 for a slot outside."""
        out = []
        for slot in slots:
            inside = 0 <= slot < self.pages * self.page_size
            p, i = divmod(int(slot) if inside else 0, self.page_size)
            x = values(self.codes[which][p, :, i], self.scales[which][p, :, i], self.bits)
            out.append(x if inside else np.zeros_like(x))
        return np.stack(out)

    def tokens(self, which, pages, length, head):
        """64-bit [tokens, dim] of one sequence's head: tokens t < length of
        pages that exist."""
        t = np.arange(min(max(length, 0), len(pages) * self.page_size))
        p = np.asarray(pages, np.int64)[t // self.page_size]
        ok = (p >= 0) & (p < self.pages)
        p, i = p[ok], (t % self.page_size)[ok]
        return values(self.codes[which][p, head, i], self.scales[which][p, head, i], self.bits)


def attention(q, cache, table, lengths, scale):
    """64-bit out [batch, heads, dim] and, for an error bound, four arrays
    [batch, heads, ...]: sum_t p |v| (per channel), the largest
    sum_i |scale q_i k_i| of a token, max |v| times the token count, and the
    largest scale max |q| sum_i |k_i| of a token."""
    q = np.asarray(q, np.float64)
    B, H, D = q.shape
    heads = cache.codes[0].shape[1]
    out, weight = np.zeros((B, H, D)), np.zeros((B, H, D))
    reach, spread, coarse = (np.zeros((B, H, 1)) for _ in range(3))
    for b in range(B):
        for h in range(heads):
            k, v = (cache.tokens(w, table[b], int(lengths[b]), h) for w in (0, 1))
            if len(k) == 0:
                continue
            for j in range(h * (H // heads), (h + 1) * (H // heads)):
                s = (k @ q[b, j]) * scale
                e = np.exp(s - s.max())
                p = e / e.sum()
                out[b, j], weight[b, j] = p @ v, p @ np.abs(v)
                reach[b, j] = (np.abs(k) @ np.abs(q[b, j])).max() * abs(scale)
                spread[b, j] = np.abs(v).max() * len(k)
                coarse[b, j] = np.abs(k).sum(-1).max() * np.abs(q[b, j]).max() * abs(scale)
    return out, weight, reach, spread, coarse
