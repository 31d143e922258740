"""The rotation, the 8-bit cache and attention over it restated in numpy: 64 bits throughout, except where the operator is
defined by fp32 roundings (scales and codes of the cache), which are made one by one."""
import numpy as np

PAGE = 64
PER127 = np.float32(1.0 / 127.0)


def row_dim(dim):
    return (dim + 63) // 64 * 64


def bf16_bits(x):
    """float32 -> bfloat16 bit patterns, round to nearest even"""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def bf16_values(bits):
    return (np.ascontiguousarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32)


def rope(x, pos, freqs, halves=True, mscale=1.0, weight=None, eps=0.0):
    x = np.asarray(x, np.float64)
    if weight is not None:
        x = x / np.sqrt(np.mean(x * x, -1, keepdims=True) + np.float64(np.float32(eps))) * np.asarray(weight, np.float64)
    rot = 2 * len(freqs)
    t = np.asarray(pos, np.float64)[:, None, None] * np.asarray(freqs, np.float64)
    z = x[..., : rot // 2] + 1j * x[..., rot // 2: rot] if halves else x[..., 0:rot:2] + 1j * x[..., 1:rot:2]
    z = z * np.exp(1j * t) * np.float64(np.float32(mscale))
    y = x.copy()
    if halves:
        y[..., : rot // 2], y[..., rot // 2: rot] = z.real, z.imag
    else:
        y[..., 0:rot:2], y[..., 1:rot:2] = z.real, z.imag
    return y


def places(dim):
    """where in a page's codes of one head the key and the value of (token, dimension) lie"""
    dp = row_dim(dim)
    t, d = np.arange(PAGE)[:, None], np.arange(dim)[None, :]
    key = (((t // 16 * (dp // 64) + d // 64) * 4 + d % 64 // 16) * 16 + t % 16) * 16 + d % 16
    value = ((d // 16 * 4 + t % 16 // 4) * 16 + d % 16) * 16 + t // 16 * 4 + t % 4
    return key, value


class Cache:
    """codes int [pages, heads, 64, dim] and scales float32 [pages, heads, 64 / block] of keys (0) and values (1)"""

    def __init__(self, n_pages, heads, dim, block):
        self.n_pages, self.heads, self.dim, self.block = n_pages, heads, dim, block
        self.codes = [np.full((n_pages, heads, PAGE, dim), -128, np.int32) for _ in range(2)]  # zeroed bytes
        self.scales = [np.zeros((n_pages, heads, PAGE // block), np.float32) for _ in range(2)]

    def write(self, row_start, kv_len, pages, k, v):
        b = self.block
        for s in range(len(kv_len)):
            n = row_start[s + 1] - row_start[s]
            first = kv_len[s] - n
            for x, codes, scales in ((k, self.codes[0], self.scales[0]), (v, self.codes[1], self.scales[1])):
                x = np.asarray(x, np.float32)
                p = first
                while p < kv_len[s]:
                    e = min(p // b * b + b, kv_len[s])  # one block's new tokens p .. e - 1
                    page, blk, t = pages[s][p // PAGE], p % PAGE // b, p % PAGE
                    rows = x[row_start[s] + p - first: row_start[s] + e - first]  # [tokens, heads, dim]
                    for h in range(self.heads):
                        mine = rows[:, h]
                        with np.errstate(all="ignore"):
                            new = np.float32(np.abs(mine).max() * PER127) if np.isfinite(mine).all() else np.float32(np.nan)
                            old = scales[page, h, blk] if p % b else np.float32(0)
                            scale = np.float32(np.nan) if np.isnan(new) or np.isnan(old) else max(new, old)
                            if p % b and scale > old:
                                f = np.float32(old / scale)
                                held = codes[page, h, blk * b: t].astype(np.float32)
                                codes[page, h, blk * b: t] = np.clip(np.rint(held * f), -127, 127).astype(np.int32)
                            q = np.zeros(mine.shape, np.int32)
                            if scale > 0:
                                q = np.clip(np.rint(mine / scale), -127, 127).astype(np.int32)
                            codes[page, h, t: t + e - p] = q
                            scales[page, h, blk] = scale
                    p = e

    def values(self, pages, count):
        """keys and values [count, heads, dim] of the first tokens behind a row of a page table, in float64; a page that
        there is not gives NaN"""
        got = []
        for codes, scales in zip(self.codes, self.scales):
            out = np.full((count, self.heads, self.dim), np.nan)
            for p in range(0, count, PAGE):
                page = pages[p // PAGE] if p // PAGE < len(pages) else -1
                if 0 <= page < self.n_pages:
                    c = codes[page].astype(np.float64) * np.repeat(scales[page].astype(np.float64), self.block, 1)[..., None]
                    out[p: p + PAGE] = c.transpose(1, 0, 2)[: count - p]
            got.append(out)
        return got

    def read(self, row_start, kv_len, pages, n_rows):
        k, v = np.zeros((n_rows, self.heads, self.dim)), np.zeros((n_rows, self.heads, self.dim))
        for s in range(len(kv_len)):
            a, b = row_start[s], row_start[s + 1]
            if b > a:
                kk, vv = self.values(pages[s], kv_len[s])
                k[a:b], v[a:b] = kk[kv_len[s] - (b - a):], vv[kv_len[s] - (b - a):]
        return k, v

    def memory(self):
        """the bytes of the cache's memory"""
        dp = row_dim(self.dim)
        parts = []
        for codes, place in zip(self.codes, places(self.dim)):
            flat = np.zeros((self.n_pages, self.heads, PAGE * dp), np.uint8)
            flat[..., place.reshape(-1)] = (codes + 128).astype(np.uint8).reshape(self.n_pages, self.heads, -1)
            parts.append(flat.reshape(-1))
        return np.concatenate(parts + [s.reshape(-1).view(np.uint8) for s in self.scales])


def attention(cache, row_start, kv_len, pages, q, scale, window=0, cap=0.0, sinks=None, causal=True, n_rows=None):
    """(outputs float64, a bound on the outputs' error in fp32 with exact operands) for q [n, heads, dim]; rows of no
    sequence are zeros.

    The bound: a score in units of log2 is off by at most d = 2^-24 (4 |z| + 32 S), S the sum of the magnitudes that the
    product adds up -- |scale| log2(e) s_k sum |q| (|code| + 128), 128 being taken out at the start -- each of the at most
    32 partial sums of the matrix instructions rounded once.  A weight is then off by the factor 2^d, and numerator and
    denominator each by that and by 2^-21 for the splitting into halves and their own sums: the output by
    max |v| * 2 (2^d - 1 + 2^-20)."""
    q = np.asarray(q, np.float64)
    n, heads, _ = q.shape
    out, bound = np.zeros_like(q), np.zeros(q.shape[:2] + (1,))
    group = heads // cache.heads
    for s in range(len(kv_len)):
        a, b, total = row_start[s], row_start[s + 1], kv_len[s]
        if b <= a:
            continue
        k, v = cache.values(pages[s], total)
        at, key = np.arange(total - (b - a), total)[:, None], np.arange(total)[None, :]
        seen = np.ones((b - a, total), bool)
        if causal:
            seen &= key <= at
        if window:
            seen &= key > at - window
        for h in range(heads):
            kk, vv = k[:, h // group], v[:, h // group]
            z = q[a:b, h] @ np.where(np.isnan(kk), 0, kk).T * scale
            sizes = np.abs(q[a:b, h]).sum(-1)[:, None] * np.abs(scale) * 1.4427 * 256
            if cap:
                z = cap * np.tanh(z / cap)
            lost = np.isnan(kk).any(-1) | np.isnan(vv).any(-1)
            z = np.where(seen, z, -np.inf)
            top = z.max(-1, initial=-np.inf)
            if sinks is not None:
                top = np.maximum(top, float(sinks[h]))
            base = np.where(np.isinf(top), 0, top)[:, None]
            w = np.exp(z - base)
            den = w.sum(-1) + (np.exp(float(sinks[h]) - base[:, 0]) if sinks is not None else 0)
            num = w @ np.where(np.isnan(vv), 0, vv)
            o = np.where(w.sum(-1)[:, None] > 0, num / np.where(den > 0, den, 1)[:, None], 0)
            o[(seen & lost[None, :]).any(-1)] = np.nan
            out[a:b, h] = o
            if total:
                ks = np.nan_to_num(np.abs(kk)).max() / 127 + 1e-30  # no scale is larger than that of the largest key's block ...
                with np.errstate(all="ignore"):
                    ks = max(ks, np.nanmax(cache.scales[0][[p for p in pages[s][: -(-total // PAGE)] if 0 <= p < cache.n_pages]], initial=0))
                d = 2.0 ** -24 * (4 * np.abs(np.where(seen, z, 0)).max(-1, keepdims=True) * 1.4427 + 32 * ks * sizes)
                vmax = np.where(seen[:, :, None], np.abs(np.nan_to_num(vv))[None], 0).max((1, 2))[:, None] if vv.size * len(z) < 3e7 else np.abs(np.nan_to_num(vv)).max()
                bound[a:b, h] = vmax * 2 * (2 ** d - 1 + 2.0 ** -20)
    return out, bound
