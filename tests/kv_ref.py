"""Plain 64-bit forms of the cache append, the paged attention and the sampler, and the element types of the cache."""
import ctypes as C

import numpy as np

import q8mi
from q8mi import hip

U = 2.0 ** -24           # half a step of fp32
HALF_STEP = {"f32": U, "bf16": 2.0 ** -8, "f16": 2.0 ** -11, "e4m3": 2.0 ** -4}
KIND = {"bf16": q8mi.KV_BF16, "f16": q8mi.KV_F16, "e4m3": q8mi.KV_E4M3}


# ---- element types -------------------------------------------------------------------------------------------------
def bf16_bits(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7fff), r)


def bf16_value(bits):
    return (np.asarray(bits, np.uint32) << 16).view(np.float32)


def _e4m3_table():
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c & 128, -v, v)


E4M3 = _e4m3_table()


def e4m3_bits(x):
    """Nearest code, ties to the even one, values beyond +-448 clamped."""
    mag = np.minimum(np.abs(np.asarray(x, np.float64)), 448.0)
    grid = E4M3[:127]
    hi = np.clip(np.searchsorted(grid, np.where(np.isnan(mag), 0, mag)), 1, 126)
    lo = hi - 1
    below, above = mag - grid[lo], grid[hi] - mag
    code = np.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
    code = np.where(np.isnan(mag), 127, code)
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def encode(x, kind):
    """Bits of x (already divided by the scale) in the cache's type."""
    return {"bf16": bf16_bits, "f16": lambda v: np.asarray(v, np.float16).view(np.uint16), "e4m3": e4m3_bits}[kind](x)


def decode(bits, kind):
    if kind == "bf16":
        return bf16_value(bits).astype(np.float64)
    if kind == "f16":
        return np.asarray(bits, np.uint16).view(np.float16).astype(np.float64)
    return E4M3[np.asarray(bits, np.uint8)]


def act_bits(x, act):
    return bf16_bits(x) if act == "bf16" else np.ascontiguousarray(x, np.float32)


def act_value(a, act):
    return (bf16_value(a) if act == "bf16" else np.asarray(a, np.float32)).astype(np.float64)


# ---- a cache on the device -----------------------------------------------------------------------------------------
class Pools:
    """Key and value pools; order "htd" = [page][head][token][dim], "thd" = [page][token][head][dim]; `gap` unused elements
    behind every token row."""

    def __init__(self, kind, pages, page_size, kv_heads, dim, order="htd", gap=0, k_scale=1.0, v_scale=1.0, fill=0xff):
        self.kind, self.pages, self.page_size, self.kv_heads, self.dim = kind, pages, page_size, kv_heads, dim
        self.dtype = np.uint8 if kind == "e4m3" else np.uint16
        row = dim + gap
        self.st, self.sh = (row, page_size * row) if order == "htd" else (kv_heads * row, row)
        self.sp = kv_heads * page_size * row
        self.scales = {"k": k_scale, "v": v_scale}
        self.host = {n: np.full(pages * self.sp, fill if kind == "e4m3" else fill * 257, self.dtype) for n in "kv"}
        self.dev = {n: hip.to_device(self.host[n]) for n in "kv"}
        self.desc = q8mi.KvCache(k=self.dev["k"].ptr, v=self.dev["v"].ptr, dtype=KIND[kind], pages=pages, page_size=page_size,
                                 kv_heads=kv_heads, head_dim=dim, stride_page=self.sp, stride_head=self.sh,
                                 stride_token=self.st, k_scale=k_scale, v_scale=v_scale)

    def at(self, page, token):
        """Element indices [kv_heads, dim] of a token's row."""
        return (page * self.sp + token * self.st + np.arange(self.kv_heads)[:, None] * self.sh + np.arange(self.dim)[None])

    def put(self, name, page, token, bits):
        self.host[name][self.at(page, token)] = bits

    def upload(self):
        for n in "kv":
            self.dev[n].upload(self.host[n])

    def download(self):
        return {n: self.dev[n].download(self.dtype) for n in "kv"}

    @property
    def ref(self):
        return C.byref(self.desc)


# ---- plain forms ---------------------------------------------------------------------------------------------------
def norm_rope(x, weight, eps, freqs, rot, interleaved, positions):
    """x [tokens, heads, dim] -> normalised and rotated, 64 bits."""
    y = x.astype(np.float64)
    if weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * weight.astype(np.float64)
    y = y.copy()
    if rot:
        i = np.arange(rot // 2)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        t = positions.astype(np.float64)[:, None, None] * freqs[None, None]
        ya, yb = y[..., a].copy(), y[..., b].copy()
        y[..., a], y[..., b] = ya * np.cos(t) - yb * np.sin(t), yb * np.cos(t) + ya * np.sin(t)
    return y


def partner_size(x, weight, eps, rot, interleaved):
    """|a| + |b| of each element's pair after the norm: what a rounding error of the rotation is relative to."""
    y = np.abs(norm_rope(x, weight, eps, None, 0, False, None))
    if rot:
        i = np.arange(rot // 2)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        s = y[..., a] + y[..., b]
        y[..., a], y[..., b] = s, s
    return y


def attention(q, k, v, scale, seen):
    """q [heads, dim], k / v [tokens, kv_heads, dim], the first `seen` of them: the output, sum_t p_t |v_t|, and
    max_t scale * sum |q k_t| (what the scores' rounding errors are relative to)."""
    heads, dim = q.shape
    group = heads // k.shape[1]
    out, mag, size = np.zeros((heads, dim)), np.zeros((heads, dim)), np.zeros(heads)
    if seen <= 0:
        return out, mag, size
    for h in range(heads):
        kk, vv = k[:seen, h // group], v[:seen, h // group]
        s = scale * (kk @ q[h])
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h], mag[h] = p @ vv, p @ np.abs(vv)
        size[h] = abs(scale) * (np.abs(kk) @ np.abs(q[h])).max()
    return out, mag, size


def sample(row, temperature, top_k, top_p, min_p, u):
    """The token of one row, weights in whole multiples of 2^-42 and sums in Python's integers."""
    z = np.where(np.isnan(row), -np.inf, row.astype(np.float64))
    if not (z > -np.inf).any():
        return -1
    order = np.argsort(-z, kind="stable")
    order = order[z[order] > -np.inf]
    if not temperature > 0:
        return int(order[0])
    top = z[order[0]]
    with np.errstate(invalid="ignore", over="ignore"):
        p = np.where(z[order] == top, 1.0, np.exp((z[order] - top) / np.float64(temperature)))
    w = [int(x) for x in np.rint(p * 2.0 ** 42)]
    kept = len(order) if top_k <= 0 else min(top_k, len(order))
    if top_p < 1:
        limit, before, n = float(np.float32(top_p)) * float(sum(w[:kept])), 0, 0
        while n < kept and (n == 0 or before < limit):
            before += w[n]
            n += 1
        kept = n
    if min_p > 0:
        kept = min(kept, int((p >= min(float(np.float32(min_p)), 1.0)).sum()))
    ids = np.argsort(order[:kept], kind="stable")
    total = sum(w[:kept])
    u = 0.0 if not u > 0 else min(1.0, float(np.float32(u)))
    target = min(int(np.floor(u * float(total))), total - 1)
    run = 0
    for i in ids:
        run += w[i]
        if run > target:
            return int(order[i])
