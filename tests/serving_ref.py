"""Packed attention, the paged cache and e4m3 with power-of-two scales in 64 bits, from their
definitions, and the bounds the 16-bit kernels are held to."""
import numpy as np

from frame_public_b200 import capi
from oracle import frame_oracle as fo

UNIT = {capi.BF16: 2.0 ** -8, capi.F16: 2.0 ** -11}   # half a step of the storage type, relative


def store(x, dt):
    """fp32 numbers as 16-bit storage."""
    return fo.from_accum(np.ascontiguousarray(x, dtype=np.float32), dt)


def load(x, dt):
    return fo.to_accum(x, dt).astype(np.float64)


def offsets(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


# ---- e4m3 ----------------------------------------------------------------------------------------
def e4m3_values():
    out = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        out[c] = (np.nan if c & 127 == 127 else v) * (-1 if c & 128 else 1)
    return out


E4M3 = e4m3_values()


def quantise(x):
    """x [..., d] -> (codes uint8, scale bytes uint8 [...])."""
    x = np.asarray(x, dtype=np.float64)
    finite = np.isfinite(x).all(-1)
    clean = np.where(finite[..., None], x, 0.0)
    amax = np.abs(clean).max(-1)
    scales = 2.0 ** np.arange(-126, 128)
    e = np.searchsorted(448.0 * scales, amax) - 126           # the smallest with amax <= 448 * 2^e
    y = clean / (2.0 ** e)[..., None]
    grid = E4M3[:127]
    at = np.clip(np.searchsorted(grid, np.abs(y)), 1, 126)
    low, high = np.abs(y) - grid[at - 1], grid[at] - np.abs(y)
    code = np.where((low < high) | ((low == high) & ((at - 1) % 2 == 0)), at - 1, at)
    code = (code + 128 * np.signbit(y)).astype(np.uint8)
    code[~finite] = 0
    return code, np.where(finite, e + 127, 255).astype(np.uint8)


def dequantise(codes, exps):
    scale = np.where(exps == 255, np.nan, 2.0 ** (exps.astype(np.float64) - 127))
    return E4M3[codes] * scale[..., None]


# ---- attention -----------------------------------------------------------------------------------
def attention(q, k, v, scale, causal):
    """One sequence: q [lq, h, d], k and v [lk, hk, d] in 64 bits.
    Returns o, lse, and per output the sum of p * |v| and the largest scale * sum |q k|."""
    lq, h, d = q.shape
    lk, hk = k.shape[0], k.shape[1]
    o, lse = np.zeros((lq, h, d)), np.full((lq, h), -np.inf)
    mag, arg = np.zeros((lq, h, d)), np.zeros((lq, h))
    seen = np.ones((lq, lk), dtype=bool)
    if causal:
        seen = np.arange(lk)[None, :] <= np.arange(lq)[:, None] + lk - lq
    some = seen.any(-1)
    for i in range(h):
        kk, vv = k[:, i // (h // hk)], v[:, i // (h // hk)]
        if lk == 0:
            continue
        s = np.where(seen, q[:, i] @ kk.T * scale, -np.inf)
        top = np.where(some, s.max(-1), 0.0)
        p = np.exp(s - top[:, None])
        total = np.where(some, p.sum(-1), 1.0)
        p = p / total[:, None]
        o[:, i], mag[:, i] = p @ vv, p @ np.abs(vv)
        lse[:, i] = np.where(some, top + np.log(total), -np.inf)
        arg[:, i] = np.where(seen, np.abs(q[:, i]) @ np.abs(kk).T * scale, 0.0).max(-1)
    return o, lse, mag, arg


def bounds(o, mag, arg, dt, dim, coded=False):
    """What the kernels may be off by.  A score is an fp32 sum of dim exact products, each addition
    rounded or truncated: dim * 2^-23 of scale * sum |q k|; the exponent's argument and ex2 add about
    8 * 2^-23 of it and 2^-21.  A probability's relative error moves O by at most twice that times
    the sum of p |v| (numerator and row sum).  P is rounded to 16 bits (bfloat16 where the values are
    e4m3), O once more; fp32 sums over the keys and the joining of parts add a few 2^-20."""
    delta = (dim + 8) * 2.0 ** -23 * arg + 2.0 ** -20
    unit_p = UNIT[capi.BF16] if coded else UNIT[dt]
    return (unit_p + 2 * delta[..., None]) * mag + UNIT[dt] * np.abs(o) + 2.0 ** -24, delta + 2.0 ** -21


class Pages:
    """A cache on the host: `lens` tokens per sequence in pages of random order."""

    def __init__(self, rng, lens, page, kv_heads, dim, dt, coded, head_major, spare=2, fill=None):
        per = [-(-n // page) for n in lens]
        self.page, self.coded, self.dt, self.head_major = page, coded, dt, head_major
        self.pages = sum(per) + spare
        self.table = np.full((len(lens), max(per + [1])), -1, dtype=np.int32)   # unused entries are never read
        order = rng.permutation(self.pages).astype(np.int32)
        at = 0
        for i, n in enumerate(per):
            self.table[i, :n] = order[at:at + n]
            at += n
        shape = (self.pages, kv_heads, page) if head_major else (self.pages, page, kv_heads)
        kind = np.uint8 if coded else np.uint16
        empty = fill if fill is not None else 0
        self.k, self.v = (np.full(shape + (dim,), empty, dtype=kind) for _ in range(2))
        self.ks, self.vs = (np.full(shape, 255, dtype=np.uint8) for _ in range(2)) if coded else (None, None)
        self.lens, self.kv_heads, self.dim = lens, kv_heads, dim

    def _at(self, arr, seq, pos):
        ids, tok = self.table[seq, pos // self.page], pos % self.page
        return (ids, slice(None), tok) if self.head_major else (ids, tok)

    def put(self, seq, first, k, v):
        """Rows k, v [n, kv_heads, dim] of storage numbers from token `first` on."""
        for x, arr, sc in ((k, self.k, self.ks), (v, self.v, self.vs)):
            pos = np.arange(first, first + len(x))
            if len(x) == 0:
                continue
            if self.coded:
                codes, exps = quantise(load(x, self.dt))
                arr[self._at(arr, seq, pos)] = codes
                sc[self._at(sc, seq, pos)] = exps
            else:
                arr[self._at(arr, seq, pos)] = x

    def values(self, seq, n):
        pos = np.arange(n)
        out = []
        for arr, sc in ((self.k, self.ks), (self.v, self.vs)):
            if n == 0:
                out.append(np.zeros((0, self.kv_heads, self.dim)))
                continue
            x = arr[self._at(arr, seq, pos)]
            out.append(dequantise(x, sc[self._at(sc, seq, pos)]) if self.coded else load(x, self.dt))
        return out

    def upload(self):
        """Device copies and the KvCache that describes them."""
        self.dev = {n: capi.DeviceBuffer.from_numpy(getattr(self, n)) for n in ("k", "v", "table")}
        c = capi.KvCache(k=self.dev["k"].ptr, v=self.dev["v"].ptr, pages=self.pages, page_size=self.page,
                         kv_heads=self.kv_heads, head_dim=self.dim, dtype=capi.U8 if self.coded else self.dt)
        st = [s // self.k.itemsize for s in self.k.strides]
        tok, head = (2, 1) if self.head_major else (1, 2)
        c.page_stride, c.token_stride, c.head_stride = st[0], st[tok], st[head]
        if self.coded:
            for n in ("ks", "vs"):
                self.dev[n] = capi.DeviceBuffer.from_numpy(getattr(self, n))
            c.k_scale, c.v_scale = self.dev["ks"].ptr, self.dev["vs"].ptr
            st = self.ks.strides
            c.scale_page_stride, c.scale_token_stride, c.scale_head_stride = st[0], st[tok], st[head]
        self.cache = c
        return c
