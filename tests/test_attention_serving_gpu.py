"""Attention of packed prompts and over a paged cache, and the cache's write and read, against plain
64-bit forms (tests/serving_ref.py, which derives the bounds)."""
import numpy as np
import pytest

import serving_ref as ref
from frame_public_b200 import capi

pytestmark = pytest.mark.gpu

BF, FH = capi.BF16, capi.F16
FILL = 0x4049   # what untouched output holds
NAN = {BF: 0x7FC0, FH: 0x7E00}


def upload(x):
    x = np.ascontiguousarray(x)
    return capi.DeviceBuffer.from_numpy(x if x.size else np.zeros(64, dtype=x.dtype))


def params(dt, heads, kv_heads, dim, q_lens, kv_lens, q_rows, causal, scale, ld=None):
    ld = ld or heads * dim
    return capi.AttentionParams(n_seqs=len(q_lens), heads=heads, kv_heads=kv_heads, head_dim=dim, q_rows=q_rows,
                                max_q=max(q_lens, default=0), max_kv=max(kv_lens, default=0), q_token_stride=ld,
                                q_head_stride=dim, o_token_stride=heads * dim, o_head_stride=dim, scale=scale,
                                causal=causal, dtype=dt)


def check_rows(got, lse, q, cu, seqs, dt, dim, scale, causal, coded=False):
    """seqs: (k, v) per sequence in 64 bits; rows outside every sequence hold FILL."""
    inside = np.zeros(len(got), dtype=bool)
    for s, (k, v) in enumerate(seqs):
        rows = slice(cu[s], cu[s + 1])
        inside[rows] = True
        o, l, mag, arg = ref.attention(ref.load(q[rows], dt), k, v, scale, causal)
        tol, tol_l = ref.bounds(o, mag, arg, dt, dim, coded)
        g = ref.load(got[rows], dt)
        assert np.all(np.abs(g - o) <= tol), (s, float(np.max(np.abs(g - o) / tol)))
        empty = np.isneginf(l)
        assert np.array_equal(np.isneginf(lse[rows]), empty)
        assert np.all(np.abs(lse[rows][~empty] - l[~empty]) <= (tol_l + 2.0 ** -22 * np.abs(l))[~empty])
        assert np.all(g[empty] == 0)
    assert np.all(got[~inside] == FILL)


PROMPTS = [
    # dtype, heads, kv_heads, dim, query lengths, key lengths (None: the same), causal
    (BF, 2, 2, 64, [1], None, 1),
    (BF, 4, 2, 64, [128, 0, 1, 129], None, 1),
    (FH, 8, 1, 128, [127, 300, 2], None, 1),
    (BF, 6, 2, 80, [65, 513, 31], None, 1),
    (FH, 3, 3, 16, [40, 257], None, 1),
    (BF, 14, 2, 96, [33, 200], None, 1),
    (BF, 10, 2, 112, [260], None, 0),
    (FH, 4, 4, 64, [5, 77, 0], [300, 12, 40], 1),      # a dense prefix; more queries than keys: empty rows
    (BF, 8, 2, 128, [100, 30], [0, 900], 1),            # no keys at all
    (BF, 8, 2, 128, [3, 200], [129, 64], 0),
    (BF, 16, 16, 64, [512, 512], None, 1),
    (BF, 64, 1, 32, [70], None, 1),
    (FH, 16, 2, 128, [1500], None, 1),
]


@pytest.mark.parametrize("case", range(len(PROMPTS)))
def test_prompt_against_64_bits(case):
    dt, h, hk, d, lq, lk, causal = PROMPTS[case]
    rng = np.random.default_rng(100 + case)
    cu, cuk = ref.offsets(lq), ref.offsets(lk or lq)
    rows, krows, pad = int(cu[-1]) + 3, int(cuk[-1]) + 5, 8
    ld = (h + 2 * hk) * d + pad
    scale = 1.3 / np.sqrt(d)
    fused = ref.store(rng.standard_normal((max(rows, krows), ld)) * 1.5, dt)
    fused[int(cu[-1]):, :h * d] = NAN[dt]             # rows behind the last sequence hold NaN
    fused[int(cuk[-1]):, h * d:] = NAN[dt]
    q = fused[:rows, :h * d].reshape(rows, h, d)
    k = fused[:, h * d:(h + hk) * d].reshape(-1, hk, d)
    v = fused[:, (h + hk) * d:(h + 2 * hk) * d].reshape(-1, hk, d)
    p = params(dt, h, hk, d, lq, lk or lq, rows, causal, scale, ld)
    p.kv_rows, p.k_token_stride, p.k_head_stride, p.v_token_stride, p.v_head_stride = krows, ld, d, ld, d
    dev, out = upload(fused), upload(np.full((rows, h, d), FILL, dtype=np.uint16))
    lse, dcu, dcuk = capi.DeviceBuffer(rows * h * 4), upload(cu), upload(cuk)
    base = dev.ptr.value
    for _ in range(2):
        capi.attention_prompt(p, base, base + h * d * 2, base + (h + hk) * d * 2, out.ptr, dcu.ptr, dcuk.ptr, lse=lse.ptr)
        capi.synchronize()
        assert capi.kernel_status(0) == 0
    seqs = [(ref.load(k[cuk[s]:cuk[s + 1]], dt), ref.load(v[cuk[s]:cuk[s + 1]], dt)) for s in range(len(lq))]
    check_rows(out.download(np.uint16, (rows, h, d)), lse.download(np.float32, (rows, h)).astype(np.float64), q, cu, seqs,
               dt, d, np.float32(scale), causal)


PAGED = [
    # dtype, heads, kv_heads, dim, query lengths, key lengths, page, e4m3, head-major, causal
    (BF, 4, 4, 64, [1, 1, 1, 0], [1, 17, 300, 5], 16, False, False, 1),
    (BF, 8, 1, 128, [1, 1], [700, 33], 32, False, True, 1),
    (FH, 12, 4, 96, [1, 2, 1], [129, 64, 1000], 64, False, True, 1),
    (BF, 8, 2, 128, [1, 1, 1], [16, 2100, 63], 16, True, True, 1),
    (FH, 14, 2, 128, [1, 1], [500, 1], 128, True, False, 1),
    (FH, 4, 2, 64, [1, 1], [31, 440], 8, True, True, 1),
    (BF, 5, 1, 80, [3, 1, 2], [3, 77, 256], 32, True, False, 1),
    (BF, 16, 2, 64, [4, 4], [900, 4], 16, False, True, 1),            # drafted tokens
    (BF, 8, 1, 128, [40, 17], [1200, 17], 16, False, False, 1),
    (BF, 8, 2, 128, [300, 5, 0, 129], [800, 1500, 40, 129], 64, False, True, 1),
    (FH, 8, 2, 128, [130, 64], [640, 64], 32, True, True, 1),
    (BF, 6, 2, 64, [100, 1], [333, 512], 256, True, False, 1),
    (BF, 8, 8, 112, [20, 70], [10, 300], 128, False, True, 1),         # more queries than keys
    (FH, 8, 2, 48, [9, 2], [0, 200], 16, False, True, 0),
    (BF, 32, 4, 128, [33], [9000], 64, False, True, 1),                # few rows over a long cache
    (BF, 32, 4, 128, [1], [20000], 64, True, True, 1),
    (BF, 64, 1, 16, [1, 2], [50, 130], 16, False, True, 1),
    (FH, 8, 1, 128, [40], [5000], 32, True, True, 1),                  # keys cut into parts, e4m3
    (BF, 32, 2, 64, [40, 3], [3000, 2500], 16, True, False, 1),
    (BF, 32, 2, 80, [2, 600], [4000, 1900], 64, False, True, 1),       # one block with parts, others without
    (FH, 24, 2, 96, [3, 1], [2049, 1024], 16, True, True, 0),
]


@pytest.mark.parametrize("case", range(len(PAGED)))
def test_paged_against_64_bits(case):
    dt, h, hk, d, lq, lk, page, coded, head_major, causal = PAGED[case]
    rng = np.random.default_rng(200 + case)
    # stale 16-bit places hold NaN: what lies behind a sequence's last token must not reach it
    pages = ref.Pages(rng, lk, page, hk, d, dt, coded, head_major, fill=0 if coded else NAN[dt])
    gain = np.exp2(rng.integers(-6, 4, (hk, 1)))
    for s, n in enumerate(lk):
        pages.put(s, 0, ref.store(rng.standard_normal((n, hk, d)) * 1.5, dt), ref.store(rng.standard_normal((n, hk, d)) * gain, dt))
    cu = ref.offsets(lq)
    rows = int(cu[-1]) + 2
    q = ref.store(rng.standard_normal((rows, h, d)) * 1.5, dt)
    q[cu[-1]:] = NAN[dt]
    scale = 1.3 / np.sqrt(d)
    p = params(dt, h, hk, d, lq, lk, rows, causal, scale)
    cache = pages.upload()
    size = capi.attention_paged_workspace(p, cache)
    work = upload(np.zeros(max(size, 1), dtype=np.uint8))
    dq, out = upload(q), upload(np.full((rows, h, d), FILL, dtype=np.uint16))
    lse, dcu, dlen = capi.DeviceBuffer(rows * h * 4), upload(cu), upload(np.array(lk, dtype=np.int32))
    first = None
    for _ in range(2):
        capi.attention_paged(p, cache, dq.ptr, out.ptr, dcu.ptr, dlen.ptr, pages.dev["table"].ptr, pages.table.shape[1],
                             work.ptr, size, lse=lse.ptr)
        capi.synchronize()
        assert capi.kernel_status(0) == 0
        got = out.download(np.uint16, (rows, h, d))
        assert first is None or np.array_equal(first, got)
        first = got
    seqs = [tuple(pages.values(s, n)) for s, n in enumerate(lk)]
    check_rows(got, lse.download(np.float32, (rows, h)).astype(np.float64), q, cu, seqs, dt, d, np.float32(scale), causal, coded)


WRITES = [
    # dtype, kv_heads, dim, new, kv lengths (the new ones counted), page, e4m3, head-major
    (BF, 2, 64, [1, 1, 1], [1, 17, 40], 16, True, True),
    (BF, 3, 128, [40, 0, 5], [40, 9, 70], 16, True, False),
    (FH, 1, 80, [33, 2], [50, 2], 8, True, True),
    (FH, 4, 16, [7], [130], 64, True, False),
    (BF, 8, 128, [130, 1], [200, 300], 128, False, True),
    (FH, 2, 112, [20, 3, 4], [20, 30, 4], 32, False, False),
]


@pytest.mark.parametrize("case", range(len(WRITES)))
def test_write_and_read_back_bit_for_bit(case):
    dt, hk, d, new, lens, page, coded, head_major = WRITES[case]
    rng = np.random.default_rng(300 + case)
    pages = ref.Pages(rng, lens, page, hk, d, dt, coded, head_major, fill=7)
    cache = pages.upload()
    cu = ref.offsets(new)
    rows = int(cu[-1]) + 2
    ld = hk * d + 16
    both = [ref.store(rng.standard_normal((rows, ld)) * np.exp2(rng.integers(-30, 12, (rows, 1))), dt) for _ in range(2)]
    flat = both[0].reshape(-1)
    flat[:d] = 0                                                   # a row of zeros
    if coded and rows > 4:
        both[0][1, 3], both[1][2, d - 1] = NAN[dt], 0x7F80 if dt == BF else 0x7C00   # a NaN, an infinity
        both[1][3, :d] = ref.store(np.linspace(-448, 448, d), dt)                     # the largest scale-1 row
        both[1][4, :d] = ref.store(np.full(d, 1.76 * 256), dt)
    k, v = (b[:, :hk * d].reshape(rows, hk, d) for b in both)
    dk, dv, dcu, dlen = upload(both[0]), upload(both[1]), upload(cu), upload(np.array(lens, dtype=np.int32))
    capi.kv_cache_write(cache, dk.ptr, ld, d, dv.ptr, ld, d, dcu.ptr, dlen.ptr, pages.dev["table"].ptr, pages.table.shape[1],
                        len(new), rows, dt)
    capi.synchronize()
    assert capi.kernel_status(0) == 0
    for s, n in enumerate(new):
        pages.put(s, lens[s] - n, k[cu[s]:cu[s + 1]], v[cu[s]:cu[s + 1]])
    for name in ("k", "v") + (("ks", "vs") if coded else ()):
        want = getattr(pages, name)
        assert np.array_equal(pages.dev[name].download(want.dtype, want.shape), want), name   # other places untouched
    # and back: the last tokens are left out of the second sequence on, rows behind stay
    keep = [max(0, n - 2 * (s > 0)) for s, n in enumerate(lens)]
    cuk = ref.offsets(keep)
    rows = int(cuk[-1]) + 3
    outs = [upload(np.full((rows, hk, d), FILL, dtype=np.uint16)) for _ in range(2)]
    dcuk = upload(cuk)
    capi.kv_cache_read(cache, outs[0].ptr, hk * d, d, outs[1].ptr, hk * d, d, dcuk.ptr, pages.dev["table"].ptr,
                       pages.table.shape[1], len(keep), rows, dt)
    capi.synchronize()
    assert capi.kernel_status(0) == 0
    for i, out in enumerate(outs):
        got = out.download(np.uint16, (rows, hk, d))
        assert np.all(got[cuk[-1]:] == FILL)
        for s, n in enumerate(keep):
            with np.errstate(over="ignore"):
                want = ref.store(pages.values(s, n)[i], dt)
            g = got[cuk[s]:cuk[s + 1]]
            nan = np.isnan(ref.load(want, dt))
            assert np.array_equal(np.isnan(ref.load(g, dt)), nan)
            assert np.array_equal(g[~nan], want[~nan])


def test_bad_pages_and_lengths_are_recorded_and_stay_inside():
    dt, hk, d, page = BF, 2, 64, 16
    rng = np.random.default_rng(7)
    pages = ref.Pages(rng, [40], page, hk, d, dt, False, True, fill=7)
    pages.table[0, 1] = 1 << 30
    cache = pages.upload()
    x = upload(ref.store(rng.standard_normal((40, hk, d)), dt))
    cu, lens = upload(np.array([0, 40], dtype=np.int32)), upload(np.array([40], dtype=np.int32))
    capi.kv_cache_write(cache, x.ptr, hk * d, d, x.ptr, hk * d, d, cu.ptr, lens.ptr, pages.dev["table"].ptr, 3, 1, 40, dt)
    capi.synchronize()
    assert capi.kernel_status(0) == 321 and capi.kernel_status(0) == 0
    src = x.download(np.uint16, (40, hk, d))
    got = pages.dev["k"].download(np.uint16, pages.k.shape)
    pages.put(0, 0, src[:16], src[:16])
    pages.table[0, 1] = pages.table[0, 2]
    pages.put(0, 16, src[32:40], src[32:40])          # token 32.. lies in the third page
    assert np.array_equal(got, pages.k)
    # a length past the table: tokens outside are skipped, the others stored; negative places too
    for n in (400, 10):
        far = upload(np.array([n], dtype=np.int32))
        capi.kv_cache_write(cache, x.ptr, hk * d, d, x.ptr, hk * d, d, cu.ptr, far.ptr, pages.dev["table"].ptr, 3, 1, 40, dt)
        capi.synchronize()
        assert capi.kernel_status(0) in (321, 322)
        assert np.array_equal(pages.dev["k"].download(np.uint16, pages.k.shape)[pages.table[0, 0]][:, 10:],
                              pages.k[pages.table[0, 0]][:, 10:]) or n == 10
    p = params(dt, 4, hk, d, [1], [40], 1, 1, 0.1)
    size = capi.attention_paged_workspace(p, cache)
    work, q = upload(np.zeros(max(size, 1), dtype=np.uint8)), upload(ref.store(rng.standard_normal((1, 4, d)), dt))
    out, one = upload(np.zeros((1, 4, d), dtype=np.uint16)), upload(np.array([0, 1], dtype=np.int32))
    capi.attention_paged(p, cache, q.ptr, out.ptr, one.ptr, lens.ptr, pages.dev["table"].ptr, 3, work.ptr, size)
    capi.synchronize()
    assert capi.kernel_status(0) == 321


def test_one_workspace_serves_calls_of_either_kind_and_a_short_max_kv():
    """Decoding and split chunks in turn through one workspace; max_kv only shapes the schedule."""
    dt, h, hk, d, page = BF, 16, 2, 128, 64
    rng = np.random.default_rng(11)
    lens = [3000, 2100]
    pages = ref.Pages(rng, lens, page, hk, d, dt, False, True)
    for s, n in enumerate(lens):
        pages.put(s, 0, ref.store(rng.standard_normal((n, hk, d)), dt), ref.store(rng.standard_normal((n, hk, d)), dt))
    cache, scale = pages.upload(), 1.0 / np.sqrt(d)
    dlen = upload(np.array(lens, dtype=np.int32))
    steps = [[1, 1], [20, 30], [1, 1], [2, 1], [64, 1], [1, 1]]
    calls = []
    for i, step in enumerate(steps):
        cu = ref.offsets(step)
        q = ref.store(rng.standard_normal((int(cu[-1]), h, d)), dt)
        p = params(dt, h, hk, d, step, lens if i % 2 else [1100], len(q), 1, scale)
        calls.append((step, cu, q, p, capi.attention_paged_workspace(p, cache)))
    size = max(c[4] for c in calls)
    work = upload(np.zeros(size, dtype=np.uint8))
    for step, cu, q, p, _ in calls:
        dq, dcu, out = upload(q), upload(cu), upload(np.full(q.shape, FILL, dtype=np.uint16))
        lse = capi.DeviceBuffer(len(q) * h * 4)
        capi.attention_paged(p, cache, dq.ptr, out.ptr, dcu.ptr, dlen.ptr, pages.dev["table"].ptr, pages.table.shape[1],
                             work.ptr, size, lse=lse.ptr)
        capi.synchronize()
        assert capi.kernel_status(0) == 0
        seqs = [tuple(pages.values(s, n)) for s, n in enumerate(lens)]
        check_rows(out.download(np.uint16, q.shape), lse.download(np.float32, q.shape[:2]).astype(np.float64), q, cu, seqs,
                   dt, d, np.float32(scale), 1)


@pytest.mark.parametrize("coded", [False, True], ids=["same", "e4m3"])
def test_a_conversation_prompt_then_chunks_then_single_tokens(coded):
    """Write, attend, write, attend: every token's row equals causal attention over the whole text, with
    the keys and values as the cache holds them."""
    dt, h, hk, d, page = BF, 8, 2, 128, 16
    rng = np.random.default_rng(9)
    steps = [[37, 150], [64, 3], [1, 1], [1, 1], [5, 1], [200, 140]]
    total = [sum(s[i] for s in steps) for i in range(2)]
    pages = ref.Pages(rng, total, page, hk, d, dt, coded, True)
    cache = pages.upload()
    text = [[ref.store(rng.standard_normal((n, heads, d)), dt) for heads in (h, hk, hk)] for n in total]
    done, scale = [0, 0], 1.0 / np.sqrt(d)
    stream = capi.c_void_p()
    capi.check(capi.load().fb200_stream_create(0, capi.byref(stream)))
    work = None
    rows_of = [[], []]
    for step in steps:
        cu = ref.offsets(step)
        q, k, v = (np.concatenate([text[s][i][done[s]:done[s] + n] for s, n in enumerate(step)]) for i in range(3))
        done = [a + b for a, b in zip(done, step)]
        dq, dk, dv, dcu = upload(q), upload(k), upload(v), upload(cu)
        dlen, out = upload(np.array(done, dtype=np.int32)), upload(np.zeros(q.shape, dtype=np.uint16))
        p = params(dt, h, hk, d, step, total, len(q), 1, scale)
        size = capi.attention_paged_workspace(p, cache)
        if work is None or work.nbytes < size:
            work = upload(np.zeros(max(size, 1), dtype=np.uint8))
        capi.kv_cache_write(cache, dk.ptr, hk * d, d, dv.ptr, hk * d, d, dcu.ptr, dlen.ptr, pages.dev["table"].ptr,
                            pages.table.shape[1], 2, len(k), dt, stream=stream)
        capi.attention_paged(p, cache, dq.ptr, out.ptr, dcu.ptr, dlen.ptr, pages.dev["table"].ptr, pages.table.shape[1],
                             work.ptr, work.nbytes, stream=stream)
        capi.synchronize(0, stream)
        assert capi.kernel_status(0) == 0
        got = out.download(np.uint16, q.shape)
        for s in range(2):
            rows_of[s].append(got[cu[s]:cu[s + 1]])
    capi.check(capi.load().fb200_stream_destroy(0, stream))
    for s in range(2):
        pages.put(s, 0, text[s][1], text[s][2])
        k, v = pages.values(s, total[s])
        o, _, mag, arg = ref.attention(ref.load(text[s][0], dt), k, v, np.float32(scale), True)
        tol, _ = ref.bounds(o, mag, arg, dt, d, coded)
        got = ref.load(np.concatenate(rows_of[s]), dt)
        assert np.all(np.abs(got - o) <= tol), float(np.max(np.abs(got - o) / tol))


# ---- how the calls are made ---------------------------------------------------------------------------
class Call:
    """A paged call whose pieces stay on the device."""

    def __init__(self, rng, dt, h, hk, d, lq, lk, page=16, coded=False, rows=None):
        self.dt, self.h, self.d, self.lq, self.lk, self.coded = dt, h, d, lq, lk, coded
        self.pages = ref.Pages(rng, lk, page, hk, d, dt, coded, True)
        for s, n in enumerate(lk):
            self.pages.put(s, 0, ref.store(rng.standard_normal((n, hk, d)), dt), ref.store(rng.standard_normal((n, hk, d)), dt))
        self.cu, self.scale = ref.offsets(lq), 1.0 / np.sqrt(d)
        self.rows = rows or int(self.cu[-1])
        self.q = ref.store(rng.standard_normal((self.rows, h, d)), dt)
        self.p = params(dt, h, hk, d, lq, lk, self.rows, 1, self.scale)
        self.cache = self.pages.upload()
        self.size = capi.attention_paged_workspace(self.p, self.cache)
        self.work = upload(np.zeros(max(self.size, 1), dtype=np.uint8))
        self.dq, self.dcu, self.dlen = upload(self.q), upload(self.cu), upload(np.array(lk, dtype=np.int32))
        self.out, self.lse = upload(np.full(self.q.shape, FILL, dtype=np.uint16)), capi.DeviceBuffer(self.rows * h * 4)

    def run(self, stream=None):
        capi.attention_paged(self.p, self.cache, self.dq.ptr, self.out.ptr, self.dcu.ptr, self.dlen.ptr,
                             self.pages.dev["table"].ptr, self.pages.table.shape[1], self.work.ptr, self.size,
                             lse=self.lse.ptr, stream=stream)

    def got(self):
        return self.out.download(np.uint16, self.q.shape)

    def check(self, lk=None):
        seqs = [tuple(self.pages.values(s, n)) for s, n in enumerate(lk or self.lk)]
        check_rows(self.got(), self.lse.download(np.float32, self.q.shape[:2]).astype(np.float64), self.q, self.cu, seqs, self.dt,
                   self.d, np.float32(self.scale), 1, self.coded)


@pytest.mark.parametrize("lq", [1, 30], ids=["decode", "chunk"])
@pytest.mark.parametrize("coded", [False, True], ids=["same", "e4m3"])
def test_many_sequences(lq, coded):
    """More sequences than a warp has lanes, some without rows, some without keys."""
    rng = np.random.default_rng(21)
    lens = [int(n) for n in rng.integers(0, 260, 101)]
    call = Call(rng, BF, 4, 2, 64, [0 if i % 7 == 3 else min(lq, 1 + i % lq) for i in range(101)], lens, coded=coded)
    call.run()
    capi.synchronize()
    assert capi.kernel_status(0) == 0
    call.check()


def test_many_prompts():
    dt, h, hk, d = FH, 4, 2, 64
    rng = np.random.default_rng(22)
    lens = [int(n) for n in rng.integers(0, 300, 77)]
    cu = ref.offsets(lens)
    rows = int(cu[-1])
    q, k, v = (ref.store(rng.standard_normal((rows, n, d)), dt) for n in (h, hk, hk))
    p = params(dt, h, hk, d, lens, lens, rows, 1, 0.125)
    p.kv_rows, p.k_token_stride, p.k_head_stride, p.v_token_stride, p.v_head_stride = rows, hk * d, d, hk * d, d
    dq, dk, dv, dcu, out = upload(q), upload(k), upload(v), upload(cu), upload(np.full(q.shape, FILL, dtype=np.uint16))
    lse = capi.DeviceBuffer(rows * h * 4)
    capi.attention_prompt(p, dq.ptr, dk.ptr, dv.ptr, out.ptr, dcu.ptr, dcu.ptr, lse=lse.ptr)
    capi.synchronize()
    assert capi.kernel_status(0) == 0
    seqs = [(ref.load(k[cu[s]:cu[s + 1]], dt), ref.load(v[cu[s]:cu[s + 1]], dt)) for s in range(len(lens))]
    check_rows(out.download(np.uint16, q.shape), lse.download(np.float32, (rows, h)).astype(np.float64), q, cu, seqs, dt, d,
               np.float32(0.125), 1)


def test_calls_on_two_streams_do_not_disturb_each_other():
    rng = np.random.default_rng(23)
    calls = [Call(rng, BF, 16, 2, 128, [1] * 5, [2000, 30, 900, 5, 1500]), Call(rng, BF, 16, 2, 128, [40, 3], [3000, 1100])]
    streams = []
    for _ in calls:
        streams.append(capi.c_void_p())
        capi.check(capi.load().fb200_stream_create(0, capi.byref(streams[-1])))
    for _ in range(20):
        for c, s in zip(calls, streams):
            c.run(s)
    for c, s in zip(calls, streams):
        capi.synchronize(0, s)
        c.check()
        capi.check(capi.load().fb200_stream_destroy(0, s))
    assert capi.kernel_status(0) == 0


@pytest.mark.parametrize("lq", [[1, 1, 1], [40, 1, 17]], ids=["decode", "chunk"])
def test_captured_and_replayed_with_lengths_that_grow_on_the_device(lq):
    """The launches depend on max_q and max_kv only: a captured step is replayed while kv_len changes."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(24)
    top = [1800, 700, 60]
    call = Call(rng, BF, 8, 2, 128, lq, top)
    call.run()
    capi.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        call.run(torch.cuda.current_stream().cuda_stream)
    for lens in ([40, 1, 17], [900, 300, 18], top):
        call.dlen.upload(np.array(lens, dtype=np.int32))
        for _ in range(2):
            graph.replay()
        torch.cuda.synchronize()
        assert capi.kernel_status(0) == 0
        call.check(lens)


def test_more_rows_than_max_q_are_recorded_and_offsets_are_cut():
    rng = np.random.default_rng(25)
    for lq, most in ([3, 2], 1), ([40, 2], 20):            # the bound of either kernel
        call = Call(rng, BF, 4, 2, 64, lq, [50, 20])
        call.p.max_q = most
        call.run()
        capi.synchronize()
        assert capi.kernel_status(0) == 322
    call = Call(rng, BF, 4, 2, 64, [3, 2], [50, 20])
    for cu in ([0, 3, 1 << 30], [-7, 3, 5], [4, 2, 5]):    # past the rows, negative, falling
        call.dcu.upload(np.array(cu, dtype=np.int32))
        call.dlen.upload(np.array([1 << 30, -4], dtype=np.int32))
        call.run()
        capi.synchronize()
        capi.kernel_status(0)
    call = Call(rng, BF, 4, 2, 64, [3, 2], [50, 20])       # and the device is as it was
    call.run()
    capi.synchronize()
    assert capi.kernel_status(0) == 0
    call.check()


@pytest.mark.parametrize("dt", [BF, FH])
@pytest.mark.parametrize("lq", [1, 20], ids=["decode", "chunk"])
def test_what_a_row_does_not_see_does_not_reach_it(dt, lq):
    """NaN and infinity in K of later tokens, and in K and V of tokens behind the sequence's length."""
    rng = np.random.default_rng(26)
    n, h, hk, d = 300, 8, 2, 64
    call = Call(rng, dt, h, hk, d, [lq], [n])
    clean = [x.copy() for x in call.pages.values(0, n)]
    at = call.pages.put
    k, v = (ref.store(x, dt) for x in clean)
    bad = k.copy()
    bad[n - 1] = NAN[dt]                                   # the last query alone sees it
    at(0, 0, bad, v)
    call.pages.dev["k"].upload(call.pages.k)
    call.run()
    capi.synchronize()
    got = ref.load(call.got(), dt)
    assert np.all(np.isnan(got[lq - 1]))
    o, _, mag, arg = ref.attention(ref.load(call.q, dt), clean[0], clean[1], np.float32(call.scale), True)
    tol, _ = ref.bounds(o, mag, arg, dt, d)
    assert np.all(np.abs(got[:lq - 1] - o[:lq - 1]) <= tol[:lq - 1])
    bad_v = v.copy()
    bad_v[n - 5:] = NAN[dt]                                # behind the length from now on
    at(0, 0, bad, bad_v)
    for name in "kv":
        call.pages.dev[name].upload(getattr(call.pages, name))
    call.dlen.upload(np.array([n - 5], dtype=np.int32))
    call.run()
    capi.synchronize()
    o, _, mag, arg = ref.attention(ref.load(call.q, dt), clean[0][:n - 5], clean[1][:n - 5], np.float32(call.scale), True)
    tol, _ = ref.bounds(o, mag, arg, dt, d)
    assert np.all(np.abs(ref.load(call.got(), dt) - o) <= tol)
    assert capi.kernel_status(0) == 0


def test_an_e4m3_token_stored_as_not_finite_makes_the_rows_that_see_it_nan():
    rng = np.random.default_rng(27)
    for lq in (1, 20):
        call = Call(rng, BF, 8, 2, 64, [lq, lq], [300, 200], coded=True)
        ids, tok = call.pages.table[0, 7 // 16], 7
        call.pages.vs[ids, :, tok] = 255                   # value of token 7 of the first sequence
        call.pages.dev["vs"].upload(call.pages.vs)
        call.run()
        capi.synchronize()
        got = ref.load(call.got(), BF)
        assert np.all(np.isnan(got[:lq])) and not np.any(np.isnan(got[lq:]))


@pytest.mark.parametrize("lq", [1, 20], ids=["decode", "chunk"])
@pytest.mark.parametrize("dt", [BF, FH])
def test_value_scales_far_apart_keep_their_precision(dt, lq):
    """e4m3 values whose scales span 2^20: each row is as near as its own weights allow."""
    rng = np.random.default_rng(28)
    n, h, hk, d = 400, 8, 2, 128
    call = Call(rng, dt, h, hk, d, [lq], [n], coded=True)
    gain = np.exp2(rng.integers(-14, 6, (n, hk, 1)))
    v = ref.store(rng.standard_normal((n, hk, d)) * gain, dt)
    v[5] = 0                                               # a row of zeros: scale 2^-126
    call.pages.put(0, 0, ref.store(rng.standard_normal((n, hk, d)), dt), v)
    for name in ("k", "v", "ks", "vs"):
        call.pages.dev[name].upload(getattr(call.pages, name))
    call.run()
    capi.synchronize()
    assert capi.kernel_status(0) == 0
    call.check()


@pytest.mark.parametrize("lq", [1, 40], ids=["decode", "chunk"])
@pytest.mark.parametrize("coded", [False, True], ids=["same", "e4m3"])
def test_pages_whose_offsets_pass_32_bits(lq, coded):
    """Pages 2^28 bytes apart, the last at 5 GiB; keys and values in the same memory."""
    dt, h, hk, d, page, n = BF, 8, 2, 128, 64, 200
    rng = np.random.default_rng(29)
    near = ref.Pages(rng, [n], page, hk, d, dt, coded, True, spare=0)
    x = ref.store(rng.standard_normal((n, hk, d)), dt)
    near.put(0, 0, x, x)
    item = 1 if coded else 2
    far = capi.DeviceBuffer((20 << 28) + (1 << 20))
    spots = np.array([20, 3, 17, 9], dtype=np.int32)       # where the sequence's four pages go
    for i, at in enumerate(spots):
        one = np.ascontiguousarray(near.k[near.table[0, i]])
        capi.check(capi.load().fb200_memcpy(0, far.ptr.value + (int(at) << 28), one.ctypes.data, one.nbytes, capi.H2D, None, 1))
    cache = near.upload()
    cache.k = cache.v = far.ptr
    cache.pages, cache.page_stride = 21, (1 << 28) // item
    if coded:                                              # the scales' pages move with them
        scales = np.full((21, hk, page), 255, dtype=np.uint8)
        scales[spots] = near.ks[near.table[0, :4]]
        dscale = upload(scales)
        cache.k_scale = cache.v_scale = dscale.ptr
    table = upload(spots[None])
    q = ref.store(rng.standard_normal((lq, h, d)), dt)
    p = params(dt, h, hk, d, [lq], [n], lq, 1, 0.09)
    size = capi.attention_paged_workspace(p, cache)
    work, dq, out = upload(np.zeros(max(size, 1), dtype=np.uint8)), upload(q), upload(np.zeros(q.shape, dtype=np.uint16))
    cu, dlen, lse = upload(np.array([0, lq], dtype=np.int32)), upload(np.array([n], dtype=np.int32)), capi.DeviceBuffer(lq * h * 4)
    capi.attention_paged(p, cache, dq.ptr, out.ptr, cu.ptr, dlen.ptr, table.ptr, 4, work.ptr, size, lse=lse.ptr)
    capi.synchronize()
    assert capi.kernel_status(0) == 0
    k, v = near.values(0, n)
    check_rows(out.download(np.uint16, q.shape), lse.download(np.float32, (lq, h)).astype(np.float64), q, [0, lq], [(k, v)], dt, d,
               np.float32(0.09), 1, coded)
