"""Attention of packed prompts and over a paged cache where numbers and lengths are at their edges: NaN at
every place of a tile, parts that hold nothing else, the top and the bottom of the types, more rows than
max_q, lengths that leave the extents, calls large enough for the wide forms of the cache's write and read."""
import numpy as np
import pytest

import serving_ref as ref
from frame_public_b200 import capi
from test_attention_serving_gpu import BF, FH, FILL, NAN, Call, check_rows, params, upload

pytestmark = pytest.mark.gpu


class Prompt:
    """A prompt call whose pieces stay on the device; k and v default to random numbers."""

    def __init__(self, rng, dt, h, hk, d, lq, lk=None, scale=None, causal=1, q=None, k=None, v=None):
        lk = lk or lq
        self.dt, self.d, self.lq, self.lk, self.causal = dt, d, lq, lk, causal
        self.cu, self.cuk = ref.offsets(lq), ref.offsets(lk)
        rows, krows = int(self.cu[-1]), int(self.cuk[-1])
        self.q = ref.store(rng.standard_normal((rows, h, d)), dt) if q is None else q
        self.k = ref.store(rng.standard_normal((krows, hk, d)), dt) if k is None else k
        self.v = ref.store(rng.standard_normal((krows, hk, d)), dt) if v is None else v
        self.scale = scale or 1.0 / np.sqrt(d)
        self.p = params(dt, h, hk, d, lq, lk, rows, causal, self.scale)
        self.p.kv_rows = krows
        self.p.k_token_stride, self.p.k_head_stride, self.p.v_token_stride, self.p.v_head_stride = hk * d, d, hk * d, d
        self.dcu, self.dcuk = upload(self.cu), upload(self.cuk)

    def run(self):
        dq, dk, dv = upload(self.q), upload(self.k), upload(self.v)
        out, lse = upload(np.full(self.q.shape, FILL, dtype=np.uint16)), capi.DeviceBuffer(self.q.shape[0] * self.q.shape[1] * 4)
        capi.attention_prompt(self.p, dq.ptr, dk.ptr, dv.ptr, out.ptr, self.dcu.ptr, self.dcuk.ptr, lse=lse.ptr)
        capi.synchronize()
        return out.download(np.uint16, self.q.shape), lse.download(np.float32, self.q.shape[:2]).astype(np.float64)


def resend(call):
    """The call's cache as it stands on the host, and its query rows."""
    for name in ("k", "v") + (("ks", "vs") if call.coded else ()):
        call.pages.dev[name].upload(getattr(call.pages, name))
    call.dq.upload(call.q)


def run(call, status=0):
    call.run()
    capi.synchronize()
    assert capi.kernel_status(0) == status
    return ref.load(call.got(), call.dt), call.lse.download(np.float32, call.q.shape[:2]).astype(np.float64)


def near(got, lse, q, k, v, dt, d, scale, coded=False, causal=True):
    """Rows of one sequence against 64 bits."""
    o, l, mag, arg = ref.attention(ref.load(q, dt), k, v, np.float32(scale), causal)
    tol, tol_l = ref.bounds(o, mag, arg, dt, d, coded)
    assert np.all(np.abs(got - o) <= tol), float(np.max(np.abs(got - o) / tol))
    assert np.all(np.abs(lse - l) <= tol_l + 2.0 ** -22 * np.abs(l))


def poison_key(call, seq, key, value_too=False):
    """Token `key` of a sequence as one whose K is not finite; its V stays finite, zero on demand."""
    at = call.pages._at(call.pages.k, seq, np.array([key]))
    if call.coded:
        call.pages.ks[at] = 255
        call.pages.k[at] = 0
    else:
        call.pages.k[at] = NAN[call.dt]
    if value_too:
        call.pages.v[at] = 0
        if call.coded:
            call.pages.vs[at] = 1


# ---- NaN ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("lq", [1, 3, 20], ids=["decode", "draft", "chunk"])
@pytest.mark.parametrize("dt,d,coded", [(BF, 64, False), (FH, 128, False), (BF, 128, True), (FH, 64, True)])
def test_a_key_that_is_not_finite_makes_the_rows_that_see_it_nan_at_every_place(dt, d, coded, lq):
    """Places 32 .. 47 of a tile in turn, one sequence each; half of the values are zero."""
    rng = np.random.default_rng(31)
    call = Call(rng, dt, 8, 2, d, [lq] * 17, [200] * 17, coded=coded)
    for r in range(16):
        poison_key(call, r, 32 + r, r % 2 == 1)
    resend(call)
    got, lse = run(call)
    for r in range(16):
        rows = slice(r * lq, (r + 1) * lq)
        assert np.all(np.isnan(got[rows])) and np.all(np.isnan(lse[rows])), r
    rows = slice(16 * lq, 17 * lq)                         # and the last sequence does not know of it
    near(got[rows], lse[rows], call.q[rows], *call.pages.values(16, 200), dt, d, call.scale, coded)


@pytest.mark.parametrize("dt,d", [(BF, 64), (FH, 64), (BF, 128), (FH, 96)])
def test_a_nan_key_of_a_prompt_reaches_the_rows_from_its_own_on(dt, d):
    rng = np.random.default_rng(32)
    n = 150
    call = Prompt(rng, dt, 4, 2, d, [n] * 16)
    for r in range(16):
        call.k[r * n + 33 + r] = NAN[dt]
    got, lse = call.run()
    assert capi.kernel_status(0) == 0
    got = ref.load(got, dt)
    for r in range(16):
        rows, at = slice(r * n, (r + 1) * n), 33 + r
        assert np.all(np.isnan(got[rows][at:])) and np.all(np.isnan(lse[rows][at:])), r
        near(got[rows][:at], lse[rows][:at], call.q[rows][:at], ref.load(call.k[rows][:at], dt), ref.load(call.v[rows][:at], dt),
             dt, d, call.scale)


@pytest.mark.parametrize("dt,coded", [(BF, False), (FH, False), (BF, True), (FH, True)])
def test_parts_that_hold_nothing_but_nan_are_not_taken_for_empty(dt, coded):
    """A chunk whose keys are cut into parts: a NaN query row, and NaN in every key of some part."""
    rng = np.random.default_rng(33)
    h, hk, d, n, lq = 8, 2, 128, 6000, 20
    call = Call(rng, dt, h, hk, d, [lq], [n], page=64, coded=coded)
    assert call.size > 4096                                # the parts' room: this call is cut
    clean = call.q.copy()
    call.q[5, 3] = NAN[dt]
    resend(call)
    got, lse = run(call)
    nan = np.zeros((lq, h), dtype=bool)
    nan[5, 3] = True
    assert np.array_equal(np.isnan(lse), nan) and np.array_equal(np.isnan(got), np.broadcast_to(nan[..., None], got.shape))
    o, l, mag, arg = ref.attention(ref.load(clean, dt), *call.pages.values(0, n), np.float32(call.scale), True)
    tol, tol_l = ref.bounds(o, mag, arg, dt, d, coded)
    assert np.all((np.abs(got - o) <= tol)[~nan]) and np.all((np.abs(lse - l) <= tol_l + 2.0 ** -22 * np.abs(l))[~nan])
    call.q = clean
    for key in range(2048, 4096):                          # whole parts of 1024 and 2048 keys
        poison_key(call, 0, key)
    resend(call)
    got, lse = run(call)
    assert np.all(np.isnan(got)) and np.all(np.isnan(lse))


# ---- more rows than max_q ----------------------------------------------------------------------------
@pytest.mark.parametrize("h,lq,most,lk", [(4, [3, 1, 2], 1, [50, 20, 300]), (4, [40, 2, 70], 20, [50, 20, 90]),
                                          (8, [400, 30, 64], 64, [500, 60, 64]), (8, [400, 30, 1], 64, [3000, 1500, 2000]),
                                          (8, [30, 400], 64, [20, 9000])],
                         ids=["decode", "one block", "blocks", "parts", "long last"])
@pytest.mark.parametrize("coded", [False, True], ids=["same", "e4m3"])
def test_a_sequence_past_max_q_costs_no_other_its_rows(h, lq, most, lk, coded):
    rng = np.random.default_rng(34)
    call = Call(rng, BF, h, 2, 64, lq, lk, coded=coded)
    call.p.max_q = most
    call.size = capi.attention_paged_workspace(call.p, call.cache)
    call.work = upload(np.zeros(max(call.size, 1), dtype=np.uint8))
    if call.size > 4096:                                   # what an earlier call left there
        call.work.upload(np.concatenate([np.zeros(4096, dtype=np.uint8), np.full(call.size - 4096, 0x41, dtype=np.uint8)]))
    got, lse = run(call, 322)
    for s, n in enumerate(lq):
        rows = slice(call.cu[s], call.cu[s] + min(n, most))
        k, v = call.pages.values(s, lk[s])
        o, l, mag, arg = ref.attention(ref.load(call.q[call.cu[s]:call.cu[s + 1]], BF), k, v, np.float32(call.scale), True)
        tol, tol_l = ref.bounds(o, mag, arg, BF, 64, coded)
        m = min(n, most)
        assert np.all(np.abs(got[rows] - o[:m]) <= tol[:m]), s
        seen = np.isfinite(l[:m])
        assert np.all(np.isneginf(lse[rows][~seen]))
        assert np.all(np.abs(lse[rows][seen] - l[:m][seen]) <= (tol_l + 2.0 ** -22 * np.abs(l))[:m][seen])
        assert np.all(call.got()[call.cu[s] + m:call.cu[s + 1]] == FILL), s       # not computed


@pytest.mark.parametrize("most", [64, 100, 0])
@pytest.mark.parametrize("causal", [1, 0])
def test_a_prompt_past_max_q_costs_no_other_its_rows(most, causal):
    rng = np.random.default_rng(35)
    lq = [700, 33, 100, 1]
    call = Prompt(rng, BF, 8, 2, 64, lq, causal=causal)
    call.p.max_q = most
    got, lse = call.run()
    assert capi.kernel_status(0) == 322
    for s, n in enumerate(lq):
        a, m = call.cu[s], min(n, most)
        rows = slice(a, a + n)
        o, l, mag, arg = ref.attention(ref.load(call.q[rows], BF), ref.load(call.k[rows], BF), ref.load(call.v[rows], BF),
                                       np.float32(call.scale), bool(causal))
        tol, tol_l = ref.bounds(o, mag, arg, BF, 64)
        assert np.all(np.abs(ref.load(got[a:a + m], BF) - o[:m]) <= tol[:m]), s
        assert np.all(np.abs(lse[a:a + m] - l[:m]) <= (tol_l + 2.0 ** -22 * np.abs(l))[:m])
        assert np.all(got[a + m:a + n] == FILL), s


# ---- the ends of the types ---------------------------------------------------------------------------
TOP = {BF: 2.0 ** 128 - 2.0 ** 120, FH: 65504.0}


def finite_values(pages, seq, n, dt):
    """What an e4m3 cache's finite numbers read as: rounded to the type, the largest finite number at most."""
    return [np.where(np.isnan(x), x, np.clip(x, -TOP[dt], TOP[dt])) for x in pages.values(seq, n)]


@pytest.mark.parametrize("dt", [BF, FH])
def test_finite_numbers_at_the_top_of_the_type_read_back_finite(dt):
    """A row's largest number may round up to 256 * 2^e, which is past the 16-bit type at its very top."""
    rng = np.random.default_rng(36)
    h, hk, d, n = 4, 2, 64, 40
    call = Call(rng, dt, h, hk, d, [1], [n], coded=True)
    x = ref.store(rng.uniform(0.9, 1.0, (n, hk, d)) * rng.choice([-1.0, 1.0], (n, hk, d)) * TOP[dt], dt)
    x[3, 0, :2] = ref.store(np.array([TOP[dt], -TOP[dt]]), dt)
    x[4, 1] = 0x7F80 if dt == BF else 0x7C00                # an infinity reads as NaN
    call.pages.put(0, 0, x, x)
    resend(call)
    outs, cu = [upload(np.full((n, hk, d), FILL, dtype=np.uint16)) for _ in range(2)], upload(np.array([0, n], dtype=np.int32))
    capi.kv_cache_read(call.cache, outs[0].ptr, hk * d, d, outs[1].ptr, hk * d, d, cu.ptr, call.pages.dev["table"].ptr,
                       call.pages.table.shape[1], 1, n, dt)
    capi.synchronize()
    assert np.abs(np.nan_to_num(call.pages.values(0, n)[0])).max() > TOP[dt]     # the case it is about
    for out, want in zip(outs, finite_values(call.pages, 0, n, dt)):
        got = ref.load(out.download(np.uint16, (n, hk, d)), dt)
        assert np.array_equal(np.isnan(got), np.isnan(want)) and np.all(np.isnan(want[4, 1]))
        fine = ~np.isnan(want)
        assert np.array_equal(got[fine], ref.load(ref.store(want, dt), dt)[fine])


@pytest.mark.parametrize("lq,n", [(1, 40), (20, 40), (20, 3000)], ids=["decode", "chunk", "parts"])
@pytest.mark.parametrize("dt", [BF, FH])
def test_attention_over_e4m3_values_at_the_top_of_the_type_stays_finite(dt, lq, n):
    """All values equal the largest finite number, so every row does, whatever the weights."""
    rng = np.random.default_rng(37)
    call = Call(rng, dt, 8, 2, 64, [lq], [n], coded=True)
    k = ref.store(rng.standard_normal((n, 2, 64)), dt)
    call.pages.put(0, 0, k, ref.store(np.full((n, 2, 64), TOP[dt]), dt))
    resend(call)
    got, lse = run(call)
    assert np.all(np.isfinite(got)) and np.all(np.isfinite(lse))
    unit = ref.UNIT[dt]
    assert np.all(got >= TOP[dt] * (1 - 2 * unit))


def score_error(arg, d):
    return (d + 8) * 2.0 ** -23 * arg + 2.0 ** -20


def small_weights_bound(o, mag, arg, dt, d, n, weights, values, smallest=2.0 ** -24):
    """Probabilities are held in float16 for float16 and e4m3 caches, the largest as 2^7 or more: half a step
    is 2^-11 of a probability, and at least 2^-25, which is 2^-32 of the row's largest weight.  (`weights`:
    that largest one per row, p times the value's scale; `values`: the sum over the keys of what it is
    multiplied with, codes or numbers.)  A score is an fp32 sum of d products, as in ref.bounds; O and the row
    sum grow in fp32 by 16 keys at a time or more, each addition truncated at worst."""
    delta, steps = score_error(arg, d), n / 16 * 2.0 ** -23
    return (2.0 ** -11 + 2 * delta[..., None] + 2 * steps) * mag + ref.UNIT[dt] * np.abs(o) + smallest + 2.0 ** -32 * weights * values


@pytest.mark.parametrize("form,dt,coded", [("prompt", FH, False)] +
                         [(f, dt, c) for f in ("decode", "draft", "chunk") for dt, c in ((FH, False), (BF, True), (FH, True))])
def test_many_small_probabilities_beside_a_large_one_are_not_lost(form, dt, coded):
    """One key outweighs each of 2^17 others by 2^26, and in all columns but one their values are 2^10 as large:
    together the others make most of the result.  Over a cache so many sequences share the pages that one CTA
    walks all keys of a sequence."""
    rng = np.random.default_rng(38)
    h, hk, d, n = 2, 1, 64, 1 << 17
    copies, lq = {"decode": (300, 1), "draft": (300, 6), "chunk": (150, 20), "prompt": (1, 20)}[form]
    scale = 0.125
    q = ref.store(np.full((lq, h, d), 1.5), dt)
    k = np.zeros((n, hk, d))
    k[7] = 1.5                                              # 2.25 * 64 / 8 = 18 = 25.97 in powers of two
    v = np.full((n, hk, d), 8.0) * rng.choice([0.875, 1.0, 1.125], (n, hk, d))
    v[7] = 2.0 ** -7
    v[7, :, 0] = 8.0                                        # its scale is the others'
    k, v = ref.store(k, dt), ref.store(v, dt)
    e = np.zeros(n)
    if form == "prompt":
        got, lse = Prompt(rng, dt, h, hk, d, [lq], [n], scale, 0, q, k, v).run()
        kk, vv = ref.load(k, dt), ref.load(v, dt)
    else:
        pages = ref.Pages(rng, [n], 128, hk, d, dt, coded, True)
        pages.put(0, 0, k, v)
        cache, table = pages.upload(), upload(np.repeat(pages.table, copies, 0))
        p = params(dt, h, hk, d, [lq] * copies, [n], lq * copies, 0, scale)
        size = capi.attention_paged_workspace(p, cache)
        work, dq = upload(np.zeros(max(size, 1), dtype=np.uint8)), upload(np.tile(q, (copies, 1, 1)))
        out, dlse = upload(np.full((lq * copies, h, d), FILL, dtype=np.uint16)), capi.DeviceBuffer(lq * copies * h * 4)
        dcu, dlen = upload(ref.offsets([lq] * copies)), upload(np.full(copies, n, dtype=np.int32))
        capi.attention_paged(p, cache, dq.ptr, out.ptr, dcu.ptr, dlen.ptr, table.ptr, pages.table.shape[1], work.ptr, size, lse=dlse.ptr)
        capi.synchronize()
        got = out.download(np.uint16, (copies, lq, h, d))
        lse = dlse.download(np.float32, (copies, lq, h)).astype(np.float64)
        kk, vv = pages.values(0, n)
        if coded:
            e = np.maximum(pages.vs[pages._at(pages.vs, 0, np.arange(n))][:, 0].astype(np.float64) - 127, -60)
    assert capi.kernel_status(0) == 0
    got = ref.load(got, dt)
    o, l, mag, arg = ref.attention(ref.load(q, dt), kk, vv, scale, False)
    p = np.exp(ref.load(q, dt)[0, 0] @ kk[:, 0].T * scale - l[0, 0])
    tol = small_weights_bound(o, mag, arg, dt, d, n, np.max(p * 2.0 ** e), (np.abs(vv[:, 0]) * 2.0 ** -e[:, None]).sum(0))
    assert np.all(tol < 0.1 * np.abs(o))                    # the bound says something
    assert np.all(np.abs(got - o) <= tol), float(np.max(np.abs(got - o) / tol))
    assert np.all(np.abs(lse - l) <= score_error(arg, d) + 2.0 ** -21 + 2.0 ** -22 * np.abs(l) + n / 16 * 2.0 ** -23)


@pytest.mark.parametrize("lq", [1, 3, 20], ids=["decode", "draft", "chunk"])
@pytest.mark.parametrize("dt,d", [(BF, 64), (FH, 128)])
def test_probabilities_over_an_e4m3_cache_keep_the_bits_of_float16(dt, d, lq):
    """Ordinary numbers, held to half a step of float16 in P (serving_ref's bound allows bfloat16's)."""
    rng = np.random.default_rng(45)
    n, h, hk = 500, 8, 2
    call = Call(rng, dt, h, hk, d, [lq], [n], coded=True)
    got, lse = run(call)
    kk, vv = call.pages.values(0, n)
    o, l, mag, arg = ref.attention(ref.load(call.q, dt), kk, vv, np.float32(call.scale), True)
    e = call.pages.vs[call.pages._at(call.pages.vs, 0, np.arange(n))].astype(np.float64) - 127      # [n, hk]
    codes = (np.abs(vv) * 2.0 ** -e[..., None]).sum(0).repeat(h // hk, 0)                           # [h, d]
    tol = small_weights_bound(o, mag, arg, dt, d, n, 2.0 ** e.max(), codes)
    assert np.all(np.abs(got - o) <= tol), float(np.max(np.abs(got - o) / tol))


@pytest.mark.parametrize("lq", [1, 3, 20], ids=["decode", "draft", "chunk"])
@pytest.mark.parametrize("gain", [2.0 ** -40, 2.0 ** -66, 2.0 ** 100])
def test_values_of_any_size_keep_their_bits_over_an_e4m3_cache(gain, lq):
    """Scales from below the smallest one that rows are normalised with (2^-60) to large ones."""
    rng = np.random.default_rng(50)
    n, h, hk, d, dt = 500, 8, 2, 64, BF
    call = Call(rng, dt, h, hk, d, [lq], [n], coded=True)
    call.pages.put(0, 0, ref.store(rng.standard_normal((n, hk, d)), dt), ref.store(rng.standard_normal((n, hk, d)) * gain, dt))
    resend(call)
    got, _ = run(call)
    kk, vv = call.pages.values(0, n)
    o, l, mag, arg = ref.attention(ref.load(call.q, dt), kk, vv, np.float32(call.scale), True)
    e = np.maximum(call.pages.vs[call.pages._at(call.pages.vs, 0, np.arange(n))].astype(np.float64) - 127, -60)
    codes = (np.abs(vv) / gain).sum(0).repeat(h // hk, 0) * gain / 2.0 ** e.min()                   # at least the sum of them
    # without the term for float16's smallest numbers, which the result's bfloat16 does not have (adding 2^-24 and
    # taking it away again would leave a multiple of 2^-76 of a bound near 2^-78)
    tol = small_weights_bound(o, mag, arg, dt, d, n, 2.0 ** e.max(), codes, 0.0)
    assert np.all(np.abs(got - o) <= tol), float(np.max(np.abs(got - o) / tol))
    assert np.median(tol / np.abs(o)) < 0.05


@pytest.mark.parametrize("lq,n", [(1, 100), (20, 100)], ids=["decode", "chunk"])
@pytest.mark.parametrize("top", [2.0 ** -126, 2.0 ** -127, 2.0 ** -131])
def test_the_smallest_bfloat16_queries_over_an_e4m3_cache(lq, n, top):
    """Query rows below or near the smallest normal number, keys near the largest: scores of a few units."""
    rng = np.random.default_rng(39)
    h, hk, d, dt = 8, 2, 64, BF
    call = Call(rng, dt, h, hk, d, [lq], [n], coded=True)
    q = np.round(rng.uniform(-1, 1, (lq, h, d)) * top / 2.0 ** -133) * 2.0 ** -133
    q[..., 0] = top                                         # multiples of the smallest subnormal number
    call.q = ref.store(q, dt)
    assert np.array_equal(ref.load(call.q, dt), q)
    call.scale = call.p.scale = 2.0 ** -126 / top
    call.pages.put(0, 0, ref.store(rng.standard_normal((n, hk, d)) * 2.0 ** 124, dt), ref.store(rng.standard_normal((n, hk, d)), dt))
    resend(call)
    got, lse = run(call)
    near(got, lse, call.q, *call.pages.values(0, n), dt, d, call.scale, True)


# ---- lengths that leave the extents ------------------------------------------------------------------
@pytest.mark.parametrize("lq", [[1, 1], [20, 30]], ids=["decode", "chunk"])
@pytest.mark.parametrize("what,cu,lens", [("past the table", None, [300, 1 << 20]), ("negative", None, [-3, 200]),
                                          ("past the rows", [0, 1, 1 << 28], None), ("before the rows", [-5, 1, 2], None),
                                          ("falling", [0, 2, 1], None), ("nothing left", [9, 9, 3], None)])
def test_lengths_that_are_cut_are_recorded(lq, what, cu, lens):
    """The rows are those of the lengths that remain (the second sequence's table row holds its 200 tokens)."""
    rng = np.random.default_rng(40)
    call = Call(rng, BF, 8, 2, 64, lq, [208, 208])
    if cu is not None:
        call.dcu.upload(np.array(cu, dtype=np.int32))
    if lens is not None:
        call.dlen.upload(np.array(lens, dtype=np.int32))
    run(call, 322)
    if lens is None:
        return
    lk = [max(0, min(n, 208)) for n in lens]
    seqs = [tuple(call.pages.values(s, n)) for s, n in enumerate(lk)]
    check_rows(call.got(), call.lse.download(np.float32, call.q.shape[:2]).astype(np.float64), call.q, call.cu, seqs, BF, 64,
               np.float32(call.scale), 1)


@pytest.mark.parametrize("lq", [[1, 0, 1, 0, 0], [20, 0, 30, 0, 0]], ids=["decode", "chunk"])
def test_empty_places_of_a_padded_batch_are_not_recorded(lq):
    """A captured step keeps its number of sequences: places without rows, whose length is not looked at."""
    rng = np.random.default_rng(51)
    call = Call(rng, BF, 8, 2, 64, lq, [100, 0, 300, 0, 0])
    call.dlen.upload(np.array([100, -1, 300, 1 << 30, -1], dtype=np.int32))
    run(call, 0)
    call.check()


@pytest.mark.parametrize("cu,cuk", [([0, 40, 1 << 28], None), ([-1, 40, 70], None), (None, [0, 40, 71]), (None, [0, 60, 40])])
def test_prompt_offsets_that_are_cut_are_recorded(cu, cuk):
    rng = np.random.default_rng(41)
    call = Prompt(rng, BF, 4, 2, 64, [40, 30])
    if cu is not None:
        call.dcu.upload(np.array(cu, dtype=np.int32))
    if cuk is not None:
        call.dcuk.upload(np.array(cuk, dtype=np.int32))
    call.run()
    assert capi.kernel_status(0) == 322
    call = Prompt(rng, BF, 4, 2, 64, [40, 30])
    call.run()
    assert capi.kernel_status(0) == 0


@pytest.mark.parametrize("cu", [[0, 3, 9], [-2, 3, 5]])
@pytest.mark.parametrize("coded", [False, True], ids=["same", "e4m3"])
def test_cache_offsets_that_leave_the_rows_are_recorded(cu, coded):
    rng = np.random.default_rng(42)
    hk, d = 2, 64
    pages = ref.Pages(rng, [20, 20], 16, hk, d, BF, coded, True)
    cache = pages.upload()
    x, dcu = upload(ref.store(rng.standard_normal((5, hk, d)), BF)), upload(np.array(cu, dtype=np.int32))
    lens = upload(np.array([20, 20], dtype=np.int32))
    table, stride = pages.dev["table"].ptr, pages.table.shape[1]
    capi.kv_cache_write(cache, x.ptr, hk * d, d, x.ptr, hk * d, d, dcu.ptr, lens.ptr, table, stride, 2, 5, BF)
    capi.synchronize()
    assert capi.kernel_status(0) == 322
    capi.kv_cache_read(cache, x.ptr, hk * d, d, x.ptr, hk * d, d, dcu.ptr, table, stride, 2, 5, BF)
    capi.synchronize()
    assert capi.kernel_status(0) == 322


def test_tokens_without_a_place_are_not_stored():
    """More new tokens than the length counts: the first ones would lie before the sequence."""
    rng = np.random.default_rng(43)
    hk, d, page, dt = 2, 64, 16, BF
    pages = ref.Pages(rng, [40], page, hk, d, dt, False, True, fill=7)
    cache = pages.upload()
    x = ref.store(rng.standard_normal((40, hk, d)), dt)
    dx, cu, lens = upload(x), upload(np.array([0, 40], dtype=np.int32)), upload(np.array([10], dtype=np.int32))
    capi.kv_cache_write(cache, dx.ptr, hk * d, d, dx.ptr, hk * d, d, cu.ptr, lens.ptr, pages.dev["table"].ptr, 3, 1, 40, dt)
    capi.synchronize()
    assert capi.kernel_status(0) == 322
    pages.put(0, 0, x[30:], x[30:])
    for name in ("k", "v"):
        assert np.array_equal(pages.dev[name].download(np.uint16, pages.k.shape), getattr(pages, name))


# ---- calls large enough for four heads per lane group --------------------------------------------------
@pytest.mark.parametrize("dt,hk,d,page,coded,head_major", [
    (BF, 4, 64, 16, True, True), (FH, 5, 80, 32, True, False), (BF, 7, 128, 64, False, True), (BF, 8, 128, 16, True, True),
    (FH, 6, 48, 8, False, False), (BF, 8, 96, 128, False, False)])
def test_large_writes_and_reads_bit_for_bit(dt, hk, d, page, coded, head_major):
    """Rows x heads x lanes of a row pass two per thread slot of the GPU (2 * 148 * 2048)."""
    rng = np.random.default_rng(44)
    rows = -(-2 * 148 * 2048 // (hk * (8 if d <= 64 else 16))) + 37
    new = [rows // 3, 0, 1, rows - rows // 3 - 1]
    lens = [new[0] + 11, 5, 40, new[3]]
    pages = ref.Pages(rng, lens, page, hk, d, dt, coded, head_major, fill=7)
    cache, cu = pages.upload(), ref.offsets(new)
    ld = hk * d + 16
    both = [ref.store(rng.standard_normal((rows, ld)) * np.exp2(rng.integers(-30, 8, (rows, 1))), dt) for _ in range(2)]
    k, v = (b[:, :hk * d].reshape(rows, hk, d) for b in both)
    dk, dv, dcu, dlen = upload(both[0]), upload(both[1]), upload(cu), upload(np.array(lens, dtype=np.int32))
    table, stride = pages.dev["table"].ptr, pages.table.shape[1]
    capi.kv_cache_write(cache, dk.ptr, ld, d, dv.ptr, ld, d, dcu.ptr, dlen.ptr, table, stride, len(new), rows, dt)
    capi.synchronize()
    assert capi.kernel_status(0) == 0
    for s, n in enumerate(new):
        pages.put(s, lens[s] - n, k[cu[s]:cu[s + 1]], v[cu[s]:cu[s + 1]])
    for name in ("k", "v") + (("ks", "vs") if coded else ()):
        want = getattr(pages, name)
        assert np.array_equal(pages.dev[name].download(want.dtype, want.shape), want), name
    keep = [new[0] + 3, 2, 40, new[3]]                       # some of the sequences in part
    cuk = ref.offsets(keep)
    total = int(cuk[-1]) + 3
    old = hk * d + 8
    outs = [upload(np.full((total, old), FILL, dtype=np.uint16)) for _ in range(2)]
    dcuk = upload(cuk)
    capi.kv_cache_read(cache, outs[0].ptr, old, d, outs[1].ptr, old, d, dcuk.ptr, table, stride, len(keep), total, dt)
    capi.synchronize()
    assert capi.kernel_status(0) == 0
    for i, out in enumerate(outs):
        got = out.download(np.uint16, (total, old))
        assert np.all(got[cuk[-1]:] == FILL) and np.all(got[:, hk * d:] == FILL)
        for s, n in enumerate(keep):
            want = ref.store(pages.values(s, n)[i], dt).reshape(n, hk * d)
            g = got[cuk[s]:cuk[s + 1], :hk * d]
            nan = np.isnan(ref.load(want, dt))
            assert np.array_equal(np.isnan(ref.load(g, dt)), nan) and np.array_equal(g[~nan], want[~nan])


# ---- layouts -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt,h,hk,d", [(BF, 8, 2, 64), (FH, 6, 2, 128), (BF, 4, 4, 80)])
def test_prompts_whose_heads_lie_apart(dt, h, hk, d):
    """[head, token, dim] instead of [token, head, dim], for every operand."""
    rng = np.random.default_rng(46)
    lens = [130, 0, 61]
    call = Prompt(rng, dt, h, hk, d, lens)
    rows = sum(lens)
    q, k, v = (upload(x.transpose(1, 0, 2)) for x in (call.q, call.k, call.v))
    out, lse = upload(np.full((h, rows + 3, d), FILL, dtype=np.uint16)), capi.DeviceBuffer(rows * h * 4)
    p = call.p
    p.q_token_stride = p.k_token_stride = p.v_token_stride = p.o_token_stride = d
    p.q_head_stride = p.k_head_stride = p.v_head_stride = rows * d
    p.o_head_stride = (rows + 3) * d
    capi.attention_prompt(p, q.ptr, k.ptr, v.ptr, out.ptr, call.dcu.ptr, call.dcuk.ptr, lse=lse.ptr)
    capi.synchronize()
    assert capi.kernel_status(0) == 0
    got = out.download(np.uint16, (h, rows + 3, d))
    assert np.all(got[:, rows:] == FILL)
    seqs = [(ref.load(call.k[a:b], dt), ref.load(call.v[a:b], dt)) for a, b in zip(call.cu, call.cu[1:])]
    check_rows(got[:, :rows].transpose(1, 0, 2), lse.download(np.float32, (rows, h)).astype(np.float64), call.q, call.cu, seqs,
               dt, d, np.float32(call.scale), 1)


@pytest.mark.parametrize("lq", [[1, 1, 1], [20, 3, 100]], ids=["decode", "chunk"])
@pytest.mark.parametrize("dt,h,hk,d,page,coded", [(BF, 8, 2, 16, 8, True), (FH, 4, 2, 48, 8, True), (BF, 8, 2, 128, 8, True),
                                                  (BF, 8, 2, 128, 8, False), (FH, 8, 2, 32, 8, False), (BF, 6, 2, 112, 512, True),
                                                  (FH, 32, 2, 16, 16, True)])
def test_small_pages_and_small_heads(dt, h, hk, d, page, coded, lq):
    """Query and output rows with their heads apart, lengths that end inside a page and a tile."""
    rng = np.random.default_rng(47)
    call = Call(rng, dt, h, hk, d, lq, [1, 267, 777], page=page, coded=coded)
    rows = call.rows
    q, out = upload(call.q.transpose(1, 0, 2)), upload(np.full((h, rows, d), FILL, dtype=np.uint16))
    call.p.q_token_stride = call.p.o_token_stride = d
    call.p.q_head_stride = call.p.o_head_stride = rows * d
    call.dq, call.out = q, out
    call.run()
    capi.synchronize()
    assert capi.kernel_status(0) == 0
    got = out.download(np.uint16, (h, rows, d)).transpose(1, 0, 2)
    seqs = [tuple(call.pages.values(s, n)) for s, n in enumerate(call.lk)]
    check_rows(got, call.lse.download(np.float32, (rows, h)).astype(np.float64), call.q, call.cu, seqs, dt, d, np.float32(call.scale),
               1, coded)


@pytest.mark.parametrize("coded", [False, True], ids=["same", "e4m3"])
def test_writes_and_reads_of_rows_whose_heads_lie_apart(coded):
    """k and v with strides of their own."""
    rng = np.random.default_rng(48)
    dt, hk, d, n = FH, 3, 64, 45
    pages = ref.Pages(rng, [n], 16, hk, d, dt, coded, True, fill=7)
    cache = pages.upload()
    k, v = (ref.store(rng.standard_normal((n, hk, d)), dt) for _ in range(2))
    dk = upload(k.transpose(1, 0, 2))
    wide = np.full((n, hk, d + 24), FILL, dtype=np.uint16)
    wide[..., :d] = v
    dv, cu, lens = upload(wide), upload(np.array([0, n], dtype=np.int32)), upload(np.array([n], dtype=np.int32))
    strides = d, n * d, hk * (d + 24), d + 24
    capi.kv_cache_write(cache, dk.ptr, strides[0], strides[1], dv.ptr, strides[2], strides[3], cu.ptr, lens.ptr, pages.dev["table"].ptr,
                        pages.table.shape[1], 1, n, dt)
    capi.synchronize()
    pages.put(0, 0, k, v)
    for name in ("k", "v") + (("ks", "vs") if coded else ()):
        want = getattr(pages, name)
        assert np.array_equal(pages.dev[name].download(want.dtype, want.shape), want), name
    ok, ov = upload(np.full((hk, n, d), FILL, dtype=np.uint16)), upload(np.full(wide.shape, FILL, dtype=np.uint16))
    capi.kv_cache_read(cache, ok.ptr, strides[0], strides[1], ov.ptr, strides[2], strides[3], cu.ptr, pages.dev["table"].ptr,
                       pages.table.shape[1], 1, n, dt)
    capi.synchronize()
    assert capi.kernel_status(0) == 0
    want_k, want_v = (ref.store(x, dt) for x in pages.values(0, n))
    assert np.array_equal(ok.download(np.uint16, (hk, n, d)).transpose(1, 0, 2), want_k)
    got = ov.download(np.uint16, wide.shape)
    assert np.array_equal(got[..., :d], want_v) and np.all(got[..., d:] == FILL)


def test_two_captured_calls_share_a_workspace_in_turn():
    """A decoding step and a chunk cut into parts, captured apart, replayed one after the other."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(49)
    calls = [Call(rng, BF, 16, 2, 128, [1, 2], [1500, 900]), Call(rng, FH, 16, 2, 128, [30, 4], [2500, 1100], coded=True)]
    size = max(c.size for c in calls)
    assert min(c.size for c in calls) > 4096
    work = upload(np.zeros(size, dtype=np.uint8))
    graphs, stream = [], torch.cuda.Stream()
    for c in calls:
        c.work, c.size = work, size
        c.run()
        capi.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            c.run(torch.cuda.current_stream().cuda_stream)
        c.out.upload(np.full(c.q.shape, FILL, dtype=np.uint16))
    with torch.cuda.stream(stream):
        for i in (0, 1, 1, 0, 1, 0):
            graphs[i].replay()
    torch.cuda.synchronize()
    assert capi.kernel_status(0) == 0
    for c in calls:
        c.check()
