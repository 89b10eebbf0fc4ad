"""Refusals of the serving attention entry points (they come before any CUDA call), and the host-side
statement of the e4m3 scale rule, without a GPU."""
import numpy as np
import pytest

import serving_ref as ref
from frame_public_b200 import capi

PTR = 1 << 20   # never dereferenced: every call here is refused first


def good_params(**kw):
    p = dict(n_seqs=2, heads=8, kv_heads=2, head_dim=64, q_rows=10, kv_rows=10, max_q=5, max_kv=9, q_token_stride=512,
             q_head_stride=64, o_token_stride=512, o_head_stride=64, k_token_stride=128, k_head_stride=64,
             v_token_stride=128, v_head_stride=64, scale=0.125, causal=1, dtype=capi.BF16)
    p.update(kw)
    return capi.AttentionParams(**p)


def good_cache(**kw):
    c = dict(k=PTR, v=PTR, pages=4, page_size=16, kv_heads=2, head_dim=64, page_stride=2048, token_stride=64,
             head_stride=1024, dtype=capi.BF16)
    if kw.get("dtype") == capi.U8:
        c.update(k_scale=PTR, v_scale=PTR, scale_page_stride=32, scale_token_stride=1, scale_head_stride=16)
    c.update(kw)
    return capi.KvCache(**c)


def prompt(p, q=PTR, k=PTR, v=PTR, o=PTR, cu_q=PTR, cu_kv=PTR):
    capi.attention_prompt(p, q, k, v, o, cu_q, cu_kv)


def paged(p, c, q=PTR, o=PTR, cu_q=PTR, kv_len=PTR, table=PTR, stride=4, work=PTR, size=1 << 40):
    capi.attention_paged(p, c, q, o, cu_q, kv_len, table, stride, work, size)


def write(c, k=PTR, v=PTR, cu=PTR, kv_len=PTR, table=PTR, ts=128, hs=64, n=2, rows=5, dt=capi.BF16, stride=4):
    capi.kv_cache_write(c, k, ts, hs, v, ts, hs, cu, kv_len, table, stride, n, rows, dt)


def read(c, k=PTR, v=PTR, cu=PTR, table=PTR, ts=128, hs=64, n=2, rows=5, dt=capi.BF16, stride=4):
    capi.kv_cache_read(c, k, ts, hs, v, ts, hs, cu, table, stride, n, rows, dt)


def refused(code, what, call, *args, **kw):
    with pytest.raises(capi.Fb200Error) as e:
        call(*args, **kw)
    assert e.value.code == code and what in str(e.value), str(e.value)


BAD_PARAMS = [(1, dict(n_seqs=-1)), (1, dict(q_rows=1 << 31)), (1, dict(kv_rows=-1)), (1, dict(max_q=-1)),
              (1, dict(heads=7)), (1, dict(kv_heads=0)), (1, dict(heads=0)), (4, dict(dtype=capi.F32)),
              (4, dict(head_dim=72)), (4, dict(head_dim=8)), (4, dict(head_dim=144)), (4, dict(heads=130)),
              (1, dict(scale=0.0)), (1, dict(scale=float("nan"))), (1, dict(scale=float("inf"))), (1, dict(scale=-1.0)),
              (1, dict(q_token_stride=508)), (1, dict(q_head_stride=56)), (1, dict(o_token_stride=1 + 512)),
              (1, dict(o_head_stride=0))]


@pytest.mark.parametrize("code,change", BAD_PARAMS, ids=lambda x: str(x))
def test_params_are_checked_by_every_attention_call(code, change):
    refused(code, "attention_prompt", prompt, good_params(**change))
    refused(code, "attention_paged", paged, good_params(**change), good_cache())
    refused(code, "attention_paged_workspace", capi.attention_paged_workspace, good_params(**change), good_cache())


BAD_CACHE = [(1, dict(pages=-1)), (1, dict(pages=1 << 31)), (1, dict(kv_heads=0)), (4, dict(head_dim=24)),
             (4, dict(head_dim=256)), (4, dict(page_size=24)), (4, dict(page_size=4)), (4, dict(page_size=0)),
             (1, dict(page_stride=2052)), (1, dict(token_stride=32)), (1, dict(head_stride=0)), (1, dict(k=None)),
             (1, dict(v=PTR + 8)), (4, dict(dtype=capi.F16)), (4, dict(dtype=capi.F32)),
             (1, dict(dtype=capi.U8, k_scale=None)), (1, dict(dtype=capi.U8, scale_head_stride=0)),
             (1, dict(dtype=capi.U8, token_stride=72))]


@pytest.mark.parametrize("code,change", BAD_CACHE, ids=lambda x: str(x))
def test_the_cache_is_checked_by_every_call_that_takes_it(code, change):
    refused(code, "attention_paged", paged, good_params(), good_cache(**change))
    refused(code, "kv_cache_write", write, good_cache(**change))
    refused(code, "kv_cache_read", read, good_cache(**change))


@pytest.mark.parametrize("name", ["q", "k", "v", "o", "cu_q", "cu_kv"])
def test_prompt_refuses_null_and_unaligned(name):
    refused(1, "null", prompt, good_params(), **{name: None})
    if not name.startswith("cu"):
        refused(1, "aligned", prompt, good_params(), **{name: PTR + 2})
    refused(1, "strides", prompt, good_params(k_token_stride=63))
    refused(1, "strides", prompt, good_params(v_head_stride=0))


@pytest.mark.parametrize("name", ["q", "o", "cu_q", "kv_len", "table"])
def test_paged_refuses_null_unaligned_and_foreign_caches(name):
    refused(1, "null", paged, good_params(), good_cache(), **{name: None})
    if name in "qo":
        refused(1, "aligned", paged, good_params(), good_cache(), **{name: PTR + 2})
    refused(1, "heads", paged, good_params(), good_cache(kv_heads=4))
    refused(1, "heads", paged, good_params(), good_cache(head_dim=128, token_stride=128))
    refused(1, "stride", paged, good_params(), good_cache(), stride=-1)
    refused(1, "without pages", paged, good_params(), good_cache(pages=0, k=None, v=None))


def test_paged_refuses_a_small_or_unaligned_workspace():
    size = capi.attention_paged_workspace(good_params(), good_cache())
    if size > 0:
        refused(1, "workspace", paged, good_params(), good_cache(), size=size - 1)
        refused(1, "workspace", paged, good_params(), good_cache(), work=None)
        refused(1, "workspace", paged, good_params(), good_cache(), work=PTR + 16)


@pytest.mark.parametrize("call", [write, read])
def test_write_and_read_refuse(call):
    for name in ("k", "v", "cu", "table") + (("kv_len",) if call is write else ()):
        refused(1, "null", call, good_cache(), **{name: None})
    for change in (dict(ts=60), dict(ts=130), dict(hs=0), dict(k=PTR + 8), dict(v=PTR + 4)):
        refused(1, "aligned", call, good_cache(), **change)
    for change in (dict(n=-1), dict(rows=-1), dict(rows=1 << 31), dict(stride=-1)):
        refused(1, "bad size", call, good_cache(), **change)
    refused(4, "bfloat16", call, good_cache(), dt=capi.F32)


def test_empty_calls_do_nothing():
    prompt(good_params(n_seqs=0), q=None)
    prompt(good_params(q_rows=0), o=None)
    paged(good_params(q_rows=0), good_cache())
    write(good_cache(), k=None, n=0)
    read(good_cache(), k=None, rows=0)


def test_the_scale_rule_by_exponent_bits_is_the_smallest_power_of_two():
    """The kernel takes the scale from the exponent field and one comparison of the mantissa; the same
    arithmetic in numpy against the definition, over every bfloat16 and the neighbours of 448 * 2^e."""
    bits = (np.arange(0x7F80, dtype=np.uint32) << 16)
    edges = (np.float32(448.0) * np.exp2(np.arange(-140, 119, dtype=np.float64))).astype(np.float32).view(np.uint32)
    bits = np.concatenate([bits, edges, edges + 1, edges - 1])
    byte = np.maximum((bits >> 23).astype(np.int64) - 8 + ((bits & 0x7FFFFF) > 0x600000), 1)
    amax = bits.view(np.float32).astype(np.float64)
    assert np.array_equal(byte, ref.quantise(amax[:, None])[1])
    assert np.all(amax <= 448.0 * 2.0 ** (byte - 127.0)) and byte.max() < 254


def test_every_code_reads_back_as_itself():
    codes = np.array([c for c in range(256) if c & 127 != 127], dtype=np.uint8)
    again, byte = ref.quantise(np.concatenate([ref.E4M3[codes], [448.0]])[None])
    assert byte[0] == 127 and np.array_equal(again[0, :-1], codes)
