"""Attention for serving: whole prompts, and new tokens over a paged key/value cache, with the
cache's quantising write and its read-back.  Each case is one call a serving loop makes:

  prompt   causal attention of packed prompts of different lengths, grouped heads
           (fb200_attention_prompt)
  write    storing the keys and values of new tokens into cache pages, as 16-bit numbers or as
           e4m3 codes with one power-of-two scale per token and head (fb200_kv_cache_write)
  read     the cached tokens of every sequence back as one dense 16-bit tensor
           (fb200_kv_cache_read)
  paged    one to many new tokens per sequence attending to everything the cache holds of it
           (fb200_attention_paged)

`run` computes the operator from elementary torch operations in 32 bits, or, where `own` is true,
with this repository's kernels.  Sequence lengths follow from the case alone, values and the pages'
order in memory from the seed.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
E4M3_MAX = 448.0


# ---- cases ---------------------------------------------------------------------------------------
def listed():
    return [
        # one short chat turn on a small model: the latency of a call
        dict(name="prompt one short", kind="prompt", dtype="bf16", n=1, heads=16, kv_heads=16, dim=64,
             q_min=100, q_max=100),
        # the heads, batch and length of this repository's transformer block workload, made causal
        dict(name="prompt 8x512 d64", kind="prompt", dtype="bf16", n=8, heads=16, kv_heads=16, dim=64,
             q_min=512, q_max=512),
        # a server's batch of prompts of very different lengths, packed without padding
        dict(name="prompt ragged", kind="prompt", dtype="f16", n=24, heads=20, kv_heads=4, dim=128,
             q_min=9, q_max=2000),
        # two long documents
        dict(name="prompt 2x8192", kind="prompt", dtype="bf16", n=2, heads=16, kv_heads=2, dim=128,
             q_min=8192, q_max=8192),
        # one decoding step of a batch: one token each
        dict(name="write step e4m3", kind="write", dtype="bf16", n=32, heads=8, kv_heads=8, dim=128,
             q_min=1, q_max=1, kv_min=40, kv_max=4000, page=16, cache="e4m3", order="head"),
        # the prompts of a batch on their way into the cache
        dict(name="write prompts e4m3", kind="write", dtype="bf16", n=16, heads=8, kv_heads=8, dim=128,
             q_min=200, q_max=4000, kv_min=200, kv_max=4000, page=64, cache="e4m3", order="head"),
        # a cached prefix read back for a dense prompt pass, head size of the transformer block workload
        dict(name="read few f16", kind="read", dtype="f16", n=3, heads=16, kv_heads=16, dim=64,
             q_min=1, q_max=1, kv_min=70, kv_max=700, page=32, cache="same", order="token"),
        # a whole batch's cache read back
        dict(name="read batch e4m3", kind="read", dtype="bf16", n=32, heads=8, kv_heads=8, dim=128,
             q_min=1, q_max=1, kv_min=300, kv_max=5000, page=64, cache="e4m3", order="head"),
        # decoding at a small batch and short contexts: the latency of a call
        dict(name="decode 4 short", kind="paged", dtype="bf16", n=4, heads=16, kv_heads=16, dim=64,
             q_min=1, q_max=1, kv_min=33, kv_max=513, page=16, cache="same", order="token"),
        # decoding at a large batch over a 16-bit cache
        dict(name="decode 64", kind="paged", dtype="bf16", n=64, heads=32, kv_heads=8, dim=128,
             q_min=1, q_max=1, kv_min=500, kv_max=8000, page=64, cache="same", order="head"),
        # decoding a few long conversations over a quantised cache
        dict(name="decode 8 long e4m3", kind="paged", dtype="bf16", n=8, heads=32, kv_heads=8, dim=128,
             q_min=1, q_max=1, kv_min=8000, kv_max=32000, page=32, cache="e4m3", order="head"),
        # the next chunk of some long prompts
        dict(name="chunk 4x512", kind="paged", dtype="bf16", n=4, heads=32, kv_heads=4, dim=128,
             q_min=512, q_max=512, kv_min=2500, kv_max=12000, page=64, cache="same", order="head"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["prompt", "write", "read", "paged", "paged", "chunk"])
    dim = rng.choice([64, 64, 128, 128, 80, 96])
    group = rng.choice([1, 2, 4, 8, 3, 5, 7])
    kv_heads = rng.choice([1, 2, 4, 8])
    case = dict(kind="paged" if kind == "chunk" else kind, dtype=rng.choice(["bf16", "bf16", "f16"]),
                heads=kv_heads * group, kv_heads=kv_heads, dim=dim)
    if kind == "prompt":
        hi = _log(rng, 1, 5000)
        room = int(4.0e8 / (hi * hi * case["heads"])) + 1    # padded scores of the plain form
        case.update(n=min(_log(rng, 1, 48), room), q_min=_log(rng, 1, hi), q_max=hi)
        return case
    hi = _log(rng, 1, 16000)
    case.update(kv_min=_log(rng, 1, hi), kv_max=hi, page=rng.choice([16, 32, 64, 128]),
                cache=rng.choice(["same", "e4m3"]), order=rng.choice(["head", "token"]))
    new = 1 if kind in ("paged", "read") else _log(rng, 1, min(hi, 1024))
    if kind == "paged" and rng.random() < 0.4:
        new = _log(rng, 1, min(hi, 16))
    case.update(q_min=min(new, case["kv_min"]), q_max=new)
    room = int(6.0e7 / (hi * kv_heads * dim)) + 1             # padded keys of the plain form
    room = min(room, int(4.0e8 / (new * hi * case["heads"])) + 1)
    case["n"] = min(_log(rng, 1, 96), room)
    return case


def _spread(lo, hi, n, turn):
    """n lengths between lo and hi, evenly over the logarithm in a scattered order; the first is hi."""
    fracs = [1.0 - ((i * turn) % 1.0) for i in range(n)]
    return [max(lo, min(hi, int(round(lo * (hi / lo) ** f)))) for f in fracs]


def _lengths(case):
    q = _spread(case["q_min"], case["q_max"], case["n"], 0.7548776662)
    if case["kind"] == "prompt":
        return q, q
    kv = _spread(case["kv_min"], case["kv_max"], case["n"], 0.6180339887)
    if case["kind"] == "write" and case["q_max"] > 1 and case["q_min"] == case["kv_min"]:
        q = kv                                                # whole prompts
    return [min(a, b) for a, b in zip(q, kv)], kv


# ---- inputs --------------------------------------------------------------------------------------
def _prefix(lens, device):
    out = [0]
    for v in lens:
        out.append(out[-1] + v)
    return torch.tensor(out, dtype=torch.int32, device=device)


def _activations(gen, rows, heads, dim, dtype, device):
    """Projections as a trained layer gives them: normal values, some channels larger than others."""
    gain = torch.exp(0.4 * torch.randn(heads, dim, generator=gen, device=device))
    return (torch.randn(rows, heads, dim, generator=gen, device=device) * gain).to(dtype)


def prepare(case, seed):
    device = "cuda"
    gen = torch.Generator(device=device).manual_seed(int(seed))
    dtype, heads, kv_heads, dim = DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]
    q_lens, kv_lens = _lengths(case)
    n, rows = case["n"], sum(q_lens)
    s = dict(kind=case["kind"], case=case, scale=1.0 / math.sqrt(dim), cu_q=_prefix(q_lens, device),
             max_q=max(q_lens), max_kv=max(kv_lens))
    if case["kind"] == "prompt":
        # one fused projection, as a model's QKV matrix leaves it
        fused = _activations(gen, rows, heads + 2 * kv_heads, dim, dtype, device)
        s.update(q=fused[:, :heads], k=fused[:, heads:heads + kv_heads], v=fused[:, heads + kv_heads:],
                 o=torch.zeros(rows, heads, dim, dtype=dtype, device=device))
    else:
        page = case["page"]
        per_seq = [-(-v // page) for v in kv_lens]
        pages = sum(per_seq) + 3
        order = torch.randperm(pages, generator=gen, device=device).to(torch.int32)
        table = torch.zeros(n, max(per_seq), dtype=torch.int32, device=device)
        at = 0
        for i, c in enumerate(per_seq):
            table[i, :c] = order[at:at + c]
            at += c
        s.update(kv_len=torch.tensor(kv_lens, dtype=torch.int32, device=device), table=table,
                 cu_kv=_prefix(kv_lens, device))
        if case["kind"] == "write":
            s.update(k=_activations(gen, rows, kv_heads, dim, dtype, device),
                     v=_activations(gen, rows, kv_heads, dim, dtype, device))
        elif case["kind"] == "paged":
            s.update(q=_activations(gen, rows, heads, dim, dtype, device),
                     o=torch.zeros(rows, heads, dim, dtype=dtype, device=device))
        else:
            total = sum(kv_lens)
            s.update(k_out=torch.zeros(total, kv_heads, dim, dtype=dtype, device=device),
                     v_out=torch.zeros(total, kv_heads, dim, dtype=dtype, device=device))
        shape = (pages, kv_heads, page, dim) if case["order"] == "head" else (pages, page, kv_heads, dim)

        def stored():
            x = _activations(gen, pages * page, kv_heads, dim, dtype, device)
            x = x.view(pages, page, kv_heads, dim)
            x = x.transpose(1, 2).contiguous() if case["order"] == "head" else x
            if case["cache"] == "same":
                return x, None
            codes, exps = _quantise(x.float())
            return codes, exps

        s["k_cache"], s["k_scale"] = stored()
        s["v_cache"], s["v_scale"] = stored()
        assert tuple(s["k_cache"].shape) == shape
        s["head_major"] = case["order"] == "head"
    if own:
        _prepare_own(s)
    return s


# ---- the plain form ------------------------------------------------------------------------------
def _pow2(e):
    """2^e in fp32 from its exponent bits, -126 <= e <= 127 (128: infinity)."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantise(x):
    """e4m3 codes (bytes) and exponent bytes of fp32 rows: the scale is the smallest power of two
    2^e, e >= -126, with max|row| <= 448 * 2^e; byte e + 127, and 255 where a row is not finite."""
    amax = x.abs().amax(-1)
    mant, ex = torch.frexp(amax)
    e = torch.where(mant > 0.875, ex - 8, ex - 9).clamp(min=-126)
    e = torch.where(amax > 0, e, torch.full_like(e, -126))
    fine = torch.isfinite(amax)
    e = torch.where(fine, e, torch.zeros_like(e))
    y = torch.where(fine[..., None], x * _pow2(-e)[..., None], torch.zeros_like(x))
    codes = y.to(torch.float8_e4m3fn).view(torch.uint8)
    exps = torch.where(fine, e + 127, torch.full_like(e, 255)).to(torch.uint8)
    return codes, exps


def _values(codes, exps):
    """What a cache holds, in fp32."""
    if exps is None:
        return codes.float()
    return codes.view(torch.float8_e4m3fn).float() * _pow2(exps.to(torch.int32) - 127)[..., None]


def _padded(cu, length):
    """Row numbers [n, length] of packed sequences, and which of them exist."""
    cu = cu.long()
    i = torch.arange(length, device=cu.device)
    there = i[None, :] < (cu[1:] - cu[:-1])[:, None]
    return torch.where(there, cu[:-1, None] + i[None, :], torch.zeros_like(cu[:-1, None])), there


def _gather_pages(cache, s, length):
    """[n, length, kv_heads, ...] of every sequence's first `length` cached tokens."""
    page = s["case"]["page"]
    i = torch.arange(length, device=cache.device)
    ids = s["table"].long()[:, (i // page).clamp(max=s["table"].shape[1] - 1)]
    tok = (i % page)[None, :].expand_as(ids)
    return cache[ids, :, tok] if s["head_major"] else cache[ids, tok]


def _attend(q, k, v, seen, scale):
    """q [n, lq, h, d], k and v [n, lk, hk, d] in fp32, seen [n, lq, lk]: softmax over the seen keys."""
    n, lq, h, d = q.shape
    hk = k.shape[2]
    qg = q.view(n, lq, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(n, hk, (h // hk) * lq, d)
    sc = torch.matmul(qg, k.permute(0, 2, 3, 1)).view(n, hk, h // hk, lq, -1) * scale
    sc = sc.masked_fill(~seen[:, None, None], float("-inf"))
    top = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(top > float("-inf"), top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, hk, (h // hk) * lq, -1), v.permute(0, 2, 1, 3)).view(n, hk, h // hk, lq, d)
    o = o / torch.where(total > 0, total, torch.ones_like(total))
    return o.permute(0, 3, 1, 2, 4).reshape(n, lq, h, d)


def _plain_attention(s, k, v, kv_len):
    """k, v [n, lk, hk, d] fp32, zero where a sequence has ended."""
    rows, there = _padded(s["cu_q"], s["max_q"])
    q_len = (s["cu_q"][1:] - s["cu_q"][:-1]).long()
    i = torch.arange(s["max_q"], device=k.device)
    j = torch.arange(k.shape[1], device=k.device)
    last = i[None, :] + (kv_len - q_len)[:, None]               # the last key that query i may see
    seen = (j[None, None, :] <= last[:, :, None]) & (j[None, None, :] < kv_len[:, None, None])
    o = _attend(s["q"].float()[rows], k, v, seen, s["scale"])
    out = torch.zeros_like(s["o"])
    out[rows[there]] = o[there].to(out.dtype)
    return out


def _run_plain(s):
    if s["kind"] == "prompt":
        rows, there = _padded(s["cu_q"], s["max_q"])
        k, v = (torch.where(there[:, :, None, None], s[t].float()[rows], torch.zeros((), device=rows.device))
                for t in ("k", "v"))
        return _plain_attention(s, k, v, (s["cu_q"][1:] - s["cu_q"][:-1]).long())
    if s["kind"] == "write":
        page = s["case"]["page"]
        q_len = (s["cu_q"][1:] - s["cu_q"][:-1]).long()
        rows, there = _padded(s["cu_q"], s["max_q"])
        pos = torch.arange(s["max_q"], device=rows.device)[None, :] + (s["kv_len"].long() - q_len)[:, None]
        ids = torch.gather(s["table"].long(), 1, (pos // page).clamp(0, s["table"].shape[1] - 1))[there]
        tok, rows = (pos % page)[there], rows[there]
        out = []
        for name in ("k", "v"):
            x, cache, scale = s[name][rows], s[name + "_cache"], s[name + "_scale"]
            if scale is None:
                if s["head_major"]:
                    cache[ids, :, tok] = x
                else:
                    cache[ids, tok] = x
                out.append(cache)
                continue
            codes, exps = _quantise(x.float())
            if s["head_major"]:
                cache[ids, :, tok] = codes
                scale[ids, :, tok] = exps
            else:
                cache[ids, tok] = codes
                scale[ids, tok] = exps
            out += [cache.view(torch.float8_e4m3fn), scale]
        return out
    length = s["max_kv"]
    got = []
    for name in ("k", "v"):
        codes = _gather_pages(s[name + "_cache"], s, length)
        exps = _gather_pages(s[name + "_scale"], s, length) if s[name + "_scale"] is not None else None
        got.append(_values(codes, exps))
    kv_len = s["kv_len"].long()
    there = torch.arange(length, device=kv_len.device)[None, :] < kv_len[:, None]
    if s["kind"] == "read":
        rows, _ = _padded(s["cu_kv"], length)
        out = []
        for x, name in zip(got, ("k_out", "v_out")):
            dense = torch.zeros_like(s[name])
            dense[rows[there]] = x[there].to(dense.dtype)
            out.append(dense)
        return out
    k, v = (torch.where(there[:, :, None, None], x, torch.zeros((), device=x.device)) for x in got)
    return _plain_attention(s, k, v, kv_len)


# ---- the framework's calls -----------------------------------------------------------------------
def _prepare_own(s):
    """What a serving program keeps beside its tensors: the call's description and a workspace."""
    from frame_public_b200 import capi
    case = s["case"]
    dt = {"bf16": capi.BF16, "f16": capi.F16}[case["dtype"]]
    s["dt"], s["capi"] = dt, capi
    if case["kind"] in ("prompt", "paged"):
        q, o = s["q"], s["o"]
        p = capi.AttentionParams(n_seqs=case["n"], heads=case["heads"], kv_heads=case["kv_heads"],
                                 head_dim=case["dim"], q_rows=q.shape[0], max_q=s["max_q"], max_kv=s["max_kv"],
                                 q_token_stride=q.stride(0), q_head_stride=q.stride(1),
                                 o_token_stride=o.stride(0), o_head_stride=o.stride(1),
                                 scale=s["scale"], causal=1, dtype=dt)
        if case["kind"] == "prompt":
            p.kv_rows = s["k"].shape[0]
            p.k_token_stride, p.k_head_stride = s["k"].stride(0), s["k"].stride(1)
            p.v_token_stride, p.v_head_stride = s["v"].stride(0), s["v"].stride(1)
        s["params"] = p
    if case["kind"] != "prompt":
        c = s["k_cache"]
        tok, head = (2, 1) if s["head_major"] else (1, 2)
        s["cache"] = capi.KvCache(k=c.data_ptr(), v=s["v_cache"].data_ptr(), pages=c.shape[0],
                                  page_size=case["page"], kv_heads=case["kv_heads"], head_dim=case["dim"],
                                  page_stride=c.stride(0), token_stride=c.stride(tok), head_stride=c.stride(head),
                                  dtype=dt if case["cache"] == "same" else capi.U8)
        if s["k_scale"] is not None:
            e = s["k_scale"]
            s["cache"].k_scale, s["cache"].v_scale = e.data_ptr(), s["v_scale"].data_ptr()
            s["cache"].scale_page_stride = e.stride(0)
            s["cache"].scale_token_stride, s["cache"].scale_head_stride = e.stride(tok), e.stride(head)
    if case["kind"] == "paged":
        size = capi.attention_paged_workspace(s["params"], s["cache"])
        s["work"] = torch.zeros(max(size, 1), dtype=torch.uint8, device=s["q"].device)


def _run_own(s):
    capi = s["capi"]
    stream = torch.cuda.current_stream().cuda_stream
    if s["kind"] == "prompt":
        capi.attention_prompt(s["params"], s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(),
                              s["o"].data_ptr(), s["cu_q"].data_ptr(), s["cu_q"].data_ptr(), stream=stream)
        return s["o"]
    table = s["table"]
    if s["kind"] == "paged":
        capi.attention_paged(s["params"], s["cache"], s["q"].data_ptr(), s["o"].data_ptr(), s["cu_q"].data_ptr(),
                             s["kv_len"].data_ptr(), table.data_ptr(), table.stride(0), s["work"].data_ptr(),
                             s["work"].numel(), stream=stream)
        return s["o"]
    if s["kind"] == "write":
        k, v = s["k"], s["v"]
        capi.kv_cache_write(s["cache"], k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
                            v.stride(1), s["cu_q"].data_ptr(), s["kv_len"].data_ptr(), table.data_ptr(),
                            table.stride(0), s["case"]["n"], k.shape[0], s["dt"], stream=stream)
        if s["k_scale"] is None:
            return [s["k_cache"], s["v_cache"]]
        return [s["k_cache"].view(torch.float8_e4m3fn), s["k_scale"],
                s["v_cache"].view(torch.float8_e4m3fn), s["v_scale"]]
    k, v = s["k_out"], s["v_out"]
    capi.kv_cache_read(s["cache"], k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
                       s["cu_kv"].data_ptr(), table.data_ptr(), table.stride(0), s["case"]["n"], k.shape[0],
                       s["dt"], stream=stream)
    return [k, v]


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


# ---- work and exact values -----------------------------------------------------------------------
def work(case):
    q_lens, kv_lens = _lengths(case)
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    pairs = sum(a * b - a * (a - 1) // 2 for a, b in zip(q_lens, kv_lens))
    per_token = hk * (d + 1) if case.get("cache") == "e4m3" else hk * d * 2    # one of K and V
    if case["kind"] == "prompt":
        return dict(bytes=2 * sum(q_lens) * d * (2 * h + 2 * hk), flops=4 * h * d * pairs)
    if case["kind"] == "paged":
        return dict(bytes=2 * sum(q_lens) * d * 2 * h + 2 * sum(kv_lens) * per_token, flops=4 * h * d * pairs)
    tokens = sum(q_lens) if case["kind"] == "write" else sum(kv_lens)
    return dict(bytes=2 * tokens * (per_token + 2 * hk * d), flops=0)


def _e4m3_values(device):
    """The 256 values of the format in 64 bits: sign, four exponent bits (bias 7), three of mantissa."""
    vals = []
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        x = math.nan if c & 127 == 127 else x
        vals.append(-x if c & 128 else x)
    return torch.tensor(vals, dtype=torch.float64, device=device)


def _nearest_e4m3(x):
    """The format's value nearest to each of x (64 bits, at most 448), ties to the even code."""
    grid = _e4m3_values(x.device)[:127]
    at = torch.searchsorted(grid, x.abs().contiguous()).clamp(1, 126)
    low, high = x.abs() - grid[at - 1], grid[at] - x.abs()
    at = torch.where((low < high) | ((low == high) & ((at - 1) % 2 == 0)), at - 1, at)
    return torch.copysign(grid[at], x)


def exact(case, seed):
    if own:
        return None
    s = prepare(case, seed)
    q_lens, kv_lens = _lengths(case)
    if case["kind"] == "write":
        out = []
        for t in ("k", "v"):
            coded, at = s[t + "_scale"] is not None, 0
            cache = s[t + "_cache"]
            cache = _e4m3_values(cache.device)[cache.long()] if coded else cache.double()
            by_token = cache.transpose(1, 2) if s["head_major"] else cache
            for i, (lq, lk) in enumerate(zip(q_lens, kv_lens)):
                x = s[t][at:at + lq].double()
                at += lq
                if coded:                       # the smallest 2^e with max|x| <= 448 * 2^e
                    amax = x.abs().amax(-1, keepdim=True)
                    tries = torch.arange(-126, 128, device=x.device)
                    scales = ((tries + 1023) << 52).view(torch.float64)
                    x = _nearest_e4m3(x / scales[torch.searchsorted(E4M3_MAX * scales, amax)])
                pos = torch.arange(lk - lq, lk, device=x.device)
                by_token[s["table"][i].long()[pos // case["page"]], pos % case["page"]] = x
            out += [cache, None] if coded else [cache]
        return out
    pairs = sum(a * b for a, b in zip(q_lens, kv_lens)) * case["heads"] * case["dim"]
    if pairs > 8e11:
        return None
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]

    def cached(name, i):
        page = case["page"]
        ids = s["table"][i, :-(-kv_lens[i] // page)].long()
        x, e = s[name + "_cache"][ids], s[name + "_scale"]
        x = _e4m3_values(x.device)[x.long()] if e is not None else x.double()
        if e is not None:
            x = x * ((e[ids].long() - 127 + 1023) << 52).view(torch.float64)[..., None]
        x = x.transpose(1, 2) if s["head_major"] else x
        return x.reshape(-1, hk, d)[:kv_lens[i]]

    if case["kind"] == "read":
        return [torch.cat([cached(t, i) for i in range(case["n"])]) for t in ("k", "v")]
    parts, at = [], 0
    for i, (lq, lk) in enumerate(zip(q_lens, kv_lens)):
        q = s["q"][at:at + lq].double()
        if case["kind"] == "prompt":
            k, v = s["k"][at:at + lq].double(), s["v"][at:at + lq].double()
        else:
            k, v = cached("k", i), cached("v", i)
        at += lq
        hidden = torch.ones(lq, lk, dtype=torch.bool, device=q.device).triu(lk - lq + 1)
        out = torch.empty(lq, h, d, dtype=torch.float64, device=q.device)
        for j in range(h):
            sc = (q[:, j] @ k[:, j // (h // hk)].T * s["scale"]).masked_fill(hidden, -math.inf)
            out[:, j] = torch.softmax(sc, -1) @ v[:, j // (h // hk)]
        parts.append(out)
    return torch.cat(parts)
