"""Cases of the 8-bit paged KV cache and of sliding-window attention, with their plain forms.

Three operators:

* ``append`` -- keys (rotated to their positions on the way) and values go into a paged cache
  held in e4m3 with one scale for each page, plane (K | V) and KV head; the pages that the call
  touched come back as the values they stand for;
* ``attn`` with ``cache="e4m3"`` -- paged attention that reads such a cache, for single new
  tokens, for chunks and whole prompts, and for beams that share a prompt (two cascade levels);
* ``attn`` with ``window >= 0`` -- a query sees the ``window`` tokens before its own and the first
  ``sinks`` tokens of its sequence, over a 16-bit or an 8-bit cache.

The scale of a block is a power of two: the smallest one under which the largest finite value of
the block is at most 448, never under 2**-40 or over 2**40 and never under the block's scale
before the call, unless the call writes the page's first slot, which begins the block anew.
Where the scale grows, the tokens that were there are rounded to the new one.

Shapes: the 8B decoder's heads (32 query, 8 KV, 128 wide), the 70B decoder's (64, 8, 128), the
tiny model's (4, 2, 64), pages of 16 tokens and, in the drawn cases, of 8 and 32.
"""
import math

import numpy as np
import torch

own = False

E4M3_MAX = 448.0
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _append(name, requests, new, old, hq=32, hkv=8, d=128, page=16, dtype="bf16"):
    return dict(name=name, op="append", requests=requests, new=new, old=old, hq=hq, hkv=hkv, d=d,
                page=page, dtype=dtype)


def _attn(name, requests, new, kv, hq=32, hkv=8, d=128, page=16, dtype="bf16", cache="e4m3",
          window=-1, sinks=0, beams=1, prefix=0, ragged=True):
    return dict(name=name, op="attn", requests=requests, new=new, kv=kv, hq=hq, hkv=hkv, d=d,
                page=page, dtype=dtype, cache=cache, window=window, sinks=sinks, beams=beams,
                prefix=prefix, ragged=ragged)


def listed():
    return [
        # one decode step of 8 prompts x 16 beams: a token each, into partly filled pages
        _append("append-beams", 128, 1, 1024),
        # 8 prompts of 1024 tokens, written by one prefill
        _append("append-prompts", 8, 1024, 0),
        # a few short continuations of the tiny model's heads
        _append("append-tiny", 5, 7, 19, hq=4, hkv=2, d=64, dtype="f16"),
        # a serving batch that decodes one token each, contexts of 2K to 4K
        _attn("cache8-decode", 64, 1, 4096),
        # one long document: a single row, split over the whole GPU
        _attn("cache8-long", 1, 1, 131072),
        # beams: 8 prompts of 1024 tokens x 16 beams with suffixes of their own
        _attn("cache8-beams", 128, 1, 1088, beams=16, prefix=1024),
        # a whole prompt against the cache that it has just filled
        _attn("cache8-prompt", 1, 4096, 4096),
        # three short requests of the tiny model's heads: latency alone
        _attn("cache8-tiny", 3, 1, 33, hq=4, hkv=2, d=64, dtype="f16"),
        # decode with a window: long contexts of which 4096 tokens and 4 sinks are seen
        _attn("window-decode", 64, 1, 16000, cache="same", window=4096, sinks=4),
        # a long prompt under a window of 1024
        _attn("window-prompt", 1, 8192, 8192, cache="same", window=1024, sinks=4),
        # chunks of new tokens after long contexts, window over an 8-bit cache
        _attn("window-chunk8", 3, 517, 6001, window=2048, sinks=16),
        # the tiny model's heads under a short window
        _attn("window-tiny", 2, 5, 77, hq=4, hkv=2, d=64, dtype="f16", cache="same", window=20,
              sinks=3),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    hq, hkv, d = rng.choice([(32, 8, 128), (64, 8, 128), (8, 8, 128), (16, 1, 128), (4, 2, 64),
                             (12, 4, 128), (32, 4, 64), (20, 4, 128)])
    page = rng.choice([8, 16, 16, 32])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    kind = rng.choice(["append", "decode", "decode", "chunk", "beams"])
    if kind == "append":
        requests = _log(rng, 1, 128)
        new = _log(rng, 1, max(1, min(2048, 8192 // requests)))
        return _append("", requests, new, _log(rng, 1, 2000) - 1, hq, hkv, d, page, dtype)
    cache = rng.choice(["e4m3", "same"])
    window = _log(rng, 1, 8192) if cache == "same" or rng.random() < 0.4 else -1
    sinks = rng.choice([0, 1, 4, 16, 100]) if window >= 0 else 0
    if kind == "decode":
        requests = _log(rng, 1, 96)
        kv = _log(rng, 1, max(1, min(65536, 160000 // requests)))
        return _attn("", requests, 1, kv, hq, hkv, d, page, dtype, cache, window, sinks)
    if kind == "beams":
        prompts, beams = rng.randint(1, 6), rng.randint(2, 24)
        prefix = page * _log(rng, 1, 1500 // page)
        return _attn("", prompts * beams, 1, prefix + rng.randint(1, 100), hq, hkv, d, page, dtype,
                     cache, window, sinks, beams, prefix)
    requests = rng.randint(1, 4)
    kv = _log(rng, 2, 6000 // requests)
    new = min(kv, _log(rng, 2, 3000))
    return _attn("", requests, new, kv, hq, hkv, d, page, dtype, cache, window, sinks)


def _lengths(case):
    """(new tokens, tokens in the cache before or with them) of each request; the same for every
    seed, since they are the case's work."""
    n = case["requests"]
    if case["op"] == "append":
        new = [max(1, case["new"] - (i * 13) % (case["new"] // 4 + 1)) for i in range(n)]
        return new, [case["old"] - (i * 29) % (case["old"] // 2 + 1) for i in range(n)]
    if not case["ragged"]:
        return [case["new"]] * n, [case["kv"]] * n
    if case["beams"] > 1:
        tail = case["kv"] - case["prefix"]
        return [1] * n, [case["prefix"] + tail - (i * 7) % ((tail + 1) // 2) for i in range(n)]
    kv = [case["kv"] - (i * 977) % (case["kv"] // 2 + 1) for i in range(n)]
    return [max(1, min(k, case["new"] - (i * 31) % (case["new"] // 2 + 1)))
            for i, k in enumerate(kv)], kv


def work(case):
    new, kv = _lengths(case)
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    elt = 1 if case.get("cache", "e4m3") == "e4m3" else 2
    if case["op"] == "append":
        touched = sum((o + m - 1) // page - o // page + 1 for m, o in zip(new, kv))
        block = 2 * page * hkv * d
        return {"bytes": 2 * sum(new) * hkv * d * (2 + 1) + touched * (block * 3 + 2 * hkv * 8),
                "flops": 3 * sum(new) * hkv * d}
    w, s = case["window"], case["sinks"]
    pairs = tokens = 0
    for i, (m, k) in enumerate(zip(new, kv)):
        lo = k - m                                       # position of the first new token
        p = np.arange(lo, k)
        seen = p + 1 if w < 0 else np.minimum(p + 1, w + 1 + np.minimum(s, np.maximum(p - w, 0)))
        pairs += int(seen.sum())
        read = k if w < 0 else min(k, m + w + s)
        shared = case["prefix"] if case["beams"] > 1 and i % case["beams"] else 0
        tokens += max(0, read - min(read, shared))
    scales = 2 * hkv * 4 * tokens // page if elt == 1 else 0
    return {"bytes": tokens * hkv * 2 * d * elt + scales + sum(new) * hq * (4 * d + 4),
            "flops": 4 * d * hq * pairs}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _rows(counts, total=None):
    """For counts per request: (request of each row, rank of the row in its request)."""
    counts = torch.as_tensor(counts, device="cuda")
    total = int(counts.sum()) if total is None else total
    req = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), counts,
                                  output_size=total)
    return req, torch.arange(total, device="cuda") - (torch.cumsum(counts, 0) - counts)[req]


def _pow2_scale(amax):
    """The block's scale for its largest value (2**-40 for a block of zeros)."""
    m, e = torch.frexp(amax.double())
    e = torch.where(amax == 0, torch.full_like(e, -40), e - 8 - (m <= 0.875).int())
    return torch.ldexp(torch.ones_like(m), e.clamp(-40, 40)).float()


def _page_lists(case, kv, g):
    """Each request's pages, drawn without order from a pool; beams of one prompt share the
    prefix's pages.  Returns (page lists as one tensor, indptr list, pool size)."""
    page, beams, shared = case["page"], case.get("beams", 1), case.get("prefix", 0) // case["page"]
    n_of = [-(-k // page) for k in kv]
    need = sum(n if i % beams == 0 else n - shared for i, n in enumerate(n_of))
    pool = need + need // 8 + 2
    perm = torch.randperm(pool, generator=g, device="cuda").tolist()
    lists, at, head = [], 0, None
    for i, n in enumerate(n_of):
        have = [] if i % beams == 0 or not shared else head[:shared]
        take = n - len(have)
        lists.append(have + perm[at:at + take])
        at += take
        if i % beams == 0:
            head = lists[-1]
    ptr = np.concatenate([[0], np.cumsum(n_of)]).astype(np.int32)
    return [p for row in lists for p in row], lists, ptr, pool


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    new, kv = _lengths(case)
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    dt = DTYPES[case["dtype"]]
    total_kv = [o + m for m, o in zip(new, kv)] if case["op"] == "append" else kv
    flat, lists, ptr, pool = _page_lists(case, total_kv, g)
    st = dict(case=case, flat=torch.tensor(flat, dtype=torch.int32, device="cuda"),
              ptr=torch.tensor(ptr, device="cuda"))
    e4m3 = case["op"] == "append" or case["cache"] == "e4m3"

    if case["op"] == "append":
        # the cache as earlier calls left it: valid tokens rounded to their block's scale
        n = sum(new)
        cache = torch.zeros((pool, 2, page, hkv, d), device="cuda")
        last = torch.tensor([o // page for o in kv], device="cuda") + st["ptr"][:-1]
        tail = st["flat"][last.long()].long()
        fill = torch.tensor([o % page for o in kv], device="cuda")
        live = torch.arange(page, device="cuda")[None, :] < fill[:, None]
        old = torch.randn((len(kv), 2, page, hkv, d), generator=g, device="cuda")
        cache[tail] = old * live[:, None, :, None, None]
        scale = _pow2_scale(cache.abs().amax((2, 4)))
        scale[tail[fill == 0]] = 0
        safe = torch.where(scale > 0, scale, torch.ones_like(scale))
        st["cache"] = (cache / safe[:, :, None, :, None]).to(torch.float8_e4m3fn)
        st["scale"] = scale
        # keys and values in place inside the fused projection's rows, not yet rotated
        qkv = torch.randn((n, (hq + 2 * hkv) * d), generator=g, device="cuda")
        spread = torch.exp(0.5 * torch.randn(((hq + 2 * hkv) * d,), generator=g, device="cuda"))
        st["qkv"] = (qkv * spread).to(dt)
        st["k"] = st["qkv"][:, hq * d:(hq + hkv) * d].view(n, hkv, d)
        st["v"] = st["qkv"][:, (hq + hkv) * d:].view(n, hkv, d)
        req, rank = _rows(new, n)
        st["batch"] = req.int()
        st["pos"] = (rank + torch.tensor(kv, device="cuda")[req]).int()
        st["inv_freq"] = (1.0 / (500000.0 ** (torch.arange(0, d, 2, dtype=torch.int64).float() / d))
                          ).cuda()
        touched = [p for r, (m, o) in zip(lists, zip(new, kv))
                   for p in r[o // page:(o + m - 1) // page + 1]]
        st["touched"] = torch.tensor(touched, dtype=torch.int32, device="cuda")
        if own:
            from beam_engine_b200.page import append_paged_kv_cache, read_paged_kv_cache
            st["append"], st["read"] = append_paged_kv_cache, read_paged_kv_cache
        return st

    # attention: a filled cache, queries inside the fused projection's rows
    n = sum(new)
    cache = torch.randn((pool, 2, page, hkv, d), generator=g, device="cuda")
    spread = torch.exp(0.4 * torch.randn((2, 1, hkv, d), generator=g, device="cuda"))
    cache *= spread
    if e4m3:
        st["scale"] = _pow2_scale(cache.abs().amax((2, 4)))
        cache /= st["scale"][:, :, None, :, None]
        st["cache"] = cache.to(torch.float8_e4m3fn)
    else:
        st["scale"], st["cache"] = None, cache.to(dt)
    del cache
    qkv = 1.5 * torch.randn((n, (hq + 2 * hkv) * d), generator=g, device="cuda")
    st["qkv"] = qkv.to(dt)
    st["q"] = st["qkv"][:, :hq * d].view(n, hq, d)
    st["req"], st["rank"] = _rows(new, n)
    st["new"] = torch.tensor(new, device="cuda")
    st["kv"] = torch.tensor(kv, device="cuda")
    st["most"] = (max(new), -(-max(kv) // page))
    if own:
        st["wrapper"] = _plan(case, new, kv, lists, ptr, dt, e4m3)
    return st


def _plan(case, new, kv, lists, ptr, dt, e4m3):
    from beam_engine_b200.cascade import (BatchPrefillWithPagedKVCacheWrapper,
                                          MultiLevelCascadeAttentionWrapper)
    page = case["page"]
    ws = torch.empty(256 << 20, dtype=torch.uint8, device="cuda")
    last = [(k - 1) % page + 1 for k in kv]
    qo = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    flat = np.asarray([p for row in lists for p in row], np.int32)
    more = dict(causal=True, kv_data_type=torch.float8_e4m3fn if e4m3 else dt,
                window_left=case["window"], num_sinks=case["sinks"])
    if case["beams"] <= 1:
        w = BatchPrefillWithPagedKVCacheWrapper(ws)
        w.plan(qo, ptr, flat, last, case["hq"], case["hkv"], case["d"], page, **more)
        return w
    beams, shared = case["beams"], case["prefix"] // page
    heads = lists[::beams]
    w = MultiLevelCascadeAttentionWrapper(2, ws)
    own_pages = [row[shared:] for row in lists]
    w.plan([np.arange(0, len(kv) + 1, beams, dtype=np.int32), qo],
           [np.arange(0, len(heads) + 1, dtype=np.int32) * shared,
            np.concatenate([[0], np.cumsum([len(r) for r in own_pages])]).astype(np.int32)],
           [np.asarray([p for r in heads for p in r[:shared]], np.int32),
            np.asarray([p for r in own_pages for p in r], np.int32)],
           [[page] * len(heads), last], case["hq"], case["hkv"], case["d"], page, **more)
    return w


# ---------------------------------------------------------------------------
# the operators
# ---------------------------------------------------------------------------
def run(st):
    if st["case"]["op"] == "append":
        return _run_append(st)
    if own:
        out, lse = st["wrapper"].run(st["q"], st["cache"], return_lse=True, kv_scale=st["scale"])
        return {"out": out, "lse": lse}
    return _plain_attention(st)


def _run_append(st):
    if own:
        st["append"](st["k"], st["v"], st["batch"], st["pos"], st["cache"], st["flat"], st["ptr"],
                     kv_scale=st["scale"], rope_inv_freq=st["inv_freq"])
        return {"pages": st["read"](st["cache"], st["touched"], kv_scale=st["scale"])}
    page, cache, scale = st["case"]["page"], st["cache"].view(torch.uint8), st["scale"]
    d, t = st["case"]["d"], st["touched"].long()
    pos = st["pos"].long()
    pages = st["flat"][st["ptr"][st["batch"].long()].long() + pos // page].long()
    slot = pos % page
    # rotation: angles of far positions and values next to a rounding border need 64 bits
    ang = pos.double()[:, None] * st["inv_freq"].double()
    cos, sin = ang.cos()[:, None], ang.sin()[:, None]
    k = st["k"].double()
    lo, hi = k[..., :d // 2], k[..., d // 2:]
    rows = torch.stack([torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1),
                        st["v"].double()], 1)                              # [n, 2, hkv, d]
    amax = torch.zeros_like(scale, dtype=torch.float64)
    amax.index_reduce_(0, pages, rows.abs().amax(-1), "amax")
    fresh = torch.zeros(scale.shape[0], dtype=torch.bool, device="cuda")
    fresh[pages[slot == 0]] = True
    before = torch.where(fresh[t][:, None, None], torch.zeros_like(scale[t]), scale[t])
    after = torch.maximum(before, _pow2_scale(amax[t]))
    # tokens that were there are rounded to the scale where it grew (not in a page begun anew)
    ratio = torch.where(fresh[t][:, None, None], torch.ones_like(after), before / after)
    kept = cache[t].view(torch.float8_e4m3fn).float() * ratio[:, :, None, :, None]
    cache[t] = kept.to(torch.float8_e4m3fn).view(torch.uint8)
    scale[t] = after
    codes = (rows / scale[pages][..., None]).float().to(torch.float8_e4m3fn).view(torch.uint8)
    cache[pages, :, slot] = codes
    back = cache[t].view(torch.float8_e4m3fn).float() * after[:, :, None, :, None]
    return {"pages": back.to(torch.bfloat16)}


def _plain_attention(st):
    case = st["case"]
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    most_q, most_p = st["most"]
    n_req, dt = len(st["new"]), st["q"].dtype
    # every request's pages, padded: [requests, tokens, kv heads, d] in 32 bits
    at = st["ptr"][:-1, None].long() + torch.arange(most_p, device="cuda")
    ids = st["flat"][at.clamp(max=st["flat"].numel() - 1)].long()
    if st["scale"] is None:
        kv = st["cache"][ids].float()
    else:
        kv = st["cache"].view(torch.uint8)[ids].view(torch.float8_e4m3fn).float()
        kv *= st["scale"][ids][:, :, :, None, :, None]
    k, v = (kv[:, :, i].reshape(n_req, most_p * page, hkv, d) for i in (0, 1))
    q = torch.zeros((n_req, most_q, hq, d), device="cuda")
    q[st["req"], st["rank"]] = st["q"].float()
    tok = torch.arange(most_p * page, device="cuda")
    p = (st["kv"] - st["new"])[:, None] + torch.arange(most_q, device="cuda")     # positions
    see = (tok <= p[..., None]) & (tok < st["kv"][:, None, None])
    if case["window"] >= 0:
        see &= (tok >= p[..., None] - case["window"]) | (tok < case["sinks"])
    v = torch.where((tok < st["kv"][:, None])[..., None, None], v, torch.zeros_like(v))
    q = q.view(n_req, most_q, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4) * d ** -0.5
    s = torch.matmul(q.reshape(n_req, hkv, -1, d), k.permute(0, 2, 3, 1))
    s = s.view(n_req, hkv, hq // hkv, most_q, -1)
    s.masked_fill_(~see[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp_min(-3e38)
    s.sub_(top).exp_()
    den = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(n_req, hkv, -1, s.shape[-1]), v.permute(0, 2, 1, 3))
    o = o.view(n_req, hkv, hq // hkv, most_q, d) / torch.where(den > 0, den, torch.ones_like(den))
    lse = (top + den.log()).squeeze(-1).permute(0, 3, 1, 2).reshape(n_req, most_q, hq)
    o = o.permute(0, 3, 1, 2, 4).reshape(n_req, most_q, hq, d)
    return {"out": o[st["req"], st["rank"]].to(dt), "lse": lse[st["req"], st["rank"]]}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _round_e4m3(x):
    """Values in 64 bits rounded to the nearest of 4 significant bits, ties to even: exponents
    from -6 (below it steps of 2**-9) to 8, at most 448."""
    e = torch.frexp(x)[1].clamp_min(-5) - 1
    step = torch.ldexp(torch.ones_like(x), e - 3)
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def exact(case, seed):
    st = prepare(dict(case), seed)
    page, d, hkv = case["page"], case["d"], case["hkv"]
    g = case["hq"] // hkv
    flat, ptr = st["flat"].tolist(), st["ptr"].tolist()
    new, kv = _lengths(case)
    if case["op"] == "append":
        steps = torch.ldexp(torch.ones(81, dtype=torch.float64, device="cuda"),
                            torch.arange(-40, 41, device="cuda"))
        value = st["cache"].double() * st["scale"].double()[:, :, None, :, None]
        pos = st["pos"].double()
        turn = torch.outer(pos, st["inv_freq"].double())
        z = torch.polar(torch.ones_like(turn), turn)[:, None]
        k, at = st["k"].double(), 0
        z = torch.complex(k[..., :d // 2], k[..., d // 2:]) * z
        rows = torch.stack([torch.cat([z.real, z.imag], -1), st["v"].double()], 1)
        out = []
        for i, (m, o) in enumerate(zip(new, kv)):
            for j in range(o // page, (o + m - 1) // page + 1):
                p, lo, hi = flat[ptr[i] + j], max(o, j * page), min(o + m, (j + 1) * page)
                r = rows[at + lo - o:at + hi - o]                            # [t, 2, hkv, d]
                top = r.abs().amax((0, 3))[..., None] / E4M3_MAX
                scale = steps[(steps >= top).double().argmax(-1)]     # the first that holds it
                if lo % page:
                    scale = torch.maximum(scale, st["scale"][p].double())
                b = scale[:, None, :, None]
                value[p] = _round_e4m3(value[p] / b) * b
                value[p, :, lo % page:(hi - 1) % page + 1] = (
                    _round_e4m3(r / scale[None, :, :, None]) * scale[None, :, :, None]
                ).transpose(0, 1)
                out.append(value[p])
            at += m
        return {"pages": torch.stack(out)}
    out, lse, at = [], [], 0
    for i, (m, k) in enumerate(zip(new, kv)):
        ids = torch.tensor(flat[ptr[i]:ptr[i + 1]], device="cuda")
        block = st["cache"].view(torch.uint8 if st["scale"] is not None else st["cache"].dtype)[ids]
        if st["scale"] is not None:
            block = block.view(torch.float8_e4m3fn).double()
            block = block * st["scale"][ids].double()[:, :, None, :, None]
        block = block.double().transpose(0, 1).reshape(2, -1, hkv, d)[:, :k]
        t = torch.arange(k, device="cuda")
        p = torch.arange(k - m, k, device="cuda")[:, None]
        see = t <= p
        if case["window"] >= 0:
            see &= (p - t <= case["window"]) | (t < case["sinks"])
        q = st["q"][at:at + m].double().view(m, hkv, g, d)
        o = torch.empty((m, hkv, g, d), dtype=torch.float64, device="cuda")
        e = torch.empty((m, hkv, g), dtype=torch.float64, device="cuda")
        for h in range(hkv):
            x = torch.einsum("mgd,td->mgt", q[:, h], block[0, :, h]) / math.sqrt(d)
            x = torch.where(see[:, None], x, torch.full_like(x, -math.inf))
            e[:, h] = torch.logsumexp(x, -1)
            o[:, h] = torch.einsum("mgt,td->mgd", torch.exp(x - e[:, h, :, None]), block[1, :, h])
        out.append(o.reshape(m, hkv * g, d))
        lse.append(e.reshape(m, hkv * g))
        at += m
    return {"out": torch.cat(out), "lse": torch.cat(lse)}
