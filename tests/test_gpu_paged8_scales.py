"""Attention over 8-bit pools whose V scales lie far apart, against the 64-bit definition, dim by dim:
a page's scale may come from another dim or from a token that no query sees, so it says nothing
of what the page adds to a dim, and no page may take precision from the others.

Tolerance, per output: half a step of its type; A (2^-11 + 2.4e-4) for the probabilities, which are fp16
whatever the query's type, and the scores (the bound of D + 4 fp32 roundings that
tests/test_gpu_paged8.py derives); 2^-25 B for probabilities below fp16's normal range, whose steps
are 2^-24 of the row's largest; A = sum p |v| and B = sum |v| over the tokens of that dim alone.  There is
no constant: outputs of 2^-40 count as much as those of 2^40 (fp16 outputs end at steps of 2^-24)."""
import numpy as np
import pytest
import torch

from test_gpu_paged8 import F8, clean_status, make_pool, reference  # noqa: F401

pytestmark = pytest.mark.gpu


def check(out, lse, ref, dt):
    o, e, a, b = ref
    bad = torch.isnan(o)
    assert torch.equal(torch.isnan(out), bad)
    tol = torch.finfo(dt).eps / 2 * o.abs() + (2.0 ** -11 + 2.4e-4) * a + 2.0 ** -25 * b
    if dt == torch.float16:
        tol = tol + 2.0 ** -25
    err = (out.double() - o).abs()
    assert (err <= tol)[~bad].all(), (err / tol)[~bad].max().item()
    none = torch.isinf(e)                            # queries that see no token
    assert torch.equal(lse.double()[none], e[none])
    assert ((lse.double() - e)[~none].abs() <= 2e-5).all()


def run(dt, pool, scale, pages, kv, qlen, hq, window=-1, sinks=0):
    from beam_engine_b200.cascade import BatchPrefillWithPagedKVCacheWrapper
    ps, hkv, d = pool.shape[2:]
    q = torch.randn((qlen, hq, d), device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)).to(dt)
    w = BatchPrefillWithPagedKVCacheWrapper(torch.empty(64 << 20, dtype=torch.uint8, device="cuda"))
    w.plan([0, qlen], [0, len(pages)], pages, [(kv - 1) % ps + 1], hq, hkv, d, ps, causal=True,
           window_left=window, num_sinks=sinks, kv_data_type=F8)
    out, lse = w.run(q, pool, return_lse=True, kv_scale=scale)
    return out, lse, reference(q, pool, scale, [0, len(pages)], pages, [kv], [0, qlen], True, window, sinks,
                               d ** -0.5)


def far_first(r, n=8):
    return [r - 8] + [-8] * (n - 1)


SPREADS = {"20 first": far_first(20), "24 first": far_first(24), "26 first": far_first(26),
           "30 first": far_first(30), "48 first": far_first(48),
           "30 last": far_first(30)[::-1], "30 inside": [-8, -8, -8, 22, -8, -8, -8, -8],
           "low first": [-38] + [-8] * 7, "low inside": [-8, -8, -31, -8, -8, -38, -8, -8],
           "ends": [40, -40, 0, -20, 20, -40, 40, 7], "up": list(range(-40, 41, 11)),
           "down": list(range(-40, 41, 11))[::-1], "window edges": [0, -15, -16, 7, 8, -38, -39, 30]}


@pytest.mark.parametrize("qlen", [1, 4, 40, 70])
@pytest.mark.parametrize("d,ps", [(64, 16), (128, 16), (128, 8), (64, 5), (128, 1), (128, 32)])
@pytest.mark.parametrize("spread", sorted(SPREADS))
def test_each_page_in_dims_of_its_own(qlen, d, ps, spread):
    """Eighth j of the dims holds codes of the pages with exponent j alone: what such a dim loses no other
    page covers."""
    exps = SPREADS[spread]
    n, hkv = (8 if ps >= 8 else 24 if ps > 1 else 80), 2
    pool, scale = make_pool(n + 2, ps, hkv, d, torch.bfloat16, True, 1)
    pages = np.random.default_rng(3).permutation(n + 2)[:n].tolist()
    for at, p in enumerate(pages):
        mask = torch.zeros(d, device="cuda")
        mask[at % 8 * (d // 8):(at % 8 + 1) * (d // 8)] = 1
        pool[p, 1] = (pool[p, 1].float() * mask).to(F8)
        scale[p, 1] = 2.0 ** exps[at % 8]
    out, lse, ref = run(torch.bfloat16, pool, scale, pages, n * ps - (ps > 2), qlen, 8)
    check(out, lse, ref, torch.bfloat16)


@pytest.mark.parametrize("qlen", [1, 40])
@pytest.mark.parametrize("ps", [16, 8])
@pytest.mark.parametrize("order", ["first", "last"])
def test_fp16_outputs(qlen, ps, order):
    """fp16 outputs reach from 2^-24 to 2^16: 448 * 2^6 in some dims, 448 * 2^-20 in the others."""
    exps = [6] + [-20] * 7
    exps = exps if order == "first" else exps[::-1]
    pool, scale = make_pool(8, ps, 2, 128, torch.float16, True, 2)
    for p in range(8):
        keep = torch.zeros(128, device="cuda")
        keep[:64 if exps[p] == 6 else 128] = 1
        keep[:64] = 1 if exps[p] == 6 else 0
        pool[p, 1] = (pool[p, 1].float() * keep).to(F8)
        scale[p, 1] = 2.0 ** exps[p]
    out, lse, ref = run(torch.float16, pool, scale, list(range(8)), 8 * ps, qlen, 8)
    check(out, lse, ref, torch.float16)


@pytest.mark.parametrize("qlen", [1, 40])
@pytest.mark.parametrize("r", [20, 26, 40])
@pytest.mark.parametrize("by", ["window", "causal"])
def test_a_scale_that_a_hidden_token_set(qlen, r, by):
    """The far page's wide value is of a token that no query sees: before the window in the first
    page, or in a slot behind the sequence's end in the last."""
    ps, n = 16, 8
    pool, scale = make_pool(n, ps, 2, 128, torch.bfloat16, True, 3)
    scale[:, 1] = 2.0 ** -8
    far, hidden = (0, 3) if by == "window" else (n - 1, 13)
    scale[far, 1] = 2.0 ** (r - 8)
    raw = pool.view(torch.uint8)
    raw[far, 1] = 0
    raw[far, 1, hidden] = 0x7e                      # 448
    kv = n * ps if by == "window" else n * ps - 6
    window = kv - qlen - 8 if by == "window" else -1
    out, lse, ref = run(torch.bfloat16, pool, scale, list(range(n)), kv, qlen, 8, window)
    check(out, lse, ref, torch.bfloat16)


@pytest.mark.parametrize("qlen", [1, 4, 40, 300])
@pytest.mark.parametrize("ps", [16, 5])
@pytest.mark.parametrize("power", [True, False])
def test_exponents_over_the_whole_range(qlen, ps, power):
    """Codes in every dim, exponents from -40 to 40 by page and head (and scales that are no powers of two)."""
    n = 40 if ps == 16 else 130
    pool, scale = make_pool(n, ps, 2, 128, torch.bfloat16, True, 4)
    g = torch.Generator(device="cuda").manual_seed(6)
    scale[:, 1] = torch.ldexp(torch.ones((n, 2), device="cuda"),
                              torch.randint(-40, 40, (n, 2), generator=g, device="cuda"))
    if not power:
        scale[:, 1] *= 1 + torch.rand((n, 2), generator=g, device="cuda")
    out, lse, ref = run(torch.bfloat16, pool, scale, list(range(n)), n * ps, qlen, 8)
    check(out, lse, ref, torch.bfloat16)


@pytest.mark.parametrize("qlen", [1, 40])
def test_long_contexts_split_and_merged(qlen):
    """A far page in one part of a sequence that is split over many CTAs."""
    n, ps = 300, 16
    pool, scale = make_pool(n, ps, 2, 128, torch.bfloat16, True, 5)
    raw = pool.view(torch.uint8)
    for p, e in ((0, 30), (120, 25), (121, -40), (299, 12)):
        scale[p, 1] = 2.0 ** e
        raw[p, 1, :, :, 1:] = 0
        raw[:p, 1, :, :, 0] = 0
    out, lse, ref = run(torch.bfloat16, pool, scale, list(range(n)), n * ps - 3, qlen, 8)
    check(out, lse, ref, torch.bfloat16)


@pytest.mark.parametrize("qlen", [1, 40])
def test_pages_of_zeros_and_pages_never_written(qlen):
    n, ps = 12, 16
    pool, scale = make_pool(n, ps, 2, 64, torch.bfloat16, True, 6)
    scale[:, 1] = 2.0 ** 3
    pool.view(torch.uint8)[::3, 1] = 0
    scale[::3, 1] = 2.0 ** -40
    scale[3, 1] = 0
    out, lse, ref = run(torch.bfloat16, pool, scale, list(range(n)), n * ps, qlen, 8)
    check(out, lse, ref, torch.bfloat16)


@pytest.mark.parametrize("qlen", [1, 3, 7, 40, 150])
@pytest.mark.parametrize("ps", [16, 5])
@pytest.mark.parametrize("at", [0, 90, -3])
@pytest.mark.parametrize("window", [True, False])
def test_nan_in_a_far_page_reaches_the_queries_that_see_it(qlen, ps, at, window):
    kv = 192 if ps == 16 else 200
    at %= kv
    pool, scale = make_pool(kv // ps, ps, 2, 64, torch.bfloat16, True, 7)
    scale[:, 1] = 2.0 ** -8
    scale[at // ps, 1] = 2.0 ** 24
    pool.view(torch.uint8)[at // ps, 1, at % ps, :, 9] = 0x7f
    out, lse, ref = run(torch.bfloat16, pool, scale, list(range(kv // ps)), kv, qlen, 8,
                        window=qlen + 3 if window else -1, sinks=2 if window else 0)
    ok = ~torch.isnan(ref[0])
    assert torch.equal(torch.isnan(out), ~ok)
    check(torch.where(ok, out, torch.zeros_like(out)), lse,
          tuple(torch.where(ok, x, torch.zeros_like(x)) if x.shape == ok.shape else x for x in ref), torch.bfloat16)
