"""8-bit and windowed attention: layouts of queries, the merge of many rows, and probabilities of wide
tiles over 8-bit caches held to fp16 (the bounds are those of tests/test_gpu_paged8_scales.py)."""
import numpy as np
import pytest
import torch

from test_gpu_paged8 import F8, clean_status, make_pool, reference, status  # noqa: F401
from test_gpu_paged8_scales import check, run

from beam_engine_b200 import _lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qlen", [1, 40])
@pytest.mark.parametrize("shift", [1, 4, 8])
@pytest.mark.parametrize("form", ["contiguous", "rows apart", "heads apart", "dims apart"])
def test_queries_of_any_layout(qlen, shift, form):
    """Queries that start off a 16-byte border, and strides of every kind, give what a copy gives."""
    from beam_engine_b200.cascade import BatchPrefillWithPagedKVCacheWrapper
    pool, scale = make_pool(6, 16, 2, 64, torch.bfloat16, True, 1)
    g = torch.Generator(device="cuda").manual_seed(1)
    flat = torch.randn(qlen * 8 * 64 * 4 + 64, generator=g, device="cuda").bfloat16()[shift:]
    q = {"contiguous": lambda: flat[:qlen * 512].view(qlen, 8, 64),
         "rows apart": lambda: flat.as_strided((qlen, 8, 64), (520 + shift, 64, 1), flat.storage_offset()),
         "heads apart": lambda: flat.as_strided((qlen, 8, 64), (8 * 72, 72, 1), flat.storage_offset()),
         "dims apart": lambda: flat.as_strided((qlen, 8, 64), (1024, 128, 2), flat.storage_offset())}[form]()
    w = BatchPrefillWithPagedKVCacheWrapper(torch.empty(8 << 20, dtype=torch.uint8, device="cuda"))
    w.plan([0, qlen], [0, 6], list(range(6)), [7], 8, 2, 64, 16, causal=True, kv_data_type=F8)
    want = w.run(q.clone(memory_format=torch.contiguous_format), pool, return_lse=True, kv_scale=scale)
    got = w.run(q, pool, return_lse=True, kv_scale=scale)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("hq,d,ps,qlen,kv,window,sinks", [
    (8, 128, 16, 300, 1100, -1, 0), (8, 128, 16, 300, 1100, 300, 130), (8, 64, 8, 129, 700, 77, 5),
    (8, 128, 5, 70, 333, -1, 0), (16, 64, 32, 256, 256, 40, 0), (8, 128, 16, 40, 4000, -1, 0)])
def test_wide_tiles_hold_probabilities_in_fp16(hq, d, ps, qlen, kv, window, sinks):
    """bf16 queries over 8 bits: 2^-11 per probability, not the query type's 2^-8."""
    n = -(-kv // ps)
    pool, scale = make_pool(n, ps, 2, d, torch.bfloat16, True, 3)
    pages = np.random.default_rng(0).permutation(n).tolist()
    out, lse, ref = run(torch.bfloat16, pool, scale, pages, kv, qlen, hq, window, sinks)
    check(out, lse, ref, torch.bfloat16)


@pytest.mark.parametrize("cache8", [True, False])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_merge_of_many_rows(cache8, dt):
    """8 prompts x 32 beams at 32 heads: 8192 merged rows, past the kernel that takes a CTA per row."""
    from beam_engine_b200.cascade import MultiLevelCascadeAttentionWrapper
    ps, hq, hkv, d, prompts, beams = 16, 32, 8, 64, 8, 32
    n = prompts * beams
    own = np.random.default_rng(1).integers(1, 17, n)
    pool, scale = make_pool(2 * prompts + n, ps, hkv, d, dt, cache8, 4)
    ids = np.random.default_rng(2).permutation(2 * prompts + n).tolist()
    heads, tails = ids[:2 * prompts], ids[2 * prompts:]
    q = torch.randn((n, hq, d), device="cuda", generator=torch.Generator(device="cuda").manual_seed(4)).to(dt)
    w = MultiLevelCascadeAttentionWrapper(2, torch.empty(64 << 20, dtype=torch.uint8, device="cuda"))
    w.plan([list(range(0, n + 1, beams)), list(range(n + 1))],
           [list(range(0, 2 * prompts + 1, 2)), list(range(n + 1))], [heads, tails],
           [[ps] * prompts, own.tolist()], hq, hkv, d, ps, causal=True,
           kv_data_type=F8 if cache8 else dt, **({} if cache8 else dict(window_left=10 ** 6)))
    assert w._plan.info.n_merge * hq > 148 * 32
    out, lse = w.run(q, pool, return_lse=True, kv_scale=scale)
    lists = [heads[2 * (i // beams):2 * (i // beams) + 2] + [tails[i]] for i in range(n)]
    ref = reference(q, pool, scale, list(range(0, 3 * n + 1, 3)), [p for x in lists for p in x],
                    [32 + int(k) for k in own], list(range(n + 1)), True, -1, 0, d ** -0.5)
    if cache8:
        check(out, lse, ref, dt)
    else:                          # probabilities in the query's type
        o, e, a, b = ref
        u = torch.finfo(dt).eps / 2
        tol = u * o.abs() + (u + 2.4e-4) * a + 2.0 ** -25 * (b + 1)
        assert ((out.double() - o).abs() <= tol).all()
        assert ((lse.double() - e).abs() <= 2e-5).all()
    assert status() == 0


@pytest.mark.parametrize("qlen", [1, 40])
@pytest.mark.parametrize("missing", [8, 9, 17])
def test_no_page_in_the_first_steps(qlen, missing):
    """The first pages are out of range: flagged, and the rest is attended as if it were all (its scales far
    apart: nothing was there to set the unit by)."""
    n, ps = 24, 16
    pool, scale = make_pool(n, ps, 2, 128, torch.bfloat16, True, 8)
    scale[:, 1] = torch.ldexp(torch.ones(n, device="cuda"), torch.arange(n, device="cuda") * 3 - 40)[:, None]
    pages = [n + 5] * missing + list(range(missing, n))
    from beam_engine_b200.cascade import BatchPrefillWithPagedKVCacheWrapper
    q = torch.randn((qlen, 8, 128), device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)).bfloat16()
    w = BatchPrefillWithPagedKVCacheWrapper(torch.empty(64 << 20, dtype=torch.uint8, device="cuda"))
    w.plan([0, qlen], [0, n], pages, [ps], 8, 2, 128, ps, causal=True, kv_data_type=F8)
    out, lse = w.run(q, pool, return_lse=True, kv_scale=scale)
    ref = reference(q, pool, scale, [0, n - missing], pages[missing:], [(n - missing) * ps],
                    [0, qlen], True, -1, 0, 128 ** -0.5)
    check(out, lse, ref, torch.bfloat16)
    assert status() == _lib.BE_EDEVICE_RANGE
