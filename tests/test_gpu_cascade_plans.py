"""One wrapper over caches of several types: a run over one type leaves the plan, the kernels and the
captured graphs of the others as they were."""
import numpy as np
import pytest
import torch

from test_gpu_paged8 import F8, clean_status, make_pool, reference, status  # noqa: F401

pytestmark = pytest.mark.gpu
PS, HQ, HKV, D = 16, 8, 2, 128
PTR, PAGES, LAST, QO, KV = [0, 3, 7], [1, 0, 3, 6, 2, 5, 4], [9, 2], [0, 1, 2], [41, 50]


def wrapper(**kw):
    from beam_engine_b200.cascade import BatchPrefillWithPagedKVCacheWrapper
    w = BatchPrefillWithPagedKVCacheWrapper(torch.empty(4 << 20, dtype=torch.uint8, device="cuda"))
    w.plan(QO, PTR, PAGES, LAST, HQ, HKV, D, PS, causal=True, **kw)
    return w


def caches():
    pool8, scale = make_pool(8, PS, HKV, D, torch.bfloat16, True, 1)
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn((8, 2, PS, HKV, D), generator=g, device="cuda")
    q = torch.randn((2, HQ, D), generator=g, device="cuda")
    return {"8": (q.bfloat16(), pool8, scale), "16": (q.bfloat16(), x.bfloat16(), None), "32": (q, x, None)}


def launched(fn):
    """Names of the kernels that a call launches."""
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        fn()
        torch.cuda.synchronize()
    return {e.name for e in prof.events() if e.device_type == torch.autograd.DeviceType.CUDA}


@pytest.mark.parametrize("order", [("8", "16", "32"), ("16", "8", "16", "32", "8"), ("32", "8", "32", "16"),
                                   ("8", "32", "8", "16", "8")])
def test_runs_over_caches_of_several_types_on_one_plan(order):
    """Each run gives, bit for bit, what it gives on a wrapper that met only its type (the tile kernel
    for 16 bits until an fp32 cache has come, work items for fp32)."""
    sets = caches()
    only = {k: wrapper().run(*sets[k][:2], return_lse=True, kv_scale=sets[k][2]) for k in sets}
    w = wrapper()
    met32 = False
    for k in order:
        q, pool, scale = sets[k]
        out, lse = w.run(q, pool, return_lse=True, kv_scale=scale)
        met32 |= k == "32"
        if k == "16" and met32:     # half a bf16 step for the probabilities and for the output
            ref = reference(q, pool, None, PTR, PAGES, KV, QO, True, -1, 0, D ** -0.5)
            assert (out.double() - ref[0]).abs().max() <= 2.0 ** -8 * (ref[0].abs() + ref[2]).max()
        else:
            assert torch.equal(out, only[k][0]) and torch.equal(lse, only[k][1])
    assert status() == 0


def test_a_16_bit_run_keeps_the_tile_kernel_after_an_8_bit_run():
    sets = caches()
    w = wrapper()
    w.run(*sets["8"][:2], kv_scale=sets["8"][2])
    names = launched(lambda: w.run(*sets["16"][:2]))
    assert any("attn_tile_kernel" in n for n in names) and not any("paged" in n for n in names), names


def test_a_graph_captured_over_16_bits_outlives_runs_over_8_bits():
    sets = caches()
    w = wrapper()
    q, pool, _ = sets["16"]
    want = w.run(q, pool)
    out = torch.empty_like(want)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        w.run(q, pool, out=out)
    q8, pool8, scale = sets["8"]
    first = w.run(q8, pool8, kv_scale=scale)
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    # and one over 8 bits, on the plan that the run before it made
    out8 = torch.empty_like(first)
    g8 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g8):
        w.run(q8, pool8, kv_scale=scale, out=out8)
    for graph, o, expect in ((g8, out8, first), (g, out, want), (g8, out8, first)):
        o.zero_()
        w.run(q, pool)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, expect)
    assert status() == 0


def test_a_new_plan_is_made_again_for_8_bits():
    sets = caches()
    w = wrapper()
    q, pool, scale = sets["8"]
    w.run(q, pool, kv_scale=scale)
    w.plan([0, 1, 2], [0, 2, 4], [7, 6, 5, 4], [16, 3], HQ, HKV, D, PS, causal=True)
    out, lse = w.run(q, pool, return_lse=True, kv_scale=scale)
    fresh = wrapper()
    fresh.plan([0, 1, 2], [0, 2, 4], [7, 6, 5, 4], [16, 3], HQ, HKV, D, PS, causal=True, kv_data_type=F8)
    a, b = fresh.run(q, pool, return_lse=True, kv_scale=scale)
    assert torch.equal(out, a) and torch.equal(lse, b)


GOOD = dict(qo=QO, ptr=PTR, pages=PAGES, last=LAST, hq=HQ, hkv=HKV, d=D, ps=PS)


@pytest.mark.parametrize("kind", ["tiles", "items", "8 bits", "window"])
@pytest.mark.parametrize("bad", [dict(qo=[0, 2, 1]), dict(last=[17, 2]), dict(hq=7), dict(d=80, window_left=3),
                                 dict(num_sinks=-1), dict(big=True, window_left=5), dict(big=True),
                                 dict(big=True, kv_data_type=F8)])
def test_a_plan_that_is_refused_leaves_the_one_before(kind, bad):
    from beam_engine_b200.cascade import BatchPrefillWithPagedKVCacheWrapper
    sets = caches()
    q, pool, scale = sets["8" if kind == "8 bits" else "32" if kind == "items" else "16"]
    kw = {"8 bits": dict(kv_data_type=F8), "window": dict(window_left=20)}.get(kind, {})
    w = BatchPrefillWithPagedKVCacheWrapper(torch.empty(1 << 16, dtype=torch.uint8, device="cuda"))
    w.plan(QO, PTR, PAGES, LAST, HQ, HKV, D, PS, causal=True, split_tokens=int(kind == "items") * 4096, **kw)
    want, lse = w.run(q, pool, return_lse=True, kv_scale=scale)
    a = dict(GOOD, **bad)
    if a.pop("big", False):                    # a plan that the workspace of 64 KB does not hold
        n = 20000
        a.update(qo=[0, 1], ptr=[0, n], pages=[0] * n, last=[16])
    with pytest.raises((ValueError, RuntimeError)):
        w.plan(*[a.pop(k) for k in ("qo", "ptr", "pages", "last", "hq", "hkv", "d", "ps")], causal=True, **a)
    got, e = w.run(q, pool, return_lse=True, kv_scale=scale)
    assert torch.equal(got, want) and torch.equal(e, lse)
    assert status() == 0
