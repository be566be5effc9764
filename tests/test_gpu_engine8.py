"""The engine on an 8-bit pool: the same beams from the step graph and the eager path, logits
against attention computed in fp32 over the values that the pool holds, and refusals."""
import numpy as np
import pytest
import torch

from beam_engine_b200.beam import BeamSearchGenerator
from beam_engine_b200.beam_state import BeamState
from beam_engine_b200.beam_strategy import VanillaBeamSearchStrategy
from beam_engine_b200.configs import TINY
from beam_engine_b200.llama import BeamLlama

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn
PROMPTS = [[int(x) for x in np.random.default_rng(i).integers(0, 1024, n)] for i, n in enumerate((70, 33, 16))]


def engine(dt=torch.bfloat16, **kw):
    model = BeamLlama(TINY, dtype=dt, seed=3)
    kw.setdefault("store_dtype", F8)
    return BeamSearchGenerator(model, None, VanillaBeamSearchStrategy(), max_num_pages=1024, **kw)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page_size", [16, 8])
def test_graph_steps_equal_eager_steps(dt, page_size):
    res = [engine(dt, page_size=page_size, use_graph=g).generate_ids(PROMPTS, 4, max_new_tokens=24)
           for g in (True, False)]
    assert [[t for t, _ in r] for r in res[0]] == [[t for t, _ in r] for r in res[1]]
    for a, b in zip(res[0], res[1]):
        np.testing.assert_allclose([x for _, x in a], [x for _, x in b], atol=1e-4)


class PoolAttention:
    """Attention in fp32 over the pool's values: per query a list of (page, tokens) and how many of
    the last tokens it does not see."""

    def __init__(self, gen, lists):
        self.gen, self.lists = gen, lists

    def run(self, layer, qkv, out):
        m, pt = self.gen.model, self.gen.page_table
        vals = pt.read_pages(layer, list(range(pt.max_num_pages)), torch.float32)
        q = qkv[:, :m.Hq * m.D].float().view(-1, m.Hkv, m.Hq // m.Hkv, m.D)
        for i, pages in enumerate(self.lists):
            kv = torch.cat([vals[p, :, :n] for p, n in pages], 1)             # [2, t, hkv, d]
            x = torch.einsum("hgd,thd->hgt", q[i], kv[0]) * m.D ** -0.5
            out[i] = torch.einsum("hgt,thd->hgd", torch.softmax(x, -1), kv[1]).reshape(-1).to(out.dtype)


def seen(levels, nq, ps, causal_last):
    lists = [[] for _ in range(nq)]
    for li, lv in enumerate(levels):
        qo, kp, ki, ll = (lv[k] for k in ("qo_indptr", "kv_indptr", "kv_indices", "kv_last_page_len"))
        for g in range(len(qo) - 1):
            pages = [int(x) for x in ki[kp[g]:kp[g + 1]]]
            full = [(p, ps if j + 1 < len(pages) else int(ll[g])) for j, p in enumerate(pages)]
            for q in range(qo[g], qo[g + 1]):
                drop = qo[g + 1] - q - 1 if causal_last and li == len(levels) - 1 else 0
                rows = list(full)
                while drop and rows:                     # the last `drop` tokens are not seen
                    p, n = rows.pop()
                    if n > drop:
                        rows.append((p, n - drop))
                        drop = 0
                    else:
                        drop -= n
                lists[q] += rows
    return lists


@pytest.mark.parametrize("page_size", [16, 8])
def test_logits_against_attention_over_the_pools_values(page_size):
    """Prompt and one decode step: the engine's logits against the same forward with attention in
    fp32 over what the pool holds (the second forward writes the same tokens again).  The
    attention outputs differ by half a bf16 step and the probabilities' rounding; two layers of
    bf16 residuals and norms carry that to the logits: 2e-2 of their spread covers it as it does for
    the 16-bit pools."""
    gen = engine(page_size=page_size, use_graph=False)
    state = BeamState(4, gen.page_table)
    state.defer_copies = True
    run = gen.model.forward
    kept = {}

    def spy(ids, pos, pt, wp, wpos, attention, logits_rows=None, layer_hook=None):
        kept.update(args=(ids, pos, pt, wp, wpos), rows=logits_rows)
        return run(ids, pos, pt, wp, wpos, attention, logits_rows=logits_rows, layer_hook=layer_hook)
    gen.model.forward = spy

    def check(logits, lists):
        before = gen.page_table.kv_cache.view(torch.uint8).clone()
        want = run(*kept["args"], PoolAttention(gen, lists), logits_rows=kept["rows"])
        assert torch.equal(gen.page_table.kv_cache[0].view(torch.uint8), before[0])   # same rows again
        gen.page_table.kv_cache.view(torch.uint8).copy_(before)
        assert (logits - want).abs().max() <= 2e-2 * want.std() * 4

    logits = gen.prefill(state, PROMPTS)
    ps = page_size
    lists = []
    pages = iter(range(1024))
    tables = [[next(pages) for _ in range(-(-len(p) // ps))] for p in PROMPTS]
    for p, tab in zip(PROMPTS, tables):
        for i in range(len(p)):
            lists.append([(pg, min(ps, i + 1 - j * ps)) for j, pg in enumerate(tab) if i + 1 > j * ps])
    check(logits, lists)
    vals, idx = gen._topk(logits, 8, 1.0)
    gen._apply(state, np.arange(4, dtype=np.int32) * 4, idx[:, :4].reshape(-1), vals[:, :4].reshape(-1))
    gen._flush_fork()
    logits = gen.decode_step(state)
    check(logits, seen(state.cascade_levels(), len(state.leaves), ps, True))


def test_pool_holds_what_a_16_bit_pool_holds():
    """The first layer's keys and values after a prompt, in both kinds of pool: the rounding to a
    block's scale, at most 2^-4 of the value or half the smallest step, beside bf16's own 2^-8."""
    vals = []
    for store in (F8, torch.bfloat16):
        gen = engine(store_dtype=store, page_size=16, use_graph=False)
        gen.prefill(BeamState(4, gen.page_table), [PROMPTS[0]])
        vals.append((gen.page_table.read_pages(0, [0, 1, 2, 3], torch.float32),
                     None if gen.page_table.kv_scale is None else gen.page_table.kv_scale[0, :4]))
    (a, s), (b, _) = vals
    tol = b.abs() * (2.0 ** -4 + 2.0 ** -8) * 1.01 + s[:, :, None, :, None] * 2.0 ** -10
    assert ((a - b).abs() <= tol).all()


def test_refusals():
    model = BeamLlama(TINY, dtype=torch.bfloat16, seed=0)
    for kind in ("fasttree", "auto"):
        with pytest.raises(ValueError, match="cascade"):
            BeamSearchGenerator(model, None, VanillaBeamSearchStrategy(), kernel_type=kind, store_dtype=F8)
    with pytest.raises(ValueError, match="bf16"):
        BeamSearchGenerator(BeamLlama(TINY, dtype=torch.float32, seed=0), None,
                            VanillaBeamSearchStrategy(), store_dtype=F8)


def test_prompts_of_more_rows_than_one_scan():
    """600 prompt rows in one call (the append sorts them into runs first): the pool's first layer
    holds the codes and scales that the same prompts leave one by one."""
    long = [[int(x) for x in np.random.default_rng(9 + i).integers(0, 1024, 300)] for i in range(2)]
    both = engine(page_size=16, use_graph=False)
    both.prefill(BeamState(4, both.page_table), long)
    for i, p in enumerate(long):
        one = engine(page_size=16, use_graph=False)
        one.prefill(BeamState(4, one.page_table), [p])
        n = 18                                             # 18 full pages of 19
        a = both.page_table.kv_cache[0, i * 19:i * 19 + n].view(torch.uint8)
        sa, sb = both.page_table.kv_scale[0, i * 19:i * 19 + n], one.page_table.kv_scale[0, :n]
        # the projections of 600 and of 300 rows may be summed in another order: nearly all codes agree
        assert (sa == sb).float().mean() > 0.99
        assert (a == one.page_table.kv_cache[0, :n].view(torch.uint8)).float().mean() > 0.97
    res = engine(page_size=16).generate_ids(long, 4, max_new_tokens=4)
    assert len(res) == 2
