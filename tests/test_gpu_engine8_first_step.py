"""The first step graph of a generation over an 8-bit pool: the step takes effect once."""
import numpy as np
import pytest
import torch

from test_gpu_engine8 import PROMPTS, engine

from beam_engine_b200.beam_state import BeamState

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page_size", [16, 8])
@pytest.mark.parametrize("down", [1, 6, 20])
def test_a_first_step_that_forks_a_page_and_raises_its_scale(dt, page_size, down):
    """The prompts' last pages are made 2^-down as large before the first decode step, so each beam's
    new token raises the scale of its page and rounds the tokens there.  The step forks those
    pages: every beam's copy is of the tokens as they were, and codes, scales and top-k are those
    of the eager step, bit for bit (the same kernels on the same inputs)."""
    got = []
    for graph in (True, False):
        gen = engine(dt, page_size=page_size, use_graph=graph)
        state = BeamState(4, gen.page_table)
        state.defer_copies = True
        logits = gen.prefill(state, [p[:-1] for p in PROMPTS])       # partly filled last pages
        gen.page_table.kv_scale.mul_(2.0 ** -down)
        vals, idx = gen._topk(logits, 8, 1.0)
        gen._apply(state, np.arange(4, dtype=np.int32) * 4, idx[:, :4].reshape(-1), vals[:, :4].reshape(-1))
        assert len(state.leaves) == 12
        steps = []
        for _ in range(3):                                           # the recorded step is replayed after it
            v, i = gen.decode_topk(state, 8, 1.0)
            steps.append((v.copy(), i.copy()))
            gen._apply(state, np.arange(13, dtype=np.int32), i[:, 0].copy(), v[:, 0].copy())
        gen._flush_fork()
        torch.cuda.synchronize()
        got.append((gen.page_table.kv_cache.view(torch.uint8).clone(), gen.page_table.kv_scale.clone(), steps))
    (c0, s0, t0), (c1, s1, t1) = got
    assert torch.equal(s0, s1)
    assert torch.equal(c0, c1)
    for (v0, i0), (v1, i1) in zip(t0, t1):
        assert np.array_equal(i0, i1) and np.array_equal(v0, v1)
