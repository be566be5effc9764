"""Pages of an 8-bit pool that are freed and taken again: what they held before, scales included, is
gone."""
import numpy as np
import pytest
import torch

from test_gpu_engine8 import F8, PROMPTS

from beam_engine_b200.beam import BeamSearchGenerator
from beam_engine_b200.beam_strategy import VanillaBeamSearchStrategy
from beam_engine_b200.configs import TINY
from beam_engine_b200.llama import BeamLlama

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page_size,pages", [(16, 56), (8, 110)])
@pytest.mark.parametrize("graph", [True, False])
def test_a_small_pool_full_of_old_codes_and_scales(page_size, pages, graph):
    """A pool that the generation goes round in (free pages are taken first in, first out) and that
    starts with large scales and arbitrary codes gives the beams of a large new one."""
    model = BeamLlama(TINY, dtype=torch.bfloat16, seed=3)
    got = []
    for n in (1024, pages):
        gen = BeamSearchGenerator(model, None, VanillaBeamSearchStrategy(), page_size=page_size,
                                  max_num_pages=n, store_dtype=F8, use_graph=graph)
        if n == pages:
            g = torch.Generator(device="cuda").manual_seed(0)
            raw = gen.page_table.kv_cache.view(torch.uint8)
            raw.copy_(torch.randint(0, 256, raw.shape, generator=g, device="cuda", dtype=torch.uint8))
            gen.page_table.kv_scale.fill_(2.0 ** 20)
        got.append(gen.generate_ids(PROMPTS, 4, max_new_tokens=40))
    for a, b in zip(*got):
        assert [t for t, _ in a] == [t for t, _ in b]
        np.testing.assert_array_equal([s for _, s in a], [s for _, s in b])
