"""PageTable.read_pages over pools without scales."""
import pytest
import torch


def table(device, dt=torch.bfloat16):
    from beam_engine_b200.page_table import PageTable
    pt = PageTable(2, 4, 6, 2, 8, device=device, store_dtype=dt)
    pt.kv_cache.copy_(torch.randn(pt.kv_cache.shape, generator=torch.Generator().manual_seed(0)).to(dt))
    return pt


DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("pages", [[], [5, 0, 5], [-1, 2, 6, 2 ** 31 - 1, -2 ** 31, 3]])
@pytest.mark.parametrize("as_tensor", [True, False])
def test_pages_out_of_range_read_as_zeros(device, pages, as_tensor):
    pt = table(device)
    ids = torch.tensor(pages, dtype=torch.int32, device=device) if as_tensor else pages
    got = pt.read_pages(1, ids, torch.float32)
    assert got.shape == (len(pages), 2, 4, 2, 8) and got.dtype == torch.float32
    for i, p in enumerate(pages):
        want = pt.kv_cache[1, p].float() if 0 <= p < 6 else torch.zeros_like(got[i])
        assert torch.equal(got[i], want)


@pytest.mark.parametrize("device", DEVICES)
def test_a_copy_and_a_shape(device):
    pt = table(device, torch.float32)
    before = pt.kv_cache.clone()
    got = pt.read_pages(0, [1, 2], torch.float32)
    got.zero_()
    assert torch.equal(pt.kv_cache, before)
    with pytest.raises(ValueError, match="pages"):
        pt.read_pages(0, torch.zeros((2, 2), dtype=torch.int32, device=device))
