"""Speculative and sparse decoding at their limits: page entries that are no pages, lengths that overlap, rows of very unlike sizes."""
import math

import pytest
import torch

from paged_reference import D, PAGE, append_rows, attend64, bounds64, check_attention, filled_cache, rows64

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


@pytest.mark.parametrize("bits", [8, 4])
def test_bounds_of_pages_that_are_none(bits):
    """Entries outside the pool raise the status bit and write nothing: the bounds of every page, page 0 among them, stay those of
    the stream that holds it."""
    import pikv_b200
    gen = torch.Generator(device="cuda").manual_seed(bits)
    n_kv, lens = 2, [160, 147, 80]
    cache = pikv_b200.PagedKVCache(3, 160, n_kv, bits=bits, symmetric=bits == 8)
    for s in range(3):
        append_rows(cache, s, 0, *(torch.randn(160, n_kv * D, generator=gen, device="cuda").bfloat16() for _ in range(2)))
    length = torch.tensor(lens, dtype=torch.int32, device="cuda")
    assert int(cache.page_table[0, 0]) == 0
    bounds = cache.page_bounds()
    bounds.codes.fill_(99)
    bounds.scale.fill_(-1)
    cache.update_bounds(bounds, seq_len=length)
    cache.check_status()
    k, _ = rows64(cache, 0, PAGE)
    codes, scale = bounds64(k)
    assert torch.equal(bounds.codes[0].double(), codes) and torch.equal(bounds.scale[0].double(), scale)
    want = bounds.codes.clone(), bounds.scale.clone()
    # a full page and the partial last one of stream 1; all pages of stream 2
    cache.page_table[1, 4] = -1
    cache.page_table[1, 9] = cache.num_pages
    cache.page_table[2] = -7
    for ids in (None, torch.tensor([1], dtype=torch.int32, device="cuda"), torch.tensor([2, 0], dtype=torch.int32, device="cuda")):
        cache.update_bounds(bounds, seq_ids=ids, seq_len=length if ids is None else length[ids.long()].contiguous())
        assert int(cache.status) == 2
        cache.status.zero_()
        assert torch.equal(bounds.codes, want[0]) and torch.equal(bounds.scale, want[1])


def test_accept_with_a_part_of_the_lengths():
    """Contexts given as a slice of the cache's own lengths, of other streams than the entries' own: read as they were."""
    S, N = 40, 5
    lens = [17 + 3 * s for s in range(S)]
    cache, gen = filled_cache([max(lens) + 3 + N] * S, 1, 8, seed=3)
    length = torch.tensor(lens, dtype=torch.int32, device="cuda")
    path = torch.tensor([[1, 2, 4]] * (S - 1), dtype=torch.int32, device="cuda")
    saved = {n: t.clone() for n, t in cache.named_buffers()}
    for ids in (None, torch.arange(S - 2, -1, -1, dtype=torch.int32, device="cuda")):
        got = []
        for ctx in (length[1:].clone(), cache.length[1:]):
            for n, t in cache.named_buffers():
                t.copy_(saved[n])
            cache.length.copy_(length)
            new = cache.accept_tree(path, seq_ids=ids, ctx_len=ctx)
            cache.check_status()
            assert torch.equal(new, length[1:] + 3)
            got.append([new] + [t.clone() for _, t in cache.named_buffers()])
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(*got))
