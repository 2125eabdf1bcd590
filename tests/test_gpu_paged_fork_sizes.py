"""fork_pages: page sizes that caches rule out, and rows that begin a sequence."""

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,size", [(128, 64), (64, 64), (128, 16), (64, 48)])
def test_a_page_size_that_a_cache_has_not(cuda, dim, size):
    """A smaller one would share a page that is still written, a larger one count keys that are not there."""
    from sfu_repro import paged_cache

    cache = paged_cache.fp4_cache(8, 2, dim, size, device=cuda)
    other = torch.zeros(8, 48, device=cuda)
    table = torch.tensor([[1, 2, -1, -1]], dtype=torch.int32, device=cuda)
    lens, parents = torch.tensor([size + 1], dtype=torch.int32, device=cuda), torch.zeros(2, dtype=torch.int32, device=cuda)
    got, _, short = paged_cache.fork_pages([cache, other], table, lens, parents, tokens=1, page_size=size)
    assert got[:, 0].tolist() == [1, 1] and got[0, 1] != got[1, 1] and short.tolist() == [0]
    same = size * 2 if dim == 128 else size // 2  # rows of the other head dimension: the same bytes
    for wrong in (16, 32, 48, 64, 128, 17, size + 1, 4 * size):
        if wrong in (size, same):
            continue
        with pytest.raises(RuntimeError, match=f"page_size {wrong} is not that of a cache"):
            paged_cache.fork_pages([other, cache], table, lens, parents, tokens=1, page_size=wrong)
    paged_cache.fork_pages([other], table, lens, parents, tokens=1, page_size=17)  # tells nothing of its rows
    eights = torch.zeros(8, 2, 2, 24 * 96, dtype=torch.uint8, device=cuda)  # a cache of another kind
    paged_cache.fork_pages([eights], table, lens, parents, tokens=1, page_size=24)
    alike = torch.zeros(8, 2, 2, 16 * 136, dtype=torch.uint8, device=cuda)
    paged_cache.fork_pages([alike.flatten(1)], table, lens, parents, tokens=1, page_size=16)


def test_new_sequences(cuda):
    """They continue a row of no keys, several the same one, each with pages of its own; a place that nothing
    uses gets none and wants none."""
    from sfu_repro import paged_cache

    size, prompt = 16, 40
    cache = paged_cache.fp4_cache(13, 2, 64, size, device=cuda)
    new = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    table, lens = torch.full((2, 4), -1, dtype=torch.int32, device=cuda), new(20, 0)
    table[0, :2] = new(3, 7)
    table, lens, short = paged_cache.fork_pages([cache], table, lens, new(0, 1, 1, -1, 1), tokens=prompt, page_size=size)
    assert lens.tolist() == [20, 0, 0, 0, 0] and short.tolist() == [0]
    held = table.cpu()
    assert (held[3] == -1).all() and (held[[1, 2, 4], :3] >= 0).all() and (held[[1, 2, 4], 3] == -1).all()
    named = held[held >= 0].tolist()
    assert len(set(named)) == len(named) == 4 + 3 * 3
    k = torch.randn(5, prompt, 2, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(cuda)
    lens = lens + new(prompt, prompt, prompt, 0, prompt)
    paged_cache.store_fp4(cache, k, k, table, lens)
    got = paged_cache.load_fp4(cache, table, lens, prompt, 64)[0]
    for i in range(5):
        ref.same(got[i], torch.zeros_like(got[i]) if i == 3 else ref.nearest(k[i].cpu()))
