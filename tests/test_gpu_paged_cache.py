"""Storing into, reading from, forking and compacting a cache in pages of 4-bit numbers:
every stored number is the definition's, and pages and tables are whole numbers, so all
comparisons are for equality."""

import math

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu


def _table(b, entries, size, lens, seed, extra=5):
    g = torch.Generator().manual_seed(seed)
    pages = b * entries + extra
    order = torch.randperm(pages, generator=g).to(torch.int32)
    return order[: b * entries].view(b, entries).clone(), torch.tensor(lens, dtype=torch.int32), pages


def _noise(*shape, seed):
    return torch.randint(0, 256, shape, generator=torch.Generator().manual_seed(seed), dtype=torch.uint8)


# dtype, batch, tokens, hkv, dim, page_size, lens
STORES = [
    ("bf16", 1, 1, 1, 128, 16, [1]),
    ("f16", 3, 1, 2, 64, 32, [70, 1, 33]),
    ("bf16", 4, 5, 3, 128, 16, [5, 64, 3, 0]),          # left-padded, and an empty one
    ("f16", 2, 100, 8, 128, 64, [100, 190]),
    ("bf16", 2, 33, 4, 64, 48, [200, 20]),              # past the table's 4 * 48
]


@pytest.mark.parametrize("case", STORES, ids=lambda c: "-".join(map(str, c[:6])))
def test_store_and_load(cuda, case):
    from sfu_repro import paged_cache

    dtype, b, t, hkv, dim, size, lens = case
    dt = torch.bfloat16 if dtype == "bf16" else torch.float16
    table, n, pages = _table(b, 4, size, lens, 1)
    table[0, 0] = pages if len(lens) > 3 else table[0, 0]  # no page there
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(b, t, hkv, dim, generator=g) * torch.exp2(torch.randint(-8, 9, (b, t, hkv, dim), generator=g))
            for _ in range(2))
    k, v = k.to(dt), v.to(dt)
    before = _noise(pages, 2, hkv, size * (dim // 2 + dim // 32), seed=3)
    cache = before.to(cuda)
    paged_cache.store_fp4(cache, k.to(cuda), v.to(cuda), table.to(cuda), n.to(cuda))
    after = ref.numbers(cache.cpu(), dim)
    want = ref.numbers(before, dim)
    held = [torch.zeros(b, t, hkv, dim, dtype=torch.float64) for _ in range(2)]
    stored = [ref.nearest(x) for x in (k, v)]
    for i in range(b):
        for j in range(t):
            x = max(0, lens[i]) - t + j
            if 0 <= x < 4 * size and 0 <= int(table[i, x // size]) < pages:
                for kv in range(2):
                    want[int(table[i, x // size]), kv, :, x % size] = held[kv][i, j] = stored[kv][i, j]
    ref.same(after, want)  # also what was not stored
    got = paged_cache.load_fp4(cache, table.to(cuda), n.to(cuda), t, dim, dtype=dt)
    for a, w in zip(got, held):
        assert a.dtype == dt
        ref.same(a, w.to(dt))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_every_number_of_a_type(cuda, dtype):
    """Each 16-bit number as the largest of its block, with its halves, thirds and neighbours beside
    it; infinities and NaN make their block NaN."""
    from sfu_repro import paged_cache

    dt = torch.bfloat16 if dtype == "bf16" else torch.float16
    top = torch.arange(-32768, 32768).to(torch.int16).view(dt)
    parts = torch.linspace(-1, 1, 31)
    x = torch.cat([top[:, None], (top.float()[:, None] * parts).to(dt)], -1).view(512, 1, -1, 128)  # 32 heads
    x = x.nan_to_num(nan=math.nan, posinf=math.inf, neginf=-math.inf)
    cache = paged_cache.fp4_cache(512 // 64, 32, 128, 64, device=cuda)
    table, lens = torch.arange(8, dtype=torch.int32, device=cuda)[None], torch.tensor([512], dtype=torch.int32, device=cuda)
    k = x.view(1, 512, 32, 128).to(cuda)
    paged_cache.store_fp4(cache, k, -k, table, lens)
    want = ref.nearest(x.view(512, 32, 128))
    got = ref.numbers(cache.cpu(), 128).transpose(2, 3).reshape(8, 2, 64, 32, 128)
    for kv, sign in ((0, 1), (1, -1)):
        ref.same(got[:, kv].reshape(512, 32, 128), want * sign)
    assert int(want.isnan().any(-1).sum()) > 0
    read, _ = paged_cache.load_fp4(cache, table, lens, 512, 128, dtype=dt)
    w = want.view(1, 512, 32, 128)
    w = (w.clamp(-65504, 65504) if dtype == "f16" else w).to(dt)
    ref.same(read, w)


def test_loads_every_byte(cuda):
    """All codes under all exponents, those above 252 as NaN."""
    from sfu_repro import paged_cache

    cache = torch.zeros(16, 2, 1, 64 * 17 * 2, dtype=torch.uint8)  # 64 rows of 64 elements a page
    cache[..., : 64 * 32] = torch.arange(256, dtype=torch.uint8).repeat(8)
    cache[..., 64 * 32:] = torch.arange(16 * 128, dtype=torch.int64).view(16, 1, 1, 128).remainder(256).to(torch.uint8)
    want = ref.numbers(cache, 64)[:, :, 0].transpose(0, 1).reshape(2, 1024, 1, 64)
    table, lens = torch.arange(16, dtype=torch.int32, device=cuda)[None], torch.tensor([1024], dtype=torch.int32, device=cuda)
    for dt in (torch.bfloat16, torch.float16):
        got = paged_cache.load_fp4(cache.to(cuda), table, lens, 1024, 64, dtype=dt)
        for a, w in zip(got, want):
            w = (w.clamp(-65504, 65504) if dt == torch.float16 else w).to(dt)
            ref.same(a[0], w)


def test_store_layouts(cuda):
    """Views of a packed projection, operands that have to be copied, one head for all: the same bytes."""
    from sfu_repro import paged_cache

    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn(2, 9, 4, 128, generator=g).to(torch.bfloat16).to(cuda) for _ in range(2))
    table = torch.tensor([[1, 2], [0, 3]], dtype=torch.int32, device=cuda)
    lens = torch.tensor([20, 9], dtype=torch.int32, device=cuda)

    def stored(k, v, table=table, lens=lens):
        cache = paged_cache.fp4_cache(4, 4, 128, 16, device=cuda)
        paged_cache.store_fp4(cache, k, v, table, lens)
        return cache

    want = stored(k, v)
    packed = torch.cat([k, v], 2)
    ref.same(stored(packed[:, :, :4], packed[:, :, 4:]), want)
    odd = torch.zeros(2, 9, 4, 131, dtype=k.dtype, device=cuda)
    odd[..., 3:] = k
    ref.same(stored(odd[..., 3:], v.transpose(1, 2).contiguous().transpose(1, 2)), want)
    ref.same(stored(k, v, table.t().contiguous().t(), torch.stack([lens, lens], 1)[:, 1]), want)
    same = k[:, :, :1].expand(-1, -1, 4, -1)
    ref.same(stored(same, same), stored(same.contiguous(), same.contiguous()))


def _state(rows, entries, size, pages, lens, seed, layers=2):
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((rows, entries), -1, dtype=torch.int32)
    for i, n in enumerate(lens):
        for j in range(min(entries, -(-max(0, n) // size))):
            table[i, j] = order.pop()
    caches = [_noise(pages, 48 * (i + 1), seed=seed + i) for i in range(layers)]
    return caches, table, torch.tensor(lens, dtype=torch.int32)


def _check_fork(cuda, caches, table, lens, parents, tokens, size):
    from sfu_repro import paged_cache

    pages = caches[0].shape[0]
    on = [c.to(cuda) for c in caches]
    given = table.to(cuda), lens.to(cuda)
    got = paged_cache.fork_pages(on, *given, None if parents is None else parents.to(cuda), tokens=tokens, page_size=size)
    out, n, short, moves = ref.fork(table, lens, parents, tokens, size, pages)
    assert torch.equal(got[0].cpu(), out) and torch.equal(got[1].cpu(), n) and got[2].tolist() == [short]
    for c, before in zip(on, caches):
        want = before.clone()
        for s, d in moves:
            want[d] = before[s]
        ref.same(c, want)
    assert torch.equal(given[0].cpu(), table) and torch.equal(given[1].cpu(), lens)
    return short, moves


def test_fork(cuda):
    size, lens = 16, [40, 32, 1, 0, 17, 95]
    caches, table, n = _state(6, 6, size, 40, lens, 1)
    new = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    for parents in (new(0, 0, 1, 1, 5, 5, 5), new(5, 4, 3, 2, 1, 0), new(2), new(0, -1, 7, 2 ** 31 - 1, 0), new(),
                    new(*[0] * 9), None):
        for tokens in (0, 1, 16, 33):
            short, moves = _check_fork(cuda, caches, table, n, parents, tokens, size)
    assert ref.fork(table, n, new(0, 0, 1, 1, 5, 5, 5), 1, size, 40)[3]  # there are copies


def test_fork_of_shared_pages(cuda):
    """Rows that share full pages, and one whose length was taken back into a shared page: a row that
    writes into what another holds gets a copy, whichever comes first."""
    size = 16
    caches, table, n = _state(2, 4, size, 20, [64, 50], 2)
    table = torch.cat([table, table[:1], table[:1], table[1:]])
    for lens in ([64, 50, 30, 30, 50], [30, 50, 64, 64, 50], [30, 50, 20, 64, 48]):
        n = torch.tensor(lens, dtype=torch.int32)
        for parents in (None, torch.tensor([4, 3, 2, 1, 0], dtype=torch.int32)):
            for tokens in (0, 1, 20):
                _check_fork(cuda, caches, table, n, parents, tokens, size)


def test_fork_without_enough_pages(cuda):
    """What is missing is counted: copies, new pages, entries past the table, last pages that are not there."""
    size = 16
    caches, table, n = _state(4, 3, size, 9, [40, 20, 33, 16], 3)
    table[1, 1] = 9
    parents = torch.tensor([0, 0, 0, 1, 2, 2, 3], dtype=torch.int32)
    for tokens in (0, 1, 17, 100, 2 ** 20):
        short, _ = _check_fork(cuda, caches, table, n, parents, tokens, size)
        assert short > 0 or tokens == 0


def test_fork_of_any_lengths(cuda):
    caches, table, n = _state(4, 3, 16, 16, [48, 20, 16, 3], 4)
    n = torch.tensor([2 ** 31 - 1, -5, -2 ** 31, 49], dtype=torch.int32)
    for tokens in (0, 3):
        _check_fork(cuda, caches, table, n, torch.tensor([0, 1, 2, 3, 0], dtype=torch.int32), tokens, 16)


@pytest.mark.parametrize("pages", [1, 31, 32, 33, 64, 5000])
def test_pages_at_the_ends_of_words(cuda, pages):
    """Caches whose pages end inside a word of a bitmap; many rows."""
    from sfu_repro import paged_cache

    g = torch.Generator().manual_seed(pages)
    rows = min(pages, 1500)
    lens = (torch.randint(1, 32, (rows,), generator=g) if pages > 64 else torch.full((rows,), 5)).tolist()
    caches, table, n = _state(rows, 3, 16, pages, lens, 5, layers=1)
    parents = torch.randint(0, rows, (rows + 3,), generator=g).to(torch.int32)
    _check_fork(cuda, caches, table, n, parents, 1, 16)
    for keep in (rows, rows // 2, 1, 0):
        sub = table[torch.randperm(rows, generator=g)[:keep]]
        out, used, moves = ref.compact(sub, pages)
        cache = caches[0].to(cuda)
        got, count = paged_cache.compact_pages([cache], sub.to(cuda))
        assert torch.equal(got.cpu(), out) and count.tolist() == [used]
        want = caches[0].clone()
        for s, d in moves:
            want[d] = caches[0][s]
        ref.same(cache, want)


def test_compact(cuda):
    """Shared pages, entries that name no page, several caches of different kinds, more than a launch takes."""
    from sfu_repro import paged_cache

    table = torch.tensor([[9, 3, -1, 17], [9, 19, 20, -7], [2 ** 31 - 1, 3, 18, 0]], dtype=torch.int32)
    caches = [_noise(20, 16 * (1 + i % 3), seed=i) for i in range(70)] + [torch.randn(20, 3, 8)]
    on = [c.to(cuda) for c in caches]
    given = table.to(cuda)
    got, used = paged_cache.compact_pages(on, given)
    out, n, moves = ref.compact(table, 20)
    assert torch.equal(got.cpu(), out) and used.tolist() == [n] and torch.equal(given.cpu(), table)
    for c, before in zip(on, caches):
        want = before.clone()
        for s, d in moves:
            want[d] = before[s]
        ref.same(c, want)
    again, used = paged_cache.compact_pages(on, got)  # nothing left to move
    assert torch.equal(again, got) and used.tolist() == [n]


def test_large_pages_past_32_bits(cuda):
    """Pages of odd sizes above a block's step, in a cache of more than 2^32 bytes."""
    from sfu_repro import paged_cache

    page = 16 * (1024 * 5 + 3)
    pages = 2 ** 32 // page + 40
    cache = torch.zeros(pages, page, dtype=torch.uint8, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(1)
    ids = [pages - 1 - 3 * i for i in range(10)]
    for i in ids:
        cache[i] = torch.randint(0, 256, (page,), generator=g, device=cuda, dtype=torch.uint8)
    before = {i: cache[i].clone() for i in ids}
    table = torch.tensor([ids], dtype=torch.int32, device=cuda)
    got, used = paged_cache.compact_pages([cache], table)
    assert used.tolist() == [10] and sorted(got[0].tolist()) == list(range(10))
    for new, old in zip(got[0].tolist(), ids):
        assert torch.equal(cache[new], before[old])
    parents = torch.zeros(2, dtype=torch.int32, device=cuda)
    lens = torch.tensor([16 * 10 - 3], dtype=torch.int32, device=cuda)
    forked, _, short = paged_cache.fork_pages([cache], table, lens, parents, page_size=16)
    assert short.tolist() == [0] and forked[1, 9] != forked[0, 9]
    assert torch.equal(cache[int(forked[1, 9])], before[ids[9]])


def test_graph_of_a_decoding_step(cuda):
    """Room for a token, its store and the attention in one graph, replayed over several tokens: the
    same as eager calls, and as the attention of all of them at the end."""
    from sfu_repro import fa4_runtime, paged_cache

    size, hkv, hq, dim, rows = 16, 2, 8, 128, 3
    g = torch.Generator().manual_seed(6)
    caches = [paged_cache.fp4_cache(24, hkv, dim, size, device=cuda) for _ in range(2)]
    table = torch.full((rows, 4), -1, dtype=torch.int32, device=cuda)
    lens = torch.zeros(rows, dtype=torch.int32, device=cuda)
    prompts = torch.tensor([14, 30, 1], dtype=torch.int32, device=cuda)
    k0, v0 = (torch.randn(rows, 30, hkv, dim, generator=g).to(torch.bfloat16).to(cuda) for _ in range(2))
    table, _, short = paged_cache.fork_pages(caches, table, lens, tokens=30, page_size=size)
    for c in caches:
        paged_cache.store_fp4(c, k0, v0, table, prompts)
    state = [table.clone(), prompts.clone()]
    k, v, q = (torch.zeros(rows, 1, h, dim, dtype=torch.bfloat16, device=cuda) for h in (hkv, hkv, hq))

    def step():
        t, n, missing = paged_cache.fork_pages(caches, state[0], state[1], tokens=1, page_size=size)
        n = n + 1
        out = []
        for c in caches:
            paged_cache.store_fp4(c, k, v, t, n)
            out += fa4_runtime.flash_attn_paged_fp4(q, c, t, n)
        return t, n, missing, out

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t, n, missing, out = step()
    queries = []
    for _ in range(20):
        for x in (k, v, q):
            x.copy_(torch.randn(x.shape, generator=g).to(torch.bfloat16))
        graph.replay()
        want = step()  # stores the same once more
        torch.cuda.synchronize()
        assert torch.equal(want[0], t) and torch.equal(want[1], n) and missing.tolist() == [0]
        assert all(torch.equal(a, b) for a, b in zip(out, want[3]))
        queries.append((q.clone(), [x.clone() for x in out]))
        state[0].copy_(t)
        state[1].copy_(n)
    assert state[1].tolist() == [34, 50, 21]
    every = torch.cat([x for x, _ in queries], 1)
    whole, lse = fa4_runtime.flash_attn_paged_fp4(every, caches[0], *state)
    for i, (step_q, o) in enumerate(queries):
        ref.check(o[:2], ref.attention(step_q.cpu(), caches[0].cpu(), state[0].cpu(), state[1].cpu() - 19 + i, 1 / math.sqrt(dim)))
    ref.check((whole, lse), ref.attention(every.cpu(), caches[0].cpu(), state[0].cpu(), state[1].cpu(), 1 / math.sqrt(dim)))


def test_beams_share_their_prompt(cuda):
    """A prompt forked into beams that go on apart and are forked again: each beam's attention is that
    of its own tokens."""
    from sfu_repro import fa4_runtime, paged_cache

    size, hkv, hq, dim = 16, 2, 4, 64
    g = torch.Generator().manual_seed(7)
    new = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    cache = paged_cache.fp4_cache(30, hkv, dim, size, device=cuda)
    table, lens, _ = paged_cache.fork_pages([cache], torch.full((1, 6), -1, dtype=torch.int32, device=cuda), new(0),
                                            tokens=37, page_size=size)
    prompt = torch.randn(2, 1, 37, hkv, dim, generator=g).to(torch.float16)
    paged_cache.store_fp4(cache, *prompt.to(cuda), table, new(37))
    lens, beams = new(37), [prompt[:, 0]]
    for parents in ([0, 0, 0, 0], [1, 1, 3, 0], [0, 2, 2, 3], [3, 2, 1, 0], [0, 0, 1, 2]):
        for _ in range(9):
            table, lens, short = paged_cache.fork_pages([cache], table, lens, new(*parents), tokens=1, page_size=size)
            beams = [beams[p] for p in parents]
            parents = list(range(len(parents)))
            kv = torch.randn(2, len(beams), 1, hkv, dim, generator=g).to(torch.float16)
            lens = lens + 1
            paged_cache.store_fp4(cache, *kv.to(cuda), table, lens)
            beams = [torch.cat([x, kv[:, i]], 1) for i, x in enumerate(beams)]
            assert short.tolist() == [0]
        table, used = paged_cache.compact_pages([cache], table)
        assert int(table.max()) == int(used) - 1
    q = torch.randn(4, 1, hq, dim, generator=g).to(torch.float16)
    out, _ = fa4_runtime.flash_attn_paged_fp4(q.to(cuda), cache, table, lens)
    for i, x in enumerate(beams):
        k, v = paged_cache.load_fp4(cache, table[i:i + 1], lens[i:i + 1], x.shape[1], dim, dtype=torch.float16)
        assert torch.equal(k[0].cpu().double(), ref.nearest(x[0])) and torch.equal(v[0].cpu().double(), ref.nearest(x[1]))
    ref.check((out, _), ref.attention(q, cache.cpu(), table.cpu(), lens.cpu(), 1 / 8))


def test_empty_calls(cuda):
    from sfu_repro import paged_cache

    cache = _noise(4, 2, 2, 16 * 68, seed=1).to(cuda)
    before = cache.clone()
    table, lens = torch.tensor([[0, 1]], dtype=torch.int32, device=cuda), torch.tensor([20], dtype=torch.int32, device=cuda)
    k = torch.zeros(1, 3, 2, 128, dtype=torch.bfloat16, device=cuda)
    paged_cache.store_fp4(cache, k[:, :0], k[:, :0], table, lens)
    paged_cache.store_fp4(cache, k[:0], k[:0], table[:0], lens[:0])
    paged_cache.store_fp4(cache, k, k, table[:, :0], lens)
    paged_cache.store_fp4(cache[:0], k, k, table, lens)
    assert torch.equal(cache, before)
    assert not bool(paged_cache.load_fp4(cache, table[:, :0], lens, 3, 128)[0].any())
    assert paged_cache.load_fp4(cache, table, lens, 0, 128)[0].shape == (1, 0, 2, 128)
    t, n, short = paged_cache.fork_pages([cache], table[:0], lens[:0], tokens=4, page_size=16)
    assert t.shape == (0, 2) and n.shape == (0,) and short.tolist() == [0]
    t, n, short = paged_cache.fork_pages([cache[:0]], table, lens, tokens=1, page_size=16)
    assert t.tolist() == [[-1, -1]] and short.tolist() == [1]
    t, n, short = paged_cache.fork_pages([cache], table[:, :0], lens, tokens=1, page_size=16)
    assert t.shape == (1, 0) and n.tolist() == [0] and short.tolist() == [1]
    t, used = paged_cache.compact_pages([cache], table[:0])
    assert t.shape == (0, 2) and used.tolist() == [0]
    assert torch.equal(cache, before)


def test_refusals(cuda):
    from sfu_repro import paged_cache

    cache = paged_cache.fp4_cache(4, 2, 128, 16, device=cuda)
    table, lens = torch.zeros(1, 2, dtype=torch.int32, device=cuda), torch.zeros(1, dtype=torch.int32, device=cuda)
    k = torch.zeros(1, 1, 2, 128, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(RuntimeError, match="no backward"):
        paged_cache.store_fp4(cache, k.clone().requires_grad_(True), k, table, lens)
    for args, message in (((cache, k, k.half(), table, lens), "same shape, dtype"), ((cache, k[:, :, :1], k[:, :, :1], table, lens), "kv heads"),
                          ((cache, k.float(), k.float(), table, lens), "float16 or bfloat16"), ((cache, k, k[:, :0], table, lens), "same shape"),
                          ((cache[:, :1], k, k, table, lens), "uint8 tensor"), ((cache, k, k, table[0], lens), "table must have shape"),
                          ((cache, k, k, table, lens.cpu()), "same CUDA device")):
        with pytest.raises(RuntimeError, match=message):
            paged_cache.store_fp4(*args)
    with pytest.raises(RuntimeError, match="dtype"):
        paged_cache.load_fp4(cache, table, lens, 1, 128, dtype=torch.float32)
    with pytest.raises(RuntimeError, match="tokens"):
        paged_cache.load_fp4(cache, table, lens, -1, 128)
    fork = lambda caches=(cache,), table=table, lens=lens, parents=None, **kw: paged_cache.fork_pages(  # noqa: E731
        caches, table, lens, parents, **{"page_size": 16, **kw})
    for call, message in ((lambda: fork(()), "at least one cache"), (lambda: fork((cache, cache[:3])), "same pages"),
                          (lambda: fork((cache[:, :, :1],)), "contiguous"), (lambda: fork((cache.cpu(),)), "same CUDA device"),
                          (lambda: fork((torch.zeros(4, 5, device=cuda),)), "16 bytes"),
                          (lambda: fork((torch.zeros(4, 16, device=cuda, requires_grad=True),)), "require gradients"),
                          (lambda: fork(table=table.long()), "int32"), (lambda: fork(lens=lens.long()), "int32"),
                          (lambda: fork(parents=lens.long()), "parents"), (lambda: fork(page_size=0), "page_size"),
                          (lambda: fork(tokens=-1), "tokens"), (lambda: fork(tokens=2 ** 31), "too many"),
                          (lambda: fork(page_size=2 ** 20), "too many"),
                          (lambda: paged_cache.compact_pages([cache], table.float()), "int32")):
        with pytest.raises(RuntimeError, match=message):
            call()


def test_a_written_cache_is_not_what_autograd_saved(cuda):
    from sfu_repro import paged_cache

    cache = paged_cache.fp4_cache(4, 2, 128, 16, device=cuda)
    wide = torch.randn(4, 2, 16, device=cuda)
    table, lens = torch.tensor([[0, 3]], dtype=torch.int32, device=cuda), torch.tensor([20], dtype=torch.int32, device=cuda)
    k = torch.zeros(1, 1, 2, 128, dtype=torch.bfloat16, device=cuda)
    for call, changed in ((lambda: paged_cache.store_fp4(cache, k, k, table, lens), (cache,)),
                          (lambda: paged_cache.fork_pages((cache, wide), table, lens, page_size=16), (cache, wide)),
                          (lambda: paged_cache.compact_pages((cache, wide), table), (cache, wide))):
        before = [t._version for t in changed]
        call()
        assert all(t._version > v for t, v in zip(changed, before))
    version = cache._version
    paged_cache.load_fp4(cache, table, lens, 1, 128)
    assert cache._version == version
    x = torch.ones(4, 2, 16, device=cuda, requires_grad=True)
    y = (x * wide).sum()
    paged_cache.fork_pages((wide,), table, lens, page_size=16)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():  # such tensors have no version
        cache = paged_cache.fp4_cache(4, 2, 128, 16, device=cuda)
    paged_cache.store_fp4(cache, k, k, table, lens)
    paged_cache.fork_pages((cache,), table, lens, page_size=16)
    paged_cache.compact_pages((cache,), table)


def test_a_cache_that_is_named_twice(cuda):
    """Its pages are copied twice, from where they were to where they go."""
    from sfu_repro import paged_cache

    before = _noise(9, 2, 2, 16 * 68, seed=5).to(cuda)
    table = torch.tensor([[8, 2], [7, 6]], dtype=torch.int32, device=cuda)
    lens, parents = torch.tensor([20, 31], dtype=torch.int32, device=cuda), torch.tensor([0, 0, 1, 1], dtype=torch.int32, device=cuda)
    for call in (lambda caches: paged_cache.fork_pages(caches, table, lens, parents, tokens=17, page_size=16),
                 lambda caches: paged_cache.compact_pages(caches, table)):
        one, two = before.clone(), before.clone()
        for a, b in zip(call([one]), call([two, two])):
            assert torch.equal(a, b)
        assert torch.equal(one, two) and not torch.equal(one, before)
