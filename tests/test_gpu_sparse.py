"""Bounds of pages and attention over the pages they select, against 64 bits; speculative and sparse decoding together."""
import math

import pytest
import torch

from paged_reference import D, PAGE, append_rows, attend64, bounds64, check_attention, chosen64, filled_cache, rows64, step64

pytestmark = pytest.mark.gpu
# a logit: the query in 15 bits of its head's largest entry (2^-14 of it, summed against the keys: 2^-14 of the sum of sizes with the largest
# entry in every channel; a normal query's mean size is a fifth of its largest entry, its smallest ratio here 1 / 12), or in f16 exactly
LOGIT = 12 * 2.0 ** -14


@pytest.fixture(autouse=True)
def device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def check_bounds(cache, bounds, stream, n, first=0):
    k, _ = rows64(cache, stream, n)
    for p in range(first, (n + PAGE - 1) // PAGE):
        codes, scale = bounds64(k[p * PAGE:(p + 1) * PAGE])
        page = int(cache.page_table[stream, p])
        assert torch.equal(bounds.codes[page].double(), codes) and torch.equal(bounds.scale[page].double(), scale)
        real = bounds.codes[page].double() * bounds.scale[page].double()[:, None, None]
        rows = k[p * PAGE:(p + 1) * PAGE]
        assert bool((rows <= real[:, 0]).all() and (rows >= real[:, 1]).all())


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n_kv", [1, 3])
def test_bounds(bits, n_kv):
    rows = [1, 15, 16, 17, 100, 0, 333]
    cache, gen = filled_cache(rows, n_kv, bits, seed=n_kv)
    cache.length.copy_(torch.tensor(rows, dtype=torch.int32))
    bounds = cache.page_bounds()
    bounds.codes.fill_(99)
    cache.update_bounds(bounds)
    cache.check_status()
    for s, n in enumerate(rows):
        check_bounds(cache, bounds, s, n)
    held = set(cache.page_table[s, p].item() for s, n in enumerate(rows) for p in range((n + PAGE - 1) // PAGE))
    spare = [p for p in range(cache.num_pages) if p not in held]
    assert bool((bounds.codes[spare] == 99).all()) and not bounds.scale[spare].any()       # pages of no stream stay as they were
    # shorter streams: the last page's bounds are of fewer rows
    lens = torch.tensor([50, 18], dtype=torch.int32, device="cuda")
    cache.update_bounds(bounds, seq_ids=torch.tensor([4, 6], dtype=torch.int32, device="cuda"), seq_len=lens)
    check_bounds(cache, bounds, 4, 50)
    check_bounds(cache, bounds, 6, 18)


@pytest.mark.parametrize("bits", [8, 4])
def test_bounds_from_a_position(bits):
    cache, gen = filled_cache([100, 40, 64, 80], 2, bits, seed=7)
    lens = torch.tensor([100, 40, 64, 80], dtype=torch.int32, device="cuda")
    start = torch.tensor([37, 39, 64, -5], dtype=torch.int32, device="cuda")
    bounds = cache.page_bounds()
    bounds.scale.fill_(-1)
    cache.update_bounds(bounds, start=start, seq_len=lens)
    for s, (n, first) in enumerate(((100, 2), (40, 2), (64, 4), (80, 0))):
        check_bounds(cache, bounds, s, n, first)
        assert bool((bounds.scale[cache.page_table[s, :first].long()] == -1).all())


def test_bounds_extremes():
    """A page of zeros, one with values of many sizes, and ones that hold something not finite."""
    cache, gen = filled_cache([64], 1, 8, seed=9)
    k = torch.randn(64, D, generator=gen, device="cuda") * 2.0 ** torch.arange(-60, 68, device="cuda").float()
    k[:16] = 0
    append_rows(cache, 0, 0, k.bfloat16(), k.bfloat16())
    cache.k_scale[int(cache.page_table[0, 2]), 0, 3] = math.inf
    cache.k_scale[int(cache.page_table[0, 3]), 0, 15] = math.nan
    bounds = cache.page_bounds()
    cache.update_bounds(bounds, seq_len=torch.tensor([64], dtype=torch.int32, device="cuda"))
    # the reference's quantiser gives a row of zeros the scale of a range of 1e-5
    check_bounds(cache, bounds, 0, 32)
    for p in (2, 3):
        page = int(cache.page_table[0, p])
        assert float(bounds.scale[page]) == math.inf and not bounds.codes[page].any()
    cache.check_status()


def sparse_check(cache, q, bounds, pages, lens, first, recent, ids=None):
    out, lse, chosen = cache.decode_attention_sparse(q, bounds, pages, seq_ids=ids, seq_len=lens, first=first, recent=recent, want_lse=True, want_pages=True)
    n_kv, G = cache.n_kv, q.shape[1] // cache.n_kv
    for b in range(q.shape[0]):
        n, s = int(lens[b]), b if ids is None else int(ids[b])
        P = (n + PAGE - 1) // PAGE
        if n == 0:
            assert not out[b].any() and bool((lse[b] == -math.inf).all()) and bool((chosen[b] == -1).all())
            continue
        at = cache.page_table[s, :P].long()
        want = chosen64(q[b], bounds.codes[at], bounds.scale[at], pages, first, recent)
        k, v = rows64(cache, s, n)
        for h in range(n_kv):
            got = chosen[b, h].tolist()
            assert got[:len(want[h])] == want[h] and all(x == -1 for x in got[len(want[h]):])
            sees = torch.zeros(P, PAGE, dtype=torch.bool, device="cuda")
            sees[want[h]] = True
            sees = sees.view(1, -1)[:, :n]
            heads = slice(h * G, (h + 1) * G)
            w, wl, big, size = attend64(q[b:b + 1, heads], k[:, h:h + 1], v[:, h:h + 1], sees)
            check_attention(out[b:b + 1, heads], lse[b:b + 1, heads], w, wl, big, size, LOGIT)
    return out, lse, chosen


# budgets of one page, of less than a stream, of all of it and more; sinks and recent pages, also filling the budget; lengths of
# zero and one and at page edges; group sizes on both sides of four; many pages (several rounds of a CTA's keys)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("rows,pages,first,recent,G,n_kv", [
    ([1, 16, 17, 0, 33, 200], 1, 0, 1, 1, 2), ([300, 100, 16, 31, 32, 33], 2, 0, 1, 4, 2), ([500, 7, 160, 161], 10, 1, 2, 8, 1),
    ([500, 1000], 10, 3, 7, 3, 1), ([700, 80], 64, 0, 1, 4, 1), ([9000, 4000, 20], 50, 2, 5, 4, 2), ([40000], 300, 0, 1, 4, 1)])
def test_sparse_attention(bits, rows, pages, first, recent, G, n_kv):
    cache, gen = filled_cache(rows, n_kv, bits, seed=pages)
    lens = torch.tensor(rows, dtype=torch.int32, device="cuda")
    bounds = cache.page_bounds()
    cache.update_bounds(bounds, seq_len=lens)
    q = torch.randn(len(rows), G * n_kv, D, generator=gen, device="cuda").bfloat16()
    out, lse, chosen = sparse_check(cache, q, bounds, pages, lens, first, recent)
    cache.length.copy_(lens)
    assert torch.equal(cache.decode_attention_sparse(q, bounds, pages, first=first, recent=recent), out)
    cache.check_status()
    ids = torch.arange(len(rows) - 1, -1, -1, dtype=torch.int32, device="cuda")
    sparse_check(cache, q, bounds, pages, lens.flip(0).contiguous(), first, recent, ids)


def test_sparse_budget_past_every_stream_is_dense():
    cache, gen = filled_cache([333, 90], 2, 8, seed=1)
    cache.length.copy_(torch.tensor([333, 90], dtype=torch.int32))
    bounds = cache.page_bounds()
    cache.update_bounds(bounds)
    q = torch.randn(2, 8, D, generator=gen, device="cuda").bfloat16()
    out = cache.decode_attention_sparse(q, bounds, 100)
    off = (out.float() - cache.decode_attention(q).float()).abs()       # split elsewhere: two roundings of the same sum
    assert bool((off <= 2.0 ** -7 * out.float().abs() + 2.0 ** -9).all())


def test_sparse_ties_and_signs():
    """Pages with equal scores: the lower ones are taken; pages whose scores are negative, and zeros of both signs."""
    n_kv, P = 1, 40
    cache, gen = filled_cache([P * PAGE], n_kv, 8, seed=6)
    lens = torch.tensor([P * PAGE], dtype=torch.int32, device="cuda")
    bounds = cache.page_bounds()
    cache.update_bounds(bounds, seq_len=lens)
    at = cache.page_table[0].long()
    q = torch.randn(1, 2, D, generator=gen, device="cuda").bfloat16()
    bounds.codes[at] = bounds.codes[at[:1]].clone()
    bounds.scale[at] = bounds.scale[at[:1]].clone()
    assert sparse_check(cache, q, bounds, 7, lens, 0, 1)[2].tolist() == [[[0, 1, 2, 3, 4, 5, 39]]]
    bounds.codes[at[20:]] = 0
    for sign in (1, -1):                                               # equal scores above or below the zeros
        bounds.codes[at[:20], 0, 0] = sign
        bounds.codes[at[:20], 0, 1] = sign
        x = torch.full((1, 2, D), 1.0, device="cuda").bfloat16()
        x[0, 1] = 0                                                    # the second head's scores are zero everywhere
        sparse_check(cache, x[:, :1].contiguous(), bounds, 25, lens, 0, 1)
        sparse_check(cache, -x, bounds, 25, lens, 0, 1)
    cache.check_status()


def test_sparse_values_that_are_not_finite():
    cache, gen = filled_cache([640], 1, 8, seed=12)
    lens = torch.tensor([640], dtype=torch.int32, device="cuda")
    bounds = cache.page_bounds()
    cache.update_bounds(bounds, seq_len=lens)
    q = torch.randn(1, 4, D, generator=gen, device="cuda").bfloat16()
    clean = sparse_check(cache, q, bounds, 6, lens, 0, 1)
    # a head that is not finite leaves the choice to the others
    q2 = q.clone()
    q2[0, 1, 7] = math.nan
    q2[0, 2, 9] = -math.inf
    at = cache.page_table[0].long()
    out, chosen = cache.decode_attention_sparse(q2, bounds, 6, seq_len=lens, want_pages=True)
    assert chosen[0, 0].tolist() == chosen64(q2[0], bounds.codes[at], bounds.scale[at], 6, 0, 1)[0]
    assert bool(torch.isfinite(out[0, [0, 3]]).all()) and bool(torch.isnan(out[0, 1]).all())
    q2[:] = math.nan
    assert cache.decode_attention_sparse(q2, bounds, 6, seq_len=lens, want_pages=True)[1].tolist() == [[[0, 1, 2, 3, 4, 39]]]
    # a page that holds something not finite is taken, and its rows reach the result
    page = next(p for p in range(39) if p not in clean[2][0, 0].tolist())
    cache.k_scale[int(at[page]), 0, 5] = math.nan
    cache.update_bounds(bounds, seq_len=lens)
    out, chosen = cache.decode_attention_sparse(q, bounds, 6, seq_len=lens, want_pages=True)
    assert page in chosen[0, 0].tolist() and bool(torch.isnan(out).all())
    cache.check_status()


def test_sparse_bad_streams_and_pages():
    cache, gen = filled_cache([320, 320, 320], 2, 8, seed=13)
    lens = torch.tensor([320, 300, 320, 100], dtype=torch.int32, device="cuda")
    bounds = cache.page_bounds()
    cache.update_bounds(bounds, seq_len=lens[:3].contiguous())
    q = torch.randn(4, 4, D, generator=gen, device="cuda").bfloat16()
    ids = torch.tensor([0, -1, 2, 9], dtype=torch.int32, device="cuda")
    out, lse, chosen = cache.decode_attention_sparse(q, bounds, 4, seq_ids=ids, seq_len=lens, want_lse=True, want_pages=True)
    assert int(cache.status) == 1 and not out[[1, 3]].any() and bool((chosen[[1, 3]] == -1).all()) and bool((lse[[1, 3]] == -math.inf).all())
    cache.status.zero_()
    cache.update_bounds(bounds, seq_ids=ids, seq_len=lens)
    assert int(cache.status) == 1
    cache.status.zero_()
    cache.page_table[0, 3] = -1
    again = cache.decode_attention_sparse(q, bounds, 4, seq_ids=ids, seq_len=lens)
    assert int(cache.status) == 3 and torch.equal(again[2], out[2])
    cache.status.zero_()


def test_sparse_many_streams():
    S = 530
    rows = [20 + (i * 53) % 180 for i in range(S)]
    cache, gen = filled_cache(rows, 1, 4, seed=21)
    lens = torch.tensor(rows, dtype=torch.int32, device="cuda")
    cache.length.copy_(lens)
    bounds = cache.page_bounds()
    cache.update_bounds(bounds)
    for s in (0, 511, 512, 529):
        check_bounds(cache, bounds, s, rows[s])
    q = torch.randn(S, 2, D, generator=gen, device="cuda").bfloat16()
    out, lse, chosen = cache.decode_attention_sparse(q, bounds, 3, want_lse=True, want_pages=True)
    for ids in ([0, 1, 2], [510, 511, 512], [513, 529]):
        at = torch.tensor(ids, dtype=torch.int32, device="cuda")
        o, l, c = sparse_check(cache, q[ids].contiguous(), bounds, 3, lens[ids].contiguous(), 0, 1, at)
        assert torch.equal(c, chosen[ids])
        assert bool(((o.float() - out[ids].float()).abs() <= 2.0 ** -7 * o.float().abs() + 2.0 ** -9).all())
    cache.check_status()


# ---- together -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [8, 4])
def test_speculative_and_sparse_steps(bits):
    """Prompts, then steps of a decode loop: draft (appended behind the context), verify, accept a path, bring the bounds up to date,
    and a sparse step; after each the cache equals one that never held the rejected rows."""
    n_kv, G, N, B = 2, 4, 7, 3
    rows = [150, 40, 203]
    cache, gen = filled_cache([r + 40 for r in rows], n_kv, bits, seed=31)
    plain, _ = filled_cache([r + 40 for r in rows], n_kv, bits, seed=31)
    for c in (cache, plain):
        c.length.copy_(torch.tensor(rows, dtype=torch.int32))
    bounds, plain_bounds = cache.page_bounds(), plain.page_bounds()
    cache.update_bounds(bounds)
    mask = torch.zeros(N, N, dtype=torch.bool, device="cuda")
    for i, parent in enumerate([-1, 0, 0, 1, 2, 3, 4]):
        if parent >= 0:
            mask[i] = mask[parent]
        mask[i, i] = True
    path = torch.tensor([[0, 2, 4, 6], [0, 1, 3, 5], [0, 2, 4, 6]], dtype=torch.int32, device="cuda")
    for step in range(3):
        k, v = (torch.randn(B * N, n_kv * D, generator=gen, device="cuda").bfloat16() for _ in range(2))
        slot = (cache.length[:, None] + torch.arange(N, device="cuda")).int().reshape(-1)
        seq = torch.arange(B, dtype=torch.int32, device="cuda").repeat_interleave(N)
        cache.append(k, v, seq, slot)
        q = torch.randn(B, N, n_kv * G, D, generator=gen, device="cuda").bfloat16()
        out = cache.decode_attention_tree(q, mask)
        count = torch.tensor([4, 1 + step, 3], dtype=torch.int32, device="cuda")
        start = cache.length.clone()
        new = cache.accept_tree(path, count)
        assert torch.equal(new, start + count) and torch.equal(cache.length, new)
        cache.update_bounds(bounds, start=start)
        # the other cache: only the accepted rows, one after the other, with a plain decode step for each
        for b in range(B):
            for i in range(int(count[b])):
                node = int(path[b, i])
                append_rows(plain, b, int(start[b]) + i, k[b * N + node][None], v[b * N + node][None])
                at = torch.tensor([b], dtype=torch.int32, device="cuda")
                want = plain.decode_attention(q[b, node][None], seq_ids=at, seq_len=(start[b] + i + 1).int().view(1))
                # the same rows in another order: two bf16 roundings, f16 weights, the query's 15 bits
                assert float((want[0].float() - out[b, node].float()).abs().max()) <= 1e-2 * float(want.float().abs().max())
        plain.length.copy_(new)
        plain.update_bounds(plain_bounds)
        for b in range(B):
            n = int(new[b])
            at = cache.page_table[b, :(n + 15) // 16].long()
            assert torch.equal(bounds.codes[at], plain_bounds.codes[at]) and torch.equal(bounds.scale[at], plain_bounds.scale[at])
        x = q[:, 0].contiguous()
        got = cache.decode_attention_sparse(x, bounds, 4, first=1, want_pages=True)
        want = plain.decode_attention_sparse(x, plain_bounds, 4, first=1, want_pages=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    cache.check_status()


def test_captured_and_on_another_stream():
    """The step of the loop as a CUDA graph, replayed on new inputs, and eagerly on a stream of its own."""
    n_kv, G, N, B = 2, 4, 5, 4
    cache, gen = filled_cache([500 + 40 * i for i in range(B)], n_kv, 8, seed=41)
    ctx = torch.tensor([480 + 40 * i for i in range(B)], dtype=torch.int32, device="cuda")
    cache.length.copy_(ctx)
    bounds = cache.page_bounds()
    cache.update_bounds(bounds)
    mask = torch.ones(N, N, dtype=torch.bool, device="cuda").tril()
    path = torch.tensor([[0, 1, 3]] * B, dtype=torch.int32, device="cuda")
    q = torch.randn(B, N, n_kv * G, D, generator=gen, device="cuda").bfloat16()

    def step():
        start = cache.length.clone()
        tree = cache.decode_attention_tree(q, mask)
        cache.accept_tree(path)
        cache.update_bounds(bounds, start=start)
        return tree, cache.decode_attention_sparse(q[:, 0].contiguous(), bounds, 9, recent=2)

    saved = {n: t.clone() for n, t in cache.named_buffers()}

    def reset():
        for n, t in cache.named_buffers():
            t.copy_(saved[n])
        cache.update_bounds(bounds)

    want = []
    for seed in range(3):
        q.copy_(torch.randn(q.shape, generator=gen, device="cuda"))
        reset()
        want.append((q.clone(), [t.clone() for t in step()], cache.length.clone()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        reset()
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[-1][1]))
    reset()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for x, outs, length in want:
        q.copy_(x)
        reset()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(held, outs)) and torch.equal(cache.length, length)
    cache.check_status()


def test_two_streams_at_once():
    """Two caches stepped on two CUDA streams, their kernels side by side on the GPU, against the same steps one after the other."""
    n_kv, G, N, B = 2, 4, 24, 6
    made = []
    for seed, bits in ((51, 8), (52, 4)):
        cache, gen = filled_cache([3000 + 100 * i for i in range(B)], n_kv, bits, seed=seed)
        cache.length.copy_(torch.tensor([2900 + 100 * i for i in range(B)], dtype=torch.int32))
        q = torch.randn(B, N, n_kv * G, D, generator=gen, device="cuda").bfloat16()
        made.append((cache, cache.page_bounds(), q, torch.rand(B, N, N, generator=gen, device="cuda") < 0.4))

    def step(cache, bounds, q, mask):
        cache.update_bounds(bounds)
        return [cache.decode_attention_tree(q, mask), cache.decode_attention_sparse(q[:, 0].contiguous(), bounds, 40, first=1), bounds.codes.clone()]

    want = [step(*m) for m in made]
    streams = [torch.cuda.Stream() for _ in made]
    for _ in range(5):
        for m in made:
            m[1].codes.zero_()
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        got = []
        for s, m in zip(streams, made):
            with torch.cuda.stream(s):
                got.append(step(*m))
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        assert all(torch.equal(x, y) for a, b in zip(got, want) for x, y in zip(a, b))
    for m in made:
        m[0].check_status()


@pytest.mark.parametrize("bits", [8, 4])
def test_bounds_repeats(bits):
    """Long enough for every warp to go round its ring of copied pages many times, into stages that it has just read: the same
    bounds every time, those of 64 bits at both ends and in between."""
    rows = [20000 + 331 * i for i in range(6)]
    cache, gen = filled_cache(rows, 8, bits, seed=61)
    cache.length.copy_(torch.tensor(rows, dtype=torch.int32))
    first = cache.page_bounds()
    cache.update_bounds(first)
    for s, n in enumerate(rows):
        k, _ = rows64(cache, s, n)
        full = n // PAGE
        pages = k[:full * PAGE].view(full, PAGE, 8, D)
        hi, lo = pages.amax(1), pages.amin(1)
        step = step64(torch.maximum(hi.abs(), lo.abs()).amax(-1))
        at = cache.page_table[s, :full].long()
        assert torch.equal(first.scale[at].double(), step)
        assert torch.equal(first.codes[at].double(), torch.stack((torch.ceil(hi / step[..., None]), torch.floor(lo / step[..., None])), 2))
    again = cache.page_bounds()
    for _ in range(20):
        again.codes.fill_(1)
        cache.update_bounds(again)
        assert torch.equal(again.codes * (again.scale > 0)[..., None, None], first.codes) and torch.equal(again.scale, first.scale)
    cache.check_status()


# an infinite page among ordinary ones stretches the range that the selection cuts into bins, so that nearly all of them lie in one bin
# and are cut again, by several orders; all of them equal, too; several of them; more than there is room for
@pytest.mark.parametrize("pages", [60, 700, 1500])
@pytest.mark.parametrize("infinite", [1, 3, 1900])
@pytest.mark.parametrize("equal", [False, True])
def test_selection_with_infinite_pages(pages, infinite, equal):
    P = 2048
    cache, gen = filled_cache([P * PAGE], 1, 8, seed=pages + infinite)
    lens = torch.tensor([P * PAGE], dtype=torch.int32, device="cuda")
    bounds = cache.page_bounds()
    cache.update_bounds(bounds, seq_len=lens)
    at = cache.page_table[0].long()
    if equal:
        bounds.codes[at] = bounds.codes[at[:1]].clone()
        bounds.scale[at] = bounds.scale[at[:1]].clone()
    bounds.scale[at[torch.randperm(P, generator=gen, device="cuda")[:infinite]]] = math.inf
    for size in (1.0, 1e-4):                                           # scores of both signs, and small ones
        q = (torch.randn(1, 4, D, generator=gen, device="cuda") * size).bfloat16()
        for first, recent in ((0, 1), (2, 5)):
            got = cache.decode_attention_sparse(q, bounds, pages, seq_len=lens, first=first, recent=recent, want_pages=True)[1]
            assert got[0, 0].tolist() == chosen64(q[0], bounds.codes[at], bounds.scale[at], pages, first, recent)[0]
    cache.check_status()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("rows,pages,n_kv,G", [([9000, 3001, 777], 300, 1, 4), ([40000], 600, 2, 4), ([5000, 5016], 40, 3, 8)])
def test_sparse_reads_the_chosen_pages(bits, rows, pages, n_kv, G):
    """Each page's values are its own number (K alike, so that all rows weigh the same): the result is the mean over the pages
    read, and one page more, less or another one shows."""
    cache, gen = filled_cache(rows, n_kv, bits, seed=71)
    lens = torch.tensor(rows, dtype=torch.int32, device="cuda")
    bounds = cache.page_bounds()
    cache.update_bounds(bounds, seq_len=lens)
    q = torch.randn(len(rows), n_kv * G, D, generator=gen, device="cuda").bfloat16()
    # the choice is by these bounds; then all keys become 0 and a page's values a pattern of its number in base 2
    bit = 2 ** (torch.arange(D, device="cuda") % 12)
    for s, n in enumerate(rows):
        page = torch.arange(n, device="cuda") // PAGE
        v = torch.where((page[:, None] & bit) > 0, 1.0, -1.0).repeat(1, n_kv)
        append_rows(cache, s, 0, torch.zeros(n, n_kv * D, device="cuda").bfloat16(), v.bfloat16())
    out, lse, chosen = cache.decode_attention_sparse(q, bounds, pages, seq_len=lens, want_lse=True, want_pages=True)
    cache.check_status()
    for b, n in enumerate(rows):
        at = cache.page_table[b, :(n + PAGE - 1) // PAGE].long()
        want = chosen64(q[b], bounds.codes[at], bounds.scale[at], pages, 0, 1)
        _, v = rows64(cache, b, n)
        for h in range(n_kv):
            sees = torch.zeros(len(at), PAGE, dtype=torch.bool, device="cuda")
            sees[want[h]] = True
            seen = sees.view(-1)[:n]
            L = int(seen.sum())
            mean = v[seen, h].mean(0)
            heads = slice(h * G, (h + 1) * G)
            # Logits are exactly 0, so all weights are equal: their rounding and that of their product with the values' scale to f16 are
            # 2^-11 each of the mean (at most 1), sums in fp32 far below; then the rounding to bf16.  A page more or less moves the
            # log-sum-exp by 1 / pages and a channel whose mean is near 0 by as much, another page the channels in which they differ by twice that
            assert bool(((out[b, heads].double() - mean).abs() <= 2.0 ** -8 * mean.abs() + 2.0 ** -10).all())
            assert bool(((lse[b, heads].double() - math.log(L)).abs() <= 2.0 ** -20 * math.log(L)).all())


def test_dense_decode_with_garbage_behind_the_end():
    """Rows behind a stream's end on its last page, with scales and zero points that are not finite, do not reach decode_attention."""
    for bits in (8, 4):
        rows = [1, 17, 100, 333, 2000]
        cache, gen = filled_cache(rows, 2, bits, seed=81)              # what it leaves unwritten is NaN
        clean, _ = filled_cache(rows, 2, bits, seed=81)
        for name, t in clean.named_buffers():
            if name.endswith(("_scale", "_zp")):
                t.nan_to_num_(0)
        lens = torch.tensor(rows, dtype=torch.int32, device="cuda")
        for G in (1, 4, 8):
            q = torch.randn(len(rows), 2 * G, D, generator=gen, device="cuda").bfloat16()
            for fill in (math.nan, math.inf, -math.inf):
                for name in ("k_scale", "v_scale") + (("k_zp", "v_zp") if bits == 4 else ()):
                    t = getattr(cache, name)
                    t[torch.isnan(t) | torch.isinf(t)] = fill
                got, want = cache.decode_attention(q, seq_len=lens), clean.decode_attention(q, seq_len=lens)
                assert bool(torch.isfinite(got).all()) and torch.equal(got, want)
                for name in ("k_scale", "v_scale") + (("k_zp", "v_zp") if bits == 4 else ()):
                    t = getattr(cache, name)
                    t[torch.isinf(t)] = math.nan
        cache.check_status()
