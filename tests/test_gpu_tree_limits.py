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


@pytest.mark.parametrize("bits", [8, 4])
def test_bounds_of_unlike_rows(bits):
    """A channel whose keys are so far below the page's largest that their quotient by a step is no float: bounds still lie outside."""
    cache, gen = filled_cache([48], 1, bits, seed=29)
    k = torch.randn(48, D, generator=gen, device="cuda") * 2.0 ** -70
    k[3] = torch.randn(D, generator=gen, device="cuda") * 2.0 ** 100
    k[20] = k[3] * 2.0 ** -100
    k[3, 40:60], k[20, 40:60] = 0, 0
    k[16:32, 50:] = k[16:32, 50:].abs()
    k[16:32, :10] = -k[16:32, :10].abs()
    append_rows(cache, 0, 0, k.bfloat16(), k.bfloat16())
    if bits == 4:                                                      # the quantiser has no scales that small
        page = int(cache.page_table[0, 0])
        cache.k_scale[page, 0, [i for i in range(16) if i != 3]] *= 2.0 ** -60
    bounds = cache.page_bounds()
    cache.update_bounds(bounds, seq_len=torch.tensor([48], dtype=torch.int32, device="cuda"))
    cache.check_status()
    rows, _ = rows64(cache, 0, 48)
    for p in range(3):
        codes, scale = bounds64(rows[p * PAGE:(p + 1) * PAGE])
        page = int(cache.page_table[0, p])
        assert torch.equal(bounds.scale[page].double(), scale) and torch.equal(bounds.codes[page].double(), codes)


# ---- rows of unlike sizes -------------------------------------------------------------------------------------------
# K and V of a row enter as f16: 2^-11 of each entry, and 2^-25 of a unit (2^9 times the power of two above the tile's largest scale, or
# the row's own) where the entry is below f16's normal range.  Rows up to 2^8 (8 bit; largest entry 127 scales) or 2^4 (4 bit; 7.5 scales)
# below their tile's largest scale share its unit, so that this is at most 2^-25 2^9 2^9 / 127 < 2^-13, or 2^-25 2^9 2^5 / 7.5 < 2^-13,
# of the row's largest entry.  A weight: 2^-11, and 2^-25 of a reference that the largest weighted row exceeds by 2^7 / 2^9 at least.
def weighted_bound(q, k, v, sees):
    """want [R, n_q, 128] and how far a kernel may be off it, relative to what each row really brings in: a logit's error is that of
    its own key, a value's that of its own row."""
    R, n_q, _ = q.shape
    L, n_kv, _ = k.shape
    x = q.double().view(R, n_kv, n_q // n_kv, D)
    shut = ~sees[:, None, None]
    s = torch.einsum("rhgd,lhd->rhgl", x, k).masked_fill(shut, -math.inf) / math.sqrt(D)
    p = torch.softmax(s, -1)
    slip = torch.einsum("rhgd,lhd->rhgl", x.abs(), (2.0 ** -11 + 264 * 2.0 ** -24) * k.abs() + 2.0 ** -13 * k.abs().amax(-1, keepdim=True)) / math.sqrt(D)
    slip = torch.minimum(slip + 2.0 ** -20 * (1 + s.abs().nan_to_num(posinf=0)), torch.ones_like(slip)).masked_fill(shut, 0)
    size = v.abs().amax(-1).permute(1, 0)[None, :, None]                                              # [1, n_kv, 1, L]
    whole = (p * size).sum(-1)
    off = (2.0 ** -11 + 2.0 ** -11 + 2.0 ** -13 + L * 2.0 ** -23 + 2.0 ** -20) * whole + (p * slip * size).sum(-1) + (p * slip).sum(-1) * whole
    want = torch.einsum("rhgl,lhd->rhgd", p, v).reshape(R, n_q, D)
    return want, 2.0 ** -8 * want.abs() + 1.1 * off.reshape(R, n_q, 1)


def check_weighted(cache, q, mask, ctx, out, nodes=None):
    for b in range(q.shape[0]):
        n, N = int(ctx[b]), q.shape[1]
        k, v = rows64(cache, b, n + N)
        sees = torch.cat([torch.ones(N, n, dtype=torch.bool, device="cuda"), mask[b] if mask.dim() == 3 else mask], 1)
        want, far = weighted_bound(q[b], k, v, sees)
        off = (out[b].double() - want).abs()
        assert bool((off <= far).all()), f"stream {b}: off by {float((off / far).max())} of what its roundings allow"


def grow(cache, stream, pos, factor, which):
    """A row times a power of two, exactly."""
    getattr(cache, which + "_scale")[int(cache.page_table[stream, pos // PAGE]), :, pos % PAGE] *= factor


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("size", [4, 8, 9, 14, 20, 30, 70])
@pytest.mark.parametrize("n_kv,G,N", [(2, 4, 8), (1, 8, 64)])
def test_tree_row_that_is_not_seen(bits, which, size, n_kv, G, N):
    """A drafted row that most nodes do not see, 2^size times the others: those nodes' results are as exact as without it."""
    ctx = [150, 1000]
    cache, gen = filled_cache([n + N for n in ctx], n_kv, bits, seed=size)
    q = torch.randn(2, N, n_kv * G, D, generator=gen, device="cuda").bfloat16()
    mask = torch.eye(N, dtype=torch.bool, device="cuda")
    mask[5, 4] = True
    length = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    for b, n in enumerate(ctx):
        grow(cache, b, n + 4, 2.0 ** size, which)
    out, lse = cache.decode_attention_tree(q, mask, ctx_len=length, want_lse=True)
    cache.check_status()
    check_weighted(cache, q, mask, length, out)
    for b, n in enumerate(ctx):
        k, v = rows64(cache, b, n + N)
        sees = torch.cat([torch.ones(N, n, dtype=torch.bool, device="cuda"), mask], 1)
        rest = [i for i in range(N) if i not in (4, 5)]
        want = attend64(q[b], k, v, sees)[1]
        assert bool(((lse[b].double() - want).abs()[rest] <= 2.0 ** -7).all())


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("size", [6, 16, 24, 40])
def test_tree_rows_of_unlike_sizes(bits, size):
    """Context rows whose keys and values lie up to 2^size apart, in every tile and in tiles of their own; large values under small
    weights, so that rows of all sizes have their share in the result; rows of zeros."""
    n_kv, G, N, ctx = 2, 4, 12, [700, 64, 130]
    cache, gen = filled_cache([n + N for n in ctx], n_kv, bits, seed=size + 100)
    for b, n in enumerate(ctx):
        L = n + N
        k, v = (torch.randn(L, n_kv, D, generator=gen, device="cuda") for _ in range(2))
        e = torch.randint(0, size + 1, (L, 1, 1), generator=gen, device="cuda").float()
        if b == 0:
            e[:320] = torch.randint(0, size + 1, (5, 1, 1), generator=gen, device="cuda").float().repeat_interleave(64, 0)
        # the key's first channel makes a logit smaller by e ln 2 with a query of -sqrt(128) there: a value 2^e larger weighs the same
        k[..., 0] = e[..., 0] * math.log(2)
        v = v * 2.0 ** e
        k[3::17] *= 2.0 ** -size
        k[5::23], v[5::23] = 0, 0
        append_rows(cache, b, 0, k.reshape(L, -1).bfloat16(), v.reshape(L, -1).bfloat16())
    q = torch.randn(len(ctx), N, n_kv * G, D, generator=gen, device="cuda")
    q[..., 0] = -math.sqrt(D)
    q = q.bfloat16()
    mask = torch.rand(len(ctx), N, N, generator=gen, device="cuda") < 0.5
    length = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    out = cache.decode_attention_tree(q, mask, ctx_len=length)
    cache.check_status()
    check_weighted(cache, q, mask, length, out)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("size", [1e31, 1e33, 1e35])
def test_tree_large_values(bits, size):
    """Keys and values up to the size where a row counts as not finite (scales of 2^117), queries that bring the logits back."""
    N, n_kv, G = 6, 2, 4
    cache, gen = filled_cache([300], n_kv, bits, seed=17)
    k, v = (torch.randn(300, n_kv * D, generator=gen, device="cuda") * size for _ in range(2))
    append_rows(cache, 0, 0, k.bfloat16(), v.bfloat16())
    q = (torch.randn(1, N, n_kv * G, D, generator=gen, device="cuda") / size).bfloat16()
    mask = torch.ones(N, N, dtype=torch.bool, device="cuda").tril()
    ctx = torch.tensor([300 - N], dtype=torch.int32, device="cuda")
    out = cache.decode_attention_tree(q, mask, ctx_len=ctx)
    cache.check_status()
    check_weighted(cache, q, mask, ctx, out)
    # one row of them, seen by none of the others, among rows of 1
    n = 300 - N
    append_rows(cache, 0, 0, torch.randn(n, n_kv * D, generator=gen, device="cuda").bfloat16(), torch.randn(n, n_kv * D, generator=gen, device="cuda").bfloat16())
    q = torch.randn(1, N, n_kv * G, D, generator=gen, device="cuda").bfloat16()
    mask = torch.zeros(N, N, dtype=torch.bool, device="cuda")
    out = cache.decode_attention_tree(q, mask, ctx_len=ctx)
    check_weighted(cache, q, mask, ctx, out)


@pytest.mark.parametrize("bits,N", [(8, 32), (4, 32), (8, 64), (4, 50)])
def test_tree_repeats_of_unlike_rows(bits, N):
    """Exponents of the rows' own in many tiles of long contexts, next to tiles without: the same bits every time."""
    ctx = [4000 + 37 * i for i in range(12)]
    cache, gen = filled_cache([n + N for n in ctx], 8, bits, seed=N + bits)
    for name in ("k_scale", "v_scale"):
        t = getattr(cache, name)
        few = torch.rand(t.shape, generator=gen, device="cuda") < 0.01
        t[few] *= 2.0 ** torch.randint(-30, 14, (int(few.sum()),), generator=gen, device="cuda").float()
    q = torch.randn(len(ctx), N, 32, D, generator=gen, device="cuda").bfloat16()
    mask = torch.rand(len(ctx), N, N, generator=gen, device="cuda") < 0.4
    length = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    first = cache.decode_attention_tree(q, mask, ctx_len=length)
    for _ in range(12):
        assert torch.equal(cache.decode_attention_tree(q, mask, ctx_len=length), first)
    cache.check_status()
    check_weighted(cache, q[:2], mask[:2], length, first)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("N,G", [(9, 4), (64, 8)])
def test_tree_unlike_rows_that_are_not_finite(bits, N, G):
    """Rows that are not finite next to rows of unlike sizes, in one tile: what a node does not see does not reach it."""
    n_kv, ctx = 1, torch.tensor([200], dtype=torch.int32, device="cuda")
    cache, gen = filled_cache([200 + N], n_kv, bits, seed=N)
    q = torch.randn(1, N, n_kv * G, D, generator=gen, device="cuda").bfloat16()
    mask = torch.eye(N, dtype=torch.bool, device="cuda")
    mask[6, 3] = mask[7, 5] = True
    for which in ("k", "v"):
        grow(cache, 0, 150, 2.0 ** -12, which)
        grow(cache, 0, 204, 2.0 ** 15, which)
    want, want_lse = cache.decode_attention_tree(q, mask, ctx_len=ctx, want_lse=True)
    check_weighted(cache, q, mask, ctx, want)
    for which in ("k_scale", "v_scale"):
        for node, x in ((3, math.nan), (5, math.inf)):
            getattr(cache, which)[int(cache.page_table[0, (200 + node) // PAGE]), 0, (200 + node) % PAGE] = x
        out, lse = cache.decode_attention_tree(q, mask, ctx_len=ctx, want_lse=True)
        hit = [3, 5, 6, 7]
        rest = [i for i in range(N) if i not in hit]
        assert torch.equal(out[0, rest], want[0, rest]) and torch.equal(lse[0, rest], want_lse[0, rest])
        assert bool((~torch.isfinite(out[0, hit])).any(-1).all())
    cache.check_status()


# ---- the choice of pages ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("key,query", [(-60, -118), (108, 10), (-100, -40), (100, 100)])
def test_page_scores_of_any_size(key, query):
    """Scores whose sizes are beyond fp32's are ranked all the same: only their ratios matter."""
    P, G = 300, 4
    cache, gen = filled_cache([P * PAGE], 2, 8, seed=23)
    lens = torch.tensor([P * PAGE], dtype=torch.int32, device="cuda")
    bounds = cache.page_bounds()
    cache.update_bounds(bounds, seq_len=lens)
    q = torch.randn(1, 2 * G, D, generator=gen, device="cuda").bfloat16()
    q[:, 1] *= 2.0 ** -9                                               # heads of a group of unlike sizes
    _, want = cache.decode_attention_sparse(q, bounds, 20, seq_len=lens, want_pages=True)
    bounds.scale *= 2.0 ** key
    _, got = cache.decode_attention_sparse((q.float() * 2.0 ** query).bfloat16(), bounds, 20, seq_len=lens, want_pages=True)
    cache.check_status()
    assert torch.equal(got, want)


# ---- the largest cache ------------------------------------------------------------------------------------------------
def test_positions_next_to_2_31():
    """A stream whose pages end 16 rows before 2^31 (all of them one page of the pool): trees and paths that do not fit there."""
    import pikv_b200
    most = 2 ** 31 - 16
    cache = pikv_b200.PagedKVCache(1, most, 1, num_pages=1, identity_table=False)
    cache.page_table.zero_()
    gen = torch.Generator(device="cuda").manual_seed(37)
    v = torch.randn(16, D, generator=gen, device="cuda").bfloat16()
    append_rows(cache, 0, 0, torch.zeros_like(v), v)
    k, v = rows64(cache, 0, 16)
    N = 20
    q = torch.randn(1, N, 2, D, generator=gen, device="cuda").bfloat16()
    mask = torch.ones(N, N, dtype=torch.bool, device="cuda")
    out, lse = cache.decode_attention_tree(q, mask, ctx_len=torch.tensor([most - 10], dtype=torch.int32, device="cuda"), want_lse=True)
    assert int(cache.status) == 8 and not out[0, 10:].any() and bool((lse[0, 10:] == -math.inf).all())
    cache.status.zero_()
    # Every row weighs the same.  A block adds up 2^31 / 64 / 296 tiles of four products each in fp32, 2^-23 a sum at most
    off = 2 ** 31 / 64 / 296 * 4 * 2.0 ** -23
    assert bool(((out[0, :10].double() - v.mean(0)).abs() <= (2 * off + 2.0 ** -8) * v.abs().max()).all())
    assert bool(((lse[0, :10].double() - math.log(most)).abs() <= off).all())
    assert not cache.decode_attention_tree(q, mask, ctx_len=torch.tensor([2 ** 31 - 1], dtype=torch.int32, device="cuda"),
                                           nodes=torch.zeros(1, dtype=torch.int32, device="cuda")).any()
    # nothing of these paths fits, is ascending, or is a length
    held = [t.clone() for _, t in cache.named_buffers()]
    path = torch.arange(40, dtype=torch.int32, device="cuda")[None].contiguous()
    for ctx, p in ((most - 10, path), (most, path), (most - 30, path.flip(1).contiguous()), (most - 5, torch.zeros_like(path)), (2 ** 31 - 1, path)):
        new = cache.accept_tree(p, ctx_len=torch.tensor([ctx], dtype=torch.int32, device="cuda"))
        assert int(cache.status) == 8 and int(new[0]) == ctx
        cache.status.zero_()
        assert all(torch.equal(a, t) for a, (_, t) in zip(held, cache.named_buffers()))
