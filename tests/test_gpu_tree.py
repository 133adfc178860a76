"""Attention for a tree of drafted tokens and the acceptance of a path, against 64 bits on the cache's own rows."""
import math

import pytest
import torch

from paged_reference import D, append_rows, attend64, check_attention, filled_cache, rows64

pytestmark = pytest.mark.gpu
# K and V enter as f16 in units of 2^(e - 9), 2^e above the largest scale of 64 rows: a rounding of 2^-11 of the entry, and of
# 2^-25 units = 2^-16 2^e, at most 2^-15 of the largest scale, where the entry is below f16's normal range.  Rows of one size have
# entries of 40 scales in the mean (127 at most), their scales lie within a factor of two: 2^-15 / 20 < 2^-19 of a mean entry.
# A logit: that of each of its 128 products, which are then summed in fp32 (2^-24 each at most, of the sum of their sizes; tensor
# cores truncate, twice that), the scalings behind them and the exponential's argument (a few times 2^-24 of a value below that sum)
VALUE = 2.0 ** -11 + 2.0 ** -19
LOGIT = VALUE + (2 * 128 + 8) * 2.0 ** -24


@pytest.fixture(autouse=True)
def device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def random_trees(gen, B, N):
    """Masks [B, N, N] of random trees: every node sees itself and its ancestors."""
    mask = torch.zeros(B, N, N, dtype=torch.bool)
    cpu = torch.Generator().manual_seed(int(torch.randint(1 << 30, (1,), generator=gen, device="cuda")))
    for b in range(B):
        for i in range(N):
            if i:
                mask[b, i] = mask[b, int(torch.randint(i, (1,), generator=cpu))]
            mask[b, i, i] = True
    return mask.cuda()


def compare(cache, q, mask, ctx, nodes, out, lse, ids=None):
    B, N = q.shape[:2]
    for b in range(B):
        s = b if ids is None else int(ids[b])
        n, t = int(ctx[b]), N if nodes is None else int(nodes[b])
        assert not out[b, t:].any()
        if lse is not None:
            assert bool((lse[b, t:] == -math.inf).all())
        if t == 0:
            continue
        k, v = rows64(cache, s, n + t)
        m = mask[b] if mask.dim() == 3 else mask
        sees = torch.cat([torch.ones(t, n, dtype=torch.bool, device="cuda"), m[:t, :t]], 1)
        check_attention(out[b, :t], None if lse is None else lse[b, :t], *attend64(q[b, :t], k, v, sees), LOGIT, VALUE)


# one row alone; contexts at the edges of pages and of 64-row tiles; row counts (nodes x group) of one, of a ragged tile, of two and
# four tiles of 128, of a group wider than a tile; contexts over many splits
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("ctx,N,G,n_kv", [
    ([0], 1, 1, 1), ([1], 1, 1, 2), ([0, 1, 15, 16, 17, 47, 48, 49, 63, 64, 65, 127, 128, 129, 500], 5, 4, 2), ([300, 60, 0], 33, 3, 1),
    ([1000, 0, 777], 64, 4, 1), ([130, 700], 64, 8, 1), ([90], 3, 64, 1), ([64, 200], 7, 48, 2), ([20000, 3], 16, 4, 2), ([9000], 64, 4, 2)])
def test_tree_attention(bits, ctx, N, G, n_kv):
    cache, gen = filled_cache([n + N for n in ctx], n_kv, bits, seed=len(ctx) + N)
    B = len(ctx)
    q = torch.randn(B, N, G * n_kv, D, generator=gen, device="cuda").bfloat16()
    mask = random_trees(gen, B, N)
    length = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    out, lse = cache.decode_attention_tree(q, mask, ctx_len=length, want_lse=True)
    cache.check_status()
    compare(cache, q, mask, length, None, out, lse)
    cache.length.copy_(length)                                     # the default is the cache's own lengths
    assert torch.equal(cache.decode_attention_tree(q, mask), out)


# any pattern is a mask: rows that see no drafted row, not even their own, and with no context nothing at all; streams named in any
# order and more than once; trees of different sizes, none among them; one mask for all
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("N,G,n_kv", [(6, 4, 2), (64, 2, 1), (40, 8, 1)])
@pytest.mark.parametrize("shared", [False, True])
def test_tree_masks_and_sizes(bits, N, G, n_kv, shared):
    rows = [N + 70, N, N + 16, N + 333, N + 1]
    cache, gen = filled_cache(rows, n_kv, bits, seed=N)
    ids = torch.tensor([3, 1, 1, 0, 4, 2, 3], dtype=torch.int32, device="cuda")
    ctx = torch.tensor([333, 0, 0, 70, 0, 16, 40], dtype=torch.int32, device="cuda")
    nodes = torch.tensor([N, 1, N, 0, N // 2, N - 1, N], dtype=torch.int32, device="cuda")
    B = len(ids)
    q = (torch.randn(B, N, G * n_kv, D, generator=gen, device="cuda") * torch.randn(B, N, G * n_kv, 1, generator=gen, device="cuda").exp()).bfloat16()
    mask = torch.rand(*((N, N) if shared else (B, N, N)), generator=gen, device="cuda") < 0.3
    mask[..., 0, :] = False
    out, lse = cache.decode_attention_tree(q, mask, seq_ids=ids, ctx_len=ctx, nodes=nodes, want_lse=True)
    cache.check_status()
    assert bool((lse[1, 0] == -math.inf).all())                    # no context and an empty mask row
    compare(cache, q, mask, ctx, nodes, out, lse, ids)


# long enough for copies, conversions and products of many tiles to run into one another where a wait or a fence is missing
@pytest.mark.parametrize("bits,N", [(8, 32), (4, 32), (8, 64), (4, 50)])
def test_tree_repeats(bits, N):
    ctx = [6000 + 37 * i for i in range(12)]
    cache, gen = filled_cache([n + N for n in ctx], 8, bits, seed=N)
    q = torch.randn(len(ctx), N, 32, D, generator=gen, device="cuda").bfloat16() * 3
    mask = random_trees(gen, len(ctx), N)
    length = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    first = cache.decode_attention_tree(q, mask, ctx_len=length)
    for _ in range(12):
        assert torch.equal(cache.decode_attention_tree(q, mask, ctx_len=length), first)
    compare(cache, q[-1:], mask[-1:], length[-1:], None, first[-1:], None, ids=[len(ctx) - 1])
    cache.check_status()


def test_tree_next_to_other_kernels():
    """Wide and narrow trees and a projection, which take tensor memory too, behind one another and on streams side by side."""
    import pikv_b200
    made = []
    for N, bits in ((64, 8), (16, 8), (60, 4)):
        cache, gen = filled_cache([2000 + 300 * i + N for i in range(6)], 4, bits, seed=N)
        cache.length.copy_(torch.tensor([2000 + 300 * i for i in range(6)], dtype=torch.int32))
        made.append((cache, torch.randn(6, N, 16, D, generator=gen, device="cuda").bfloat16(), random_trees(gen, 6, N)))
    x = torch.randn(8192, 1024, generator=gen, device="cuda").bfloat16()
    w = torch.randn(64, 1024, generator=gen, device="cuda").bfloat16()

    def steps(first):
        got = []
        for i in range(3):
            cache, q, mask = made[(first + i) % 3]
            got += [pikv_b200.ops.lowrank_project(x, w), cache.decode_attention_tree(q, mask)]
        return got

    want = [steps(i) for i in range(3)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        got = []
        for i, s in enumerate(streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(steps(i))
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        assert all(torch.equal(a, b) for x_, y_ in zip(got, want) for a, b in zip(x_, y_))
    for cache, _, _ in made:
        cache.check_status()


def test_tree_zero_points():
    """4-bit rows of one value, whose zero points are millions, between ordinary ones; zero points that are not whole numbers."""
    ctx, N, n_kv = [150, 64], 9, 2
    cache, gen = filled_cache([n + N for n in ctx], n_kv, 4, seed=11)
    for s, n in enumerate(ctx):
        k, v = (torch.randn(n, n_kv * D, generator=gen, device="cuda") for _ in range(2))
        k[1::3] = torch.randn(len(k[1::3]), 1, generator=gen, device="cuda")
        v[2::3] = 30 * torch.randn(len(v[2::3]), 1, generator=gen, device="cuda")
        k[5], v[7] = 0, 0
        append_rows(cache, s, 0, k.bfloat16(), v.bfloat16())
    assert float(torch.nan_to_num(cache.k_zp).abs().max()) > 1e5
    q = torch.randn(2, N, 4 * n_kv, D, generator=gen, device="cuda").bfloat16()
    mask = random_trees(gen, 2, N)
    length = torch.tensor(ctx, dtype=torch.int32, device="cuda")

    def check():
        out, lse = cache.decode_attention_tree(q, mask, ctx_len=length, want_lse=True)
        cache.check_status()
        for b, n in enumerate(ctx):
            k, v = rows64(cache, b, n + N)
            sees = torch.cat([torch.ones(N, n, dtype=torch.bool, device="cuda"), mask[b]], 1)
            # An entry (code - zero point) scale is rounded twice here, by 2^-11 each (the difference, where it is above 2048 steps, and
            # the entry), and what a factor lost comes back rounded by 2^-11 of at most 2^-10 of it; the dequantised rows that it is
            # compared with are rounded to fp32 twice.  Units: 2^-25 where the tile's largest row has entries above 2^-6, of its own
            value = 2.0 ** -10 + 2.0 ** -20 + 2.0 ** -19
            check_attention(out[b], lse[b], *attend64(q[b], k, v, sees), value + (2 * 128 + 8) * 2.0 ** -24, value)

    check()
    for zp in (cache.k_zp, cache.v_zp):
        zp.add_(torch.rand(zp.shape, generator=gen, device="cuda") - 0.5)
    check()


def test_tree_layouts():
    """Strided and unaligned queries, a strided mask."""
    N, n_q, n_kv = 9, 8, 2
    cache, gen = filled_cache([200, 77], n_kv, 8, seed=5)
    ctx = torch.tensor([191, 60], dtype=torch.int32, device="cuda")
    q = torch.randn(2, N, n_q, D, generator=gen, device="cuda").bfloat16()
    mask = random_trees(gen, 2, N)
    want = cache.decode_attention_tree(q, mask, ctx_len=ctx)
    odd = torch.empty(q.numel() + 3, dtype=torch.bfloat16, device="cuda")[3:].view_as(q)
    odd.copy_(q)
    assert torch.equal(cache.decode_attention_tree(odd, mask, ctx_len=ctx), want)
    wide = torch.zeros(2, n_q, N, D, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    wide.copy_(q)
    assert torch.equal(cache.decode_attention_tree(wide, mask.transpose(1, 2).contiguous().transpose(1, 2), ctx_len=ctx), want)
    assert cache.decode_attention_tree(q[:0], mask[:0], ctx_len=ctx[:0]).shape == (0, N, n_q, D)
    assert cache.decode_attention_tree(q[:, :0], mask[:, :0, :0], ctx_len=ctx).shape == (2, 0, n_q, D)


def test_tree_many_streams():
    """More streams than one launch takes, with and without ids."""
    S, N, n_kv = 600, 3, 1
    rows = [5 + (i * 37) % 90 + N for i in range(S)]
    cache, gen = filled_cache(rows, n_kv, 8, seed=8)
    ctx = torch.tensor([r - N for r in rows], dtype=torch.int32, device="cuda")
    q = torch.randn(S, N, 2, D, generator=gen, device="cuda").bfloat16()
    mask = random_trees(gen, S, N)
    out, lse = cache.decode_attention_tree(q, mask, ctx_len=ctx, want_lse=True)
    some = torch.tensor([0, 1, 511, 512, 513, 599], device="cuda")
    for b in some.tolist():
        k, v = rows64(cache, b, rows[b])
        sees = torch.cat([torch.ones(N, rows[b] - N, dtype=torch.bool, device="cuda"), mask[b]], 1)
        check_attention(out[b], lse[b], *attend64(q[b], k, v, sees), LOGIT, VALUE)
    ids = torch.randperm(S, generator=gen, device="cuda")
    cache.length.copy_(ctx)
    again = cache.decode_attention_tree(q[ids].contiguous(), mask[ids].contiguous(), seq_ids=ids.int())
    off = (again.float() - out[ids].float()).abs()                 # split elsewhere: two roundings of the same sum
    assert bool((off <= 2.0 ** -7 * out[ids].float().abs() + 2.0 ** -9).all())
    cache.check_status()


@pytest.mark.parametrize("bits", [8, 4])
def test_tree_values_that_are_not_finite(bits):
    """What a row does not see does not reach it, whatever it holds; what it sees does."""
    N, n_kv, G = 8, 2, 4
    cache, gen = filled_cache([100 + N], n_kv, bits, seed=11)
    q = torch.randn(1, N, n_kv * G, D, generator=gen, device="cuda").bfloat16()
    mask = torch.eye(N, dtype=torch.bool, device="cuda")
    mask[5, 4] = True
    ctx = torch.tensor([100], dtype=torch.int32, device="cuda")
    want, want_lse = cache.decode_attention_tree(q, mask, ctx_len=ctx, want_lse=True)
    page, row = int(cache.page_table[0, 104 // 16]), 104 % 16
    for name in ("k_scale", "v_scale"):
        for x in (math.nan, math.inf):
            kept = getattr(cache, name)[page, 0, row].clone()
            getattr(cache, name)[page, 0, row] = x                  # node 4, KV head 0
            out, lse = cache.decode_attention_tree(q, mask, ctx_len=ctx, want_lse=True)
            getattr(cache, name)[page, 0, row] = kept
            hit = torch.zeros(N, n_kv * G, dtype=torch.bool, device="cuda")
            hit[4:6, :G] = True
            assert torch.equal(out[0][~hit], want[0][~hit]) and torch.equal(lse[0][~hit], want_lse[0][~hit])
            assert bool((~torch.isfinite(out[0][hit])).any(-1).all())
    q[0, 2, 3] = math.nan
    q[0, 6, 7, 5] = math.inf
    out = cache.decode_attention_tree(q, mask, ctx_len=ctx)
    hit = torch.zeros(N, n_kv * G, dtype=torch.bool, device="cuda")
    hit[2, 3] = hit[6, 7] = True
    assert torch.equal(out[0][~hit], want[0][~hit]) and bool(torch.isnan(out[0][2, 3]).all())
    cache.check_status()


@pytest.mark.parametrize("size", [1e-6, 1e-3, 1e4, 1e30])
def test_tree_value_ranges(size):
    """Values far from 1, keys with them, and queries that bring the logits back: the weights' 16 bits are relative."""
    N, n_kv, G = 4, 1, 2
    cache, gen = filled_cache([300], n_kv, 8, seed=3)
    k, v = (torch.randn(300, D, generator=gen, device="cuda") * size for _ in range(2))
    v *= torch.randn(300, 1, generator=gen, device="cuda").exp()
    append_rows(cache, 0, 0, k.bfloat16(), v.bfloat16())
    q = (torch.randn(1, N, G, D, generator=gen, device="cuda") / size).bfloat16()
    mask = torch.ones(N, N, dtype=torch.bool, device="cuda")
    ctx = torch.tensor([300 - N], dtype=torch.int32, device="cuda")
    out, lse = cache.decode_attention_tree(q, mask, ctx_len=ctx, want_lse=True)
    compare(cache, q, mask, ctx, None, out, lse)


def test_tree_bad_streams_and_pages():
    """Ids outside the cache, trees that do not fit behind their context and pages that the table does not hold raise status bits;
    the other streams' results stay."""
    N, n_kv = 4, 2
    cache, gen = filled_cache([90, 33, 64], n_kv, 8, seed=2, capacity=96)
    q = torch.randn(4, N, 8, D, generator=gen, device="cuda").bfloat16()
    mask = random_trees(gen, 4, N)
    ids = torch.tensor([0, -1, 2, 3], dtype=torch.int32, device="cuda")
    ctx = torch.tensor([86, 5, 60, 7], dtype=torch.int32, device="cuda")
    out, lse = cache.decode_attention_tree(q, mask, seq_ids=ids, ctx_len=ctx, want_lse=True)
    assert int(cache.status) == 1 and not out[[1, 3]].any() and bool((lse[[1, 3]] == -math.inf).all())
    cache.status.zero_()
    for b in (0, 2):
        compare(cache, q[b:b + 1], mask[b:b + 1], ctx[b:b + 1], None, out[b:b + 1], lse[b:b + 1], ids[b:b + 1])
    good = out[0].clone()
    cache.page_table[2, 1] = cache.num_pages
    out = cache.decode_attention_tree(q, mask, seq_ids=torch.tensor([0, 0, 2, 0], dtype=torch.int32, device="cuda"), ctx_len=ctx)
    assert int(cache.status) == 2 and torch.equal(out[0], good)
    cache.status.zero_()
    cache.decode_attention_tree(q[:1], mask[:1], ctx_len=torch.tensor([cache.max_pages * 16 - 2], dtype=torch.int32, device="cuda"))
    assert int(cache.status) & 8
    cache.status.zero_()


# ---- acceptance ---------------------------------------------------------------------------------------------------
def buffers(cache):
    return {n: t.clone() for n, t in cache.named_buffers() if n != "status"}


# paths at page edges, whole and of one node, across two pages; deeper than a batch of sixteen rows; every format
@pytest.mark.parametrize("bits,sym", [(8, True), (4, False), (8, False), (4, True)])
@pytest.mark.parametrize("ctx,N,depth", [([0, 1, 14, 15, 16, 31], 9, 5), ([100], 1, 1), ([5, 250], 64, 40), ([7], 200, 33)])
def test_accept_moves_rows(bits, sym, ctx, N, depth):
    import pikv_b200
    gen = torch.Generator(device="cuda").manual_seed(N + depth)
    n_kv, B = 3, len(ctx)
    cap = max(ctx) + N
    cache = pikv_b200.PagedKVCache(B + 1, cap, n_kv, bits=bits, symmetric=sym)
    cache.page_table.copy_(torch.randperm(cache.num_pages, generator=gen, device="cuda").int().view_as(cache.page_table))
    for s in range(B + 1):
        append_rows(cache, s, 0, *(torch.randn(cap, n_kv * D, generator=gen, device="cuda").bfloat16() for _ in range(2)))
    ids = torch.randperm(B + 1, generator=gen, device="cuda")[:B].int()
    path = torch.stack([torch.randperm(N, generator=gen, device="cuda")[:depth].sort().values for _ in range(B)]).int()
    count = torch.randint(0, depth + 1, (B,), generator=gen, device="cuda").int()
    count[-1] = depth
    length = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    before = [[cache.gather(torch.full((cap,), s, dtype=torch.int32, device="cuda"), torch.arange(cap, dtype=torch.int32, device="cuda"), w, codes=True) for w in "kv"]
              for s in range(B + 1)]
    cache.length.copy_(torch.full((B + 1,), -7, dtype=torch.int32))
    new = cache.accept_tree(path, count, seq_ids=ids, ctx_len=length)
    cache.check_status()
    assert torch.equal(new, length + count)
    named = {int(s): b for b, s in enumerate(ids)}
    for s in range(B + 1):
        at = torch.arange(cap, device="cuda")
        if s in named:
            b = named[s]
            c = int(count[b])
            at[ctx[b]:ctx[b] + c] = ctx[b] + path[b, :c].long()
            assert int(cache.length[s]) == ctx[b] + c
        else:
            assert int(cache.length[s]) == -7
        for w, (rows, codes) in zip("kv", before[s]):
            got = cache.gather(torch.full((cap,), s, dtype=torch.int32, device="cuda"), torch.arange(cap, dtype=torch.int32, device="cuda"), w, codes=True)
            assert torch.equal(got[0], rows[at]) and torch.equal(got[1], codes[at])


def test_accept_refused_paths():
    """A path that does not ascend, leaves the cache or meets a bad page, and a stream named twice: nothing moves, and the status
    word says so; the other streams of the call are carried out."""
    cache, gen = filled_cache([60] * 4, 2, 8, seed=4, capacity=64)
    ctx = torch.tensor([40, 41, 42, 50], dtype=torch.int32, device="cuda")
    cache.length.copy_(ctx)
    start = buffers(cache)
    for path, bit in (([2, 2, 3], 8), ([3, 1, 4], 8), ([-1, 0, 1], 8), ([0, 5, 24], 8), ([0, 5, 2**31 - 1], 8)):
        p = torch.tensor([[0, 1, 2], path, [0, 1, 2], [0, 1, 2]], dtype=torch.int32, device="cuda")
        new = cache.accept_tree(p)
        assert int(cache.status) == bit
        cache.status.zero_()
        assert new.tolist() == [43, 41, 45, 53]
        for n, t in buffers(cache).items():
            assert torch.equal(t.view(torch.uint8), start[n].view(torch.uint8)) or n == "length"      # 0, 1, 2 move onto themselves
        cache.length.copy_(ctx)
    p = torch.tensor([[1, 2, 4]] * 3, dtype=torch.int32, device="cuda")
    for count in (4, -1):
        new = cache.accept_tree(p[:1], torch.tensor([count], dtype=torch.int32, device="cuda"))
        assert int(cache.status) == 8 and new.tolist() == [40]
        cache.status.zero_()
    new = cache.accept_tree(p, seq_ids=torch.tensor([2, 4, 2], dtype=torch.int32, device="cuda"))
    assert int(cache.status) == 1 and new.tolist() == [45, 0, 0] and cache.length.tolist() == [40, 41, 45, 50]
    cache.status.zero_()
    new = cache.accept_tree(p[:, :0], seq_ids=torch.tensor([3, 0, 2], dtype=torch.int32, device="cuda"))     # nothing accepted
    assert new.tolist() == [50, 40, 45] and cache.length.tolist() == [40, 41, 45, 50]
    assert cache.accept_tree(p[:0]).shape == (0,)
    cache.check_status()
    cache.page_table[1, 2] = -1
    held = buffers(cache)
    new = cache.accept_tree(p[:1], seq_ids=torch.tensor([1], dtype=torch.int32, device="cuda"))
    assert int(cache.status) == 2 and new.tolist() == [41]
    cache.status.zero_()
    assert all(torch.equal(t.view(torch.uint8), held[n].view(torch.uint8)) for n, t in buffers(cache).items())


@pytest.mark.parametrize("bits", [8, 4])
def test_accept_many_streams(bits):
    """More streams than one launch takes, without ids and with ids in any order; a stream named in both launches is carried out once."""
    S, N, n_kv = 600, 6, 1
    ctx = [3 + (i * 37) % 60 for i in range(S)]
    cache, gen = filled_cache([n + N for n in ctx], n_kv, bits, seed=18)
    length = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    path = torch.stack([torch.randperm(N, generator=gen, device="cuda")[:4].sort().values for _ in range(S)]).int()
    count = torch.randint(0, 5, (S,), generator=gen, device="cuda").int()
    saved = {n: t.clone() for n, t in cache.named_buffers()}
    before = [rows64(cache, s, ctx[s] + N) for s in range(S)]

    def check(streams, new):
        for b, s in enumerate(streams):
            c = int(count[b])
            at = torch.arange(ctx[s] + N, device="cuda")
            at[ctx[s]:ctx[s] + c] = ctx[s] + path[b, :c].long()
            assert int(new[b]) == ctx[s] + c == int(cache.length[s])
            assert all(torch.equal(x, y[at]) for x, y in zip(rows64(cache, s, ctx[s] + N), before[s]))

    cache.length.copy_(length)
    new = cache.accept_tree(path, count)                               # the cache's own lengths, read and written
    cache.check_status()
    check(range(S), new)
    for twice in (False, True):
        for n, t in cache.named_buffers():
            t.copy_(saved[n])
        cache.length.copy_(length)
        ids = torch.randperm(S, generator=gen, device="cuda").int()
        if twice:
            ids[530] = ids[7]                                          # 7 goes with the first launch, 530 with the second
        new = cache.accept_tree(path, count, seq_ids=ids, ctx_len=length[ids.long()].contiguous())
        if twice:
            assert int(cache.status) == 1 and int(new[530]) == 0
            cache.status.zero_()
            keep = [b for b in range(S) if b != 530]
            left_out = set(range(S)) - set(ids.tolist())
            assert all(torch.equal(x, y) for s in left_out for x, y in zip(rows64(cache, s, ctx[s] + N), before[s]))
            path, count, new, ids = path[keep], count[keep], new[keep], ids[keep]
        cache.check_status()
        check(ids.tolist(), new)
