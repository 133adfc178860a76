"""Operators of a speculative, long-context decode loop over the paged quantised cache, as cases that can be timed.

Four operators: attention for a tree of drafted tokens over the cache, the acceptance of one path of that tree (its rows
move up behind the context), the bounds of every page's keys, and decode attention over the pages that those bounds
select.  `run` computes them with elementary torch operations, or with the package's own calls where `own` is set.

The cache layout is the package's: pages of 16 rows, [page, head, row, bytes]; the 16-byte chunk c of an 8-bit row lies at
c ^ (row & 7), the 8-byte unit u of a 4-bit row at u ^ (row & 4), the even channel of a byte in its low nibble.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

D = 128                 # head width of the cache
PAGE = 16               # rows per page
TOPIC = 64              # neighbouring rows whose keys resemble one another


def listed():
    return [
        # one user, a short conversation, a small draft: the latency of one verification step
        dict(name="tree_single", kind="tree", streams=1, context=1500, nodes=8, n_kv=8, group=4, bits=8, ragged=False),
        # a serving batch with long contexts; 32 drafted tokens and 4 query heads fill the 128 rows of a tensor-core tile
        dict(name="tree_16x16384", kind="tree", streams=16, context=16384, nodes=32, n_kv=8, group=4, bits=8, ragged=False),
        # large trees over long contexts: two tiles of rows for every key, the most arithmetic for its bytes
        dict(name="tree_wide_8x32768", kind="tree", streams=8, context=32768, nodes=64, n_kv=8, group=4, bits=8, ragged=False),
        # requests of different lengths with trees of different sizes over the 4-bit cache
        dict(name="tree_ragged_q4", kind="tree", streams=24, context=6001, nodes=21, n_kv=8, group=4, bits=4, ragged=True),
        # the path of one user's tree
        dict(name="accept_single", kind="accept", streams=1, context=1500, nodes=8, depth=5, n_kv=8, bits=8),
        # the paths of a batch of large trees, 4-bit cache
        dict(name="accept_64_q4", kind="accept", streams=64, context=2001, nodes=64, depth=16, n_kv=8, bits=4),
        # one new token in each of 64 streams: the bounds of one page per stream and head
        dict(name="bounds_token_64", kind="bounds", streams=64, context=4099, fresh=1, n_kv=8, bits=8, ragged=True),
        # whole prompts
        dict(name="bounds_prompt_8x32768", kind="bounds", streams=8, context=32768, fresh=32768, n_kv=8, bits=8, ragged=False),
        # ragged prompts in the 4-bit cache
        dict(name="bounds_prompt_q4", kind="bounds", streams=24, context=6001, fresh=6001, n_kv=8, bits=4, ragged=True),
        # one user's long document, 64 of its 2048 pages
        dict(name="sparse_single_32768", kind="sparse", streams=1, context=32768, pages=64, first=1, recent=4, n_kv=8, group=4, bits=8, ragged=False),
        # a full decode batch over long contexts, a sixteenth of the pages
        dict(name="sparse_64x32768", kind="sparse", streams=64, context=32768, pages=128, first=1, recent=4, n_kv=8, group=4, bits=8, ragged=False),
        # requests of different lengths over the 4-bit cache, some shorter than their budget
        dict(name="sparse_ragged_q4", kind="sparse", streams=24, context=50001, pages=100, first=0, recent=1, n_kv=8, group=4, bits=4, ragged=True),
    ]


def _between(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "sparse", "sparse", "sparse", "bounds", "accept"])
    bits, n_kv = rng.choice([8, 8, 4]), rng.choice([1, 2, 4, 8, 8])
    if kind == "tree":
        streams = _between(rng, 1, 64)
        return dict(kind=kind, streams=streams, context=_between(rng, 1, min(32768, 262144 // streams)), nodes=_between(rng, 1, 64),
                    n_kv=n_kv, group=rng.choice([1, 2, 4, 4, 3]), bits=bits, ragged=rng.random() < 0.6)
    if kind == "accept":
        nodes = _between(rng, 2, 64)
        return dict(kind=kind, streams=_between(rng, 1, 64), context=_between(rng, 1, 4096), nodes=nodes, depth=_between(rng, 1, min(16, nodes)),
                    n_kv=n_kv, bits=bits)
    if kind == "bounds":
        streams = _between(rng, 1, 64)
        context = _between(rng, 1, min(32768, 262144 // streams))
        return dict(kind=kind, streams=streams, context=context, fresh=rng.choice([1, _between(rng, 1, context), context]), n_kv=n_kv, bits=bits,
                    ragged=rng.random() < 0.6)
    streams = _between(rng, 1, 64)
    context = _between(rng, 16, min(131072, 64 * 32768 // streams))
    pages = _between(rng, 4, 128)
    first = rng.choice([0, 1, 2])
    return dict(kind=kind, streams=streams, context=context, pages=pages, first=first, recent=rng.randint(1, pages - first), n_kv=n_kv,
                group=rng.choice([1, 2, 4, 4, 8]), bits=bits, ragged=rng.random() < 0.6)


# ---- sizes that a case stands for ---------------------------------------------------------------------------------
def _lengths(case):
    """Rows of each stream before its tree (or in all): ragged ones are spread over 5 % to 100 % of the longest."""
    n, longest = case["streams"], case["context"]
    if not case.get("ragged"):
        return [longest] * n
    return [max(1, longest - (longest * 19 * ((i * 7919) % n)) // (20 * n)) for i in range(n)]


def _nodes(case):
    n, most = case["streams"], case["nodes"]
    if not case.get("ragged"):
        return [most] * n
    return [max(1, most - (most * ((i * 31) % n)) // (2 * n)) for i in range(n)]


def _pages(n):
    return -(-n // PAGE)


def _row_bytes(bits):
    """One row of one head: codes, scale and, for 4 bits, zero point."""
    return D * bits // 8 + 2 + (4 if bits == 4 else 0)


def work(case):
    kind, h, row = case["kind"], case["n_kv"], _row_bytes(case["bits"])
    lens = _lengths(case)
    if kind == "tree":
        nodes = _nodes(case)
        rows = [n + t for n, t in zip(lens, nodes)]
        io = sum(2 * t * h * case["group"] * D * 2 + t * t for t in nodes)                 # queries, outputs, mask
        return {"bytes": sum(rows) * h * 2 * row + io, "flops": sum(4 * D * t * case["group"] * h * r for t, r in zip(nodes, rows))}
    if kind == "accept":
        moved = case["streams"] * case["depth"]
        return {"bytes": 2 * moved * h * 2 * row + 4 * moved, "flops": 0}
    if kind == "bounds":
        first = [max(0, n - case["fresh"]) // PAGE * PAGE for n in lens]
        rows, pages = sum(n - f for n, f in zip(lens, first)), sum(_pages(n) - f // PAGE for n, f in zip(lens, first))
        return {"bytes": rows * h * row + pages * h * (2 * D + 4), "flops": 2 * rows * h * D}
    pages = [_pages(n) for n in lens]
    kept = [min(n, case["pages"] * PAGE - (-n) % PAGE) for n in lens]
    seen = sum(max(0, p - case["first"] - case["recent"]) for p in pages if p > case["pages"])   # pages that are scored
    io = 2 * case["streams"] * h * case["group"] * D * 2
    return {"bytes": seen * h * (2 * D + 4) + sum(kept) * h * 2 * row + io,
            "flops": seen * h * case["group"] * 4 * D + sum(4 * D * case["group"] * h * k for k in kept)}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _quantise(x, bits):
    """Codes, scale (bf16) and zero point of rows [..., 128], as the cache stores them."""
    lo, hi = x.amin(-1), x.amax(-1)
    if bits == 8:
        scale = 2 * torch.maximum(lo.abs(), hi.abs()) / 255
        q = (x / scale[..., None]).round_().clamp_(-128, 127).to(torch.int8).view(torch.uint8)
        return q, scale.bfloat16(), None
    scale = (hi - lo) / 15
    zp = 0 - torch.round(lo / scale)
    q = ((x / scale[..., None]).add_(zp[..., None]).round_()).clamp_(0, 15).to(torch.uint8)
    return q[..., 0::2] | (q[..., 1::2] << 4), scale.bfloat16(), zp


def _swizzle(codes, bits):
    """Rows [..., 16, bytes] to and from their place in a page (the exchange is its own inverse)."""
    row = torch.arange(PAGE, device=codes.device)
    unit = torch.arange(8, device=codes.device)
    at = unit ^ ((row & 7) if bits == 8 else (row & 4))[:, None]
    shape = codes.shape
    return codes.reshape(*shape[:-1], 8, shape[-1] // 8)[..., row[:, None], at, :].reshape(shape)


def _trees(rng, streams, nodes):
    """Parent of every node (-1: the root, node 0), as a draft model leaves them: most branches near the root."""
    parent = np.full((streams, nodes), -1)
    for i in range(1, nodes):
        parent[:, i] = (rng.random(streams) ** 1.5 * i).astype(int)
    return parent


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = np.random.default_rng(seed)
    kind, B, H, bits = case["kind"], case["streams"], case["n_kv"], case["bits"]
    lens = _lengths(case)
    extra = case["nodes"] if kind in ("tree", "accept") else 0
    width = _pages(case["context"] + extra)
    s = dict(kind=kind, bits=bits, width=width)
    pages = B * width
    row = D * bits // 8
    order = torch.randperm(pages, generator=g, device=dev)           # pages lie anywhere in the pool
    s["page_table"] = order.int().view(B, width)
    for n in ("k", "v"):
        s[n + "_codes"] = torch.empty(pages, H, PAGE, row, dtype=torch.uint8, device=dev)
        s[n + "_scale"] = torch.empty(pages, H, PAGE, dtype=torch.bfloat16, device=dev)
        s[n + "_zp"] = torch.empty(pages, H, PAGE, device=dev) if bits == 4 else None
    # keys of neighbouring rows share a topic, some channels are larger than others; a query asks for a few topics
    topics = -(-width * PAGE // TOPIC)
    topic = torch.randn(B, topics, H, D, generator=g, device=dev)
    loud = 0.6 + torch.rand(H, D, generator=g, device=dev) ** 8 * 2
    for b in range(B):
        at = order[b * width:(b + 1) * width]
        for n in ("k", "v"):
            x = torch.randn(width * PAGE, H, D, generator=g, device=dev)
            if n == "k":
                x = (x * 0.7 + topic[b].repeat_interleave(TOPIC, 0)[:width * PAGE] * 0.7) * loud
            x = x.view(width, PAGE, H, D).transpose(1, 2).bfloat16().float()
            codes, scale, zp = _quantise(x, bits)
            s[n + "_codes"][at] = _swizzle(codes, bits)
            s[n + "_scale"][at] = scale
            if zp is not None:
                s[n + "_zp"][at] = zp
    s["length"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    if kind in ("tree", "sparse"):
        N = case["nodes"] if kind == "tree" else 1
        G = case["group"]
        want = torch.from_numpy(rng.integers(0, topics, (B, N))).to(dev)
        asked = topic[torch.arange(B, device=dev)[:, None], want] * loud                # [B, N, H, D]
        q = 0.8 * asked[:, :, :, None] + 0.8 * torch.randn(B, N, H, G, D, generator=g, device=dev)
        s["q"] = q.reshape(B, N, H * G, D).bfloat16()
    if kind in ("tree", "accept"):
        N = case["nodes"]
        parent = _trees(rng, B, N)
        mask = np.zeros((B, N, N), bool)
        every = np.arange(B)
        for i in range(N):
            mask[:, i] = np.where((parent[:, i] >= 0)[:, None], mask[every, parent[:, i]], False)
            mask[:, i, i] = True
        if kind == "tree":
            s["mask"] = torch.from_numpy(mask).to(dev)
            s["nodes"] = torch.tensor(_nodes(case), dtype=torch.int32, device=dev)
        else:
            # a path of `depth` nodes down the tree; a real tree may be shallower, so the rest are nodes in rising order
            path = np.stack([np.sort(rng.permutation(N)[:case["depth"]]) for _ in range(B)])
            s["path"] = torch.from_numpy(path).int().to(dev)
            s["path_len"] = torch.from_numpy(rng.integers(1, case["depth"] + 1, B)).int().to(dev)
            s["path_len"][0] = case["depth"]
    if kind == "bounds":
        s["start"] = torch.clamp(s["length"] - case["fresh"], min=0)
    if kind in ("bounds", "sparse"):
        s["bound_codes"] = torch.zeros(pages, H, 2, D, dtype=torch.int8, device=dev)
        s["bound_scale"] = torch.zeros(pages, H, device=dev)
    if kind == "sparse":
        s["q"] = s["q"][:, 0].contiguous()
        s["pages"], s["first"], s["recent"] = case["pages"], case["first"], case["recent"]
        for b in range(B):                                             # what a program keeps beside its cache
            n = _pages(lens[b])
            codes, scale = _bounds(s, slice(b, b + 1), torch.zeros(1, dtype=torch.int32, device=dev))
            s["bound_codes"][s["page_table"][b, :n].long()] = codes[0, :n]
            s["bound_scale"][s["page_table"][b, :n].long()] = scale[0, :n]
    if own:
        import pikv_b200
        cache = pikv_b200.PagedKVCache(B, width * PAGE, H, bits=bits, symmetric=bits == 8, device=dev, identity_table=False, num_pages=pages)
        for n, t in cache.named_buffers():
            if n in s:                                                 # one copy of the cache: its buffers are the state's
                setattr(cache, n, s[n].clone() if n == "length" else s[n])     # accept_tree writes the cache's own length
        s["cache"] = cache
        if kind in ("bounds", "sparse"):
            s["bounds"] = pikv_b200.PageBounds(s["bound_codes"], s["bound_scale"])
    return s


# ---- the plain forms -----------------------------------------------------------------------------------------------
def _values(s, name, pages, dtype=torch.float32):
    """Dequantised rows of physical pages [...]: [..., H, 16, 128].  A row's value is (code - zero point) * scale in 32 bits."""
    return _decode(s, name, s[name + "_codes"][pages], s[name + "_scale"][pages], None if s[name + "_zp"] is None else s[name + "_zp"][pages], dtype)


def _decode(s, name, codes, scale, zp, dtype=torch.float32):
    codes = _swizzle(codes, s["bits"])
    if s["bits"] == 8:
        return codes.view(torch.int8).to(dtype) * scale[..., None].to(dtype)
    both = torch.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], D)
    return (both.to(dtype) - zp[..., None].to(dtype)) * scale[..., None].to(dtype)


def _tree(s):
    """softmax(q K^T / sqrt(128)) V of every drafted token over its stream's rows and, behind them, its ancestors' rows."""
    q, mask, length, nodes = s["q"], s["mask"], s["length"].long(), s["nodes"].long()
    B, N, HQ, _ = q.shape
    k, v = (_values(s, n, s["page_table"].long()).transpose(1, 2).flatten(2, 3) for n in "kv")    # [B, H, rows, D]
    H, L = k.shape[1], k.shape[2]
    node = torch.arange(L, device=q.device) - length[:, None]                                       # [B, L], < 0 inside the context
    at = node.clamp(0, N - 1)[:, None].expand(B, N, L)
    open_ = (node < 0)[:, None] | (mask.gather(2, at) & (node < nodes[:, None])[:, None])
    open_ &= (torch.arange(N, device=q.device) < nodes[:, None])[:, :, None]                       # [B, N, L]
    x = q.float().view(B, N, H, HQ // H, D).permute(0, 2, 1, 3, 4).flatten(2, 3)                    # [B, H, N G, D]
    logit = (x @ k.transpose(2, 3)).view(B, H, N, HQ // H, L) / math.sqrt(D)
    logit = logit.masked_fill_(~open_[:, None, :, None], -math.inf)
    top = logit.amax(-1, keepdim=True)
    p = logit.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.flatten(2, 3) @ v).view(B, H, N, HQ // H, D) / torch.where(total == 0, 1.0, total)
    return out.permute(0, 2, 1, 3, 4).reshape(B, N, HQ, D).to(q.dtype)


def _accept(s):
    """Rows length + path[i] move to length + i for i < path_len, in place."""
    path, count, length = s["path"].long(), s["path_len"].long(), s["length"].long()
    i = torch.arange(path.shape[1], device=path.device)
    live = i < count[:, None]
    src, dst = (length[:, None] + path)[live], (length[:, None] + i)[live]
    b = torch.arange(path.shape[0], device=path.device)[:, None].expand_as(path)[live]
    table = s["page_table"].long()
    unit = torch.arange(8, device=path.device)
    turn = 7 if s["bits"] == 8 else 4
    out = {}
    for n in ("k", "v"):
        codes = s[n + "_codes"]
        H = codes.shape[1]
        cells = codes.view(codes.shape[0], H, PAGE, 8, -1)
        head = torch.arange(H, device=path.device)[:, None]
        place = lambda pos: (table[b, pos // PAGE][:, None, None], head, (pos % PAGE)[:, None, None], unit ^ ((pos % PAGE) & turn)[:, None, None])  # noqa: E731
        cells[place(dst)] = cells[place(src)]
        for side in (s[n + "_scale"], s[n + "_zp"]):
            if side is not None:
                side[table[b, dst // PAGE], :, dst % PAGE] = side[table[b, src // PAGE], :, src % PAGE]
        out[n] = [codes, s[n + "_scale"]] + ([] if s[n + "_zp"] is None else [s[n + "_zp"]])
    return {"cache": out, "length": (length + count).int()}


def _power(a):
    """The smallest power of two p with a <= 127 p, at least 2^-126."""
    m, e = torch.frexp(a)
    return torch.ldexp(torch.ones_like(a), torch.where(a == 0, -126, e - 7 + (m > 127 / 128)).clamp(min=-126))


def _bounds(s, streams, start):
    """Largest and smallest key of every channel over a page's rows, in whole steps of a power of two, rounded outwards."""
    table, length = s["page_table"][streams].long(), s["length"][streams]
    B, P = table.shape
    k = _values(s, "k", table)                                                                       # [B, P, H, 16, D]
    there = torch.arange(P * PAGE, device=k.device).view(P, 1, PAGE, 1) < length.view(B, 1, 1, 1, 1)
    hi = k.masked_fill(~there, -math.inf).amax(3)
    lo = k.masked_fill_(~there, math.inf).amin(3)
    step = _power(torch.maximum(hi.abs(), lo.abs()).nan_to_num(posinf=0).amax(-1))
    codes = torch.stack((torch.ceil(hi / step[..., None]), torch.floor(lo / step[..., None])), 3)
    return codes.nan_to_num(posinf=0, neginf=0).to(torch.int8), step


def _bounds_update(s):
    codes, step = _bounds(s, slice(None), s["start"])
    p = torch.arange(s["width"], device=codes.device)
    fresh = (p >= s["start"][:, None] // PAGE) & (p * PAGE < s["length"][:, None])
    at = s["page_table"][fresh].long()
    s["bound_codes"][at] = codes[fresh]
    s["bound_scale"][at] = step[fresh]
    return s["bound_codes"], s["bound_scale"]


def _chosen(s):
    """Page numbers [B, H, pages], ascending, -1 behind them: the first and the most recent pages of a stream, and of those
    between them the ones whose keys can reach the largest logit with any query head of the group."""
    q, length, m = s["q"], s["length"].long(), s["pages"]
    table = s["page_table"].long()
    B, P = table.shape
    H = s["bound_codes"].shape[1]
    x = q.float().view(B, H, -1, D)
    step = _power(x.abs().amax(-1))                                                                  # [B, H, G]
    x = torch.round(x / step[..., None])
    bound = s["bound_codes"][table].float()                                                          # [B, P, H, 2, D]
    dot = torch.einsum("bhgd,bphd->bhpg", x.clamp(min=0), bound[:, :, :, 0]) + torch.einsum("bhgd,bphd->bhpg", x.clamp(max=0), bound[:, :, :, 1])
    score = (dot * s["bound_scale"][table].transpose(1, 2)[..., None] * step[:, :, None]).amax(-1)    # [B, H, P]
    n = ((length + PAGE - 1) // PAGE)[:, None, None]
    p = torch.arange(P, device=q.device)
    score = torch.where((p < s["first"]) | (p >= n - s["recent"]), math.inf, score)
    score = torch.where(p >= n, -math.inf, score)
    rank = torch.sort(score, dim=-1, descending=True, stable=True).indices
    rank = torch.nn.functional.pad(rank, (0, max(0, m - P)), value=P)[..., :m]
    kept = torch.where(torch.arange(m, device=q.device) < torch.minimum(n, torch.full_like(n, m)), rank, P).sort(-1).values
    return torch.where(kept < P, kept, -1)


def _sparse(s):
    """Decode attention over the chosen pages."""
    q, length = s["q"], s["length"].long()
    B, HQ, _ = q.shape
    kept = _chosen(s)
    H, m = kept.shape[1:]
    at = torch.gather(s["page_table"].long()[:, None].expand(B, H, -1), 2, kept.clamp(min=0))
    head = torch.arange(H, device=q.device)[:, None]
    k, v = (_decode(s, n, s[n + "_codes"][at, head], s[n + "_scale"][at, head], None if s[n + "_zp"] is None else s[n + "_zp"][at, head]).flatten(2, 3)
            for n in "kv")
    row = kept[..., None] * PAGE + torch.arange(PAGE, device=q.device)
    shut = ((kept < 0)[..., None] | (row >= length[:, None, None, None])).flatten(2)
    logit = (q.float().view(B, H, HQ // H, D) @ k.transpose(2, 3) / math.sqrt(D)).masked_fill_(shut[:, :, None], -math.inf)
    p = (logit - logit.amax(-1, keepdim=True)).exp()
    out = (p @ v) / p.sum(-1, keepdim=True)
    return out.reshape(B, HQ, D).to(q.dtype), kept.int()


def run(state):
    s = state
    if own:
        cache = s["cache"]
        if s["kind"] == "tree":
            return cache.decode_attention_tree(s["q"], s["mask"], ctx_len=s["length"], nodes=s["nodes"])
        if s["kind"] == "accept":
            length = cache.accept_tree(s["path"], s["path_len"], ctx_len=s["length"])
            return {"cache": {n: [getattr(cache, n + x) for x in ("_codes", "_scale", "_zp") if getattr(cache, n + x) is not None] for n in "kv"},
                    "length": length}
        if s["kind"] == "bounds":
            cache.update_bounds(s["bounds"], start=s["start"], seq_len=s["length"])
            return s["bounds"].codes, s["bounds"].scale
        return cache.decode_attention_sparse(s["q"], s["bounds"], s["pages"], seq_len=s["length"], first=s["first"], recent=s["recent"], want_pages=True)
    return {"tree": _tree, "accept": _accept, "bounds": _bounds_update, "sparse": _sparse}[s["kind"]](s)


# ---- in 64 bits, from the definitions ------------------------------------------------------------------------------
def _rows64(s, name, table_row, n, head):
    """Rows 0 .. n - 1 of a list of pages and one head, in 64 bits: [n, 128]."""
    raw = s[name + "_codes"][table_row, head]                                                        # [P, 16, bytes]
    P, _, width = raw.shape
    r = torch.arange(PAGE, device=raw.device)
    byte = torch.arange(width, device=raw.device)
    if s["bits"] == 8:
        where = (byte[None] // 16 ^ (r & 7)[:, None]) * 16 + byte[None] % 16
    else:
        where = (byte[None] // 8 ^ (r & 4)[:, None]) * 8 + byte[None] % 8
    raw = torch.gather(raw, 2, where.expand(P, PAGE, width)).long()
    if s["bits"] == 8:
        x = torch.where(raw > 127, raw - 256, raw).double()
    else:
        x = torch.empty(P, PAGE, D, dtype=torch.float64, device=raw.device)
        x[..., 0::2], x[..., 1::2] = (raw % 16).double(), (raw // 16).double()
        x -= s[name + "_zp"][table_row, head].double()[..., None]
    return (x * s[name + "_scale"][table_row, head].double()[..., None]).view(P * PAGE, D)[:n]


def _step64(most):
    """The smallest power of two p >= 2^-126 with most <= 127 p."""
    e = torch.ceil(torch.log2(most.clamp(min=2.0 ** -140) / 127)).clamp(min=-126)
    return torch.ldexp(torch.ones_like(most), e.long())


def exact(case, seed):
    if case["kind"] == "accept":
        return None                                                    # rows are moved, nothing is computed
    s = prepare(case, seed)
    dev = s["length"].device
    H = case["n_kv"]
    lens = _lengths(case)
    if case["kind"] == "bounds":
        codes, scale = s["bound_codes"], s["bound_scale"].double()
        for b, n in enumerate(lens):
            p0, p1 = int(s["start"][b]) // PAGE, _pages(n)
            row = s["page_table"][b, :p1].long()
            for h in range(H):
                x = _rows64(s, "k", row, n, h)
                pad = p1 * PAGE - n
                x = torch.cat([x, x[-1:].expand(pad, D)]).view(p1, PAGE, D)[p0:]
                hi, lo = x.max(1).values, x.min(1).values
                step = _step64(x.abs().flatten(1).max(1).values)
                scale[row[p0:], h] = step
                codes[row[p0:], h, 0] = torch.ceil(hi / step[:, None]).to(torch.int8)
                codes[row[p0:], h, 1] = torch.floor(lo / step[:, None]).to(torch.int8)
        return codes, scale
    G = case["group"]
    if case["kind"] == "tree":
        N, nodes = case["nodes"], _nodes(case)
        out = torch.zeros(case["streams"], N, H * G, D, dtype=torch.float64, device=dev)
        for b, n in enumerate(lens):
            t = nodes[b]
            row = s["page_table"][b].long()
            sees = torch.cat([torch.ones(t, n, dtype=torch.bool, device=dev), s["mask"][b, :t, :t]], 1)
            for h in range(H):
                k, v = (_rows64(s, x, row, n + t, h) for x in "kv")
                q = s["q"][b, :t, h * G:(h + 1) * G].double()
                logit = torch.einsum("ngd,ld->ngl", q, k) * D ** -0.5
                out[b, :t, h * G:(h + 1) * G] = torch.softmax(logit.masked_fill(~sees[:, None], -math.inf), -1) @ v
        return out
    m = case["pages"]
    out = torch.zeros(case["streams"], H * G, D, dtype=torch.float64, device=dev)
    kept = torch.full((case["streams"], H, m), -1, dtype=torch.int32, device=dev)
    for b, n in enumerate(lens):
        P = _pages(n)
        row = s["page_table"][b, :P].long()
        for h in range(H):
            q = s["q"][b, h * G:(h + 1) * G].double()
            take = torch.arange(P, device=dev)
            if P > m:
                step = _step64(q.abs().max(1).values)
                u = torch.round(q / step[:, None])
                bound = s["bound_codes"][row, h].double() * s["bound_scale"][row, h].double()[:, None, None]
                reach = ((torch.relu(u) @ bound[:, 0].T) - (torch.relu(-u) @ bound[:, 1].T)) * step[:, None]
                mid = reach.max(0).values[case["first"]:P - case["recent"]]
                best = torch.argsort(-mid, stable=True)[:m - case["first"] - case["recent"]] + case["first"]
                take = torch.cat([take[:case["first"]], best, take[P - case["recent"]:]]).sort().values
            kept[b, h, :len(take)] = take.int()
            tail = len(take) * PAGE - (P * PAGE - n)
            k, v = (_rows64(s, x, row[take], tail, h) for x in "kv")
            out[b, h * G:(h + 1) * G] = torch.softmax(q @ k.T * D ** -0.5, -1) @ v
    return out, kept
