"""Filled caches and the operators of speculative and sparse decoding in 64 bits, for the tests of the kernels."""
import math

import torch

PAGE, D = 16, 128


def filled_cache(rows, n_kv, bits, seed, capacity=None, device="cuda"):
    """A cache whose stream s holds rows[s] rows of K and V, on pages in random order with spare pages between them, whose
    unwritten rows are left with scales that are not a number."""
    import pikv_b200
    gen = torch.Generator(device=device).manual_seed(seed)
    S, most = len(rows), max(max(rows), 1)
    width = (most + PAGE - 1) // PAGE
    pages = S * width + 3
    cache = pikv_b200.PagedKVCache(S, capacity or most, n_kv, bits=bits, symmetric=bits == 8, device=device, num_pages=pages, identity_table=False)
    cache.page_table[:, :width] = torch.randperm(pages, generator=gen, device=device)[:S * width].int().view(S, width)
    for name, t in cache.named_buffers():
        if name.endswith(("_scale", "_zp")):
            t.fill_(math.nan)
    for s, n in enumerate(rows):
        if n:
            append_rows(cache, s, 0, *(torch.randn(n, n_kv * D, generator=gen, device=device).bfloat16() for _ in range(2)))
    return cache, gen


def append_rows(cache, stream, at, k, v):
    pos = torch.arange(at, at + k.shape[0], dtype=torch.int32, device=k.device)
    cache.append(k, v, torch.full_like(pos, stream), pos)


def rows64(cache, stream, n):
    """Dequantised K and V [n, n_kv, 128] of a stream, in 64 bits."""
    pos = torch.arange(n, dtype=torch.int32, device=cache.k_codes.device)
    return tuple(cache.gather(torch.full_like(pos, stream), pos, w).view(n, cache.n_kv, D).double() for w in ("k", "v"))


def attend64(q, k, v, sees):
    """q [R, n_q, 128], k and v [L, n_kv, 128], sees [R, L] -> out [R, n_q, 128], lse [R, n_q], and per (R, n_q) the largest
    |V| seen and the largest sum of |q k| / sqrt(128) (what roundings are relative to); rows that see nothing: 0 and -inf."""
    R, n_q, _ = q.shape
    L, n_kv, _ = k.shape
    x = q.double().view(R, n_kv, n_q // n_kv, D)
    shut = ~sees[:, None, None]
    s = torch.einsum("rhgd,lhd->rhgl", x, k).masked_fill(shut, -math.inf) / math.sqrt(D)
    size = torch.einsum("rhgd,lhd->rhgl", x.abs(), k.abs()).masked_fill(shut, 0).amax(-1) / math.sqrt(D)
    lse = torch.logsumexp(s, -1)
    p = torch.where(lse[..., None] == -math.inf, 0.0, (s - torch.where(lse == -math.inf, 0.0, lse)[..., None]).exp())
    out = torch.einsum("rhgl,lhd->rhgd", p, torch.where(torch.isfinite(v), v, 0.0) if not sees.all() else v)
    big = v.abs().amax(-1)[None, :, :, None].permute(0, 2, 3, 1).expand(R, n_kv, 1, L).masked_fill(shut, 0).amax(-1)
    return out.reshape(R, n_q, D), lse.reshape(R, n_q), big.expand(R, n_kv, n_q // n_kv).reshape(R, n_q), size.reshape(R, n_q)


def attention_bound(want, big, size, logit, value):
    """How far a kernel's output and log-sum-exp may be off: the output's rounding to bf16 (2^-8 of itself), the weights' to
    f16 (2^-11, and 2^-24 of the largest where they are tiny), that of V (`value` of the largest) and an error of the logits,
    `logit` of their terms' sum, which moves a weight and the denominator by that much each; the weights add up to 1, so all but
    the first are relative to the largest V."""
    slip = logit * size + 2.0 ** -20
    return 2.0 ** -8 * want.abs() + ((2.0 ** -11 + value + 2.0 ** -20 + 2 * slip) * big)[..., None], slip + 2.0 ** -20


def check_attention(out, lse, want, want_lse, big, size, logit, value=0.0):
    far, far_lse = attention_bound(want, big, size, logit, value)
    nothing = want_lse == -math.inf
    off = (out.double() - want).abs()
    assert bool((off <= far).all()), f"output off by {float((off / far.clamp(min=1e-300)).max())} of what its roundings allow"
    if lse is not None:
        assert bool((lse[nothing] == -math.inf).all())
        off = (lse.double() - want_lse).abs()[~nothing]
        assert bool((off <= (far_lse + 2.0 ** -22 * want_lse.abs())[~nothing]).all())


def step64(a):
    """The smallest power of two p >= 2^-126 with a <= 127 p."""
    m, e = torch.frexp(a.double())
    return torch.ldexp(torch.ones_like(m), torch.where(a == 0, -126, e - 7 + (m > 127 / 128)).clamp(min=-126))


def bounds64(k):
    """Bounds of one page's rows k [rows, n_kv, 128]: codes [n_kv, 2, 128], scale [n_kv]."""
    hi, lo = k.amax(0), k.amin(0)
    s = step64(torch.maximum(hi.abs(), lo.abs()).amax(-1))
    return torch.stack((torch.ceil(hi / s[:, None]), torch.floor(lo / s[:, None])), 1), s


def chosen64(q, codes, scale, pages, first, recent):
    """Page numbers per KV head for one stream: q [n_q, 128], codes [P, n_kv, 2, 128], scale [P, n_kv]."""
    P, n_kv = scale.shape
    if P <= pages:
        return [list(range(P))] * n_kv
    x = q.double().view(n_kv, -1, D)
    got = []
    for h in range(n_kv):
        best = torch.full((P,), -math.inf, dtype=torch.float64, device=q.device)
        for row in x[h]:
            if not bool(torch.isfinite(row).all()):
                continue
            s = step64(row.abs().max())
            u = torch.round(row / s)
            dot = codes[:, h, 0].double() @ u.clamp(min=0) + codes[:, h, 1].double() @ u.clamp(max=0)
            best = torch.maximum(best, dot * scale[:, h].double() * s)
        best = torch.where(torch.isinf(scale[:, h]), math.inf, best)
        order = torch.argsort(-best[first:P - recent], stable=True)[:pages - first - recent] + first
        got.append(sorted(list(range(first)) + order.tolist() + list(range(P - recent, P))))
    return got
