"""What the speed of the operators of a drafted decoding step is measured on: one call of one operator a case.

A step that checks several drafted tokens a sequence at once calls, beside the products that this library has:

  append  the norm of each query and key head, their rotary positions, and the step's keys and values written into the
          pages of a cache, in one pass.
  attend  attention of a step's rows over the pages of a cache: each row sees its sequence's earlier tokens, and of the
          step's own those that its tree of drafts (a mask of bits) or chain has ahead of it.
  sample  a token from each row of logits: temperature, top-k, top-p and min-p, by given random numbers.

`run` computes the plain form with elementary torch operations (in 32 bits; the sampled weights and their sums in 64,
since a token is decided by which side of a border a number falls), or with `own` makes the calls of
include/transmuter_hip.h that a program makes, over buffers and a context that it keeps.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6
MAX_POSITIONS = 32768
LEAST = 2.0 ** -44  # a token of less weight (of the largest's) is not drawn

_CTX = None


def _ctx():
    """The program's one context (device and stream)."""
    global _CTX
    if _CTX is None:
        from transmuter_amd import Context

        torch.cuda.init()
        _CTX = Context(0)
    return _CTX


def _code(dtype):
    from transmuter_amd import _lib

    return {"f32": _lib.F32, "f16": _lib.F16, "bf16": _lib.BF16}[dtype]


# ---------------------------------------------------------------- the cases


def listed() -> list[dict]:
    return [
        # One user's token; a server's step of eight drafted tokens for each of 32 users; a prompt with padded rows.
        {"name": "append f16 1", "kind": "append", "rows": 1, "heads": 16, "kv_heads": 8, "dim": 128, "rotary": 128,
         "interleaved": False, "page": 16, "order": "token", "dtype": "f16", "padding": False},
        {"name": "append bf16 256", "kind": "append", "rows": 256, "heads": 32, "kv_heads": 4, "dim": 128,
         "rotary": 128, "interleaved": False, "page": 16, "order": "head", "dtype": "bf16", "padding": False},
        {"name": "append bf16 4096", "kind": "append", "rows": 4096, "heads": 32, "kv_heads": 4, "dim": 128,
         "rotary": 128, "interleaved": False, "page": 64, "order": "token", "dtype": "bf16", "padding": True},
        # One user's eight drafted tokens in a short chat; a server's ragged batch with trees of one to 32 tokens; a
        # tree of 64 tokens over one very long document; an f32 export of odd sizes with a sliding window; chunks of
        # four users' prompts.
        {"name": "attend f16 1x8 over 700", "kind": "attend", "batch": 1, "fewest": 8, "nodes": 8, "shortest": 700,
         "longest": 700, "tree": True, "heads": 16, "kv_heads": 8, "dim": 128, "page": 16, "order": "token",
         "window": 0, "dtype": "f16"},
        {"name": "attend bf16 32x32 over 8000", "kind": "attend", "batch": 32, "fewest": 1, "nodes": 32,
         "shortest": 40, "longest": 8000, "tree": True, "heads": 32, "kv_heads": 4, "dim": 128, "page": 16,
         "order": "token", "window": 0, "dtype": "bf16"},
        {"name": "attend f16 1x64 over 131072", "kind": "attend", "batch": 1, "fewest": 64, "nodes": 64,
         "shortest": 131072, "longest": 131072, "tree": True, "heads": 16, "kv_heads": 4, "dim": 128, "page": 64,
         "order": "head", "window": 0, "dtype": "f16"},
        {"name": "attend f32 3x13 over 1000", "kind": "attend", "batch": 3, "fewest": 5, "nodes": 13, "shortest": 9,
         "longest": 1000, "tree": True, "heads": 6, "kv_heads": 2, "dim": 80, "page": 20, "order": "token",
         "window": 300, "dtype": "f32"},
        {"name": "attend bf16 4x512 over 4096", "kind": "attend", "batch": 4, "fewest": 512, "nodes": 512,
         "shortest": 512, "longest": 4096, "tree": False, "heads": 32, "kv_heads": 4, "dim": 128, "page": 16,
         "order": "token", "window": 0, "dtype": "bf16"},
        # One user's token from f32 logits by the usual top-k and top-p; a decode batch by top-p alone; a large batch
        # whose users each chose something else, greedy ones among them; the nodes of many trees by min-p.
        {"name": "sample f32 1x151936", "kind": "sample", "rows": 1, "vocabulary": 151936, "dtype": "f32", "by": "kp"},
        {"name": "sample bf16 64x151936", "kind": "sample", "rows": 64, "vocabulary": 151936, "dtype": "bf16",
         "by": "p"},
        {"name": "sample f16 500x32003", "kind": "sample", "rows": 500, "vocabulary": 32003, "dtype": "f16",
         "by": "mixed"},
        {"name": "sample f32 256x151936", "kind": "sample", "rows": 256, "vocabulary": 151936, "dtype": "f32",
         "by": "m"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["append", "attend", "attend", "sample"])
    dtype = rng.choice(["f16", "f16", "bf16", "bf16", "f32"])
    if kind == "sample":
        rows, vocabulary = _log(rng, 1, 512), _log(rng, 32, 262144)
        rows = max(1, min(rows, 256 * 151936 * 4 // (vocabulary * SIZE[dtype])))
        return {"kind": kind, "rows": rows, "vocabulary": vocabulary, "dtype": dtype,
                "by": rng.choice(["", "k", "p", "m", "kp", "kpm", "mixed", "mixed"])}
    dim = rng.choice([64, 80, 96, 128, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 5, 8, 16])
    page, order = rng.choice([8, 16, 16, 32, 64, 256, 20]), rng.choice(["token", "head"])
    if kind == "append":
        rows = min(_log(rng, 1, 8192), 4096 * 40 * 128 // ((heads + 2 * kv_heads) * dim))
        return {"kind": kind, "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "rotary": rng.choice([dim, dim, dim // 2, 0]), "interleaved": rng.random() < 0.3, "page": page,
                "order": order, "dtype": dtype, "padding": rng.random() < 0.3}
    tree = rng.random() < 0.7
    batch, nodes, longest = _log(rng, 1, 64), _log(rng, 1, 80 if tree else 512), _log(rng, 1, 131072)
    # No more bytes than one long document's, no more operations than the chunks of prompts.
    longest = max(1, min(longest, 131072 * 4 * 128 * 2 // (batch * kv_heads * dim * SIZE[dtype])))
    longest = max(1, min(longest, 4 * 512 * 32 * 128 * 2304 // (batch * nodes * heads * dim)))
    nodes = min(nodes, longest)
    return {"kind": kind, "batch": batch, "fewest": rng.choice([0, 1, nodes, nodes]), "nodes": nodes,
            "shortest": rng.choice([nodes, max(nodes, longest // 2), longest]), "longest": longest, "tree": tree,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "order": order,
            "window": rng.choice([0, 0, 0, 100, 1024, 4096]), "dtype": dtype}


# ---------------------------------------------------------------- inputs


def _gen(seed, *path):
    """A generator for one input: every input of a case has its own, made from the seed."""
    x = (int(seed) + 1) * 1000003
    for p in path:
        x = (x * 1000003 + int(p) + 1) % (1 << 62)
    return torch.Generator(device=DEVICE).manual_seed(x)


def _pool(case, pages, gen):
    """A cache of random values [pages, page, kv_heads, dim], the heads of a page inside or outside its tokens."""
    shape = (pages, case["page"], case["kv_heads"], case["dim"])
    if case["order"] == "head":
        shape = (shape[0], shape[2], shape[1], shape[3])
    pool = torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).to(TORCH[case["dtype"]])
    return pool.transpose(1, 2) if case["order"] == "head" else pool


def _append_inputs(case, seed):
    t, h, g, d = case["rows"], case["heads"], case["kv_heads"], case["dim"]
    pages = -(-2 * t // case["page"]) + 3
    # Heads of other sizes, which is what the norms are for.
    qkv = torch.randn(t, h + 2 * g, d, generator=_gen(seed, 1), device=DEVICE)
    qkv *= 0.2 + 5 * torch.rand(1, h + 2 * g, 1, generator=_gen(seed, 6), device=DEVICE)
    qkv = qkv.reshape(t, -1).to(TORCH[case["dtype"]])
    gammas = [(0.5 + torch.rand(d, generator=_gen(seed, 7 + i), device=DEVICE)).to(TORCH[case["dtype"]]) for i in (0, 1)]
    k_pool, v_pool = _pool(case, pages, _gen(seed, 2)), _pool(case, pages, _gen(seed, 3))
    first = int(torch.randint(0, MAX_POSITIONS - t, (1,), generator=_gen(seed, 4), device=DEVICE))
    positions = torch.arange(first, first + t, device=DEVICE)
    order = torch.randperm(pages, generator=_gen(seed, 5), device=DEVICE)
    at = torch.arange(t, device=DEVICE)
    slots = order[at // case["page"]] * case["page"] + at % case["page"]
    if case["padding"]:
        slots[7::16] = -1  # padded rows have no place in the cache
    cos = sin = None
    if case["rotary"]:
        half = case["rotary"] // 2
        freq = 10000.0 ** (-torch.arange(half, device=DEVICE, dtype=torch.float64) / half)
        angle = torch.arange(MAX_POSITIONS, device=DEVICE, dtype=torch.float64)[:, None] * freq
        cos, sin = angle.cos().float(), angle.sin().float()
    return qkv, gammas, k_pool, v_pool, positions, slots, cos, sin


def _spread(lo, hi, n):
    """n numbers evenly from the least to the greatest."""
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _shapes(case):
    """(tokens in the cache, drafted tokens among them) of each sequence: most tokens and most drafts do not meet."""
    b = case["batch"]
    nodes = _spread(case["fewest"], case["nodes"], b)
    lengths = _spread(case["shortest"], case["longest"], b)
    return [(lengths[i], nodes[(i * 7 + 3) % b] if b % 7 else nodes[i]) for i in range(b)]


def _words(case):
    return -(-case["nodes"] // 64)


def _attend_inputs(case, seed):
    b, page, words = case["batch"], case["page"], _words(case)
    shapes = _shapes(case)
    lengths = torch.tensor([s[0] for s in shapes], device=DEVICE, dtype=torch.int32)
    nodes = torch.tensor([s[1] for s in shapes], device=DEVICE)
    starts = torch.nn.functional.pad(nodes.cumsum(0), (1, 0)).int()
    rows = sum(s[1] for s in shapes)
    need = (lengths.long() + page - 1) // page
    pages = int(need.sum()) + 5
    width = max(1, int(need.max()))
    order = torch.randperm(pages, generator=_gen(seed, 2), device=DEVICE).int()
    first = need.cumsum(0) - need
    at = torch.arange(width, device=DEVICE)
    table = order[(first[:, None] + at).clamp(max=pages - 1)]
    table = torch.where(at < need[:, None], table, -1).contiguous()
    q = torch.randn(rows, case["heads"] * case["dim"], generator=_gen(seed, 3), device=DEVICE)
    q = (q * 2).to(TORCH[case["dtype"]])  # scores of a few units: some tokens count far more than others
    mask = None
    if case["tree"]:
        # Each draft continues one of the sixteen before it; a row's bits are its ancestors and itself.
        n = case["nodes"]
        back = torch.randint(1, 17, (b, n), generator=_gen(seed, 6), device=DEVICE)
        parent = (torch.arange(n, device=DEVICE) - back).clamp(min=0)
        tree = torch.zeros(b, n, words, dtype=torch.int64, device=DEVICE)
        every = torch.arange(b, device=DEVICE)
        for i in range(n):
            if i:
                tree[:, i] = tree[every, parent[:, i]]
            tree[:, i, i // 64] |= (1 << (i % 64)) if i % 64 < 63 else -(1 << 63)
        mask = tree[torch.arange(n, device=DEVICE) < nodes[:, None]].contiguous()
    return q, _pool(case, pages, _gen(seed, 4)), _pool(case, pages, _gen(seed, 5)), table, lengths, starts, mask


def _sample_inputs(case, seed):
    t, v, by = case["rows"], case["vocabulary"], case["by"]
    logits = 2.5 * torch.randn(t, v, generator=_gen(seed, 1), device=DEVICE)
    # A few dozen candidates a row, some far ahead of the rest.
    peaks = torch.randint(0, v, (t, 48), generator=_gen(seed, 2), device=DEVICE)
    ahead = torch.rand(t, 48, generator=_gen(seed, 3), device=DEVICE).clamp(min=1e-6).log().mul(-3)
    logits.scatter_add_(1, peaks, ahead + 4)
    logits = logits.to(TORCH[case["dtype"]])
    u = torch.rand(t, 6, generator=_gen(seed, 4), device=DEVICE)
    temperature = 0.3 * 5 ** u[:, 0]
    top_k = (2 * 150 ** u[:, 1]).int()
    top_p = 0.5 + 0.5 * u[:, 2]
    min_p = 0.15 * u[:, 3]
    if by == "mixed":
        some = torch.rand(t, 4, generator=_gen(seed, 5), device=DEVICE)
        temperature = torch.where(some[:, 0] < 0.2, 0.0, temperature)
        top_k = torch.where(some[:, 1] < 0.5, 0, top_k)
        top_p = torch.where(some[:, 2] < 0.4, 1.0, top_p)
        min_p = torch.where(some[:, 3] < 0.6, 0.0, min_p)
        by = "kpm"
    return (logits, temperature, top_k if "k" in by else None, top_p if "p" in by else None,
            min_p if "m" in by else None, u[:, 5].contiguous())


# ---------------------------------------------------------------- plain forms


def _plain_rotate(x, cos, sin, rotary, interleaved):
    """x [rows, heads, dim] in 32 bits with its first `rotary` dimensions turned, pairs neighbours or half apart."""
    if not rotary:
        return x
    turned = x[..., :rotary]
    c, s = cos[:, None, :], sin[:, None, :]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
    else:
        a, b = turned[..., :rotary // 2], turned[..., rotary // 2:]
        turned = torch.cat((a * c - b * s, a * s + b * c), -1)
    return torch.cat((turned, x[..., rotary:]), -1)


def _plain_append(st):
    qkv, gammas, k_pool, v_pool, positions, slots, cos, sin = st["inputs"]
    c = st["case"]
    t, h, g, d = c["rows"], c["heads"], c["kv_heads"], c["dim"]
    x = qkv.view(t, h + 2 * g, d)
    y = x[:, :h + g].float()
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS)
    y = torch.cat((y[:, :h] * gammas[0].float(), y[:, h:] * gammas[1].float()), 1)
    if c["rotary"]:
        cos, sin = cos[positions], sin[positions]
    turned = _plain_rotate(y, cos, sin, c["rotary"], c["interleaved"]).to(qkv.dtype)
    keep = (slots >= 0).nonzero().flatten()
    page, at = slots[keep] // c["page"], slots[keep] % c["page"]
    k_pool[page, at] = turned[keep, h:]
    v_pool[page, at] = x[keep, h + g:]
    return {"q": turned[:, :h].reshape(t, h * d), "k": k_pool, "v": v_pool}


def _plain_attend(st):
    q, k_pool, v_pool, table, lengths, starts, mask = st["inputs"]
    c = st["case"]
    b, n, h, g, d = c["batch"], c["nodes"], c["heads"], c["kv_heads"], c["dim"]
    # Rows padded to the most drafts a sequence has.
    node = torch.arange(n, device=q.device)
    nodes = (starts[1:] - starts[:-1])[:, None]
    there = node < nodes
    rows = (starts[:-1, None] + node).clamp(max=max(q.shape[0] - 1, 0))
    at = torch.arange(table.shape[1] * c["page"], device=q.device)
    j = at - (lengths[:, None] - nodes)  # of the step's own tokens: which
    inside = (j >= 0) & (at < lengths[:, None])
    if mask is None:
        sees = j[:, None] <= node[:, None]
    else:
        words = mask[rows].gather(2, (j.clamp(0, 64 * mask.shape[1] - 1) // 64)[:, None].expand(b, n, -1))
        sees = (j < 0)[:, None] | ((words >> (j.clamp(min=0) % 64)[:, None]) & 1).bool()
    sees = sees & (inside | (j < 0))[:, None] & there[..., None]
    if c["window"]:
        behind = sees.flip(-1).cumsum(-1).flip(-1)  # the tokens from here on that the row sees
        sees = sees & (behind <= c["window"])
    pages = table.long().clamp(min=0)
    k = k_pool[pages].float().flatten(1, 2).permute(0, 2, 3, 1).contiguous()
    x = q.float()[rows].view(b, n, g, h // g, d).permute(0, 2, 1, 3, 4).reshape(b, g, n * (h // g), d)
    scores = ((x @ k) / math.sqrt(d)).view(b, g, n, h // g, -1)
    del k
    scores = scores.masked_fill_(~sees[:, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(scores - top)
    del scores
    total = p.sum(-1, keepdim=True)
    v = v_pool[pages].float().flatten(1, 2)
    v = v.masked_fill(~(at < lengths[:, None])[..., None, None], 0).permute(0, 2, 1, 3).contiguous()
    y = (p.flatten(2, 3) @ v).view(b, g, n, h // g, d) / torch.where(total == 0, torch.ones_like(total), total)
    y = y.permute(0, 2, 1, 3, 4).reshape(b, n, h * d)
    return {"y": y[there].to(q.dtype)}


def _plain_sample(st):
    logits, temperature, top_k, top_p, min_p, u = st["inputs"]
    t, v = logits.shape
    x = logits.double()
    top = x.amax(-1, keepdim=True)
    greedy = (x == top).int().argmax(-1)
    tau = temperature.double()[:, None]
    w = torch.exp((x - top) / torch.where(tau > 0, tau, 1.0))
    w = torch.where(w < LEAST, 0.0, w)
    if top_k is not None or top_p is not None:
        order = x.sort(dim=-1, descending=True, stable=True).indices
        ranked = w.gather(1, order)
        if top_k is not None:
            k = torch.where(top_k > 0, top_k, v)[:, None]
            ranked = torch.where(torch.arange(v, device=x.device) < k, ranked, 0.0)
        if top_p is not None:
            p = top_p.double()[:, None]
            sums = ranked.cumsum(-1)
            need = torch.where(p < 1, p * sums[:, -1:], math.inf)
            ahead = torch.nn.functional.pad(sums[:, :-1], (1, 0))
            ranked = torch.where((ahead < need) | (torch.arange(v, device=x.device) == 0), ranked, 0.0)
        w = torch.zeros_like(w).scatter_(1, order, ranked)
    if min_p is not None:
        w = torch.where(w >= min_p.double()[:, None], w, 0.0)
    sums = w.cumsum(-1)
    past = sums > u.double()[:, None] * sums[:, -1:]
    return {"tokens": torch.where(tau[:, 0] > 0, past.int().argmax(-1), greedy)}


# ---------------------------------------------------------------- the framework's calls


def _ptr(t):
    return None if t is None else t.data_ptr()


def _cache(case, k_pool, v_pool):
    from transmuter_amd._lib import PagedCacheDesc

    return PagedCacheDesc(k=_ptr(k_pool), v=_ptr(v_pool), dtype=_code(case["dtype"]), kv_heads=case["kv_heads"],
                          head_dim=case["dim"], page_size=case["page"], pages=k_pool.shape[0],
                          page_stride=k_pool.stride(0), token_stride=k_pool.stride(1), head_stride=k_pool.stride(2))


def _own_append(case, inputs):
    import ctypes

    from transmuter_amd import _lib
    from transmuter_amd._lib import lib

    qkv, gammas, k_pool, v_pool, positions, slots, cos, sin = inputs
    t, h, g, d = case["rows"], case["heads"], case["kv_heads"], case["dim"]
    out = {"q": torch.empty(t, h * d, dtype=qkv.dtype, device=DEVICE), "k": k_pool, "v": v_pool}
    pitch, at = qkv.shape[1], _ptr(qkv)
    size = SIZE[case["dtype"]]
    cache = _cache(case, k_pool, v_pool)
    return out, (lib().tmh_paged_append_norm, (
        _ctx().handle, at, pitch, at + h * d * size, pitch, at + (h + g) * d * size, pitch, t, h, _ptr(gammas[0]),
        _ptr(gammas[1]), _code(case["dtype"]), EPS, _ptr(positions), _ptr(cos), _ptr(sin), _lib.F32, MAX_POSITIONS,
        case["rotary"], int(case["interleaved"]), _ptr(slots), ctypes.byref(cache), _ptr(out["q"]), h * d, None)), cache


def _own_attend(case, inputs):
    import ctypes

    from transmuter_amd._lib import lib

    q, k_pool, v_pool, table, lengths, starts, mask = inputs
    h, d = case["heads"], case["dim"]
    out = {"y": torch.empty_like(q)}
    cache = _cache(case, k_pool, v_pool)
    return out, (lib().tmh_paged_tree_attention, (
        _ctx().handle, _ptr(q), h * d, q.shape[0], h, ctypes.byref(cache), _ptr(table), case["batch"], table.shape[1],
        _ptr(lengths), _ptr(starts), _ptr(mask), 0 if mask is None else mask.shape[1], 1 / math.sqrt(d),
        case["window"], _ptr(out["y"]), h * d, None)), cache


def _own_sample(case, inputs):
    from transmuter_amd._lib import lib

    logits, temperature, top_k, top_p, min_p, u = inputs
    t, v = logits.shape
    out = {"tokens": torch.empty(t, dtype=torch.int64, device=DEVICE)}
    return out, (lib().tmh_sample, (
        _ctx().handle, _ptr(logits), v, _code(case["dtype"]), t, v, _ptr(temperature), _ptr(top_k), _ptr(top_p),
        _ptr(min_p), _ptr(u), _ptr(out["tokens"]), None)), None


# ---------------------------------------------------------------- exact values


def _exact_append(case, seed):
    qkv, gammas, k_pool, v_pool, positions, slots, cos, sin = _append_inputs(case, seed)
    t, h, g, d, rot = case["rows"], case["heads"], case["kv_heads"], case["dim"], case["rotary"]
    x = qkv.double().view(t, -1, d)
    for part, gamma in ((x[:, :h], gammas[0]), (x[:, h:h + g], gammas[1])):
        part /= torch.sqrt(part.square().sum(-1, keepdim=True) / d + EPS)
        part *= gamma.double()
    if rot:
        z = x[:, :h + g, :rot]
        z = z.unflatten(-1, (rot // 2, 2)) if case["interleaved"] else z.unflatten(-1, (2, rot // 2)).transpose(-1, -2)
        turn = torch.complex(cos[positions].double(), sin[positions].double())[:, None]
        z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
        x[:, :h + g, :rot] = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
    k, v = k_pool.double(), v_pool.double()
    for i, slot in enumerate(slots.tolist()):
        if slot >= 0:
            k[slot // case["page"], slot % case["page"]] = x[i, h:h + g]
            v[slot // case["page"], slot % case["page"]] = x[i, h + g:]
    return {"q": x[:, :h].reshape(t, h * d), "k": k, "v": v}


def _exact_attend(case, seed):
    q, k_pool, v_pool, table, lengths, starts, mask = _attend_inputs(case, seed)
    h, g, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out = torch.zeros(q.shape[0], h, d, dtype=torch.float64, device=DEVICE)
    bits = None if mask is None else mask.cpu().numpy().astype("<i8").view(np.uint8)
    for b, (length, n) in enumerate(_shapes(case)):
        if not n:
            continue
        start = int(starts[b])
        sees = np.ones((n, length), bool)
        if mask is None:
            sees[:, length - n:] = np.tril(np.ones((n, n), bool))
        else:
            sees[:, length - n:] = np.unpackbits(bits[start:start + n], axis=1, bitorder="little")[:, :n]
        if case["window"]:
            for row in sees:
                row[np.flatnonzero(row)[:-case["window"]]] = False
        at = torch.arange(length, device=DEVICE)
        where = (table[b, at // page].long(), at % page)
        hidden = torch.from_numpy(~sees).to(DEVICE)
        for head in range(g):
            k, v = k_pool[where[0], where[1], head].double(), v_pool[where[0], where[1], head].double()
            some = slice(head * (h // g), (head + 1) * (h // g))
            x = q[start:start + n].double().view(n, h, d)[:, some]  # [nodes, group, dim]
            s = (x.reshape(-1, d) @ k.t()).view(n, h // g, length) * d ** -0.5
            s.masked_fill_(hidden[:, None], -math.inf)
            out[start:start + n, some] = (torch.softmax(s, -1).flatten(0, 1) @ v).view(n, h // g, d)
    return {"y": out.reshape(q.shape[0], h * d)}


def _exact_sample(case, seed):
    inputs = [None if v is None else v.float().cpu().numpy().astype(np.float64) for v in _sample_inputs(case, seed)]
    logits, temperature, top_k, top_p, min_p, u = inputs
    tokens = []
    for i, row in enumerate(logits):
        if temperature[i] == 0:
            tokens.append(int(np.flatnonzero(row == row.max())[0]))
            continue
        w = np.exp((row - row.max()) / temperature[i])
        w[w < LEAST] = 0
        order = np.argsort(-row, kind="stable")
        if top_k is not None and top_k[i] > 0:
            order = order[:int(top_k[i])]
        if top_p is not None and top_p[i] < 1:
            sums = np.cumsum(w[order])
            order = order[:1 + np.searchsorted(sums, top_p[i] * sums[-1])]
        if min_p is not None:
            order = order[w[order] >= min_p[i]]
        order = np.sort(order)
        sums = np.cumsum(w[order])
        tokens.append(int(order[np.searchsorted(sums, u[i] * sums[-1], side="right")]))
    return {"tokens": torch.tensor(tokens, device=DEVICE)}


# ---------------------------------------------------------------- work


def _work_append(case):
    rows, size, g = case["rows"], SIZE[case["dtype"]], case["kv_heads"]
    kept = rows - (len(range(7, rows, 16)) if case["padding"] else 0)
    q, kv = case["heads"] * case["dim"] * size, 2 * g * case["dim"] * size
    return {"bytes": 2 * rows * q + 2 * kept * kv + rows * (16 + 4 * case["rotary"]) + 2 * case["dim"] * size,
            "flops": rows * (case["heads"] + g) * (4 * case["dim"] + 3 * case["rotary"])}


def _work_attend(case):
    size, read, seen, rows = SIZE[case["dtype"]], 0, 0, 0
    for length, n in _shapes(case):
        rows += n
        most = min(length, case["window"] + n - 1) if case["window"] else length
        read += most if n else 0
        # A chain's row sees half of the step's tokens in the mean; what a tree's sees is counted as much.
        each = length - n / 2
        seen += n * (min(each, case["window"]) if case["window"] else each)
    return {"bytes": 2 * read * case["kv_heads"] * case["dim"] * size + 2 * rows * case["heads"] * case["dim"] * size,
            "flops": int(4 * seen * case["heads"] * case["dim"])}


def _work_sample(case):
    n = case["rows"] * case["vocabulary"]
    return {"bytes": n * SIZE[case["dtype"]] + 28 * case["rows"], "flops": 4 * n}


# ---------------------------------------------------------------- the interface

_INPUTS = {"append": _append_inputs, "attend": _attend_inputs, "sample": _sample_inputs}
_PLAIN = {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}
_OWN = {"append": _own_append, "attend": _own_attend, "sample": _own_sample}
_EXACT = {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}
_WORK = {"append": _work_append, "attend": _work_attend, "sample": _work_sample}


def prepare(case, seed):
    state = {"case": case, "inputs": _INPUTS[case["kind"]](case, seed)}
    if own:
        # The buffers and the arguments that a program keeps from call to call.
        state["out"], state["call"], state["keep"] = _OWN[case["kind"]](case, state["inputs"])
        state["check"] = _ctx().check
    torch.cuda.synchronize()
    return state


def run(state):
    if own:
        call, arguments = state["call"]
        state["check"](call(*arguments))
        return state["out"]
    return _PLAIN[state["case"]["kind"]](state)


def exact(case, seed):
    return _EXACT[case["kind"]](case, seed)


def work(case):
    return _WORK[case["kind"]](case)
