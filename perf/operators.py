"""What the speed of the decoder-layer operators is measured on: one call of one operator a case.

The operators are what a decoder layer with weights in 8-bit floating point needs beside the quantized
products this library already has, in the order in which such a layer calls them:

  norm      the residual's addition and the root-mean-square norm, answered in 8 bits with a scale for
            each block of 128 columns (what the 8-bit product takes), in the input's type, or both.
  matmul    the product of 8-bit rows with an 8-bit weight: a scale for each row's block of 128 of K, and
            for each 128 x 128 block of the weight.
  append    rotary positions of a step's queries and keys, and its keys and values written into the pages
            of a cache.
  attend    attention of one new token a sequence over its pages of that cache.
  quantize  rows (an attention's answer, or the gated activation of a merged gate/up product) in 8 bits
            with a scale for each block of 128 columns.

`run` computes the plain form in 32 bits with elementary torch operations, or with `own` makes the calls of
include/transmuter_hip.h that a program makes, over buffers, weights and a context that it keeps.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
F8 = torch.float8_e4m3fn
F8_MAX = 448.0  # the largest finite e4m3 value
BLOCK = 128  # columns that share a scale
EPS = 1e-6

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
        # The smallest call: one user's token ahead of a 3B decoder's q/k/v product.
        {"name": "norm f16 1x2048", "kind": "norm", "rows": 1, "cols": 2048, "dtype": "f16", "residual": True,
         "out": "q"},
        # A long prompt's rows ahead of a mixture of experts: 8 bits for the product, bf16 for the router.
        {"name": "norm bf16 4096x2048", "kind": "norm", "rows": 4096, "cols": 2048, "dtype": "bf16",
         "residual": True, "out": "both"},
        # One user's token through a merged gate/up product, a decode batch through the down product, a prompt
        # of odd length through a small f32 export of odd sizes, and a long prompt's chunk.
        {"name": "matmul f16 1x2048x22016", "kind": "matmul", "m": 1, "k": 2048, "n": 22016, "dtype": "f16",
         "bias": False},
        {"name": "matmul bf16 32x11008x2048", "kind": "matmul", "m": 32, "k": 11008, "n": 2048, "dtype": "bf16",
         "bias": False},
        {"name": "matmul f32 509x1040x2050", "kind": "matmul", "m": 509, "k": 1040, "n": 2050, "dtype": "f32",
         "bias": True},
        {"name": "matmul f16 4096x2048x22016", "kind": "matmul", "m": 4096, "k": 2048, "n": 22016, "dtype": "f16",
         "bias": False},
        # A decode batch's new token, and a prompt's tokens with a padded row here and there.
        {"name": "append f16 32", "kind": "append", "rows": 32, "heads": 16, "kv_heads": 8, "dim": 128,
         "rotary": 128, "interleaved": False, "page": 16, "order": "token", "dtype": "f16", "padding": False},
        {"name": "append bf16 4096", "kind": "append", "rows": 4096, "heads": 32, "kv_heads": 4, "dim": 128,
         "rotary": 128, "interleaved": False, "page": 64, "order": "head", "dtype": "bf16", "padding": True},
        # A short chat of one user, a server's decode batch of ragged lengths, four very long documents.
        {"name": "attend f16 1x700", "kind": "attend", "batch": 1, "shortest": 700, "longest": 700, "heads": 16,
         "kv_heads": 4, "dim": 128, "page": 16, "order": "token", "window": 0, "dtype": "f16"},
        {"name": "attend bf16 32x8000", "kind": "attend", "batch": 32, "shortest": 1, "longest": 8000, "heads": 32,
         "kv_heads": 4, "dim": 128, "page": 16, "order": "token", "window": 0, "dtype": "bf16"},
        {"name": "attend f16 4x131072", "kind": "attend", "batch": 4, "shortest": 120000, "longest": 131072,
         "heads": 16, "kv_heads": 4, "dim": 128, "page": 64, "order": "head", "window": 0, "dtype": "f16"},
        # The gated activation of a prompt ahead of the down product (an attention's answer is drawn).
        {"name": "quantize f16 2048x11008", "kind": "quantize", "rows": 2048, "cols": 11008, "dtype": "f16",
         "gate": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["norm", "matmul", "matmul", "append", "attend", "attend", "quantize"])
    dtype = rng.choice(["f16", "f16", "bf16", "bf16", "f32"])
    if kind in ("norm", "quantize"):
        cols = _log(rng, 64, 16384)
        if rng.random() < 0.7:
            cols = max(64, cols // 64 * 64)
        rows = min(_log(rng, 1, 8192), 11008 * 2048 // cols)
        if kind == "norm":
            return {"kind": kind, "rows": rows, "cols": cols, "dtype": dtype, "residual": rng.random() < 0.7,
                    "out": rng.choice(["q", "q", "y", "both"])}
        return {"kind": kind, "rows": rows, "cols": cols, "dtype": dtype, "gate": rng.random() < 0.5}
    if kind == "matmul":
        # Mostly whole blocks, as models have them; else any K and N.
        m, k, n = _log(rng, 1, 4096), _log(rng, 128, 11008), _log(rng, 64, 22016)
        if rng.random() < 0.7:
            k, n = max(128, k // 128 * 128), max(64, n // 64 * 64)
        elif rng.random() < 0.7:
            k = k // 16 * 16
        while m * k * n > 4096 * 2048 * 22016:
            m = -(-m // 2)
        return {"kind": kind, "m": m, "k": k, "n": n, "dtype": dtype, "bias": rng.random() < 0.3}
    dim = rng.choice([64, 80, 96, 128, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 5, 8, 16])
    page, order = rng.choice([8, 16, 16, 32, 64, 256, 20]), rng.choice(["token", "head"])
    if kind == "append":
        rows = min(_log(rng, 1, 8192), 4096 * 40 * 128 // ((heads + 2 * kv_heads) * dim))
        return {"kind": kind, "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "rotary": rng.choice([dim, dim, dim // 2, 0]), "interleaved": rng.random() < 0.3, "page": page,
                "order": order, "dtype": dtype, "padding": rng.random() < 0.3}
    batch, longest = _log(rng, 1, 256), _log(rng, 1, 131072)
    longest = max(1, min(longest, 120000 * 4 * 4 * 128 * 2 // (batch * kv_heads * dim * SIZE[dtype])))
    return {"kind": kind, "batch": batch, "shortest": rng.choice([0, 1, longest // 2, longest]), "longest": longest,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "order": order,
            "window": rng.choice([0, 0, 0, 100, 1024, 4096]), "dtype": dtype}


# ---------------------------------------------------------------- inputs


def _gen(seed, *path):
    """A generator for one input: every input of a case has its own, made from the seed."""
    x = (int(seed) + 1) * 1000003
    for p in path:
        x = (x * 1000003 + int(p) + 1) % (1 << 62)
    return torch.Generator(device=DEVICE).manual_seed(x)


def _activations(rows, cols, dtype, gen):
    """Normal rows with some columns 10 times the others, as a decoder's hidden state has them."""
    x = torch.randn(rows, cols, generator=gen, device=DEVICE)
    x *= 1 + 9 * (torch.rand(cols, generator=gen, device=DEVICE) < 0.02)
    return x.to(TORCH[dtype])


def _blocks(n):
    return -(-n // BLOCK)


def _norm_inputs(case, seed):
    x = _activations(case["rows"], case["cols"], case["dtype"], _gen(seed, 1))
    r = _activations(case["rows"], case["cols"], case["dtype"], _gen(seed, 2)) if case["residual"] else None
    gamma = 0.5 + torch.rand(case["cols"], generator=_gen(seed, 3), device=DEVICE)
    return x, r, gamma.to(TORCH[case["dtype"]])


def _quantize_inputs(case, seed):
    # The halves of one merged gate/up product: rows twice as long.
    x = _activations(case["rows"], case["cols"] * (2 if case["gate"] else 1), case["dtype"], _gen(seed, 1))
    return (x[:, case["cols"]:], x[:, :case["cols"]]) if case["gate"] else (x, None)


def _matmul_inputs(case, seed):
    m, k, n = case["m"], case["k"], case["n"]
    kb, nb = _blocks(k), _blocks(n)
    x = _activations(m, kb * BLOCK, "f32", _gen(seed, 1)).reshape(m, kb, BLOCK)
    a_scales = x.abs().amax(-1) / F8_MAX
    a = (x / a_scales[..., None]).reshape(m, -1)[:, :k].clamp(-F8_MAX, F8_MAX).to(F8).contiguous()
    w = torch.randn(nb * BLOCK, kb * BLOCK, generator=_gen(seed, 2), device=DEVICE) / math.sqrt(k)
    w = w.reshape(nb, BLOCK, kb, BLOCK)
    w_scales = w.abs().amax((1, 3)) / F8_MAX
    w = (w / w_scales[:, None, :, None]).reshape(nb * BLOCK, -1)[:n, :k].clamp(-F8_MAX, F8_MAX).to(F8).contiguous()
    bias = torch.randn(n, generator=_gen(seed, 3), device=DEVICE).to(TORCH[case["dtype"]]) if case["bias"] else None
    return a, a_scales.t().contiguous(), w, w_scales, bias


def _pool(case, pages, gen):
    """A cache of random values [pages, page, kv_heads, dim], the heads of a page inside or outside its tokens."""
    shape = (pages, case["page"], case["kv_heads"], case["dim"])
    if case["order"] == "head":
        shape = (shape[0], shape[2], shape[1], shape[3])
    pool = torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).to(TORCH[case["dtype"]])
    return pool.transpose(1, 2) if case["order"] == "head" else pool


MAX_POSITIONS = 32768


def _append_inputs(case, seed):
    t, h, g, d = case["rows"], case["heads"], case["kv_heads"], case["dim"]
    pages = -(-2 * t // case["page"]) + 3
    qkv = torch.randn(t, (h + 2 * g) * d, generator=_gen(seed, 1), device=DEVICE).to(TORCH[case["dtype"]])
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
    return qkv, k_pool, v_pool, positions, slots, cos, sin


def _lengths(case):
    """The lengths of a batch, evenly from the shortest to the longest."""
    lo, hi, n = case["shortest"], case["longest"], case["batch"]
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _attend_inputs(case, seed):
    b, page = case["batch"], case["page"]
    lengths = torch.tensor(_lengths(case), device=DEVICE, dtype=torch.int32)
    lengths = lengths[torch.randperm(b, generator=_gen(seed, 1), device=DEVICE)].contiguous()
    need = (lengths.long() + page - 1) // page
    pages = int(need.sum()) + 5
    width = max(1, int(need.max()))
    order = torch.randperm(pages, generator=_gen(seed, 2), device=DEVICE).int()
    first = need.cumsum(0) - need
    at = torch.arange(width, device=DEVICE)
    table = order[(first[:, None] + at).clamp(max=pages - 1)]
    table = torch.where(at < need[:, None], table, -1).contiguous()
    q = torch.randn(b, case["heads"] * case["dim"], generator=_gen(seed, 3), device=DEVICE)
    q = (q * 2).to(TORCH[case["dtype"]])  # scores of a few units: some tokens count far more than others
    return q, _pool(case, pages, _gen(seed, 4)), _pool(case, pages, _gen(seed, 5)), table, lengths


# ---------------------------------------------------------------- plain forms


def _plain_blocks(y):
    """e4m3 rows of y (f32) and the scales of their blocks of 128, [blocks, rows]."""
    rows, cols = y.shape
    kb = _blocks(cols)
    v = torch.nn.functional.pad(y, (0, kb * BLOCK - cols)).reshape(rows, kb, BLOCK)
    s = v.abs().amax(-1) / F8_MAX
    s = torch.where(s == 0, torch.ones_like(s), s)
    q = (v / s[..., None]).clamp(-F8_MAX, F8_MAX).reshape(rows, -1)[:, :cols].to(F8)
    return q, s.t()


def _plain_norm(st):
    x, r, gamma = st["inputs"]
    h = x.float() if r is None else x.float() + r.float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * gamma.float()
    out = {} if r is None else {"sum": h.to(x.dtype)}
    if st["case"]["out"] != "q":
        out["y"] = y.to(x.dtype)
    if st["case"]["out"] != "y":
        out["q"], out["scales"] = _plain_blocks(y)
    return out


def _plain_quantize(st):
    x, gate = st["inputs"]
    y = x.float()
    if gate is not None:
        g = gate.float()
        y = g / (1 + torch.exp(-g)) * y
    q, scales = _plain_blocks(y)
    return {"q": q, "scales": scales}


def _plain_matmul(st):
    a, a_scales, w, w_scales, bias = st["inputs"]
    k, n = a.shape[1], w.shape[0]
    x = a.float() * a_scales.t().repeat_interleave(BLOCK, 1)[:, :k]
    v = w.float() * w_scales.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    y = x @ v.t()
    if bias is not None:
        y = y + bias.float()
    return {"y": y.to(TORCH[st["case"]["dtype"]])}


def _plain_rotate(x, cos, sin, rotary, interleaved):
    """x [rows, heads, dim] with its first `rotary` dimensions turned, pairs neighbours or half apart."""
    v = x.float()
    if not rotary:
        return v
    turned = v[..., :rotary]
    c, s = cos[:, None, :], sin[:, None, :]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
    else:
        a, b = turned[..., :rotary // 2], turned[..., rotary // 2:]
        turned = torch.cat((a * c - b * s, a * s + b * c), -1)
    return torch.cat((turned, v[..., rotary:]), -1)


def _plain_append(st):
    qkv, k_pool, v_pool, positions, slots, cos, sin = st["inputs"]
    c = st["case"]
    t, h, g, d = c["rows"], c["heads"], c["kv_heads"], c["dim"]
    x = qkv.view(t, h + 2 * g, d)
    if c["rotary"]:
        cos, sin = cos[positions], sin[positions]
    turned = _plain_rotate(x[:, :h + g], cos, sin, c["rotary"], c["interleaved"]).to(qkv.dtype)
    keep = (slots >= 0).nonzero().flatten()
    page, at = slots[keep] // c["page"], slots[keep] % c["page"]
    k_pool[page, at] = turned[keep, h:]
    v_pool[page, at] = x[keep, h + g:]
    return {"q": turned[:, :h].reshape(t, h * d), "k": k_pool, "v": v_pool}


def _plain_attend(st):
    q, k_pool, v_pool, table, lengths = st["inputs"]
    c = st["case"]
    b, h, g, d = c["batch"], c["heads"], c["kv_heads"], c["dim"]
    at = torch.arange(table.shape[1] * c["page"], device=q.device)
    keep = at < lengths[:, None]
    if c["window"]:
        keep = keep & (at >= lengths[:, None] - c["window"])
    pages = table.long().clamp(min=0)
    k = k_pool[pages].float().flatten(1, 2).permute(0, 2, 3, 1).contiguous()
    scores = (q.float().view(b, g, h // g, d) @ k) / math.sqrt(d)
    del k
    scores = scores.masked_fill(~keep[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(scores - top)
    v = v_pool[pages].float().flatten(1, 2).masked_fill(~keep[..., None, None], 0).permute(0, 2, 1, 3).contiguous()
    total = p.sum(-1, keepdim=True)
    y = (p @ v) / torch.where(total == 0, torch.ones_like(total), total)  # no token: zeros
    return {"y": y.reshape(b, h * d).to(q.dtype)}


# ---------------------------------------------------------------- the framework's calls


def _ptr(t):
    return None if t is None else t.data_ptr()


def _own_norm(case, inputs):
    from transmuter_amd._lib import lib

    x, r, gamma = inputs
    rows, cols = x.shape
    out = {} if r is None else {"sum": torch.empty_like(x)}
    if case["out"] != "q":
        out["y"] = torch.empty_like(x)
    if case["out"] != "y":
        out["q"] = torch.empty(rows, cols, dtype=F8, device=DEVICE)
        out["scales"] = torch.empty(_blocks(cols), rows, device=DEVICE)
    code = _code(case["dtype"])
    return out, [(lib().tmh_rms_norm, (
        _ctx().handle, _ptr(x), cols, _ptr(r), cols, code, rows, cols, _ptr(gamma), code, EPS, _ptr(out.get("sum")),
        cols, _ptr(out.get("y")), cols, _ptr(out.get("q")), cols, _ptr(out.get("scales")), None))], None


def _own_quantize(case, inputs):
    from transmuter_amd._lib import lib

    x, gate = inputs
    rows, cols = x.shape
    out = {"q": torch.empty(rows, cols, dtype=F8, device=DEVICE),
           "scales": torch.empty(_blocks(cols), rows, device=DEVICE)}
    return out, [(lib().tmh_quantize_rows, (
        _ctx().handle, _ptr(x), x.stride(0), _ptr(gate), x.stride(0), _code(case["dtype"]), rows, cols,
        _ptr(out["q"]), cols, _ptr(out["scales"]), None))], None


def _own_matmul(case, inputs):
    from transmuter_amd._lib import lib
    from transmuter_amd.serving import Fp8Weight

    a, a_scales, w, w_scales, bias = inputs
    (m, k), n = a.shape, w.shape[0]
    torch.cuda.synchronize()
    weight = Fp8Weight.from_pointers(_ctx(), _ptr(w), _ptr(w_scales), k, n)
    out = {"y": torch.empty(m, n, dtype=TORCH[case["dtype"]], device=DEVICE)}
    code = _code(case["dtype"])
    return out, [(lib().tmh_matmul_fp8, (
        _ctx().handle, weight.handle, _ptr(a), m, k, _ptr(a_scales), _ptr(bias), code, _ptr(out["y"]), code, n,
        None))], weight


def _cache(case, k_pool, v_pool):
    from transmuter_amd._lib import PagedCacheDesc

    return PagedCacheDesc(k=_ptr(k_pool), v=_ptr(v_pool), dtype=_code(case["dtype"]), kv_heads=case["kv_heads"],
                          head_dim=case["dim"], page_size=case["page"], pages=k_pool.shape[0],
                          page_stride=k_pool.stride(0), token_stride=k_pool.stride(1), head_stride=k_pool.stride(2))


def _own_append(case, inputs):
    import ctypes

    from transmuter_amd import _lib
    from transmuter_amd._lib import lib

    qkv, k_pool, v_pool, positions, slots, cos, sin = inputs
    t, h, g, d = case["rows"], case["heads"], case["kv_heads"], case["dim"]
    out = {"q": torch.empty(t, h * d, dtype=qkv.dtype, device=DEVICE), "k": k_pool, "v": v_pool}
    pitch, at = qkv.shape[1], _ptr(qkv)
    size = SIZE[case["dtype"]]
    cache = _cache(case, k_pool, v_pool)
    return out, [(lib().tmh_paged_append, (
        _ctx().handle, at, pitch, at + h * d * size, pitch, at + (h + g) * d * size, pitch, t, h, _ptr(positions),
        _ptr(cos), _ptr(sin), _lib.F32, MAX_POSITIONS, case["rotary"], int(case["interleaved"]), _ptr(slots),
        ctypes.byref(cache), _ptr(out["q"]), h * d, None))], cache


def _own_attend(case, inputs):
    import ctypes

    from transmuter_amd._lib import lib

    q, k_pool, v_pool, table, lengths = inputs
    b, h, d = case["batch"], case["heads"], case["dim"]
    out = {"y": torch.empty_like(q)}
    cache = _cache(case, k_pool, v_pool)
    return out, [(lib().tmh_paged_attention, (
        _ctx().handle, _ptr(q), h * d, b, h, ctypes.byref(cache), _ptr(table), table.shape[1], _ptr(lengths),
        1 / math.sqrt(d), case["window"], _ptr(out["y"]), h * d, None))], cache


# ---------------------------------------------------------------- exact values


def _exact_scales(y):
    """The values in e4m3's range that 8 bits round, and the scales they are divided by."""
    s = torch.stack([part.abs().amax(1) for part in y.split(BLOCK, 1)], 1) / F8_MAX
    s = s + (s == 0)
    return y / s[:, torch.arange(y.shape[1], device=y.device) // BLOCK], s.t()


def _exact_norm(case, seed):
    x, r, gamma = (None if v is None else v.double() for v in _norm_inputs(case, seed))
    h = x if r is None else x + r
    y = gamma * (h / torch.sqrt(h.square().sum(1, keepdim=True) / h.shape[1] + EPS))
    out = {} if r is None else {"sum": h}
    if case["out"] != "q":
        out["y"] = y
    if case["out"] != "y":
        out["q"], out["scales"] = _exact_scales(y)
    return out


def _exact_quantize(case, seed):
    x, gate = _quantize_inputs(case, seed)
    y = x.double() if gate is None else x.double() * gate.double() * torch.sigmoid(gate.double())
    q, scales = _exact_scales(y)
    return {"q": q, "scales": scales}


def _exact_matmul(case, seed):
    a, a_scales, w, w_scales, bias = _matmul_inputs(case, seed)
    y = torch.zeros(case["m"], case["n"], dtype=torch.float64, device=DEVICE)
    column = torch.arange(case["n"], device=DEVICE) // BLOCK
    for i, (x, v) in enumerate(zip(a.double().split(BLOCK, 1), w.double().split(BLOCK, 1))):
        y.addcmul_(x @ v.t(), a_scales[i].double()[:, None] * w_scales[:, i].double()[column])
    return {"y": y if bias is None else y + bias.double()}


def _exact_append(case, seed):
    qkv, k_pool, v_pool, positions, slots, cos, sin = _append_inputs(case, seed)
    t, h, g, d, rot = case["rows"], case["heads"], case["kv_heads"], case["dim"], case["rotary"]
    x = qkv.double().view(t, -1, d)
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
    q, k_pool, v_pool, table, lengths = _attend_inputs(case, seed)
    g, d, page = case["kv_heads"], case["dim"], case["page"]
    rows = []
    for i, n in enumerate(lengths.tolist()):
        first = max(0, n - case["window"]) if case["window"] else 0
        if n == 0:
            rows.append(torch.zeros(case["heads"] * d, dtype=torch.float64, device=DEVICE))
            continue
        at = torch.arange(first, n, device=DEVICE)
        where = (table[i, at // page].long(), at % page)
        k, v = k_pool[where].double(), v_pool[where].double()  # [tokens, kv_heads, dim]
        x = q[i].double().view(g, -1, d)
        p = torch.softmax((x @ k.permute(1, 2, 0)) * d ** -0.5, -1)
        rows.append((p @ v.transpose(0, 1)).flatten())
    return {"y": torch.stack(rows)}


# ---------------------------------------------------------------- work


def _work_norm(case):
    n, size = case["rows"] * case["cols"], SIZE[case["dtype"]]
    moved = n * size * (3 if case["residual"] else 1) + case["cols"] * size
    if case["out"] != "q":
        moved += n * size
    if case["out"] != "y":
        moved += n + 4 * case["rows"] * _blocks(case["cols"])
    return {"bytes": moved, "flops": 5 * n}


def _work_quantize(case):
    n = case["rows"] * case["cols"]
    return {"bytes": n * SIZE[case["dtype"]] * (2 if case["gate"] else 1) + n + 4 * case["rows"] * _blocks(case["cols"]),
            "flops": n * (7 if case["gate"] else 2)}


def _work_matmul(case):
    m, k, n = case["m"], case["k"], case["n"]
    scales = 4 * _blocks(k) * (m + _blocks(n))
    return {"bytes": m * k + n * k + scales + SIZE[case["dtype"]] * (m * n + (n if case["bias"] else 0)),
            "flops": 2 * m * k * n}


def _work_append(case):
    rows, size = case["rows"], SIZE[case["dtype"]]
    kept = rows - (len(range(7, rows, 16)) if case["padding"] else 0)
    q, kv = case["heads"] * case["dim"] * size, 2 * case["kv_heads"] * case["dim"] * size
    return {"bytes": 2 * rows * q + 2 * kept * kv + rows * (16 + 4 * case["rotary"]),
            "flops": 3 * rows * (case["heads"] + case["kv_heads"]) * case["rotary"]}


def _work_attend(case):
    read = sum(min(n, case["window"]) if case["window"] else n for n in _lengths(case))
    size = SIZE[case["dtype"]]
    return {"bytes": 2 * read * case["kv_heads"] * case["dim"] * size + 2 * case["batch"] * case["heads"] * case["dim"] * size,
            "flops": 4 * read * case["heads"] * case["dim"]}


# ---------------------------------------------------------------- the interface

_INPUTS = {"norm": _norm_inputs, "quantize": _quantize_inputs, "matmul": _matmul_inputs, "append": _append_inputs,
           "attend": _attend_inputs}
_PLAIN = {"norm": _plain_norm, "quantize": _plain_quantize, "matmul": _plain_matmul, "append": _plain_append,
          "attend": _plain_attend}
_OWN = {"norm": _own_norm, "quantize": _own_quantize, "matmul": _own_matmul, "append": _own_append,
        "attend": _own_attend}
_EXACT = {"norm": _exact_norm, "quantize": _exact_quantize, "matmul": _exact_matmul, "append": _exact_append,
          "attend": _exact_attend}
_WORK = {"norm": _work_norm, "quantize": _work_quantize, "matmul": _work_matmul, "append": _work_append,
         "attend": _work_attend}


def prepare(case, seed):
    state = {"case": case, "inputs": _INPUTS[case["kind"]](case, seed)}
    if own:
        # The buffers, the prepared weight and the arguments that a program keeps from call to call.
        state["out"], state["calls"], state["keep"] = _OWN[case["kind"]](case, state["inputs"])
        state["check"] = _ctx().check
    torch.cuda.synchronize()
    return state


def run(state):
    if own:
        for call, arguments in state["calls"]:
            state["check"](call(*arguments))
        return state["out"]
    return _PLAIN[state["case"]["kind"]](state)


def exact(case, seed):
    return _EXACT[case["kind"]](case, seed)


def work(case):
    return _WORK[case["kind"]](case)
