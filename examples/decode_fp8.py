"""Greedy decoding of a small decoder with 8-bit floating-point weights over a paged cache, on random weights.

    python examples/decode_fp8.py [--layers 4 --hidden 2048 --batch 8 --prompt 64 --steps 32 ...]

A batch's prompts run as rows of one pass (each token attends to the tokens of its sequence up to itself: its own row of
the page table, its own length), then steps of one token a sequence run as one HIP graph, recorded once and replayed
over buffers whose contents change: tokens' embeddings, positions, slots, lengths and page tables. At the end all tokens run
again as one prompt, whose last logits have to agree with the decoded ones: sums in another order move some values by a
step of 8 bits, and such steps move more of them in later products, up to the roundings' own noise (a few per cent of
the norm); a token at a wrong position or page gives logits that have little to do with the others.
"""

from __future__ import annotations

import argparse
import ctypes
import os
import sys
import time

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from transmuter_amd import Context, serving  # noqa: E402
from transmuter_amd._lib import lib  # noqa: E402
from transmuter_amd.serving import Fp8Weight, Norm, PagedCache, Rows8  # noqa: E402


def e4m3(x: np.ndarray) -> np.ndarray:
    """Values of magnitude up to 448 as e4m3 bits, rounded to nearest, ties to even."""
    a = np.abs(x).astype(np.float32)
    exponent = np.maximum(np.frexp(a)[1] - 1, -6)  # of the leading bit; -6 and below: subnormal
    steps = np.rint(np.ldexp(a, 3 - exponent)).astype(np.int32)  # of 2^(exponent - 3); 16 carries into the exponent by itself
    bits = np.where(steps < 8, steps, (exponent + 6) * 8 + steps)
    return (bits | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def block_scaled(w: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """A weight [N, K] in e4m3 and the scales of its 128 x 128 blocks."""
    n, k = w.shape
    nb, kb = -(-n // 128), -(-k // 128)
    v = np.zeros((nb * 128, kb * 128), np.float32)
    v[:n, :k] = w
    v = v.reshape(nb, 128, kb, 128)
    scales = np.abs(v).max((1, 3)) / np.float32(448)
    scales[scales == 0] = 1
    q = e4m3(np.clip(v / scales[:, None, :, None], -448, 448))
    return q.reshape(nb * 128, kb * 128)[:n, :k].copy(), scales


class Model:
    """The weights, on the device but for the embedding."""

    def __init__(self, ctx: Context, a, rng):
        def weight(n, k):
            return Fp8Weight.prepare(ctx, *block_scaled(rng.standard_normal((n, k), np.float32) / np.float32(np.sqrt(k))))

        def gamma():
            return ctx.put((rng.random(a.hidden) + 0.5).astype(np.float16))

        self.ctx, self.a = ctx, a
        qkv = (a.heads + 2 * a.kv_heads) * a.head_dim
        self.layers = [dict(norm1=gamma(), qkv=weight(qkv, a.hidden), out=weight(a.hidden, a.heads * a.head_dim), norm2=gamma(),
                            gate_up=weight(2 * a.ffn, a.hidden), down=weight(a.hidden, a.ffn)) for _ in range(a.layers)]
        self.norm, self.head = gamma(), weight(a.vocabulary, a.hidden)
        self.embedding = rng.standard_normal((a.vocabulary, a.hidden)).astype(np.float16)
        half = a.head_dim // 2
        angle = np.arange(a.context)[:, None] * 10000.0 ** (-np.arange(half) / half)
        self.cos, self.sin = ctx.put(np.cos(angle).astype(np.float32)), ctx.put(np.sin(angle).astype(np.float32))


class Pass:
    """The buffers of a pass over `rows` tokens, and its calls."""

    def __init__(self, model: Model, caches: list[PagedCache], rows: int):
        ctx, a = model.ctx, model.a
        self.model, self.caches, self.rows = model, caches, rows
        half = lambda *shape: ctx.empty(shape, "f16")  # noqa: E731
        wide, inner = (a.heads + 2 * a.kv_heads) * a.head_dim, a.heads * a.head_dim
        self.x, self.normed = half(rows, a.hidden), Rows8.empty(ctx, (rows, a.hidden))
        self.qkv, self.q, self.attended, self.attended8 = half(rows, wide), half(rows, inner), half(rows, inner), Rows8.empty(ctx, (rows, inner))
        self.projected, self.gate_up, self.gated = half(rows, a.hidden), half(rows, 2 * a.ffn), Rows8.empty(ctx, (rows, a.ffn))
        self.logits = ctx.empty((rows, a.vocabulary), "f32")
        self.positions, self.slots = ctx.empty((rows,), "s64"), ctx.empty((rows,), "s64")
        self.table, self.lengths = ctx.empty((rows, -(-a.context // a.page)), "s32"), ctx.empty((rows,), "s32")

    def set(self, tokens, sequences, positions, tables) -> None:
        """The pass's tokens: token tokens[i] of sequence sequences[i] at positions[i]."""
        page = self.model.a.page
        table = tables[sequences].astype(np.int32)
        slots = table[np.arange(self.rows), positions // page].astype(np.int64) * page + positions % page
        for tensor, host in ((self.x, self.model.embedding[tokens]), (self.positions, positions.astype(np.int64)), (self.slots, slots),
                             (self.table, table), (self.lengths, (positions + 1).astype(np.int32))):
            host = np.ascontiguousarray(host)
            assert host.nbytes == tensor.nbytes
            tensor.ctx.check(lib().tmh_upload(tensor.ctx.handle, tensor.ptr, host.ctypes.data_as(ctypes.c_void_p), host.nbytes))

    def run(self) -> None:
        m, a = self.model, self.model.a
        normed, delta = Norm(None, self.normed, self.x), None  # x holds the residual, which each norm adds to
        for layer, cache in zip(m.layers, self.caches):
            if delta is None:
                serving.rms_norm(self.x, layer["norm1"], out=normed)
            else:
                serving.rms_norm(delta, layer["norm1"], self.x, out=normed)
            serving.matmul_fp8(self.normed, layer["qkv"], out=self.qkv)
            cache.append(self.qkv, a.heads, self.slots, self.positions, m.cos, m.sin, out=self.q)
            cache.attend(self.q, self.table, self.lengths, out=self.attended)
            serving.quantize_rows(self.attended, out=self.attended8)
            serving.matmul_fp8(self.attended8, layer["out"], out=self.projected)
            serving.rms_norm(self.projected, layer["norm2"], self.x, out=normed)
            serving.matmul_fp8(self.normed, layer["gate_up"], out=self.gate_up)
            serving.quantize_swiglu(self.gate_up, out=self.gated)
            delta = serving.matmul_fp8(self.gated, layer["down"], out=self.projected)
        serving.rms_norm(delta, m.norm, self.x, out=normed)
        serving.matmul_fp8(self.normed, m.head, y_type="f32", out=self.logits)

    def record(self) -> ctypes.c_void_p:
        """The pass as a graph. (It has run before: nothing it needs is allocated while it is recorded.)"""
        ctx, graph = self.model.ctx, ctypes.c_void_p()
        ctx.check(lib().tmh_graph_begin(ctx.handle, None))
        self.run()
        ctx.check(lib().tmh_graph_end(ctx.handle, None, ctypes.byref(graph)))
        return graph


def arguments(argv=None):
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("layers", 4), ("hidden", 2048), ("heads", 16), ("kv-heads", 4), ("head-dim", 128), ("ffn", 11008),
                          ("vocabulary", 4096), ("batch", 8), ("prompt", 64), ("steps", 32), ("context", 1024), ("page", 16), ("seed", 0)):
        p.add_argument("--" + name, type=int, default=default)
    return p.parse_args(argv)


def main(argv=None) -> dict:
    a = arguments(argv)
    if a.steps < 1 or a.prompt < 1 or a.prompt + a.steps > a.context:
        raise SystemExit("a prompt and its steps (one of each at least) have to fit the context")
    ctx, rng = Context(0), np.random.default_rng(a.seed)
    model = Model(ctx, a, rng)
    per = -(-a.context // a.page)
    caches = [PagedCache(ctx, a.batch * per, a.page, a.kv_heads, a.head_dim) for _ in range(a.layers)]
    tables = rng.permutation(a.batch * per).astype(np.int32).reshape(a.batch, per)
    tokens = rng.integers(0, a.vocabulary, (a.batch, a.prompt))

    def prompt(tokens):
        """All tokens of the batch as one pass; the logits of the last of each sequence."""
        b, n = tokens.shape
        whole = Pass(model, caches, b * n)
        whole.set(tokens.reshape(-1), np.repeat(np.arange(b), n), np.tile(np.arange(n), b), tables)
        ctx.synchronize()
        began = time.perf_counter()
        whole.run()
        ctx.synchronize()
        return whole.logits.numpy().reshape(b, n, -1)[:, -1], time.perf_counter() - began

    logits, prompt_s = prompt(tokens)
    step, graph, step_s = Pass(model, caches, a.batch), None, []
    for i in range(a.steps):
        tokens = np.concatenate([tokens, logits.argmax(-1)[:, None]], 1)
        step.set(tokens[:, -1], np.arange(a.batch), np.full(a.batch, a.prompt + i), tables)
        ctx.synchronize()
        began = time.perf_counter()
        if graph is None:
            step.run()
        else:
            ctx.check(lib().tmh_graph_launch(ctx.handle, graph, None))
        ctx.synchronize()
        step_s.append(time.perf_counter() - began)
        logits = step.logits.numpy()
        graph = graph or step.record()
    again, _ = prompt(tokens)
    ctx.synchronize()
    ctx.check(lib().tmh_graph_destroy(ctx.handle, graph))
    difference = float(np.linalg.norm(logits - again) / np.linalg.norm(again))
    return {"prompt_ms": prompt_s * 1e3, "step_ms": float(np.median(step_s[1:] or step_s)) * 1e3, "difference": difference,
            "finite": bool(np.isfinite(logits).all()), "tokens": tokens}


# Roundings to e4m3 are off by 2.6% of the norm (2^-4 over sqrt 3, at mantissas from 1 to 2), so two passes whose roundings had
# nothing in common would differ by 3.7% behind each product: by less than 4 times that behind a layer's branches and the
# head, as the residual dilutes what earlier layers add. Logits that have nothing in common differ by 1.4.
AGREES = 0.15

if __name__ == "__main__":
    result = main()
    print(f"prompt {result['prompt_ms']:.2f} ms, a step {result['step_ms']:.3f} ms, decoded and prompted logits differ by "
          f"{result['difference']:.1e} of their norm")
    sys.exit(0 if result["finite"] and result["difference"] < AGREES else 1)
