"""Beam search over a paged key/value cache: the paged operators of include/gptoss.h together.

A small attention-only model with random weights (an embedding, a few layers of projections around
gptoss_kv_append and gptoss_paged_attention, an output matrix) reads a batch of prompts of unequal length in one call
per layer, then grows `beams` continuations of each: gptoss_beam_select picks rows and tokens, gptoss_kv_fork reorders
the caches (full pages shared, part-filled last pages copied) and gives room for the next token, and now and then
gptoss_kv_compact moves the live pages together. All bookkeeping stays on the GPU.

    python examples/beam_search.py [--requests 4] [--beams 4] [--steps 24] [--check]

--check recomputes the winning beams' scores from scratch with plain matrix products and compares.
"""
import argparse
import ctypes
import math
import sys
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "gptoss-infer_b200"))
from gptoss_b200 import capi  # noqa: E402

Q_HEADS, KV_HEADS, DIM, LAYERS, PAGE, VOCAB, WIDTH, WINDOW = 16, 2, 64, 4, 16, 4096, 512, 48
P = capi.ptr


def yarn_tables(positions, rot, theta=150000.0, factor=32.0, original=4096, device="cuda"):
    """cos and sin [positions][rot / 2] of YaRN-scaled rotary frequencies, as the engine builds its own: frequencies that
    turn more than 32 times within the original context stay, those below one turn are divided by the factor."""
    half = rot // 2
    base = theta ** (np.arange(half) * 2.0 / rot)
    low, high = (rot * math.log(original / (r * 2 * math.pi)) / (2 * math.log(theta)) for r in (32.0, 1.0))
    ramp = np.clip((np.arange(half) - low) / max(high - low, 1e-3), 0, 1)
    angle = np.arange(positions)[:, None] * ((1 - ramp) / base + ramp / (factor * base))
    scale = 0.1 * math.log(factor) + 1.0
    return [torch.tensor(f(angle) * scale, dtype=torch.float32, device=device) for f in (np.cos, np.sin)]


class Model:
    def __init__(self, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        def w(*shape):
            return torch.randn(*shape, device="cuda", generator=g) / math.sqrt(shape[-1])
        self.embed, self.out = w(VOCAB, WIDTH) * 20, w(VOCAB, WIDTH) * 3
        self.qkv = [w((Q_HEADS + 2 * KV_HEADS) * DIM, WIDTH) for _ in range(LAYERS)]
        self.o = [w(WIDTH, Q_HEADS * DIM) for _ in range(LAYERS)]
        self.sinks = torch.randn(LAYERS, Q_HEADS, device="cuda", generator=g)


class Cache:
    """A pool of fp16 pages for all layers, its reference counts, and the tables of the sequences in it."""

    def __init__(self, lib, pages):
        self.lib, self.pages = lib, pages
        self.k = torch.zeros(LAYERS, pages, PAGE, KV_HEADS, DIM, dtype=torch.float16, device="cuda")
        self.v = torch.zeros_like(self.k)
        self.pool = lib.gptoss_kv_pool_create(P(self.k), P(self.v), 1, LAYERS, pages, PAGE, KV_HEADS, DIM,
                                              (ctypes.c_longlong * 4)(*self.k.stride()[:4]))
        if not self.pool:
            raise capi.GptossError(lib.gptoss_last_error().decode())
        self.refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
        self.stride = pages
        self.tables = torch.full((1, self.stride), -1, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(1, dtype=torch.int32, device="cuda")

    def fork(self, parents, extra, stream):
        """The sequences `parents` (rows of the present tables, -1: a new one) with room for `extra` more positions each
        take the place of the present ones."""
        n = parents.numel()
        tables = torch.empty(n, self.stride, dtype=torch.int32, device="cuda")
        lens = torch.empty(n, dtype=torch.int32, device="cuda")
        capi.check(self.lib.gptoss_kv_fork(self.pool, P(self.refs), P(self.tables), P(self.lens), self.lens.numel(),
                                           P(parents), P(extra), n, self.stride, P(self.refs), P(tables), P(lens), stream))
        self.tables, self.lens = tables, lens

    def compact(self, stream):
        remap, live = torch.empty_like(self.refs), torch.empty(1, dtype=torch.int32, device="cuda")
        capi.check(self.lib.gptoss_kv_compact(self.pool, P(self.refs), P(self.tables), P(self.lens), self.lens.numel(),
                                              self.stride, P(self.refs), P(self.tables), P(remap), P(live), stream))
        return live

    def status(self):
        code = ctypes.c_int()
        capi.check(self.lib.gptoss_kv_pool_status(self.pool, ctypes.byref(code)))
        return code.value

    def close(self):
        torch.cuda.synchronize()
        self.lib.gptoss_kv_pool_destroy(self.pool)


def forward(lib, model, cache, tokens, cu, most, tabs, stream):
    """Logits of each sequence's last token. Layers alternate between full and sliding-window attention."""
    x = model.embed[tokens]
    rows = tokens.numel()
    batch = capi.KvBatch(cu.numel() - 1, rows, most, cache.stride, P(cu), P(cache.lens), P(cache.tables))
    q = torch.empty(rows, Q_HEADS, DIM, device="cuda")
    a = torch.empty_like(q)
    for l in range(LAYERS):
        h = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-5)
        qkv = h @ model.qkv[l].T
        at, width = P(qkv), qkv.shape[1]
        capi.check(lib.gptoss_kv_append(cache.pool, l, ctypes.byref(batch), at, at + Q_HEADS * DIM * 4,
                                        at + (Q_HEADS + KV_HEADS) * DIM * 4, 0, width, width, Q_HEADS, P(tabs[0]), P(tabs[1]),
                                        tabs[0].shape[0], DIM, 0, P(q), 0, stream))
        capi.check(lib.gptoss_paged_attention(cache.pool, l, ctypes.byref(batch), P(q), 0, Q_HEADS * DIM, Q_HEADS,
                                              P(model.sinks[l]), DIM ** -0.5, WINDOW if l % 2 else 0, P(a), Q_HEADS * DIM,
                                              stream))
        x = x + a.view(rows, -1) @ model.o[l].T
    last = x[cu[1:].long() - 1]
    return (last * torch.rsqrt(last.pow(2).mean(-1, keepdim=True) + 1e-5)) @ model.out.T


def search(lib, model, prompts, beams, steps, compact_every=8):
    """(scores [requests][beams], tokens [requests][beams][steps]) of the best continuations."""
    stream = torch.cuda.current_stream().cuda_stream
    n = len(prompts)
    need = sum(-(-len(p) // PAGE) for p in prompts) + n * beams * (3 + steps // PAGE)
    cache = Cache(lib, need)
    tabs = yarn_tables(max(len(p) for p in prompts) + steps + 1, DIM)
    i32 = dict(dtype=torch.int32, device="cuda")
    # the prompts: one sequence per request
    cache.fork(torch.full((n,), -1, **i32), None, stream)
    cache.fork(torch.arange(n, **i32), torch.tensor([len(p) for p in prompts], **i32), stream)
    cu = torch.tensor(np.cumsum([0] + [len(p) for p in prompts]), **i32)
    logits = forward(lib, model, cache, torch.tensor(np.concatenate(prompts), device="cuda"), cu,
                     max(len(p) for p in prompts), tabs, stream)
    scores = torch.zeros(n, device="cuda")
    history = torch.empty(n * beams, 0, dtype=torch.int32, device="cuda")
    one, cu1 = torch.ones(n * beams, **i32), torch.arange(n * beams + 1, **i32)
    for step in range(steps):
        per_row = 1 if step == 0 else beams           # the first selection starts from one row per request
        picked, rows, tokens = (torch.empty(n * beams, device="cuda"), torch.empty(n * beams, **i32),
                                torch.empty(n * beams, **i32))
        capi.check(lib.gptoss_beam_select(P(logits), 0, VOCAB, P(scores), None, 0, n, per_row, VOCAB, beams, P(picked),
                                          P(rows), P(tokens), stream))
        scores = picked
        history = torch.cat([history[rows.long()] if step else history, tokens[:, None]], 1)
        if step + 1 == steps:
            break
        cache.fork(rows, one, stream)
        if step % compact_every == compact_every - 1:
            cache.compact(stream)
        logits = forward(lib, model, cache, tokens.long(), cu1, 1, tabs, stream)
    code = cache.status()
    cache.close()
    if code:
        raise RuntimeError(f"the cache's status is {code}")
    return scores.view(n, beams), history.view(n, beams, steps)


def plain_score(model, prompt, tokens):
    """The log probability of `tokens` after `prompt`, from scratch in plain matrix products (fp16 keys and values)."""
    ids = torch.tensor(np.concatenate([prompt, tokens]), device="cuda")
    n = ids.numel() - 1
    cos, sin = (t[:n, None] for t in yarn_tables(n, DIM))
    x, pos = model.embed[ids[:n]], torch.arange(n, device="cuda")
    for l in range(LAYERS):
        h = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-5)
        q, k, v = (h @ model.qkv[l].T).view(n, -1, DIM).split([Q_HEADS, KV_HEADS, KV_HEADS], 1)
        q, k = (torch.cat([t[..., :32] * cos - t[..., 32:] * sin, t[..., 32:] * cos + t[..., :32] * sin], -1) for t in (q, k))
        k, v = (t.half().float().repeat_interleave(Q_HEADS // KV_HEADS, 1) for t in (k, v))
        s = torch.einsum("thd,shd->hts", q, k) * DIM ** -0.5
        seen = pos[None] <= pos[:, None]
        if l % 2:
            seen &= pos[None] > pos[:, None] - WINDOW
        s = torch.cat([s.masked_fill(~seen, -torch.inf), model.sinks[l][:, None, None].expand(-1, n, 1)], -1)
        a = torch.einsum("hts,shd->thd", s.softmax(-1)[..., :n], v)
        x = x + a.reshape(n, -1) @ model.o[l].T
    x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-5)
    logp = torch.log_softmax((x[len(prompt) - 1:] @ model.out.T).double(), -1)
    return logp.gather(1, ids[len(prompt):, None]).sum().item()


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--requests", type=int, default=4)
    ap.add_argument("--beams", type=int, default=4)
    ap.add_argument("--steps", type=int, default=24)
    ap.add_argument("--check", action="store_true")
    a = ap.parse_args()
    lib, model, r = capi.load(), Model(), np.random.RandomState(1)
    prompts = [r.randint(0, VOCAB, r.randint(5, 200)) for _ in range(a.requests)]
    scores, tokens = search(lib, model, prompts, a.beams, a.steps)
    for i, p in enumerate(prompts):
        print(f"request {i}: {len(p)} prompt tokens, best score {scores[i, 0].item():.4f}, tokens {tokens[i, 0].tolist()[:8]} ...")
        if a.check:
            for b in range(a.beams):
                want = plain_score(model, p, tokens[i, b].cpu().numpy())
                assert abs(want - scores[i, b].item()) <= 2e-3 * max(1.0, abs(want)), (i, b, want, scores[i, b].item())
    if a.check:
        print("scores agree with the plain recomputation")


if __name__ == "__main__":
    main()
