"""Cases of the paged key/value cache operators: rotary append, chunk attention, beam selection, fork and compaction.

Each case names an operator in "op". `run` computes it in elementary torch operations, or, with `own`, through the
library's C ABI (include/gptoss.h). Lengths follow from the case alone, values from the seed.
"""
import ctypes
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

TYPES = {"f32": (0, torch.float32, 4), "f16": (1, torch.float16, 2), "bf16": (2, torch.bfloat16, 2)}


# ------------------------------------------------------------------------------------------------------- cases
def _attn(name, seqs, new, ctx, qh, kvh, dim, page, qt, kt, window=0, sinks=True, mixed=False, order="token"):
    return {"name": name, "op": "attention", "seqs": seqs, "new": new, "ctx": ctx, "q_heads": qh, "kv_heads": kvh,
            "dim": dim, "page": page, "q_type": qt, "kv_type": kt, "window": window, "sinks": sinks, "mixed": mixed,
            "order": order}


def _append(name, seqs, new, ctx, qh, kvh, dim, rot, page, it, qt, kt, interleaved=False, order="token"):
    return {"name": name, "op": "append", "seqs": seqs, "new": new, "ctx": ctx, "q_heads": qh, "kv_heads": kvh,
            "dim": dim, "rot": rot, "page": page, "in_type": it, "q_type": qt, "kv_type": kt,
            "interleaved": interleaved, "order": order, "mixed": False, "window": 0}


def _beam(name, batch, beams, vocab, picks, it, done):
    return {"name": name, "op": "beam", "batch": batch, "beams": beams, "vocab": vocab, "picks": picks,
            "in_type": it, "done": done}


def _fork(name, batch, beams, ctx, page, layers, kvh, dim, kt, extra):
    return {"name": name, "op": "fork", "batch": batch, "beams": beams, "ctx": ctx, "page": page, "layers": layers,
            "kv_heads": kvh, "dim": dim, "kv_type": kt, "extra": extra}


def _compact(name, seqs, ctx, page, layers, kvh, dim, kt, spare):
    return {"name": name, "op": "compact", "seqs": seqs, "ctx": ctx, "page": page, "layers": layers, "kv_heads": kvh,
            "dim": dim, "kv_type": kt, "spare": spare}


def listed():
    return [
        # one sequence's next token after 4096 positions, in the engine's own types: latency
        _attn("attention one token", 1, 1, 4097, 64, 8, 64, 16, "f32", "f16"),
        # 64 concurrent sequences of unequal lengths decode one token each: memory bandwidth
        _attn("attention 64 sequences", 64, 1, 8191, 64, 8, 64, 16, "bf16", "bf16"),
        # one sequence's prompt chunk beside seven that decode, heads of 128 in fives, a sliding window, head-major pages
        _attn("attention mixed window", 8, 511, 5000, 40, 8, 128, 32, "f16", "f16", window=1000, sinks=False,
              mixed=True, order="head"),
        # a 2048-token chunk late in a long prompt: tensor throughput
        _attn("attention long chunk", 1, 2048, 16384, 64, 8, 64, 64, "bf16", "bf16"),
        # the append of a 64-sequence decode step: latency
        _append("append 64 tokens", 64, 1, 4100, 64, 8, 64, 64, 16, "f32", "f16", "f16"),
        # the append of a long prompt, adjacent pairs, half of each head rotated
        _append("append prompt", 3, 5461, 5461, 32, 8, 128, 64, 32, "bf16", "bf16", "bf16", interleaved=True,
                order="head"),
        # four beams of one request over the full vocabulary
        _beam("beams of one request", 1, 4, 201088, 8, "f32", False),
        # eight beams of 32 requests, some of them finished
        _beam("beams of 32 requests", 32, 8, 201088, 16, "bf16", True),
        # reordering four beams of one request after a selection: latency
        _fork("fork four beams", 1, 4, 1003, 16, 24, 8, 64, "f16", 1),
        # reordering 32 x 8 beams, every last page copied in every layer
        _fork("fork 256 beams", 32, 8, 4007, 64, 8, 8, 128, "bf16", 1),
        # a small cache with a few holes
        _compact("compact small", 5, 700, 16, 24, 8, 64, "f16", 0.25),
        # a large cache, half of it freed
        _compact("compact large", 64, 4100, 32, 2, 8, 128, "bf16", 1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "append", "append", "beam", "beam", "fork", "compact"])
    dim, page = rng.choice([64, 128]), rng.choice([8, 16, 24, 32, 64, 128])
    kvh, order = rng.choice([1, 2, 4, 8]), rng.choice(["token", "head"])
    pair = rng.choice([("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")])
    if op == "attention":
        group = rng.choice([1, 2, 4, 5, 7, 8, 16]) if kvh < 8 else rng.choice([1, 4, 5, 8])
        seqs, ctx = _log(rng, 1, 64), _log(rng, 16, 16000)
        new = 1 if rng.random() < 0.4 else min(ctx, _log(rng, 2, 2048))
        while seqs * new * ctx * kvh * group > 2048 * 16384 * 64 // 4 or seqs * ctx > 64 * 8192:
            seqs, new = max(1, seqs // 2), max(1, new - new // 4)
            ctx = max(new, ctx - ctx // 8)
        window = rng.choice([0, 0, 128, _log(rng, 1, 4000)])
        return _attn("", seqs, new, ctx, group * kvh, kvh, dim, page, *pair, window=window, sinks=rng.random() < 0.5,
                     mixed=rng.random() < 0.3, order=order) | {"salt": rng.randrange(1 << 20)}
    if op == "append":
        group, seqs, new = rng.choice([1, 4, 7, 8]), _log(rng, 1, 64), _log(rng, 1, 8000)
        new = max(1, min(new, 12000 // seqs))
        it = rng.choice(["f32", "f16", "bf16"])
        rot = rng.choice([dim, dim, dim // 2, 24])
        return _append("", seqs, new, new + _log(rng, 1, 8000), group * kvh, kvh, dim, rot, page, it, *pair,
                       interleaved=rng.random() < 0.5, order=order) | {"salt": rng.randrange(1 << 20)}
    if op == "beam":
        batch, beams, vocab = _log(rng, 1, 32), rng.choice([1, 2, 3, 4, 5, 8]), _log(rng, 300, 201088)
        return _beam("", batch, beams, vocab, rng.choice([1, beams, 2 * beams]), rng.choice(["f32", "f16", "bf16"]),
                     rng.random() < 0.5) | {"salt": rng.randrange(1 << 20)}
    layers, kt = rng.choice([1, 2, 4, 8]), pair[1]
    if op == "fork":
        return _fork("", _log(rng, 1, 32), rng.choice([1, 2, 4, 8]), _log(rng, 1, 4000), max(page, 16), layers, kvh,
                     dim, kt, rng.choice([0, 1, 1, 17])) | {"salt": rng.randrange(1 << 20)}
    return _compact("", _log(rng, 1, 64), _log(rng, 1, 4000), max(page, 16), min(layers, 2), kvh, dim, kt,
                    rng.uniform(0.1, 1.0)) | {"salt": rng.randrange(1 << 20)}


def _spread(case, n, top, least):
    """n lengths in [least .. top], unequal, by the case alone; the first is the longest."""
    r = np.random.RandomState((top * 7919 + n * 31 + case.get("salt", 0)) % (1 << 31))
    v = r.randint(least, top + 1, n)
    v[0] = top
    return v.astype(np.int64)


def _lengths(case):
    """(new tokens, cache length after them) of each sequence."""
    n, new, ctx = case["seqs"], case["new"], case["ctx"]
    if case["mixed"]:
        q = np.ones(n, np.int64)
        q[0] = new
    else:
        q = _spread(case, n, new, max(1, new // 2))
    kv = np.maximum(_spread(case, n, ctx, max(1, ctx // 2)), q)
    return q, kv


# ------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _pages(shape, order, dtype, g):
    """[layers, pages, slots, heads, dim] of N(0, 1), stored slot-major or head-major."""
    layers, pages, slots, heads, dim = shape
    if order == "head":
        return torch.randn(layers, pages, heads, slots, dim, device="cuda", generator=g).to(dtype).transpose(2, 3)
    return torch.randn(layers, pages, slots, heads, dim, device="cuda", generator=g).to(dtype)


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def _random_tables(need, num_pages, stride, seed):
    """Tables that name each page once, in a random order; entries past a sequence's pages are -1."""
    order = np.random.RandomState(seed % (1 << 31)).permutation(num_pages)[: int(need.sum())]
    t = np.full((len(need), stride), -1, np.int64)
    t[np.arange(stride)[None, :] < need[:, None]] = order
    return t


def _prepare_batch(case, seed):
    q, kv = _lengths(case)
    need = -(-kv // case["page"])
    pages, stride = int(need.sum()) + 3, int(need.max()) + 2
    s = {"pages": pages, "stride": stride, "T": int(q.sum()), "cu": _ints(np.concatenate([[0], np.cumsum(q)])),
         "lens": _ints(kv), "tables": _ints(_random_tables(need, pages, stride, seed)), "most": int(q.max()),
         "ctx": int(kv.max())}
    return s


def _rope_table(positions, rot, seed):
    """cos and sin of YaRN-scaled frequencies (theta 150000, factor 32 over 4096 positions)."""
    half, theta, factor, original = rot // 2, 150000.0, 32.0, 4096.0
    base = theta ** (np.arange(half) * 2.0 / rot)
    low, high = (rot * math.log(original / (r * 2 * math.pi)) / (2 * math.log(theta)) for r in (32.0, 1.0))
    ramp = np.clip((np.arange(half) - low) / max(high - low, 1e-3), 0, 1)
    inv = (1 - ramp) / base + ramp / (factor * base)
    ang = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * torch.from_numpy(inv).cuda()
    m = 0.1 * math.log(factor) + 1.0
    return (ang.cos() * m).float(), (ang.sin() * m).float()


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    op = case["op"]
    if op in ("attention", "append"):
        s |= _prepare_batch(case, seed)
        kt = TYPES[case["kv_type"]][1]
        shape = (1, s["pages"], case["page"], case["kv_heads"], case["dim"])
        s["k"], s["v"] = _pages(shape, case["order"], kt, g), _pages(shape, case["order"], kt, g)
        if op == "attention":
            qt = TYPES[case["q_type"]][1]
            s["q"] = torch.randn(s["T"], case["q_heads"], case["dim"], device="cuda", generator=g).to(qt)
            s["out"] = torch.empty_like(s["q"])
            s["sinks"] = torch.randn(case["q_heads"], device="cuda", generator=g) if case["sinks"] else None
        else:
            width = (case["q_heads"] + 2 * case["kv_heads"]) * case["dim"]
            s["qkv"] = torch.randn(s["T"], width, device="cuda", generator=g).to(TYPES[case["in_type"]][1])
            s["cos"], s["sin"] = _rope_table(s["ctx"], case["rot"], seed)
            s["q_out"] = torch.empty(s["T"], case["q_heads"], case["dim"], device="cuda",
                                     dtype=TYPES[case["q_type"]][1])
    elif op == "beam":
        rows = case["batch"] * case["beams"]
        s["logits"] = (torch.randn(rows, case["vocab"], device="cuda", generator=g) * 3).to(TYPES[case["in_type"]][1])
        s["scores"] = -10 * torch.rand(rows, device="cuda", generator=g)
        s["done"] = (torch.rand(rows, device="cuda", generator=g) < 0.25).to(torch.uint8) if case["done"] else None
        n = case["batch"] * case["picks"]
        s["out"] = [torch.empty(n, device="cuda"), torch.empty(n, device="cuda", dtype=torch.int32),
                    torch.empty(n, device="cuda", dtype=torch.int32)]
    else:
        s |= _prepare_pages(case, seed, g)
    if own:
        s |= _prepare_own(s)
    return s


def _prepare_pages(case, seed, g):
    page, r = case["page"], np.random.RandomState(seed % (1 << 31))
    s = {}
    if op_is(case, "fork"):
        batch, beams = case["batch"], case["beams"]
        n = batch * beams
        # the beams of a request share its prompt's full pages (half of the context) and hold the rest on their own
        lens = np.repeat(_spread(case, batch, case["ctx"], max(1, case["ctx"] // 2)), beams)
        need = -(-lens // page)
        shared = lens // 2 // page
        grow = -(-(lens + case["extra"]) // page)
        stride = int(grow.max()) + 1
        first = np.arange(n) % beams == 0
        mine = np.where(first, need, need - shared)
        pages = int(mine.sum()) + n * (2 + -(-case["extra"] // page)) + 5
        order, tables, at = r.permutation(pages), np.full((n, stride), -1, np.int64), 0
        for i in range(n):
            lo = 0 if first[i] else shared[i]
            if lo:
                tables[i, :lo] = tables[i - i % beams, :lo]
            tables[i, lo:need[i]] = order[at:at + need[i] - lo]
            at += need[i] - lo
        # a selection names the better beams several times and drops others
        parents = (np.arange(n) // beams) * beams + np.floor(r.rand(n) ** 2 * beams).astype(np.int64)
        s |= {"parents": _ints(parents), "extra": _ints(np.full(n, case["extra"]))}
        s["order"] = None
    else:
        n = case["seqs"]
        lens = _spread(case, n, case["ctx"], max(1, case["ctx"] // 2))
        need = -(-lens // page)
        pages = int(need.sum()) + max(1, int(need.sum() * case["spare"]))
        stride = int(need.max()) + 1
        tables = _random_tables(need, pages, stride, seed)
        s |= {"remap": torch.empty(pages, device="cuda", dtype=torch.int32),
              "live": torch.empty(1, device="cuda", dtype=torch.int32)}
    refs = np.bincount(tables[tables >= 0], minlength=pages)
    kt = TYPES[case["kv_type"]][1]
    shape = (case["layers"], pages, page, case["kv_heads"], case["dim"])
    s |= {"pages": pages, "stride": stride, "tables": _ints(tables), "lens": _ints(lens), "refs": _ints(refs),
          "k": _pages(shape, "token", kt, g), "v": _pages(shape, "token", kt, g)}
    s |= {"tables_out": torch.empty_like(s["tables"]), "lens_out": torch.empty_like(s["lens"]),
          "refs_out": torch.empty_like(s["refs"])}
    return s


def op_is(case, op):
    return case["op"] == op


# ------------------------------------------------------------------------------------------------------- plain forms
def _rows_of(s):
    """(sequence, position) of every new token."""
    t = torch.arange(s["T"], device="cuda")
    cu = s["cu"].long()
    seq = torch.searchsorted(cu, t, right=True) - 1
    new = cu[1:] - cu[:-1]
    return seq, s["lens"].long()[seq] - new[seq] + (t - cu[seq])


def _plain_attention(s):
    c = s["case"]
    page, kvh, dim, group = c["page"], c["kv_heads"], c["dim"], c["q_heads"] // c["kv_heads"]
    n, most, ctx = c["seqs"], s["most"], s["ctx"]
    wide = -(-ctx // page)
    ids = s["tables"][:, :wide].long().clamp(min=0)
    inside = (torch.arange(wide * page, device="cuda") < s["lens"].long()[:, None])
    keep = inside[:, :, None, None]
    k = torch.where(keep, s["k"][0][ids].reshape(n, wide * page, kvh, dim).float(), 0.0)
    v = torch.where(keep, s["v"][0][ids].reshape(n, wide * page, kvh, dim).float(), 0.0)
    cu = s["cu"].long()
    new = cu[1:] - cu[:-1]
    i = torch.arange(most, device="cuda")
    at = (cu[:-1, None] + i).clamp(max=s["T"] - 1)
    real = i < new[:, None]
    q = s["q"][at].float().reshape(n, most, kvh, group, dim).permute(0, 2, 3, 1, 4).reshape(n, kvh, group * most, dim)
    score = torch.matmul(q, k.permute(0, 2, 3, 1)).mul_(dim ** -0.5).view(n, kvh, group, most, wide * page)
    pos = (s["lens"].long() - new)[:, None] + i
    j = torch.arange(wide * page, device="cuda")
    seen = (j <= pos[:, :, None]) & inside[:, None, :]
    if c["window"]:
        seen &= j > pos[:, :, None] - c["window"]
    score.masked_fill_(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].view(1, kvh, group, 1, 1)
        top = torch.maximum(top, sink)
    top = torch.where(torch.isinf(top), 0.0, top)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + (sink - top).exp()
    o = torch.matmul(p.view(n, kvh, group * most, wide * page), v.permute(0, 2, 1, 3)).view(n, kvh, group, most, dim)
    o = torch.where(total > 0, o / total, 0.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, most, c["q_heads"], dim)
    s["out"][at[real]] = o[real].to(s["out"].dtype)
    return s["out"]


def _plain_append(s):
    c = s["case"]
    qh, kvh, dim, rot = c["q_heads"], c["kv_heads"], c["dim"], c["rot"]
    seq, pos = _rows_of(s)
    x = s["qkv"].float().view(s["T"], qh + 2 * kvh, dim)
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    r = x[:, : qh + kvh, :rot]
    a, b = (r[..., 0::2], r[..., 1::2]) if c["interleaved"] else (r[..., : rot // 2], r[..., rot // 2:])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([ra, rb], -1).flatten(-2) if c["interleaved"] else torch.cat([ra, rb], -1)
    y = torch.cat([turned, x[:, : qh + kvh, rot:]], -1)
    s["q_out"].copy_(y[:, :qh])
    page = s["tables"][seq, pos // c["page"]].long()
    s["k"][0][page, pos % c["page"]] = y[:, qh:].to(s["k"].dtype)
    s["v"][0][page, pos % c["page"]] = x[:, qh + kvh:].to(s["v"].dtype)
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _plain_beam(s):
    c = s["case"]
    batch, beams, vocab, picks = c["batch"], c["beams"], c["vocab"], c["picks"]
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    lse = (x - top).exp().sum(-1, keepdim=True).log() + top
    score = s["scores"][:, None] + (x - lse)
    if s["done"] is not None:
        kept = torch.where(torch.arange(vocab, device="cuda") == 0, s["scores"][:, None], float("-inf"))
        score = torch.where(s["done"].bool()[:, None], kept, score)
    score = torch.where(torch.isnan(score), float("-inf"), score).view(batch, beams * vocab)
    bits = score.view(torch.int32).long()
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
    key = order * (1 << 32) + (0xFFFFFFFF - torch.arange(beams * vocab, device="cuda"))
    at = 0xFFFFFFFF - (key.topk(picks, -1).values & 0xFFFFFFFF)
    best = score.gather(1, at)
    row = at // vocab + torch.arange(batch, device="cuda")[:, None] * beams
    none = torch.isinf(best)
    return {"scores": best.reshape(-1), "rows": torch.where(none, -1, row).int().reshape(-1),
            "tokens": torch.where(none, -1, at % vocab).int().reshape(-1)}


def _plain_fork(s):
    page, m, stride = s["case"]["page"], s["parents"].numel(), s["stride"]
    lens, tables, refs_in = s["lens"].long(), s["tables"].long(), s["refs"].long()
    j = torch.arange(stride, device="cuda")
    held = j < -(-lens // page)[:, None]
    one = torch.ones(1, device="cuda", dtype=torch.long)
    refs = refs_in.clone()
    gone = tables[held]
    refs.index_add_(0, gone, -one.expand(gone.numel()))
    parents = s["parents"].long()
    named, parent = parents >= 0, parents.clamp(min=0)
    base = torch.where(named, lens[parent], 0)
    full, part = base // page, base % page > 0
    mine = tables[parent]
    kept = mine[j < full[:, None]]
    refs.index_add_(0, kept, one.expand(kept.numel()))
    child = torch.arange(m, device="cuda")
    first = torch.full_like(lens, m).scatter_reduce(0, parent[named], child[named], "amin")
    last = mine.gather(1, full.clamp(max=stride - 1)[:, None])[:, 0].clamp(min=0)
    stays = part & (first[parent] == child) & (refs_in[last] == 1)
    refs.index_add_(0, last[stays], one.expand(int(stays.sum())))
    old = full + stays.long()
    total = torch.where(named, base + s["extra"].long(), 0)
    wants = -(-total // page)
    fresh = wants - old
    starts = fresh.cumsum(0) - fresh
    free = (refs == 0).nonzero()[:, 0]
    new = (j >= old[:, None]) & (j < wants[:, None])
    pick = free[(starts[:, None] + j - old[:, None])[new]]
    refs[pick] = 1
    out = torch.where(j < old[:, None], mine, -1)
    out[new] = pick
    copies = part & ~stays
    src, dst = last[copies], out.gather(1, full.clamp(max=stride - 1)[:, None])[:, 0][copies]
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    return {"refs": refs.int(), "tables": out.int(), "lens": total.int(), "k": s["k"], "v": s["v"]}


def _plain_compact(s):
    page, stride = s["case"]["page"], s["stride"]
    refs, tables = s["refs"].long(), s["tables"].long()
    at = torch.arange(s["pages"], device="cuda")
    live = refs > 0
    count = live.sum()
    holes, movers = (~live & (at < count)).nonzero()[:, 0], (live & (at >= count)).nonzero()[:, 0]
    remap = torch.where(live, at, -1)
    remap[movers] = holes
    s["k"][:, holes] = s["k"][:, movers]
    s["v"][:, holes] = s["v"][:, movers]
    held = torch.arange(stride, device="cuda") < -(-s["lens"].long() // page)[:, None]
    out = torch.where(held, remap[tables.clamp(min=0)], -1)
    after = torch.zeros_like(refs)
    after[remap[live]] = refs[live]
    return {"refs": after.int(), "tables": out.int(), "remap": remap.int(), "live": count.int().view(1), "k": s["k"],
            "v": s["v"]}


PLAIN = {"attention": _plain_attention, "append": _plain_append, "beam": _plain_beam, "fork": _plain_fork,
         "compact": _plain_compact}


# ------------------------------------------------------------------------------------------------------- the library
class _Pool:
    """A pool handle that goes with its state."""

    def __init__(self, capi, s, c):
        self.lib = capi.load()
        k = s["k"]
        strides = (ctypes.c_longlong * 4)(*k.stride()[:4])
        self.h = self.lib.gptoss_kv_pool_create(k.data_ptr(), s["v"].data_ptr(), TYPES[c["kv_type"]][0], k.shape[0],
                                                k.shape[1], c["page"], c["kv_heads"], c["dim"], strides)
        if not self.h:
            raise capi.GptossError(self.lib.gptoss_last_error().decode())

    def __del__(self):
        self.lib.gptoss_kv_pool_destroy(self.h)


def _prepare_own(s):
    at = str(Path.cwd() / "gptoss-infer_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    from gptoss_b200 import capi
    c, P = s["case"], capi.ptr
    o = {"lib": capi.load(), "check": capi.check}
    if c["op"] == "beam":
        o["args"] = (P(s["logits"]), TYPES[c["in_type"]][0], c["vocab"], P(s["scores"]), P(s["done"]), 0, c["batch"],
                     c["beams"], c["vocab"], c["picks"], *(P(t) for t in s["out"]))
        return o
    pool = o["pool"] = _Pool(capi, s, c)
    if c["op"] in ("attention", "append"):
        b = capi.KvBatch(c["seqs"], s["T"], s["most"], s["stride"], P(s["cu"]), P(s["lens"]), P(s["tables"]))
        o["batch"] = b
    if c["op"] == "attention":
        row = c["q_heads"] * c["dim"]
        o["args"] = (pool.h, 0, ctypes.byref(b), P(s["q"]), TYPES[c["q_type"]][0], row, c["q_heads"], P(s["sinks"]),
                     c["dim"] ** -0.5, c["window"], P(s["out"]), row)
    elif c["op"] == "append":
        e, x = TYPES[c["in_type"]][2], P(s["qkv"])
        width, qw, kw = s["qkv"].shape[1], c["q_heads"] * c["dim"], c["kv_heads"] * c["dim"]
        o["args"] = (pool.h, 0, ctypes.byref(b), x, x + qw * e, x + (qw + kw) * e, TYPES[c["in_type"]][0], width, width,
                     c["q_heads"], P(s["cos"]), P(s["sin"]), s["ctx"], c["rot"], int(c["interleaved"]), P(s["q_out"]),
                     TYPES[c["q_type"]][0])
    elif c["op"] == "fork":
        o["args"] = (pool.h, P(s["refs"]), P(s["tables"]), P(s["lens"]), s["lens"].numel(), P(s["parents"]),
                     P(s["extra"]), s["parents"].numel(), s["stride"], P(s["refs_out"]), P(s["tables_out"]),
                     P(s["lens_out"]))
    else:
        o["args"] = (pool.h, P(s["refs"]), P(s["tables"]), P(s["lens"]), s["lens"].numel(), s["stride"],
                     P(s["refs_out"]), P(s["tables_out"]), P(s["remap"]), P(s["live"]))
    return o


def run(s):
    op = s["case"]["op"]
    if not own:
        return PLAIN[op](s)
    lib, stream = s["lib"], torch.cuda.current_stream().cuda_stream
    if op == "attention":
        s["check"](lib.gptoss_paged_attention(*s["args"], stream))
        return s["out"]
    if op == "append":
        s["check"](lib.gptoss_kv_append(*s["args"], stream))
        return {"q": s["q_out"], "k": s["k"], "v": s["v"]}
    if op == "beam":
        s["check"](lib.gptoss_beam_select(*s["args"], stream))
        return dict(zip(("scores", "rows", "tokens"), s["out"]))
    if op == "fork":
        s["check"](lib.gptoss_kv_fork(*s["args"], stream))
        return {"refs": s["refs_out"], "tables": s["tables_out"], "lens": s["lens_out"], "k": s["k"], "v": s["v"]}
    s["check"](lib.gptoss_kv_compact(*s["args"], stream))
    return {"refs": s["refs_out"], "tables": s["tables_out"], "remap": s["remap"], "live": s["live"], "k": s["k"],
            "v": s["v"]}


# ------------------------------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "beam":
        rows = case["batch"] * case["beams"]
        n = rows * case["vocab"]
        return {"bytes": n * TYPES[case["in_type"]][2] + 4 * rows + 12 * case["batch"] * case["picks"], "flops": 4 * n}
    e = TYPES[case["kv_type"]][2]
    if op in ("attention", "append"):
        q, kv = _lengths(case)
        tokens, qh, kvh, dim = int(q.sum()), case["q_heads"], case["kv_heads"], case["dim"]
        if op == "append":
            ins = tokens * (qh + 2 * kvh) * dim * TYPES[case["in_type"]][2] + tokens * case["rot"] * 4
            outs = tokens * qh * dim * TYPES[case["q_type"]][2] + 2 * tokens * kvh * dim * e
            return {"bytes": ins + outs, "flops": 3 * tokens * (qh + kvh) * case["rot"]}
        w = case["window"] or 1 << 40
        seen = sum(int(np.minimum(np.arange(L - n, L) + 1, w).sum()) for n, L in zip(q, kv))
        read = sum(int(min(L, n + w - 1)) for n, L in zip(q, kv))
        moved = 2 * tokens * qh * dim * TYPES[case["q_type"]][2] + 2 * read * kvh * dim * e
        return {"bytes": moved, "flops": 4 * seen * qh * dim}
    page = case["page"]
    size = 2 * case["layers"] * page * case["kv_heads"] * case["dim"] * e
    if op == "fork":
        n = case["batch"] * case["beams"]
        lens = np.repeat(_spread(case, case["batch"], case["ctx"], max(1, case["ctx"] // 2)), case["beams"])
        # about a third of the last pages have to be copied: the rest stay with the first child of their parent
        copies = int((lens % page > 0).sum() * (case["beams"] - 1) / case["beams"] / 2)
        entries = int((-(-lens // page)).sum() + (-(-(lens + case["extra"]) // page)).sum())
        return {"bytes": 2 * copies * size + 4 * entries + 16 * n, "flops": 0}
    lens = _spread(case, case["seqs"], case["ctx"], max(1, case["ctx"] // 2))
    live = int((-(-lens // page)).sum())
    total = live + max(1, int(live * case["spare"]))
    moved = live * (total - live) // total  # pages lie at random: so many of the live ones are past the live count
    return {"bytes": 2 * moved * size + 4 * (3 * total + 2 * live), "flops": 0}


# ------------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    op = case["op"]
    if op in ("fork", "compact"):
        return None  # whole numbers, and pages copied bit for bit
    s = prepare(case, seed)
    if op == "beam":
        rows, picks, vocab = case["beams"], case["picks"], case["vocab"]
        found = []
        for b in range(case["batch"]):
            x = s["logits"][b * rows:(b + 1) * rows].double()
            sc = torch.log_softmax(x, -1) + s["scores"][b * rows:(b + 1) * rows, None].double()
            if s["done"] is not None:
                for r in range(rows):
                    if int(s["done"][b * rows + r]):
                        sc[r] = float("-inf")
                        sc[r, 0] = s["scores"][b * rows + r].double()
            found.append(sc.flatten().sort(descending=True).values[:picks])
        return {"scores": torch.cat(found), "rows": None, "tokens": None}
    q_lens, kv_lens = _lengths(case)
    page, qh, kvh, dim = case["page"], case["q_heads"], case["kv_heads"], case["dim"]
    tables = s["tables"].cpu().long()
    t0 = 0
    if op == "append":
        k, v = s["k"].double(), s["v"].double()
        q = torch.empty(s["T"], qh, dim, device="cuda", dtype=torch.float64)
        half = case["rot"] // 2
        first = torch.arange(half, device="cuda") * (2 if case["interleaved"] else 1)
        second = first + (1 if case["interleaved"] else half)
        for b, (n, L) in enumerate(zip(q_lens, kv_lens)):
            pos = torch.arange(L - n, L)
            x = s["qkv"][t0:t0 + n].double().view(n, qh + 2 * kvh, dim)
            z = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]
            w = torch.complex(x[:, : qh + kvh, first], x[:, : qh + kvh, second]) * z
            y = x.clone()
            y[:, : qh + kvh, first], y[:, : qh + kvh, second] = w.real, w.imag
            q[t0:t0 + n] = y[:, :qh]
            where = tables[b][pos // page].cuda(), (pos % page).cuda()
            k[0][where], v[0][where] = y[:, qh:qh + kvh], y[:, qh + kvh:]
            t0 += n
        return {"q": q, "k": k, "v": v}
    out = torch.zeros(s["T"], qh, dim, device="cuda", dtype=torch.float64)
    for b, (n, L) in enumerate(zip(q_lens, kv_lens)):
        ids = tables[b][: -(-L // page)].cuda()
        k, v = (s[x][0][ids].reshape(-1, kvh, dim)[:L] for x in ("k", "v"))
        pos = torch.arange(L - n, L, device="cuda")[:, None]
        j = torch.arange(L, device="cuda")[None]
        hidden = (j > pos) | (j <= pos - (case["window"] or 1 << 40))
        for h in range(qh):
            a = s["q"][t0:t0 + n, h].double() @ k[:, h * kvh // qh].double().T / math.sqrt(dim)
            a[hidden] = float("-inf")
            if s["sinks"] is not None:
                a = torch.cat([a, s["sinks"][h].double().expand(n, 1)], 1)
            out[t0:t0 + n, h] = torch.softmax(a, 1)[:, :L] @ v[:, h * kvh // qh].double()
        t0 += n
    return out
