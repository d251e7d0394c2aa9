"""Paged key/value cache operators against plain 64-bit forms: rotary append, chunk attention, beam selection, fork and
compaction.

Tolerances, from the arithmetic (u = half a unit in the last place, relative: 2^-11 for fp16, 2^-8 for bf16):
  * append: |err| <= u |y| + 2^-22 (|a| + |b|) max|cos, sin| + 2^-25 (fp32 products and one rounding; u = 0 for fp32;
    2^-25: half of fp16's smallest step). Dims that are not rotated, and values: the rounded input, bit for bit.
  * attention, 16-bit: |err| <= u |out| + (u + 1e-5) A, A = sum w |v| / sum w (the output's rounding, the weights'
    rounding for the second product, fp32 statistics); fp32: |err| <= 1e-5 A (two 11-bit parts keep 2^-22 of each
    factor; a score is at most about 16 here, so its error is below 4e-6 and enters the weights twice).
  * beam scores: 1e-5 absolute beside logits of size 10 (fp32 log-sum-exp); rows and tokens equal.
  * pages: bit for bit.
"""
import ctypes

import numpy as np
import pytest
import torch

from gptoss_b200 import capi

pytestmark = pytest.mark.gpu
P = capi.ptr
TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
U = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def lib():
    return capi.load()


def ok(lib, rc):
    assert rc == 0, lib.gptoss_last_error().decode()


def stream():
    return torch.cuda.current_stream().cuda_stream


def ints(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


class Pool:
    def __init__(self, lib, k, v):
        """k, v: [layers, pages, slots, heads, dim] views."""
        self.lib, self.k, self.v = lib, k, v
        self.h = lib.gptoss_kv_pool_create(P(k), P(v), TYPES[k.dtype], k.shape[0], k.shape[1], k.shape[2], k.shape[3],
                                           k.shape[4], (ctypes.c_longlong * 4)(*k.stride()[:4]))
        assert self.h, lib.gptoss_last_error().decode()

    def status(self):
        code = ctypes.c_int(-1)
        ok(self.lib, self.lib.gptoss_kv_pool_status(self.h, ctypes.byref(code)))
        return code.value

    def __del__(self):
        self.lib.gptoss_kv_pool_destroy(self.h)


def make_pages(layers, pages, slots, heads, dim, dtype, head_major, seed, fill=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = (layers, pages, heads, slots, dim) if head_major else (layers, pages, slots, heads, dim)
    def one():
        x = torch.randn(shape, device="cuda", generator=g) if fill is None else torch.full(shape, fill, device="cuda")
        x = x.to(dtype)
        return x.transpose(2, 3) if head_major else x
    return one(), one()


class Setup:
    """Sequences with new tokens and cached lengths over a pool; pages lie in a random order, unused table entries are
    not page ids, and slots no sequence holds are NaN."""

    def __init__(self, lib, new, lens, page, kvh, dim, dtype, head_major=False, seed=0, layers=1):
        r = np.random.RandomState(seed)
        self.new, self.lens, self.page, self.kvh, self.dim = list(new), list(lens), page, kvh, dim
        need = [-(-x // page) for x in lens]
        pages = sum(need) + 2
        order = r.permutation(pages)
        stride = max(need + [0]) + 1
        self.tables = np.full((len(new), stride), 1 << 30, np.int64)
        k, v = make_pages(layers, pages, page, kvh, dim, dtype, head_major, seed, fill=float("nan"))
        g = torch.Generator(device="cuda").manual_seed(seed + 1)
        self.keys, self.values, at = [], [], 0
        for b, n in enumerate(need):
            self.tables[b, :n] = order[at:at + n]
            at += n
            kk = torch.randn(lens[b], kvh, dim, device="cuda", generator=g).to(dtype)
            vv = torch.randn(lens[b], kvh, dim, device="cuda", generator=g).to(dtype)
            pos = torch.arange(lens[b])
            where = torch.tensor(self.tables[b], dtype=torch.long)[pos // page].cuda(), (pos % page).cuda()
            for l in range(layers):
                k[l][where], v[l][where] = kk, vv
            self.keys.append(kk)
            self.values.append(vv)
        self.pool = Pool(lib, k, v)
        self.T = sum(new)
        self.cu, self.dlens, self.dtab = ints(np.cumsum([0] + self.new)), ints(lens), ints(self.tables)
        self.batch = capi.KvBatch(len(new), self.T, max(new + [0]) if isinstance(new, list) else max(new), stride,
                                  P(self.cu), P(self.dlens), P(self.dtab))


def reference_attention(s, q, sinks, scale, window):
    """(out, A) in 64 bits; q [T, heads, dim]."""
    T, H, D = q.shape
    out = torch.zeros(T, H, D, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(out)
    t = 0
    for b, n in enumerate(s.new):
        L = s.lens[b]
        if n and L:
            pos = torch.arange(L - n, L, device="cuda")[:, None]
            j = torch.arange(L, device="cuda")[None]
            seen = (j <= pos) & (j > pos - (window or 1 << 40))
            for h in range(H):
                k, v = s.keys[b][:, h * s.kvh // H].double(), s.values[b][:, h * s.kvh // H].double()
                x = (q[t:t + n, h].double() @ k.T) * scale
                x = torch.where(seen, x, -torch.inf)
                top = x.amax(1, keepdim=True)
                if sinks is not None:
                    top = torch.maximum(top, sinks[h].double())
                top = torch.where(torch.isinf(top), 0.0, top)
                w = (x - top).exp()
                z = w.sum(1, keepdim=True)
                if sinks is not None:
                    z = z + (sinks[h].double() - top).exp()
                z = torch.where(z > 0, z, 1.0)
                out[t:t + n, h], mag[t:t + n, h] = w @ v / z, w @ v.abs() / z
        t += n
    return out, mag


def check_attention(out, want, mag):
    dtype = out.dtype
    bound = U[dtype] * want.abs() + (U[dtype] + 1e-5) * mag + 1e-30
    if dtype == F16:
        bound = bound + 2.0 ** -25
    err = (out.double() - want).abs()
    assert torch.isfinite(out).all()
    worst = (err / bound).max().item() if err.numel() else 0.0
    assert worst <= 1.0, worst


def run_attention(lib, s, q, sinks=None, window=0, scale=None, layer=0, max_new=None, out=None):
    T, H, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    out = torch.full((T, H, D), float("nan"), device="cuda", dtype=q.dtype) if out is None else out
    if max_new is not None:
        s.batch.max_new = max_new
    ok(lib, lib.gptoss_paged_attention(s.pool.h, layer, ctypes.byref(s.batch), P(q), TYPES[q.dtype], q.stride(0), H,
                                       P(sinks), scale, window, P(out), out.stride(0), stream()))
    return out


def new_q(T, H, D, dtype, seed=5):
    return torch.randn(T, H, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


PAIRS = [(F32, F16), (F16, F16), (BF16, BF16)]
SHAPES = [  # new tokens, cached lengths with them
    ([1], [1]), ([1], [2]), ([1], [517]), ([1, 1, 1], [33, 1, 4096]), ([5], [5]), ([3, 0, 1, 7], [64, 9, 65, 300]),
    ([17], [17]), ([40], [1000]), ([129], [129]), ([200, 1, 33], [411, 700, 33]), ([2, 300], [2, 2500]),
]


@pytest.mark.parametrize("pair", PAIRS, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("shape", SHAPES, ids=[f"{sum(a)}of{max(b)}" for a, b in SHAPES])
def test_attention_lengths(lib, shape, dim, pair):
    s = Setup(lib, *shape, page=16, kvh=2, dim=dim, dtype=pair[1], seed=3)
    q = new_q(s.T, 16, dim, pair[0])
    sinks = torch.randn(16, device="cuda")
    out = run_attention(lib, s, q, sinks)
    check_attention(out, *reference_attention(s, q, sinks, dim ** -0.5, 0))
    assert s.pool.status() == 0


@pytest.mark.parametrize("group,kvh", [(1, 1), (1, 3), (3, 2), (7, 2), (8, 1), (16, 1), (20, 1), (71, 1)])
@pytest.mark.parametrize("shape", [([1, 1], [200, 77]), ([9, 70], [90, 203])], ids=["decode", "chunk"])
def test_attention_heads(lib, shape, group, kvh):
    s = Setup(lib, *shape, page=24, kvh=kvh, dim=64, dtype=F16, seed=4)
    q = new_q(s.T, group * kvh, 64, F16)
    out = run_attention(lib, s, q)
    check_attention(out, *reference_attention(s, q, None, 0.125, 0))


@pytest.mark.parametrize("page", [1, 3, 8, 64, 100, 256])
@pytest.mark.parametrize("head_major", [False, True])
@pytest.mark.parametrize("shape", [([1, 1], [260, 129]), ([150, 2], [333, 128])], ids=["decode", "chunk"])
def test_attention_pages(lib, shape, page, head_major):
    s = Setup(lib, *shape, page=page, kvh=2, dim=128, dtype=BF16, head_major=head_major, seed=5, layers=2)
    q = new_q(s.T, 8, 128, BF16)
    out = run_attention(lib, s, q, layer=1)
    check_attention(out, *reference_attention(s, q, None, 128 ** -0.5, 0))


@pytest.mark.parametrize("window", [1, 2, 5, 63, 64, 65, 128, 1000])
@pytest.mark.parametrize("shape", [([1, 1, 1], [1, 130, 700]), ([64, 257, 1], [64, 600, 900])], ids=["decode", "chunk"])
@pytest.mark.parametrize("pair", PAIRS[:2], ids=["f32", "f16"])
def test_attention_window(lib, pair, shape, window):
    s = Setup(lib, *shape, page=16, kvh=2, dim=64, dtype=pair[1], seed=6)
    q, sinks = new_q(s.T, 16, 64, pair[0]), torch.randn(16, device="cuda")
    out = run_attention(lib, s, q, sinks, window)
    check_attention(out, *reference_attention(s, q, sinks, 0.125, window))


@pytest.mark.parametrize("seqs", [31, 32, 33, 130, 300])
@pytest.mark.parametrize("most,window", [(1, 0), (3, 40), (150, 0)])
def test_attention_many_sequences(lib, seqs, most, window):
    """Unequal lengths, some sequences without new tokens, some without positions."""
    r = np.random.RandomState(seqs)
    new = [int(x) for x in r.randint(0, most + 1, seqs)]
    lens = [max(n, int(x)) if x > 20 else 0 for n, x in zip(new, r.randint(0, 500, seqs))]
    s = Setup(lib, new, lens, page=16, kvh=2, dim=64, dtype=F16, seed=seqs)
    q = new_q(s.T, 4, 64, F16)
    out = run_attention(lib, s, q, None, window)
    check_attention(out, *reference_attention(s, q, None, 0.125, window))


def test_attention_window_never_reads_freed_pages(lib):
    """Pages wholly before the window may be freed: their table entries are not read, and no error is flagged."""
    s = Setup(lib, [1, 40], [500, 700], page=16, kvh=2, dim=64, dtype=F16, seed=7)
    t = s.tables.copy()
    t[0, :(500 - 64) // 16] = -1
    t[1, :(660 - 64 + 1) // 16] = -1
    s.dtab.copy_(ints(t))
    q = new_q(s.T, 8, 64, F16)
    out = run_attention(lib, s, q, None, 64)
    check_attention(out, *reference_attention(s, q, None, 0.125, 64))
    assert s.pool.status() == 0


@pytest.mark.parametrize("sinks", [None, 0.5, -float("inf")])
@pytest.mark.parametrize("most", [1, 500])
def test_attention_rows_without_keys_are_zero(lib, sinks, most):
    """A sequence of no positions, and one with fewer positions than new tokens: the rows before position 0 see
    nothing."""
    s = Setup(lib, [2, 12, 1], [0, 5, 30], page=16, kvh=1, dim=64, dtype=F16, seed=8)
    q = new_q(s.T, 8, 64, F16)
    sk = None if sinks is None else torch.full((8,), sinks, device="cuda")
    out = run_attention(lib, s, q, sk, max_new=most)
    want, mag = reference_attention(s, q, sk, 0.125, 0)
    check_attention(out, want, mag)
    assert (out[:2 + 7] == 0).all()


@pytest.mark.parametrize("most", [1, 500])
def test_attention_result_does_not_depend_on_max_new(lib, most):
    """max_new steers the kernel choice only: a wrong value still gives right results."""
    s = Setup(lib, [1, 90, 3], [700, 90, 50], page=16, kvh=2, dim=64, dtype=BF16, seed=9)
    q = new_q(s.T, 16, 64, BF16)
    out = run_attention(lib, s, q, max_new=most)
    check_attention(out, *reference_attention(s, q, None, 0.125, 0))


@pytest.mark.parametrize("pair", PAIRS, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [([1] * 5, [3000, 40, 1, 900, 2000]), ([300, 5], [1500, 1400])], ids=["decode", "chunk"])
def test_attention_strided_rows_repeat_bitwise_and_stay_inside(lib, pair, shape):
    """q inside a fused projection, out inside a wider array: the rest of it is untouched, and a second run gives the
    same bits."""
    s = Setup(lib, *shape, page=16, kvh=4, dim=64, dtype=pair[1], seed=10)
    H, D = 32, 64
    fused = new_q(s.T, H + 8, D, pair[0])
    q = fused[:, 4:4 + H]
    outs = []
    for _ in range(2):
        wide = torch.full((s.T, H + 2, D), 7.0, device="cuda", dtype=pair[0])
        run_attention(lib, s, q, out=wide[:, 1:1 + H])
        assert (wide[:, 0] == 7).all() and (wide[:, -1] == 7).all()
        outs.append(wide[:, 1:1 + H].clone())
    assert torch.equal(outs[0], outs[1])
    check_attention(outs[0], *reference_attention(s, q, None, 0.125, 0))


@pytest.mark.parametrize("pair", PAIRS, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [([1, 1], [900, 50]), ([140], [600])], ids=["decode", "chunk"])
def test_attention_large_scores(lib, pair, shape):
    """Scores of several hundred: one key takes all the weight, nothing overflows."""
    s = Setup(lib, *shape, page=16, kvh=1, dim=64, dtype=pair[1], seed=11)
    q = (new_q(s.T, 8, 64, F32) * 40).to(pair[0])
    out = run_attention(lib, s, q, scale=1.0)
    want, mag = reference_attention(s, q, None, 1.0, 0)
    assert torch.isfinite(out).all()
    # a score of several hundred carries an absolute error of about 700 * 2^-21 (fp32 sums): 1e-3 of the weights
    assert ((out.double() - want).abs() <= 2 * U[pair[0]] * mag + 2e-3 * mag + 2.0 ** -24).all()


@pytest.mark.parametrize("pair", PAIRS, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [([1, 1], [90, 50]), ([140], [300])], ids=["decode", "chunk"])
def test_attention_negative_scale(lib, pair, shape):
    s = Setup(lib, *shape, page=16, kvh=1, dim=64, dtype=pair[1], seed=15)
    q, sinks = new_q(s.T, 8, 64, pair[0]), torch.randn(8, device="cuda")
    check_attention(run_attention(lib, s, q, sinks, scale=-0.1), *reference_attention(s, q, sinks, -0.1, 0))


@pytest.mark.parametrize("dim,page", [(64, 16), (64, 20), (128, 16), (128, 20)])
@pytest.mark.parametrize("window", [0, 100])
def test_attention_chunks_of_many_pieces(lib, dim, page, window):
    """Items cut over several CTAs and CTAs with several items, next to sequences of few rows; twice the same bits."""
    s = Setup(lib, [1, 300, 1, 700, 64, 2, 129], [3000, 5000, 20, 700, 3000, 3000, 1000], page=page, kvh=2, dim=dim,
              dtype=BF16, seed=16)
    q = new_q(s.T, 16, dim, BF16)
    outs = [run_attention(lib, s, q, None, window) for _ in range(3)]
    check_attention(outs[0], *reference_attention(s, q, None, dim ** -0.5, window))
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    assert s.pool.status() == 0


@pytest.mark.parametrize("pair", PAIRS[:2], ids=["f32", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 20])
def test_attention_chunks_by_type_and_page(lib, pair, dim, page):
    """Pages that are and are not multiples of 8 slots, queries of very different sizes from row to row."""
    s = Setup(lib, [150, 1, 333], [900, 300, 333], page=page, kvh=2, dim=dim, dtype=pair[1], seed=17)
    q = new_q(s.T, 6, dim, F32)
    q = (q * torch.logspace(-6, 0, s.T, device="cuda")[:, None, None]).to(pair[0])
    q[::7] = 0
    sinks = torch.randn(6, device="cuda")
    out = run_attention(lib, s, q, sinks)
    check_attention(out, *reference_attention(s, q, sinks, dim ** -0.5, 0))
    assert s.pool.status() == 0


def test_attention_on_another_stream_and_in_a_graph(lib):
    s = Setup(lib, [1, 1], [800, 333], page=16, kvh=8, dim=64, dtype=F16, seed=12)
    q = new_q(s.T, 64, 64, F32)
    want = run_attention(lib, s, q)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = run_attention(lib, s, q)
    side.synchronize()
    assert torch.equal(want, got)
    out = torch.zeros_like(want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run_attention(lib, s, q, out=out)
    for _ in range(2):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(want, out)


def test_attention_bad_tables_are_flagged(lib):
    s = Setup(lib, [1], [100], page=16, kvh=1, dim=64, dtype=F16, seed=13)
    q = new_q(1, 8, 64, F16)
    good = s.dtab.clone()
    s.dtab[0, 2] = -1
    run_attention(lib, s, q)
    assert s.pool.status() == 300
    s.dtab.copy_(good)
    s.dlens.fill_(100000)
    run_attention(lib, s, q, max_new=1)
    assert s.pool.status() != 0
    s.dlens.fill_(100)
    out = run_attention(lib, s, q)
    check_attention(out, *reference_attention(s, q, None, 0.125, 0))
    assert s.pool.status() == 0


@pytest.mark.parametrize("new", [1, 80])
def test_attention_offsets_past_32_bits(lib, new):
    """Pages 40 MB apart: byte offsets of the last ones exceed 2^32."""
    pages, page, L = 120, 16, 100
    k = torch.zeros(pages * 20_000_000 + 2048, device="cuda", dtype=F16)
    kv = k.as_strided((1, pages, page, 1, 64), (0, 20_000_000, 64, 64, 1))
    vv = k.as_strided((1, pages, page, 1, 64), (0, 20_000_000, 64, 64, 1), 1024)
    s = Setup.__new__(Setup)
    s.new, s.lens, s.page, s.kvh, s.dim, s.T = [new], [L], page, 1, 64, new
    s.tables = np.array([[119, 3, 118, 117, 116, 0, 115, 1 << 30]])
    g = torch.Generator(device="cuda").manual_seed(1)
    s.keys = [torch.randn(L, 1, 64, device="cuda", generator=g).half()]
    s.values = [torch.randn(L, 1, 64, device="cuda", generator=g).half()]
    for j in range(L):
        kv[0, s.tables[0, j // page], j % page] = s.keys[0][j]
        vv[0, s.tables[0, j // page], j % page] = s.values[0][j]
    s.pool = Pool(lib, kv, vv)
    s.cu, s.dlens, s.dtab = ints([0, new]), ints([L]), ints(s.tables)
    s.batch = capi.KvBatch(1, new, new, 8, P(s.cu), P(s.dlens), P(s.dtab))
    q = new_q(new, 8, 64, F16)
    check_attention(run_attention(lib, s, q), *reference_attention(s, q, None, 0.125, 0))


def test_attention_masked_nan_and_infinity(lib):
    """Keys outside a row's window or before its position do not reach it, whatever they hold: NaN and infinities in the
    values and keys of positions that only other rows see."""
    s = Setup(lib, [4], [400], page=16, kvh=1, dim=64, dtype=F16, seed=14)
    q = new_q(4, 8, 64, F16)
    want, mag = reference_attention(s, q, None, 0.125, 32)
    kpos, vpos = 399, 398                               # seen by the last row only; by the last two
    for pos, pages, bad in ((kpos, s.pool.k, float("inf")), (vpos, s.pool.v, float("nan"))):
        pages[0, s.tables[0, pos // 16], pos % 16] = bad
    out = run_attention(lib, s, q, None, 32)
    check_attention(out[:2], want[:2], mag[:2])


# --------------------------------------------------------------------------------------------------------- append
def rope_reference(x, cos, sin, rot, interleaved):
    """x [T, heads, dim] in 64 bits, cos/sin [T, rot / 2]; also |a| + |b| per output."""
    y, mag = x.clone(), torch.zeros_like(x)
    half = rot // 2
    i = torch.arange(half, device="cuda")
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    a, b, c, s = x[..., ia], x[..., ib], cos[:, None], sin[:, None]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia] = mag[..., ib] = a.abs() + b.abs()
    return y, mag


@pytest.mark.parametrize("tin", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("tq,tkv", PAIRS, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("rot,interleaved", [(64, False), (64, True), (32, False), (16, True), (24, False), (2, True), (0, False),
                                             (24, True), (8, False), (40, True), (20, False), (56, False)])
def test_append(lib, tin, tq, tkv, rot, interleaved):
    run_append(lib, [1, 0, 9, 3], [70, 5, 9, 33], 16, 2, 64, 8, tin, tq, tkv, rot, interleaved)


@pytest.mark.parametrize("new,lens", [([1], [1]), ([700], [700]), ([1] * 70, list(range(1, 71))), ([9600, 500], [9600, 900])])
@pytest.mark.parametrize("page,head_major,dim", [(1, False, 64), (24, True, 128), (128, False, 128)])
def test_append_lengths_and_pages(lib, new, lens, page, head_major, dim):
    run_append(lib, new, lens, page, 3, dim, 5, BF16, BF16, BF16, dim // 2, True, head_major)


def test_append_unaligned_rows(lib):
    run_append(lib, [5, 2], [40, 20], 16, 2, 64, 4, F16, F16, F16, 64, False, offset=1)


def run_append(lib, new, lens, page, kvh, dim, H, tin, tq, tkv, rot, interleaved, head_major=False, offset=0):
    s = Setup(lib, new, lens, page, kvh, dim, tkv, head_major, seed=20)
    before_k, before_v = s.pool.k.clone(), s.pool.v.clone()
    W = (H + 2 * kvh) * dim
    x = torch.randn(s.T * (W + 8 * offset) + offset, device="cuda").to(tin)
    x = x[offset:].view(s.T, W + 8 * offset)[:, :W] if offset else x.view(s.T, W)
    n_pos = max(lens)
    ang = torch.rand(n_pos, max(rot // 2, 1), device="cuda", dtype=torch.float64) * 6.28
    cos, sin = (1.35 * ang.cos()).float(), (1.35 * ang.sin()).float()
    q_out = torch.full((s.T, H, dim), float("nan"), device="cuda", dtype=tq)
    e = x.element_size()
    ok(lib, lib.gptoss_kv_append(s.pool.h, 0, ctypes.byref(s.batch), P(x), P(x) + H * dim * e,
                                 P(x) + (H + kvh) * dim * e, TYPES[tin], x.stride(0), x.stride(0), H, P(cos), P(sin),
                                 n_pos, rot, int(interleaved), P(q_out), TYPES[tq], stream()))
    assert s.pool.status() == 0
    seq = np.repeat(np.arange(len(new)), new)
    pos = np.concatenate([np.arange(L - n, L) for n, L in zip(new, lens)])
    x3 = x.double().view(s.T, H + 2 * kvh, dim) if not offset else x.double().reshape(s.T, H + 2 * kvh, dim)
    p = torch.tensor(pos, device="cuda")
    y, mag = rope_reference(x3[:, :H + kvh], cos[p].double()[:, :rot // 2], sin[p].double()[:, :rot // 2], rot, interleaved)

    def close(got, want, m):
        u = U[got.dtype]
        assert ((got.double() - want).abs() <= u * want.abs() + 2.0 ** -22 * 1.35 * m + (2.0 ** -25 if u else 0)).all()

    close(q_out, y[:, :H], mag[:, :H])
    where = torch.tensor(s.tables[seq, pos // page], device="cuda"), torch.tensor(pos % page, device="cuda")
    close(s.pool.k[0][where], y[:, H:], mag[:, H:])
    assert torch.equal(s.pool.v[0][where], x3[:, H + kvh:].to(tkv))
    for now, was in ((s.pool.k, before_k), (s.pool.v, before_v)):     # nothing else moved
        now, was = now.clone(), was.clone()
        now[0][where], was[0][where] = 0, 0
        assert torch.equal(now.view(torch.int16), was.view(torch.int16))


def test_append_positions_and_pages_out_of_range_are_flagged(lib):
    s = Setup(lib, [2], [40], 16, 1, 64, F16, seed=21)
    x = torch.randn(2, 10 * 64, device="cuda")
    cos = torch.ones(39, 32, device="cuda")
    q = torch.zeros(2, 8, 64, device="cuda")
    before = s.pool.k.clone()

    def call():
        ok(lib, lib.gptoss_kv_append(s.pool.h, 0, ctypes.byref(s.batch), P(x), P(x) + 8 * 256, P(x) + 9 * 256, 0, 640,
                                     640, 8, P(cos), P(cos), 39, 64, 0, P(q), 0, stream()))
        return s.pool.status()

    assert call() == 303                              # position 39 has no row in the table; position 38 is written
    assert (q[1] == 0).all() and not (q[0] == 0).all()
    s.pool.k.copy_(before)
    s.dlens.fill_(39)
    s.dtab[0, 2] = 10 ** 6
    assert call() == 300
    assert torch.equal(s.pool.k.view(torch.int16), before.view(torch.int16))
    s.dlens.fill_(1)                                  # the first of two new tokens would stand at -1
    assert call() == 303


# --------------------------------------------------------------------------------------------------------- beams
def reference_beams(x, scores, done, token, beams, picks):
    """x [rows, vocab] fp64 numpy."""
    x = np.where(np.isnan(x), -np.inf, x)
    rows, vocab = x.shape
    out = []
    with np.errstate(all="ignore"):
        top = x.max(1, keepdims=True)
        lse = np.log(np.exp(x - top).sum(1, keepdims=True)) + top
        sc = scores[:, None].astype(np.float64) + (x - lse)
    if done is not None:
        for r in np.flatnonzero(done):
            sc[r] = -np.inf
            sc[r, token] = scores[r]
    sc = np.where(np.isnan(sc), -np.inf, sc)
    for b in range(rows // beams):
        flat = sc[b * beams:(b + 1) * beams].reshape(-1)
        at = np.argsort(-flat, kind="stable")[:picks]
        at = np.concatenate([at, np.zeros(max(0, picks - at.size), at.dtype)])
        val = np.where(np.arange(picks) < flat.size, flat[at], -np.inf)
        none = np.isneginf(val)
        out.append((val, np.where(none, -1, at // vocab + b * beams), np.where(none, -1, at % vocab)))
    return [np.stack(o) for o in zip(*out)]


def run_beams(lib, x, scores, done, token, beams, picks, stride=None):
    rows, vocab = x.shape
    batch = rows // beams
    sc, row, tok = (torch.full((batch, picks), 7, device="cuda", dtype=t) for t in (F32, torch.int32, torch.int32))
    ok(lib, lib.gptoss_beam_select(P(x), TYPES[x.dtype], x.stride(0), P(scores), P(done), token, batch, beams, vocab,
                                   picks, P(sc), P(row), P(tok), stream()))
    return [t.cpu().numpy() for t in (sc, row, tok)]


def check_beams(lib, x, scores, done=None, token=0, beams=1, picks=1):
    got = run_beams(lib, x, scores, done, token, beams, picks)
    want = reference_beams(x.double().cpu().numpy(), scores.cpu().numpy(), None if done is None else done.cpu().numpy(),
                           token, beams, picks)
    assert np.array_equal(got[1], want[1]), (got[1], want[1])
    assert np.array_equal(got[2], want[2]), (got[2], want[2])
    live = np.isfinite(want[0])
    assert np.array_equal(np.isneginf(got[0]), np.isneginf(want[0]))
    assert np.abs(got[0][live] - want[0][live]).max(initial=0) <= 1e-5
    again = run_beams(lib, x, scores, done, token, beams, picks)
    assert all(np.array_equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("batch,beams,vocab,picks", [(1, 1, 1, 1), (1, 1, 17, 5), (3, 4, 1000, 8), (2, 5, 8193, 10),
                                                     (1, 64, 515, 64), (2, 8, 201088, 16), (40, 1, 30001, 3),
                                                     (1, 3, 32, 64), (1, 2, 16384, 64)])
def test_beams(lib, dtype, batch, beams, vocab, picks):
    g = torch.Generator(device="cuda").manual_seed(vocab + picks)
    x = (torch.randn(batch * beams, vocab + 3, device="cuda", generator=g) * 2).to(dtype)[:, :vocab]
    check_beams(lib, x, -5 * torch.rand(batch * beams, device="cuda", generator=g), None, 0, beams, picks)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("vocab", [33, 9000, 50001])
def test_beams_ties_go_to_the_lower_index(lib, dtype, vocab):
    x = torch.zeros(4, vocab, device="cuda").to(dtype)
    check_beams(lib, x, torch.zeros(4, device="cuda"), None, 0, 4, 64 if 4 * vocab >= 64 else 8)
    x[:, vocab // 2:] = 1
    x[1] = x[3]
    check_beams(lib, x, torch.tensor([0.0, 1.0, -1.0, 1.0], device="cuda"), None, 0, 2, 7)
    x = (torch.arange(vocab, device="cuda") % 7).to(dtype).repeat(2, 1)
    check_beams(lib, x, torch.zeros(2, device="cuda"), None, 0, 2, 50)


def test_beams_sorted_rows(lib):
    """Ascending and descending rows: every candidate of one row part beats all others."""
    v = torch.arange(20000, device="cuda").float() / 1000
    check_beams(lib, torch.stack([v, v.flip(0)]), torch.tensor([0.0, 0.5], device="cuda"), None, 0, 2, 64)


@pytest.mark.parametrize("vocab", [40, 20000])
def test_beams_masked_and_nan(lib, vocab):
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(6, vocab, device="cuda", generator=g)
    x[0] = -float("inf")
    x[1, 5:] = -float("inf")
    x[2, ::2] = float("nan")
    x[3, 1:] = torch.finfo(F32).min
    x[4] = float("nan")
    s = torch.tensor([0.0, -3.0, -1.0, -2.0, 0.0, -float("inf")], device="cuda")
    check_beams(lib, x, s, None, 0, 6, 32)
    check_beams(lib, x, s, None, 0, 3, 10)
    check_beams(lib, x[:2].contiguous(), s[:2], None, 0, 2, 8)    # five candidates for eight places


@pytest.mark.parametrize("vocab", [12, 9001])
def test_beams_finished_rows(lib, vocab):
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(8, vocab, device="cuda", generator=g)
    s = -torch.rand(8, device="cuda", generator=g)
    done = torch.tensor([1, 0, 0, 0, 1, 1, 1, 1], device="cuda", dtype=torch.uint8)
    check_beams(lib, x, s, done, vocab - 2, 4, 8)
    check_beams(lib, x, s, torch.ones_like(done), 3, 4, 8)
    x[0] = float("nan")
    check_beams(lib, x, s, done, 1, 4, 5)


# --------------------------------------------------------------------------------------------------------- pages
def reference_fork(refs, tables, lens, parents, extra, page, num_pages):
    refs0, refs = list(refs), list(refs)
    for b, L in enumerate(lens):
        for j in range(-(-L // page)):
            refs[tables[b][j]] -= 1
    out, taken, plan = [], set(), []
    for m, par in enumerate(parents):
        base = lens[par] if par >= 0 else 0
        full, t = base // page, [] if par < 0 else list(tables[par])
        keep, src = t[:full], None
        if base % page:
            if par not in taken and refs0[t[full]] == 1:
                keep = t[:full + 1]
            else:
                src = t[full]
        taken.add(par)
        for p in keep:
            refs[p] += 1
        plan.append((list(keep), src, base + (extra[m] if par >= 0 else 0)))
    free = [p for p in range(num_pages) if refs[p] == 0]
    moves, new_lens, short = [], [], False
    for keep, src, total in plan:
        want = -(-total // page)
        while len(keep) < want and free:
            p = free.pop(0)
            refs[p] = 1
            keep.append(p)
            if src is not None:
                moves.append((src, p))
                src = None
        short |= len(keep) < want
        new_lens.append(min(total, len(keep) * page))
        out.append(keep)
    return refs, out, new_lens, moves, short


def run_fork(lib, pool, refs, tables, lens, parents, extra, stride, alias=False):
    r, l = ints(refs), ints(lens)
    t = torch.full((len(lens), stride), 1 << 28, dtype=torch.int32, device="cuda")
    for b, row in enumerate(tables):
        t[b, :len(row)] = ints(row)
    m = len(parents)
    ro = r if alias else torch.full_like(r, 77)
    to, lo = torch.full((m, stride), 77, dtype=torch.int32, device="cuda"), torch.full((m,), 77, dtype=torch.int32, device="cuda")
    p, e = ints(parents), None if extra is None else ints(extra)
    ok(lib, lib.gptoss_kv_fork(pool.h, P(r), P(t), P(l), len(lens), P(p), P(e), m, stride, P(ro), P(to), P(lo), stream()))
    torch.cuda.synchronize()
    return ro.tolist(), to.tolist(), lo.tolist()


def make_sequences(r, seqs, page, most, share, spare):
    """Tables with shared prefixes, their counts, and a pool size."""
    tables, lens, pages = [], [], 0
    ids = list(r.permutation(seqs * (most // page + 2) + spare))
    refs = [0] * len(ids)
    for b in range(seqs):
        L = int(r.randint(0, most + 1))
        need = -(-L // page)
        row = []
        if share and b and r.rand() < 0.7:
            o = int(r.randint(0, b))
            row = tables[o][:min(lens[o] // page, need)]
        row = list(row) + [int(ids.pop()) for _ in range(need - len(row))]
        for p in row:
            refs[p] += 1
        tables.append(row)
        lens.append(L)
    return refs, tables, lens


@pytest.mark.parametrize("seqs,children,page,most,layers", [(1, 1, 16, 40, 1), (4, 4, 16, 1003, 3), (6, 9, 5, 100, 2),
                                                            (40, 70, 64, 900, 2), (3, 1, 1, 30, 1), (8, 0, 16, 200, 1),
                                                            (0, 3, 16, 0, 1), (200, 1300, 16, 60, 1)])
@pytest.mark.parametrize("head_major", [False, True])
def test_fork(lib, seqs, children, page, most, layers, head_major):
    r = np.random.RandomState(seqs * 7 + children)
    refs, tables, lens = make_sequences(r, seqs, page, most, True, 3 * children + 8)
    refs[:2] = [refs[0] + 1, refs[1] + 1]                     # held elsewhere
    parents = [int(r.randint(-1, seqs)) if seqs else -1 for _ in range(children)]
    extra = [int(r.choice([0, 1, 1, page, 2 * page + 1])) for _ in range(children)]
    stride = -(-(most + 2 * page + 1) // page) + 1
    k, v = make_pages(layers, len(refs), page, 2, 64, F16, head_major, 3)
    pool = Pool(lib, k, v)
    wk, wv = k.clone(), v.clone()
    got = run_fork(lib, pool, refs, tables, lens, parents, extra, stride, alias=bool(children % 2))
    want = reference_fork(refs, tables, lens, parents, extra, page, len(refs))
    assert pool.status() == (304 if want[4] else 0)
    assert got[0] == want[0]
    assert got[1] == [t + [-1] * (stride - len(t)) for t in want[1]]
    assert got[2] == want[2]
    for src, dst in want[3]:
        wk[:, dst], wv[:, dst] = wk[:, src].clone(), wv[:, src].clone()
    assert torch.equal(wk, k) and torch.equal(wv, v)


def test_fork_and_compact_of_different_sizes_in_turn(lib):
    """Calls of different sizes on one pool, one after another: what one launch leaves in the workspace (counts, grid-wide
    barriers) has to suit the next."""
    r = np.random.RandomState(5)
    refs, tables, lens = make_sequences(r, 30, 16, 500, False, 700)
    k, v = make_pages(2, len(refs), 16, 2, 64, F16, False, 3)
    pool = Pool(lib, k, v)
    stride = 40
    for children in (1, 200, 3, 60, 7):
        parents = [int(x) for x in r.randint(-1, 30, children)]
        got = run_fork(lib, pool, refs, tables, lens, parents, [1] * children, stride)
        want = reference_fork(refs, tables, lens, parents, [1] * children, 16, len(refs))
        assert pool.status() == (304 if want[4] else 0)
        assert got[0] == want[0] and got[2] == want[2]
        assert got[1] == [t + [-1] * (stride - len(t)) for t in want[1]]
        R, t = ints(refs), ints([row + [-1] * (stride - len(row)) for row in tables])
        remap, live = torch.empty_like(R), ints([0])
        ok(lib, lib.gptoss_kv_compact(pool.h, P(R), P(t), P(ints(lens)), children % 30, stride, P(R), P(t), P(remap),
                                      P(live), stream()))
        assert pool.status() == 0 and live.item() == sum(n > 0 for n in refs)


def test_fork_runs_out_of_pages(lib):
    k, v = make_pages(1, 6, 4, 1, 64, F16, False, 3)
    pool = Pool(lib, k, v)
    refs, tables, lens = [1, 1, 1, 0, 1, 1], [[0, 1, 2]], [10]          # pages 4, 5 held elsewhere; page 3 is free
    got = run_fork(lib, pool, refs, tables, lens, [0, 0, 0], [0, 3, 0], 5)
    want = reference_fork(refs, tables, lens, [0, 0, 0], [0, 3, 0], 4, 6)
    assert want[4] and pool.status() == 304 and pool.status() == 0
    assert got[0] == want[0] and got[2] == want[2] == [10, 12, 8]
    assert got[1] == [t + [-1] * (5 - len(t)) for t in want[1]]


def test_fork_reuses_the_pages_it_frees(lib):
    """All but one beam dropped in a full pool: their pages serve the new children."""
    k, v = make_pages(1, 8, 4, 1, 64, F16, False, 3)
    pool = Pool(lib, k, v)
    refs, tables, lens = [1] * 8, [[0, 1], [2, 3], [4, 5], [6, 7]], [7, 6, 5, 5]
    before = k.clone()
    got = run_fork(lib, pool, refs, tables, lens, [2, 2, 2, 2], None, 3)
    want = reference_fork(refs, tables, lens, [2] * 4, [0] * 4, 4, 8)
    assert got[0] == want[0] and got[2] == [5] * 4 and pool.status() == 0
    for m in range(4):
        assert torch.equal(k[0, got[1][m][1]], before[0, 5]) and got[1][m][0] == 4


def test_fork_flags_bad_parents_and_pages(lib):
    k, v = make_pages(1, 8, 4, 1, 64, F16, False, 3)
    pool = Pool(lib, k, v)
    got = run_fork(lib, pool, [1, 1] + [0] * 6, [[0, 1]], [8], [5, 0], None, 4)
    assert pool.status() == 305 and got[2] == [0, 8]
    run_fork(lib, pool, [1, 1] + [0] * 6, [[0, 99]], [6], [0], None, 4)
    assert pool.status() == 300
    run_fork(lib, pool, [1, 1] + [0] * 6, [[0, 1]], [600], [0], None, 4)
    assert pool.status() != 0


@pytest.mark.parametrize("seqs,page,most,layers,alias", [(1, 16, 30, 1, False), (5, 16, 700, 3, True), (30, 8, 90, 2, False),
                                                         (12, 64, 4000, 1, True), (0, 16, 0, 1, False)])
@pytest.mark.parametrize("head_major", [False, True])
def test_compact(lib, seqs, page, most, layers, alias, head_major):
    r = np.random.RandomState(seqs + page)
    refs, tables, lens = make_sequences(r, seqs, page, most, True, 5)
    stride = -(-most // page) + 2
    k, v = make_pages(layers, len(refs), page, 2, 128, BF16, head_major, 4)
    pool = Pool(lib, k, v)
    before = k.clone(), v.clone()
    t = torch.full((seqs, stride), -5, dtype=torch.int32, device="cuda")
    for b, row in enumerate(tables):
        t[b, :len(row)] = ints(row)
    R, L = ints(refs), ints(lens)
    ro, to = (R, t) if alias else (torch.full_like(R, 77), torch.full_like(t, 77))
    remap, live = torch.full_like(R, 77), torch.full((1,), 77, dtype=torch.int32, device="cuda")
    ok(lib, lib.gptoss_kv_compact(pool.h, P(R), P(t), P(L), seqs, stride, P(ro), P(to), P(remap), P(live), stream()))
    assert pool.status() == 0
    alive = [p for p, n in enumerate(refs) if n > 0]
    holes = [p for p in range(len(alive)) if refs[p] == 0]
    want = {p: p for p in alive if p < len(alive)} | dict(zip([p for p in alive if p >= len(alive)], holes))
    assert remap.tolist() == [want.get(p, -1) for p in range(len(refs))] and live.item() == len(alive)
    after = [0] * len(refs)
    for p in alive:
        after[want[p]] = refs[p]
        assert torch.equal(k[:, want[p]], before[0][:, p]) and torch.equal(v[:, want[p]], before[1][:, p])
    assert ro.tolist() == after
    assert to.tolist() == [[want[p] for p in row] + [-1] * (stride - len(row)) for row in tables]


# --------------------------------------------------------------------------------------------------------- refusals
def test_refusals_with_a_pool(lib):
    k, v = make_pages(2, 4, 16, 2, 64, BF16, False, 1)
    pool = Pool(lib, k, v)
    t = torch.zeros(4096, device="cuda")
    b = capi.KvBatch(1, 2, 2, 1, P(t), P(t), P(t))

    def attention(layer=0, batch=b, q=P(t), type=2, qs=256, heads=4, window=0, out=P(t), os=256, scale=1.0):
        return lib.gptoss_paged_attention(pool.h, layer, batch and ctypes.byref(batch), q, type, qs, heads, None, scale,
                                          window, out, os, None)

    def append(q=P(t), k=P(t), type=2, qs=512, ks=512, heads=4, cos=P(t), n=8, rot=64, qt=2):
        return lib.gptoss_kv_append(pool.h, 0, ctypes.byref(b), q, k, P(t), type, qs, ks, heads, cos, P(t), n, rot, 0,
                                    P(t), qt, None)

    def fork(seqs=1, refs=P(t), children=1, parents=P(t), tables_out=P(t) + 64, lens_out=P(t) + 128):
        return lib.gptoss_kv_fork(pool.h, refs, P(t), P(t), seqs, parents, None, children, 1, P(t) + 256, tables_out,
                                  lens_out, None)

    cases = [
        (lambda: attention(layer=2), b"layer"), (lambda: attention(layer=-1), b"layer"),
        (lambda: attention(batch=None), b"null batch"), (lambda: attention(type=0), b"cache's type"),
        (lambda: attention(type=1), b"cache's type"), (lambda: attention(heads=3), b"multiple"),
        (lambda: attention(heads=0), b"multiple"), (lambda: attention(window=-1), b"window"),
        (lambda: attention(q=None), b"null"), (lambda: attention(out=None), b"null"),
        (lambda: attention(qs=128), b"shorter"), (lambda: attention(q=P(t) + 2), b"aligned"),
        (lambda: attention(os=257), b"aligned"), (lambda: attention(scale=0.0), b"scale"),
        (lambda: attention(scale=float("nan")), b"scale"),
        (lambda: attention(batch=capi.KvBatch(-1, 2, 2, 1, P(t), P(t), P(t))), b"negative"),
        (lambda: attention(batch=capi.KvBatch(1, 2, 2, 1, None, P(t), P(t))), b"null pointer"),
        (lambda: append(type=9), b"type"), (lambda: append(qt=9), b"type"), (lambda: append(rot=63), b"rot_dim"),
        (lambda: append(rot=66), b"rot_dim"), (lambda: append(cos=None), b"cos/sin"), (lambda: append(n=0), b"cos/sin"),
        (lambda: append(k=None), b"null"), (lambda: append(q=None), b"null"), (lambda: append(qs=64), b"q_stride"),
        (lambda: append(ks=64), b"kv_stride"), (lambda: append(n=-1), b"positions"),
        (lambda: fork(refs=None), b"null"), (lambda: fork(parents=None), b"null"), (lambda: fork(seqs=-1), b"negative"),
        (lambda: fork(tables_out=P(t)), b"arrays of their own"), (lambda: fork(lens_out=None), b"null"),
        (lambda: lib.gptoss_kv_compact(pool.h, P(t), P(t), P(t), 1, 1, P(t), P(t), None, P(t), None), b"null"),
        (lambda: lib.gptoss_kv_compact(pool.h, P(t), P(t), P(t), -1, 1, P(t), P(t), P(t), P(t), None), b"out of range"),
        (lambda: lib.gptoss_kv_pool_status(pool.h, None), b"null"),
    ]
    for call, message in cases:
        assert call() == -1
        assert message in lib.gptoss_last_error(), (message, lib.gptoss_last_error())
    empty = capi.KvBatch(0, 0, 0, 0, None, None, None)
    assert attention(batch=empty) == 0
    assert pool.status() == 0
