"""Paged key/value cache operators where they are easily wrong: shared last pages, rows that a few keys dominate, scores
and values that are not finite or very large, lengths and sums near 2^31, zeros of both signs, failed calls and captured
ones. Helpers and tolerances: test_paged_gpu.py."""
import ctypes

import numpy as np
import pytest
import torch

from gptoss_b200 import capi
from test_paged_gpu import (F16, PAIRS, Pool, Setup, U, check_attention, check_beams, lib, make_pages,  # noqa: F401
                            ints, new_q, ok, reference_attention, run_attention, run_beams, run_fork,
                            stream)

pytestmark = pytest.mark.gpu


# --------------------------------------------------------------------------------------------------------- attention
def set_kv(s, b, at, keys=None, values=None):
    """Writes keys and values [n, heads, dim] of positions `at` of sequence b."""
    at = torch.as_tensor(at)
    where = torch.tensor(s.tables[b], dtype=torch.long)[at // s.page].cuda(), (at % s.page).cuda()
    for x, store, mine in ((keys, s.pool.k, s.keys[b]), (values, s.pool.v, s.values[b])):
        if x is not None:
            mine[at.cuda()] = x.to(mine.dtype)
            store[0][where] = x.to(mine.dtype)


@pytest.mark.parametrize("pair", PAIRS, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("new,length,dim,page", [(1, 16384, 64, 16), (1, 131072, 64, 16), (1, 9000, 128, 16),
                                                 (150, 16384, 64, 16), (150, 9000, 128, 20), (40, 131072, 64, 64)])
@pytest.mark.parametrize("rest,spread", [(0.065, 0.3), (1.1e-3, 0.3), (1.1e-3, 0.0)])
def test_attention_beside_a_dominant_key(lib, new, length, dim, page, pair, rest, spread):
    """The first key takes nearly all the weight and has no value (the sink of a long context): the others, `rest` of
    the weight together, make the whole result.

    Bound: as in test_paged_gpu.py (A = sum w |v| / sum w, here about `rest`), and for weights stored as fp16 2^-38 of
    the row's largest weight for each key: fp16 ends at 2^-24, half of that is lost at most, and the largest weight is
    stored as 2^13 or more."""
    s = Setup(lib, [new], [length], page=page, kvh=1, dim=dim, dtype=pair[1], seed=30)
    g = torch.Generator(device="cuda").manual_seed(31)
    sign = torch.where(torch.rand(dim, device="cuda", generator=g) < 0.5, -1.0, 1.0)
    keys = spread * torch.randn(length, 1, dim, device="cuda", generator=g)
    values = torch.randn(length, 1, dim, device="cuda", generator=g) + 0.5
    scale = dim ** -0.5
    keys[0, 0] = sign * (np.log(length / rest) / (dim * scale))
    values[0] = 0
    set_kv(s, 0, np.arange(length), keys, values)
    q = (sign + 0.05 * torch.randn(new, 8, dim, device="cuda", generator=g)).to(pair[0])
    out = run_attention(lib, s, q)
    want, mag = reference_attention(s, q, None, scale, 0)
    u = U[pair[0]]
    bound = u * want.abs() + (u + 1e-5) * mag + (2.0 ** -25 if pair[0] == F16 else 1e-30)
    if pair[1] == F16:
        bound = bound + 2.0 ** -38 * s.values[0].double().abs().sum(0)
    worst = ((out.double() - want).abs() / bound).max().item()
    assert worst <= 1.0, worst


@pytest.mark.parametrize("pair", PAIRS, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 20)])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("power", range(17, 25))
def test_attention_scores_in_the_millions(lib, power, new, dim, page, pair):
    """Scores near 2^power, where fp32 steps by up to 2: a second large key, some tiles on, lies 1 to 4 above the first,
    about the distance at which weights are rescaled. Nothing overflows.

    Bound: a score's rounding (three of them: product, scale, difference) is 3 steps of 2^(power - 22) at most, and the
    first key's share 1 / (1 + exp(difference)) has a slope of 1/4 at most; 0.01 for weights and outputs of 8 bits."""
    n, length = 64, 400
    s = Setup(lib, [new] * n, [length] * n, page=page, kvh=1, dim=dim, dtype=pair[1], seed=41)
    for b in range(n):
        keys, values = torch.zeros(length, 1, dim, device="cuda"), torch.zeros(length, 1, dim, device="cuda")
        keys[[3, 200 + b], 0, 0] = 2048.0
        keys[200 + b, 0, 1] = 1 + b * 3 / 64
        values[3, 0, 0], values[200 + b, 0, 1] = 1.0, 1.0
        set_kv(s, b, np.arange(length), keys, values)
    q = torch.zeros(s.T, 8, dim, device="cuda", dtype=pair[0])
    q[:, :, 0], q[:, :, 1] = 2.0 ** (power - 11), 1.0
    out = run_attention(lib, s, q, scale=1.0)
    assert torch.isfinite(out).all()
    first, later = out[:, :, 0].float(), out[:, :, 1].float()
    assert ((first + later - 1).abs() <= 0.01).all() and (first >= 0).all() and (later >= 0).all()
    above = torch.stack([k[200 + b, 0, 1].double() for b, k in enumerate(s.keys)]).repeat_interleave(new)
    share = (1 / (1 + above.exp())).float()[:, None]
    assert ((first - share).abs() <= 0.01 + 0.75 * 2.0 ** (power - 22)).all()


@pytest.mark.parametrize("pair", PAIRS, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,page", [(64, 16), (64, 20), (128, 16), (128, 20)])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("where", [0, 128])
def test_attention_visible_scores_that_are_not_finite(lib, new, dim, page, pair, where):
    """Sequence b holds a key of NaN, or one with an infinity, at position where + b, which all its rows see and whose
    neighbours none of them masks: a score of NaN or +infinity makes the row NaN, one of -infinity has no weight."""
    n, length = 32, 400
    s = Setup(lib, [new] * n, [length] * n, page=page, kvh=1, dim=dim, dtype=pair[1], seed=40)
    q = new_q(s.T, 8, dim, pair[0])
    good = [k.clone() for k in s.keys]
    for b in range(n):
        set_kv(s, b, [where + b], keys=torch.full((1, 1, dim), float("nan"), device="cuda"))
    assert torch.isnan(run_attention(lib, s, q)).all()
    for b in range(n):
        key = good[b][where + b].clone()
        key[0, 5] = float("inf")
        set_kv(s, b, [where + b], keys=key[None])
    out = run_attention(lib, s, q)
    up = q[:, :, 5] > 0
    assert torch.isnan(out[up]).all()
    if pair[0] == pair[1]:
        for b in range(n):                            # a key far below the others in the place of -infinity
            key = good[b][where + b].float()
            key[0, 5] = 3e4
            s.keys[b][where + b] = key.to(pair[1])
        low = q[:, :, 5].float() < -0.1               # 3e4 * 0.1 / sqrt(dim) below the others: weight 0 in 64 bits too
        want, mag = reference_attention(s, q, None, dim ** -0.5, 0)
        check_attention(out[low], want[low], mag[low])


@pytest.mark.parametrize("pair", PAIRS, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,page", [(64, 16), (64, 20), (128, 16), (128, 20)])
@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("new", [150, 400])
def test_attention_chunks_beside_bad_positions_of_later_rows(lib, new, window, dim, page, pair):
    """NaN and infinities in keys and values that only some rows of a chunk see, alone in a pool (items cut into pieces)
    and with other sequences: the rows that do not see them are right, those that do are not finite."""
    for shape in ([1500], [1500, 700, 1500]):
        news = [new, 33, new][:len(shape)]
        s = Setup(lib, news, shape, page=page, kvh=2, dim=dim, dtype=pair[1], seed=50)
        q = new_q(s.T, 16, dim, pair[0])
        want, mag = reference_attention(s, q, None, dim ** -0.5, window)
        first = 1500 - new
        # (position, its key or its value, what it holds)
        bad = [(first + 20, "v", float("nan")), (first + 77, "k", float("nan")), (first + 103, "v", float("inf")),
               (1499, "k", float("nan"))]
        for pos, what, x in bad:
            held = torch.full((1, 2, dim), x, device="cuda")
            set_kv(s, 0, [pos], **({"keys": held} if what == "k" else {"values": held}))
        out = run_attention(lib, s, q, None, window)
        p = torch.arange(first, 1500, device="cuda")
        sees = torch.zeros(s.T, dtype=torch.bool, device="cuda")
        for pos, *_ in bad:
            sees[:new] |= (p >= pos) & (p - pos < (window or 1 << 30))
        assert 0 < sees.sum() < new
        check_attention(out[~sees], want[~sees], mag[~sees])
        assert not torch.isfinite(out[sees]).any()
        assert s.pool.status() == 0


@pytest.mark.parametrize("page", [16, 20])
def test_attention_chunk_whose_window_begins_behind_bad_positions(lib, page):
    """Positions before the first row's window share its tile (and its page) and hold NaN: no row sees them."""
    s = Setup(lib, [300], [1000], page=page, kvh=1, dim=64, dtype=F16, seed=51)
    q = new_q(300, 8, 64, F16)
    want, mag = reference_attention(s, q, None, 0.125, 77)
    gone = np.arange(701 - 77)                        # position 700's window begins at 624
    nan = torch.full((len(gone), 1, 64), float("nan"), device="cuda")
    set_kv(s, 0, gone, nan, nan)
    check_attention(run_attention(lib, s, q, None, 77), want, mag)


@pytest.mark.parametrize("others", [1, 40])
def test_attention_of_more_than_one_call_counts_is_flagged(lib, others):
    """2^17 new tokens of 8 heads over 2^20 positions, said to be one token: 2^33 groups of 16 keys. That sequence is left
    out and flagged, the others are right."""
    new, L, page = 1 << 17, 1 << 20, 1 << 20
    g = torch.Generator(device="cuda").manual_seed(54)
    k, v = (torch.randn(1, 1, page, 1, 128, device="cuda", generator=g).half() for _ in range(2))
    s = Setup.__new__(Setup)
    s.pool, s.kvh, s.T, s.new, s.lens = Pool(lib, k, v), 1, new + 3 * others, [new] + [3] * others, [L] + [50] * others
    s.cu, s.dlens, s.dtab = ints(np.cumsum([0] + s.new)), ints(s.lens), ints([[0]] * (1 + others))
    s.batch = capi.KvBatch(1 + others, s.T, 1, 1, s.cu.data_ptr(), s.dlens.data_ptr(), s.dtab.data_ptr())
    q = new_q(s.T, 8, 128, F16)
    out = run_attention(lib, s, q)
    assert s.pool.status() == 306
    s.new, s.lens, s.keys, s.values = s.new[1:], s.lens[1:], [k[0, 0, :50]] * others, [v[0, 0, :50]] * others
    check_attention(out[new:], *reference_attention(s, q[new:], None, 128 ** -0.5, 0))


@pytest.mark.parametrize("page", [16, 20])
@pytest.mark.parametrize("most", [1, 500])
@pytest.mark.parametrize("window", [(1 << 31) - 1, (1 << 31) - 3, 1 << 30, 6])
def test_attention_windows_of_any_size_beside_rows_before_position_0(lib, window, most, page):
    """A window longer than every sequence hides nothing, also in tiles whose first rows stand before position 0."""
    s = Setup(lib, [2, 12, 1, 130], [0, 5, 30, 9], page=page, kvh=1, dim=64, dtype=F16, seed=53)
    q = new_q(s.T, 8, 64, F16)
    out = run_attention(lib, s, q, None, window, max_new=most)
    check_attention(out, *reference_attention(s, q, None, 0.125, window))
    assert s.pool.status() == 0


@pytest.mark.parametrize("new", [1, 80])
def test_lengths_up_to_31_bits(lib, new):
    """2048 pages of 2^20 slots that are all one page in memory: 2^31 - 4096 positions are right, more are flagged."""
    page, most, W = 1 << 20, (1 << 31) - 4096, 100
    g = torch.Generator(device="cuda").manual_seed(52)
    k, v = (torch.randn(page, 1, 64, device="cuda", generator=g).half() for _ in range(2))
    k, v = (x.as_strided((1, 2048, page, 1, 64), (0, 0, 64, 64, 1)) for x in (k, v))
    s = Setup.__new__(Setup)
    s.pool, s.T, s.kvh = Pool(lib, k, v), new, 1
    s.cu, s.dlens, s.dtab = ints([0, new]), ints([most]), ints([list(range(2048))])
    s.batch = capi.KvBatch(1, new, new, 2048, s.cu.data_ptr(), s.dlens.data_ptr(), s.dtab.data_ptr())
    q = new_q(new, 8, 64, F16)
    out = run_attention(lib, s, q, None, W)
    assert s.pool.status() == 0
    tail = torch.arange(most - 200, most, device="cuda") % page           # the same sum over the last 200 positions
    s.new, s.lens, s.keys, s.values = [new], [200], [k[0, 0][tail]], [v[0, 0][tail]]
    check_attention(out, *reference_attention(s, q, None, 0.125, W))
    for length in (most + 1, (1 << 31) - 1):
        s.dlens.fill_(length)
        run_attention(lib, s, q, None, W)
        assert s.pool.status() == 301
    # room past 2^31 - 4096 is not given
    refs, lens = ints([0] * 2048), ints([most - 5])
    tables, lens_out, refs_out = torch.empty(1, 2048, dtype=torch.int32, device="cuda"), ints([7]), ints([0] * 2048)
    parent, room = ints([0]), ints([0])
    for extra, want, code in ((5, most, 0), (6, most, 301), ((1 << 31) - 1, most, 301)):
        refs.fill_(1)
        room.fill_(extra)
        ok(lib, lib.gptoss_kv_fork(s.pool.h, refs.data_ptr(), s.dtab.data_ptr(), lens.data_ptr(), 1, parent.data_ptr(),
                                   room.data_ptr(), 1, 2048, refs_out.data_ptr(), tables.data_ptr(), lens_out.data_ptr(),
                                   stream()))
        assert s.pool.status() == code and lens_out.item() == want


@pytest.mark.parametrize("most", [1, 200])
def test_rows_of_no_sequence_are_left_as_they_are(lib, most):
    """A batch padded to more tokens than its sequences have, before the first and behind the last."""
    s = Setup(lib, [1, 100], [30, 120], page=16, kvh=1, dim=64, dtype=F16, seed=56)
    cu = ints([3, 4, 104])
    q, out = new_q(110, 8, 64, F16), torch.full((110, 8, 64), 7.0, device="cuda", dtype=F16)
    s.batch.cu_tokens, s.batch.tokens = cu.data_ptr(), 110
    run_attention(lib, s, q, max_new=most, out=out)
    want, mag = reference_attention(s, q[3:104], None, 0.125, 0)
    check_attention(out[3:104], want, mag)
    assert (out[:3] == 7).all() and (out[104:] == 7).all()
    x, q_out = torch.ones(110, 10 * 64, device="cuda"), torch.full((110, 8, 64), 7.0, device="cuda")
    cos = torch.ones(120, 32, device="cuda")
    p = x.data_ptr()
    ok(lib, lib.gptoss_kv_append(s.pool.h, 0, ctypes.byref(s.batch), p, p + 8 * 256, p + 9 * 256, 0, 640, 640, 8,
                                 cos.data_ptr(), cos.data_ptr(), 120, 64, 0, q_out.data_ptr(), 0, stream()))
    assert (q_out[:3] == 7).all() and (q_out[104:] == 7).all() and (q_out[3:104] != 7).all()
    assert s.pool.status() == 0


def test_status_loses_no_report_of_the_next_call(lib):
    """Reading the status clears it before it returns: what a call on another stream reports right after is kept."""
    s = Setup(lib, [1], [20], page=16, kvh=1, dim=64, dtype=F16, seed=55)
    q, side = new_q(1, 8, 64, F16), torch.cuda.Stream()
    s.dtab.fill_(-1)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(300):
            run_attention(lib, s, q)
            assert s.pool.status() == 300
    assert s.pool.status() == 0


# --------------------------------------------------------------------------------------------------------- pages
def fork_by_rule(refs, tables, lens, parents, extra, page):
    """The header's rule, by whole numbers: (counts, tables, lengths, [(source, destination)], ran short)."""
    refs = list(refs)
    for row, L in zip(tables, lens):
        for p in row[:-(-L // page)]:
            refs[p] -= 1
    for par in parents:
        if par >= 0:
            for p in tables[par][:lens[par] // page]:
                refs[p] += 1
    plan = []
    for m, par in enumerate(parents):
        if par < 0:
            plan.append(([], None, 0))
            continue
        keep, src = list(tables[par][:lens[par] // page]), None
        if lens[par] % page:
            last = tables[par][lens[par] // page]
            if refs[last] == 0:                       # no reference left: it stays with this child
                refs[last] = 1
                keep.append(last)
            else:
                src = last
        plan.append((keep, src, lens[par] + extra[m]))
    free = [p for p, n in enumerate(refs) if n == 0]
    out, out_lens, moves, short = [], [], [], False
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
        out.append(keep)
        out_lens.append(min(total, len(keep) * page))
    return refs, out, out_lens, moves, short


def check_fork(lib, refs, tables, lens, parents, extra, page, stride, layers=2, alias=False):
    k, v = make_pages(layers, len(refs), page, 2, 64, F16, False, 3)
    pool = Pool(lib, k, v)
    was_k, was_v = k.clone(), v.clone()               # every expected page is gathered from here
    got = run_fork(lib, pool, refs, tables, lens, parents, extra, stride, alias)
    want = fork_by_rule(refs, tables, lens, parents, extra, page)
    assert pool.status() == (304 if want[4] else 0)
    assert got[0] == want[0] and got[2] == want[2]
    assert got[1] == [t + [-1] * (stride - len(t)) for t in want[1]]
    src, dst = ([x[i] for x in want[3]] for i in (0, 1))
    assert not set(src) & set(dst)
    wk, wv = was_k.clone(), was_v.clone()
    wk[:, dst], wv[:, dst] = was_k[:, src], was_v[:, src]
    assert torch.equal(wk, k) and torch.equal(wv, v)
    for m, par in enumerate(parents):                 # what a child reads is what its parent held
        for j in range(min(lens[par], got[2][m]) if par >= 0 else 0):
            a, b = got[1][m][j // page], tables[par][j // page]
            assert torch.equal(k[:, a, j % page], was_k[:, b, j % page])
            assert torch.equal(v[:, a, j % page], was_v[:, b, j % page])


@pytest.mark.parametrize("parents", [[0, 1, 2, 3], [3, 1, 2, 0], [1, 1, 3, 3, 0, 2], [0, 2], [2, 0, 2, 0]])
@pytest.mark.parametrize("extra", [0, 1, 5])
def test_fork_of_sequences_that_share_their_last_page(lib, parents, extra):
    """Part-filled last pages held by two sequences each, all holders in the call: no page is overwritten while it is
    copied from."""
    refs = [2, 2] + [0] * 14
    check_fork(lib, refs, [[0], [0], [1], [1]], [3, 3, 3, 3], parents, [extra] * len(parents), 4, 6,
               alias=len(parents) == 2)


def test_fork_shared_last_pages_in_a_full_pool(lib):
    """Every page held: the shared last pages stay, and children that need a page of their own get none."""
    check_fork(lib, [2, 2, 1], [[0], [0], [1], [1]], [3, 3, 2, 2], [0, 2], [0, 0], 4, 2)
    check_fork(lib, [2, 2, 1], [[0], [0], [1], [1]], [3, 3, 2, 2], [0, 1, 2, 3], [0] * 4, 4, 2)


@pytest.mark.parametrize("seed", range(6))
def test_fork_shared_last_pages_at_random(lib, seed):
    """Sequences cut back into pages that others hold (a rollback), in a small pool, children of some of them."""
    r = np.random.RandomState(seed)
    page, seqs = int(r.choice([1, 3, 4, 16])), int(r.randint(2, 40))
    pages = 3 * seqs
    refs, tables, lens = [0] * pages, [], []
    ids = [int(x) for x in r.permutation(pages)]
    for b in range(seqs):
        row = list(tables[int(r.randint(0, b))]) if b and r.rand() < 0.7 else [ids.pop() for _ in range(r.randint(0, 3))]
        L = int(r.randint(0, len(row) * page + 1))
        row = row[:-(-L // page)]
        tables.append(row)
        lens.append(L)
    for row in tables:
        for p in row:
            refs[p] += 1
    for p in r.randint(0, pages, 2):                  # held elsewhere too
        refs[p] += 1
    children = int(r.randint(1, 3 * seqs))
    parents = [int(x) for x in r.randint(-1, seqs, children)]
    check_fork(lib, refs, tables, lens, parents, [int(x) for x in r.randint(0, 3, children)], page, 8)


def test_fork_of_children_that_ask_for_more_than_31_bits_of_pages(lib):
    """600 children of 2^22 pages each in a pool of five free ones: the first gets those, the others none."""
    n, room = 600, 1 << 22
    k, v = make_pages(1, 6, 1, 1, 64, F16, False, 3)
    pool = Pool(lib, k, v)
    refs, tables, lens = ints([0, 0, 1, 0, 0, 0]), torch.full((1, room), 2, dtype=torch.int32, device="cuda"), ints([1])
    out, lens_out = (torch.empty(shape, dtype=torch.int32, device="cuda") for shape in ((n, room), (n,)))
    parents, extra = ints([0] * n), ints([room - 1] * n)
    ok(lib, lib.gptoss_kv_fork(pool.h, refs.data_ptr(), tables.data_ptr(), lens.data_ptr(), 1, parents.data_ptr(),
                               extra.data_ptr(), n, room, refs.data_ptr(), out.data_ptr(), lens_out.data_ptr(), stream()))
    assert pool.status() == 304
    assert lens_out.tolist() == [6] + [1] * (n - 1) and refs.tolist() == [1, 1, n, 1, 1, 1]
    assert out[0, :7].tolist() == [2, 0, 1, 3, 4, 5, -1] and (out[:, 0] == 2).all() and (out[1:, 1:] == -1).all()


def test_fork_empty_children_get_no_pages(lib):
    """Parent -1: length 0 and no pages whatever its extra says; the next call gives the room. Negative extras count as
    none."""
    check_fork(lib, [1, 1] + [0] * 6, [[0, 1]], [6], [-1, 0, -1], [5, 3, 9], 4, 4)
    k, v = make_pages(1, 8, 4, 2, 64, F16, False, 3)
    pool = Pool(lib, k, v)
    got = run_fork(lib, pool, [0] * 8, [], [], [-1, -1], [5, 9], 4)
    assert got == ([0] * 8, [[-1] * 4] * 2, [0, 0])
    got = run_fork(lib, pool, got[0], [[], []], [0, 0], [0, 1], [5, -9], 4)
    assert got[1:] == ([[0, 1, -1, -1], [-1] * 4], [5, 0]) and pool.status() == 0


def test_fork_refuses_null_lengths_and_tables(lib):
    """Lengths are read for every parent, also where tables have no columns."""
    k, v = make_pages(1, 4, 4, 1, 64, F16, False, 3)
    pool, t = Pool(lib, k, v), torch.zeros(64, dtype=torch.int32, device="cuda")
    p = t.data_ptr()
    for tables, lens, stride in ((None, None, 0), (p, None, 0), (p, None, 1), (None, p, 1)):
        rc = lib.gptoss_kv_fork(pool.h, p, tables, lens, 1, p, None, 1, stride, p + 64, p + 128, p + 192, None)
        assert rc == -1 and b"null tables or lengths" in lib.gptoss_last_error()
    assert lib.gptoss_kv_fork(pool.h, p, None, p, 1, p, None, 1, 0, p + 64, None, p + 192, None) == 0
    assert pool.status() == 0 and (t == 0).all()


# --------------------------------------------------------------------------------------------------------- beams
def test_beams_captured_before_the_workspace_grows(lib):
    """A graph of a small selection gives the same picks after larger calls of the same thread, in memory that other
    tensors have been given meanwhile."""
    g = torch.Generator(device="cuda").manual_seed(60)
    x, scores = torch.randn(6, 40000, device="cuda", generator=g), -torch.rand(6, device="cuda", generator=g)
    want = run_beams(lib, x, scores, None, 0, 3, 5)
    out = [torch.zeros(10, dtype=t, device="cuda") for t in (torch.float32, torch.int32, torch.int32)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert lib.gptoss_beam_select(x.data_ptr(), 0, 40000, scores.data_ptr(), None, 0, 2, 3, 40000, 5,
                                      *(t.data_ptr() for t in out), torch.cuda.current_stream().cuda_stream) == 0
    for rows in (64, 256, 1024, 4096):
        y = torch.randn(rows, 20000, device="cuda", generator=g)
        z = torch.zeros(rows, device="cuda")
        first = run_beams(lib, y, z, None, 0, 64, 64)
        filler = [torch.full((1 << 18,), -1, device="cuda", dtype=torch.int32) for _ in range(64)]
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            assert all(np.array_equal(a.cpu().numpy(), b.reshape(-1)) for a, b in zip(out, want))
        assert all((f == -1).all() for f in filler)
        assert all(np.array_equal(a, b) for a, b in zip(first, run_beams(lib, y, z, None, 0, 64, 64)))


@pytest.mark.parametrize("dtype", [torch.float32, F16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [17, 9000, 50001])
def test_beams_zeros_of_both_signs_are_equal(lib, dtype, vocab):
    """-0.0 and +0.0 are equal scores: the lower token wins, within a part of a row, between parts and between rows."""
    x = torch.zeros(4, vocab, device="cuda", dtype=dtype)
    x[:, 0] = -0.0
    check_beams(lib, x, torch.zeros(4, device="cuda"), None, 0, 1, 1)
    x[:, ::2] = -0.0
    check_beams(lib, x, torch.zeros(4, device="cuda"), None, 0, 2, 12)
    x[:] = -0.0
    x[:, vocab // 2:] = 0.0
    check_beams(lib, x, torch.tensor([-0.0, 0.0, 0.0, -0.0], device="cuda"), None, 0, 4, 40)
    x[:, 3:] = -1.0
    x[2, 1] = 0.0
    check_beams(lib, x, torch.zeros(4, device="cuda"), None, 0, 4, 9)


def test_a_failed_allocation_does_not_fail_the_next_call(lib):
    """A selection whose workspace (4 TB) cannot be had is refused; the next calls run."""
    x, s, wide = torch.randn(2, 1000, device="cuda"), torch.zeros(2, device="cuda"), (1 << 25) - 1
    k, v = make_pages(1, 4, 4, 1, 64, F16, False, 3)
    pool, t = Pool(lib, k, v), torch.zeros(64, dtype=torch.int32, device="cuda")
    p = t.data_ptr()
    for _ in range(2):
        assert lib.gptoss_beam_select(x.data_ptr(), 0, wide, s.data_ptr(), None, 0, 1 << 16, 64, wide, 64, p, p, p,
                                      stream()) == -1
        assert b"memory" in lib.gptoss_last_error()
        check_beams(lib, x, s, None, 0, 2, 5)
    cu, one, q, out = ints([0, 1]), ints([1]), new_q(1, 8, 64, F16), new_q(1, 8, 64, F16)
    b = capi.KvBatch(1, 1, 1, 1, cu.data_ptr(), one.data_ptr(), p)
    assert lib.gptoss_beam_select(x.data_ptr(), 0, wide, s.data_ptr(), None, 0, 1 << 16, 64, wide, 64, p, p, p,
                                  stream()) == -1
    t.zero_()
    ok(lib, lib.gptoss_paged_attention(pool.h, 0, ctypes.byref(b), q.data_ptr(), 1, 512, 8, None, 0.125, 0,
                                       out.data_ptr(), 512, stream()))
    assert pool.status() == 0 and torch.equal(out, v[0, 0, 0].expand(1, 8, 64))
