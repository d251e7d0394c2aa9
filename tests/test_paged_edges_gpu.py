"""Paged key/value cache operators where they are easily wrong: shared last pages, rows that a few keys dominate, values
that are not finite, zeros of both signs. Helpers and tolerances: test_paged_gpu.py."""
import numpy as np
import pytest
import torch

from test_paged_gpu import F16, Pool, lib, make_pages, run_fork  # noqa: F401

pytestmark = pytest.mark.gpu


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
