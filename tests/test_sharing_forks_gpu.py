"""paged_fork where old rows of one call share more than whole pages: rows that were cut back into pages that others hold too. Against
a simulation in Python; everything equal."""
import random

import pytest
import torch

from test_paged_gpu import D, DEV, ints, ops

pytestmark = pytest.mark.gpu


def fork(refs, table, lens, parents, P):
    """(refs, table, lens, info, copies [(row, from, to, filled rows)]) by the definition: a partly filled page is the first new row's
    that ends in it, where nothing else holds it."""
    width, after = len(table[0]), list(refs)
    for b, n in enumerate(lens):
        for j in range(-(-n // P)):
            after[table[b][j]] -= 1
    for b in parents:
        for j in range(lens[b] // P if b >= 0 else 0):
            after[table[b][j]] += 1
    copy = []
    for b in parents:
        page = table[b][lens[b] // P] if b >= 0 and lens[b] % P else None
        copy.append(page is not None and after[page] != 0)
        if page is not None and not copy[-1]:
            after[page] = 1
    free = [p for p, r in enumerate(after) if r == 0]
    if sum(copy) > len(free):
        return list(refs), [[-1] * width for _ in parents], [0] * len(parents), [sum(copy) - len(free), sum(r == 0 for r in refs)], []
    rows, copies = [], []
    for i, (b, c) in enumerate(zip(parents, copy)):
        row = table[b][:-(-lens[b] // P)] if b >= 0 else []
        if c:
            p = free.pop(0)
            after[p] = 1
            copies.append((i, row[-1], p, lens[b] % P))
            row = row[:-1] + [p]
        rows.append(row + [-1] * (width - len(row)))
    return after, rows, [lens[b] if b >= 0 else 0 for b in parents], [0, len(free)], copies


def check_fork(refs, table, lens, parents, P):
    want = fork(refs, table, lens, parents, P)
    g = torch.Generator(device=DEV).manual_seed(len(parents))
    pools = [torch.randn(2, len(refs), 1, P, D, generator=g, device=DEV).bfloat16() for _ in range(2)]
    expect = [x.clone() for x in pools]
    for x in expect:
        for _, a, b, n in want[4]:
            x[:, b, :, :n] = x[:, a, :, :n]
    k, out = ops(), ints([-9] * len(refs))
    to, lo, info = ints([[-9] * len(table[0])] * len(parents)), ints([-9] * len(parents)), ints([-9, -9])
    k.device_error()
    k.paged_fork(ints(refs), ints(lens), ints(parents), ints(table), to, lo, *pools, refs_out=out, info=info)
    assert k.device_error() == (8 if want[3][0] else 0)
    assert (out.tolist(), to.tolist(), lo.tolist(), info.tolist()) == want[:4]
    assert all(torch.equal(a, b) for a, b in zip(pools, expect))
    r, again = ints(refs), ints([[-9] * len(table[0])] * len(parents))
    k.paged_fork(r, ints(lens), ints(parents), ints(table), again, lo, *pools)      # the counts in place
    assert r.tolist() == want[0] and again.tolist() == want[1]
    k.device_error()
    # no row of the new ones can write into another's page
    ends = [row[n // P] for row, n in zip(want[1], want[2]) if n % P]
    assert len(set(ends)) == len(ends) and all(want[0][p] == 1 for p in ends)


CASES = {   # refs, table, lens, parents: pages of 16
    "two_end_in_one": ([2, 0], [[0], [0]], [5, 5], [0, 1]),
    "the_later_one_first": ([2, 0], [[0], [0]], [5, 9], [1, 0]),
    "both_twice": ([2, 0, 0, 0], [[0], [0]], [5, 9], [0, 1, 1, 0]),
    "one_of_them_ends": ([2, 0], [[0], [0]], [5, 5], [-1, 1]),
    "cut_back_into_a_longer_rows_page": ([2, 1, 0, 0], [[0, -1], [0, 1]], [5, 20], [0, 1]),
    "the_longer_one_ends": ([2, 1, 0], [[0, -1], [0, 1]], [5, 20], [0, 0]),
    "someone_outside_too": ([3, 0, 0], [[0], [0]], [5, 5], [1, 0]),
    "one_page_too_few": ([2, 1], [[0], [0]], [5, 5], [0, 1]),
    "too_few_for_a_longer_row": ([2, 1, 0], [[0, -1], [0, 1]], [5, 20], [0, 1, 0]),
    "full_ones_need_none": ([2], [[0], [0]], [16, 16], [0, 1, 1]),
}


@pytest.mark.parametrize("name", CASES)
def test_rows_that_end_in_one_page(name):
    refs, table, lens, parents = CASES[name]
    check_fork(refs, table, lens, parents, 16)


@pytest.mark.parametrize("rows,spare", [(3, 3), (8, 2), (40, 60), (700, 500), (3000, 3500), (3000, 100)])
def test_any_rows_over_shared_pages(rows, spare):
    """Rows of any length over a few chains of pages, each cut anywhere; parents in any order, some of them several times, some none."""
    rng = random.Random(rows + spare)
    P, width = 16, 6
    chains = max(1, rows // 5)
    pages = list(range(chains * width + spare))
    rng.shuffle(pages)
    chain = [[pages.pop() for _ in range(width)] for _ in range(chains)]
    table = [chain[rng.randrange(chains)] for _ in range(rows)]
    lens = [rng.choice((rng.randrange(width * P + 1), rng.randrange(width + 1) * P)) for _ in range(rows)]
    refs = [0] * (chains * width + spare)
    for row, n in zip(table, lens):
        for p in row[:-(-n // P)]:
            refs[p] += 1
    for p in rng.sample(range(len(refs)), len(refs) // 20):      # sequences outside the call
        refs[p] += 1
    for parents in ([rng.randrange(-1, rows) for _ in range(rows + 2)], list(range(rows)), [-1] * rows, list(range(rows - 1, -1, -2))):
        check_fork(refs, table, lens, parents, P)


def test_many_rows_end_in_one_page():
    n = 5000
    check_fork([n] + [0] * n, [[0]] * n, [1 + i % 15 for i in range(n)], [(7 * i) % n for i in range(n)], 16)
