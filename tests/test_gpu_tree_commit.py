"""Committing the accepted path of drafted trees (ec_tree_commit) and copying rows between slots (ec_kv_copy), against numpy
on the host: rows and numbers equal, everything else untouched."""
from __future__ import annotations

import numpy as np
import pytest

import edgecore_b200 as ec

pytestmark = pytest.mark.gpu


class Arena:
    def __init__(self, torch, layers, dim, slots, per, seed, dtype=None, spare=3):
        self.torch = torch
        self.rs = np.random.RandomState(seed)
        self.pages = slots * per + spare
        self.table = self.rs.permutation(self.pages)[: slots * per].reshape(slots, per).astype(np.int32)
        g = torch.Generator().manual_seed(seed)
        dtype = dtype or torch.float16
        self.k, self.v = (torch.randn(layers, self.pages, 64, dim, generator=g).to(dtype).cuda() for _ in range(2))
        self.layers, self.dim = layers, dim

    def host(self):
        return [x.view(self.torch.int16).cpu().numpy().reshape(self.layers, -1, self.dim).copy() for x in (self.k, self.v)]

    def at(self, slot, p):
        return int(self.table[slot, p // 64]) * 64 + p % 64

    def dev(self, a, t=np.int32):
        return self.torch.from_numpy(np.ascontiguousarray(np.asarray(a).astype(t))).cuda()


def walk(parents, tokens, picked, most):
    path, here = [], 0 if len(parents) else None
    while here is not None and len(path) < most:
        path.append(here)
        here = next((c for c in range(here + 1, len(parents)) if parents[c] == path[-1] and tokens[c] == picked[path[-1]]), None)
    return path


def commit(a, trees, bases, most, slots=None, in_place=False):
    """trees: (parents, tokens, picked) each."""
    words = max([1] + [-(-len(t[0]) // 64) for t in trees])
    start = np.cumsum([0] + [len(t[0]) for t in trees])
    mask = np.zeros((max(1, start[-1]), words), np.uint64)
    for b, t in enumerate(trees):
        if len(t[0]):
            m = ec.tree_mask(t[0]).view(np.uint64)
            mask[start[b]:start[b + 1], : m.shape[1]] = m
    slots = list(range(len(trees))) if slots is None else slots
    n = len(trees)
    want = a.host()
    acc, cnt = np.full((n, most), -1), np.zeros(n, int)
    for b, t in enumerate(trees):
        path = walk(*t, most)
        cnt[b] = len(path)
        for step, node in enumerate(path):
            acc[b, step] = t[2][node]
            for x in want:
                x[:, a.at(slots[b], bases[b] + step)] = x[:, a.at(slots[b], bases[b] + node)]
    cat = lambda i: a.dev(np.concatenate([np.asarray(t[i], int) for t in trees] or [[0]]))  # noqa: E731
    base = a.dev(bases)
    out = [a.dev(np.full((n, most), -9)), a.dev(np.full(n, -9)), base if in_place else a.dev(np.full(n, -9))]
    ec.tree_commit(a.k, a.v, a.dev(a.table), a.dev(start), base, a.dev(mask.view(np.int64), np.int64), cat(1), cat(2), *out, slots=a.dev(slots))
    a.torch.cuda.synchronize()
    assert ec.device_error_take() == 0
    got = a.host()
    assert (out[0].cpu().numpy() == acc).all()
    assert (out[1].cpu().numpy() == cnt).all()
    assert (out[2].cpu().numpy() == np.array(bases) + cnt).all()
    for x, y in zip(got, want):
        assert (x == y).all()
    return cnt


def random_tree(rs, n, alphabet=3, back=7):
    parents = [-1] + [int(rs.randint(max(0, i - back), i)) for i in range(1, n)]
    return parents[:n], rs.randint(0, alphabet, n), rs.randint(0, alphabet, n)


@pytest.mark.parametrize("layers,dim", [(1, 8), (3, 128), (2, 72), (5, 1024), (12, 768)])
@pytest.mark.parametrize("nodes", [1, 2, 17, 64, 65, 200])
def test_random_trees(cuda, layers, dim, nodes):
    a = Arena(cuda, layers, dim, 4, 6, seed=dim + nodes)
    trees = [random_tree(a.rs, nodes) for _ in range(4)]
    commit(a, trees, [0, 37, 63, 130], 40, slots=[2, 0, 3, 1])


def test_long_chain_with_gaps_moves_every_row(cuda):
    """A path of every second node, longer than a page: each row moves, onto rows that are read before."""
    a = Arena(cuda, 2, 256, 1, 8, seed=1)
    n = 300
    parents = [-1] + [max(0, i - 2) if i % 2 == 0 else 0 for i in range(1, n)]
    tokens = np.arange(n)
    picked = np.arange(n) + 2
    cnt = commit(a, [(parents, tokens, picked)], [50], 300)
    assert cnt[0] == 150


def test_most_nodes_empty_trees_and_equal_siblings(cuda):
    a = Arena(cuda, 2, 64, 5, 3, seed=2)
    chain = ([-1, 0, 1, 2, 3], [5, 6, 7, 8, 9], [6, 7, 8, 9, 4])
    twins = ([-1, 0, 0, 1, 2], [1, 4, 4, 8, 3], [4, 8, 3, 0, 0])       # both siblings match: the first is taken
    none = ([-1, 0, 0], [1, 2, 3], [7, 7, 7])
    assert commit(a, [chain, ([], [], []), twins, none, ([], [], [])], [10, 0, 62, 100, 7], 3).tolist() == [3, 0, 3, 1, 0]
    a = Arena(cuda, 2, 64, 5, 3, seed=3)
    assert commit(a, [chain, ([], [], []), twins, none, chain], [10, 0, 62, 100, 7], 1).tolist() == [1, 0, 1, 1, 1]
    a = Arena(cuda, 2, 64, 5, 3, seed=3)
    assert commit(a, [chain, ([], [], []), twins, none, chain], [10, 0, 62, 100, 7], 9, in_place=True).tolist() == [5, 0, 3, 1, 5]


def test_many_sequences_and_other_strides(cuda):
    a = Arena(cuda, 4, 128, 150, 2, seed=4)
    commit(a, [random_tree(a.rs, int(a.rs.randint(1, 30)), alphabet=2) for _ in range(150)], a.rs.randint(0, 60, 150).tolist(), 30, slots=a.rs.permutation(150).tolist())
    # K and V side by side in one pool
    both = cuda.randn(3, 7, 64, 2, 64, device="cuda").half()
    a = Arena(cuda, 3, 64, 2, 3, seed=5, spare=1)
    both[:, :, :, 0], both[:, :, :, 1] = a.k, a.v
    a.k, a.v = both[:, :, :, 0], both[:, :, :, 1]
    a.host = lambda: [x.contiguous().view(cuda.int16).cpu().numpy().reshape(3, -1, 64).copy() for x in (a.k, a.v)]
    commit(a, [random_tree(a.rs, 20, 2), random_tree(a.rs, 33, 2)], [3, 90], 20)


def test_commit_reports_bad_indices(cuda):
    a = Arena(cuda, 2, 64, 2, 2, seed=6)
    before = a.host()
    chain = ec.tree_mask([-1, 0, 0])
    for slots, bases, start in (([0, 2], [0, 0], [0, 3, 6]), ([0, -1], [0, 0], [0, 3, 6]), ([0, 1], [0, 126], [0, 3, 6]), ([0, 1], [0, -1], [0, 3, 6]), ([0, 1], [0, 0], [0, 3, 7])):
        out = [a.dev(np.full((2, 4), -9)), a.dev([-9, -9]), a.dev([-9, -9])]
        ec.tree_commit(a.k, a.v, a.dev(a.table), a.dev(start), a.dev(bases), a.dev(np.concatenate([chain, chain]), np.int64), a.dev([1, 2, 3] * 2), a.dev([9] * 6), *out,
                       slots=a.dev(slots))
        assert ec.device_error_take() == 2
        assert out[1].cpu().tolist() == [1, 0] and out[2].cpu().tolist() == [1, bases[1]]
        assert out[0].cpu().tolist() == [[9, -1, -1, -1], [-1] * 4]
    for x, y in zip(a.host(), before):
        assert (x == y).all()


@pytest.mark.parametrize("layers,dim", [(1, 8), (3, 128), (2, 72), (12, 768)])
@pytest.mark.parametrize("start,end", [(0, 0), (0, 1), (5, 6), (0, 64), (63, 65), (10, 200), (64, 320)])
def test_copy(cuda, layers, dim, start, end):
    a = Arena(cuda, layers, dim, 5, 5, seed=dim + end)
    want = a.host()
    for d in (0, 3, 4):
        for p in range(start, end):
            for x in want:
                x[:, a.at(d, p)] = x[:, a.at(2, p)]
    ec.kv_copy(a.k, a.v, a.dev(a.table), a.dev([2] * 3), a.dev([0, 3, 4]), a.dev([start] * 3), a.dev([end] * 3))
    assert ec.device_error_take() == 0
    for x, y in zip(a.host(), want):
        assert (x == y).all()


def test_copy_jobs_of_their_own_ranges(cuda):
    """One slot fed from two others at ranges that do not meet, a chain whose ranges do not meet, an empty and a reversed range."""
    a = Arena(cuda, 2, 64, 6, 4, seed=8)
    jobs = [(0, 1, 0, 70), (2, 1, 70, 256), (1, 3, 256, 256), (3, 4, 9, 3), (4, 5, 100, 130), (5, 4, 130, 200)]
    want = a.host()
    for s, d, lo, hi in jobs:
        for p in range(lo, hi):
            for x in want:
                x[:, a.at(d, p)] = x[:, a.at(s, p)]
    ec.kv_copy(a.k, a.v, a.dev(a.table), *(a.dev(c) for c in zip(*jobs)))
    assert ec.device_error_take() == 0
    for x, y in zip(a.host(), want):
        assert (x == y).all()


def test_copy_refuses_jobs_that_meet(cuda):
    a = Arena(cuda, 2, 64, 6, 4, seed=9)
    good = (0, 1, 0, 100)
    for bad in ([(2, 3, 0, 50), (4, 3, 49, 60)], [(2, 3, 0, 50), (3, 4, 49, 60)], [(2, 2, 0, 5)], [(2, 6, 0, 5)], [(-1, 2, 0, 5)], [(2, 3, 0, 257)], [(2, 3, -1, 5)],
                [(2, 3, 5, 9), (2, 3, 5, 9)]):
        jobs = [good] + bad
        want = a.host()
        for p in range(100):
            for x in want:
                x[:, a.at(1, p)] = x[:, a.at(0, p)]
        ec.kv_copy(a.k, a.v, a.dev(a.table), *(a.dev(c) for c in zip(*jobs)))
        assert ec.device_error_take() == 2, bad
        for x, y in zip(a.host(), want):
            assert (x == y).all(), bad


def test_copy_with_an_unmapped_page(cuda):
    a = Arena(cuda, 2, 64, 3, 4, seed=10)
    a.table[1, 1] = -1
    want = a.host()
    for p in list(range(0, 64)) + list(range(128, 200)):
        for x in want:
            x[:, a.at(1, p)] = x[:, a.at(0, p)]
    ec.kv_copy(a.k, a.v, a.dev(a.table), a.dev([0]), a.dev([1]), a.dev([0]), a.dev([200]))
    assert ec.device_error_take() == 2
    for x, y in zip(a.host(), want):
        assert (x == y).all()


@pytest.mark.parametrize("back,step", [(3, 2), (700, 1), (1500, 150)])
def test_trees_of_many_nodes(cuda, back, step):
    """Paths that go on after gaps of one node, of some hundred, and of more than the nodes a block holds."""
    a = Arena(cuda, 2, 72, 2, 30, seed=11)
    trees = []
    for _ in range(2):
        parents, tokens, picked = random_tree(a.rs, 1700, 50, back)
        node = 0
        while True:                      # a path that reaches the last nodes
            to = [c for c in range(node + 1, min(1700, node + 2 * step + 1)) if c - node >= min(step, 1699 - node)]
            if not to:
                break
            child = to[int(a.rs.randint(len(to)))]
            parents[child], tokens[child] = node, picked[node]
            node = child
        trees.append((parents, tokens, picked))
    assert min(commit(a, trees, [0, 99], 900, slots=[1, 0])) > 1


def test_copies_of_many_jobs(cuda):
    """More jobs than a block judges at a time: forks of two sources in groups, ranges of their own, bad ones among them."""
    a = Arena(cuda, 2, 24, 310, 2, seed=12)
    jobs = [(0, d, 3, 100) for d in range(2, 150)] + [(1, d, 0, 64) for d in range(150, 280)] + [(1, d, d - 280, 90) for d in range(280, 305)]
    jobs = [jobs[i] for i in a.rs.permutation(len(jobs))]
    bad = [(0, 400, 3, 100), (0, 0, 3, 100), (-1, 305, 0, 9)]
    want = a.host()
    for s, d, lo, hi in jobs:
        for p in range(lo, hi):
            for x in want:
                x[:, a.at(d, p)] = x[:, a.at(s, p)]
    for extra in ([], bad):
        ec.kv_copy(a.k, a.v, a.dev(a.table), *(a.dev(c) for c in zip(*(extra + jobs))))
        assert ec.device_error_take() == (2 if extra else 0)
    for x, y in zip(a.host(), want):
        assert (x == y).all()


@pytest.mark.parametrize("many", [0, 300])
def test_copy_refused_jobs_do_not_stop_others(cuda, many):
    """A job that is refused for itself (a bad slot or range, its own source) writes and reads nothing, so it meets nobody."""
    a = Arena(cuda, 2, 24, 10 + many, 2, seed=13)
    good = [(0, 1, 0, 100), (0, 2, 0, 100), (3, 4, 7, 120)] + [(0, 10 + i, 0, 100) for i in range(many)]
    bad = [(0, 0, 0, 100), (-1, 1, 0, 100), (3, 10 + many, 7, 120), (10 + many, 4, 0, 128), (3, 4, -5, 100), (1, 0, 0, 129), (4, 4, 7, 120)]
    jobs = bad + good
    want = a.host()
    for s, d, lo, hi in good:
        for p in range(lo, hi):
            for x in want:
                x[:, a.at(d, p)] = x[:, a.at(s, p)]
    ec.kv_copy(a.k, a.v, a.dev(a.table), *(a.dev(c) for c in zip(*jobs)))
    assert ec.device_error_take() == 2
    for x, y in zip(a.host(), want):
        assert (x == y).all()


def test_copy_skips_both_of_two_jobs_that_meet(cuda):
    """A chain 0 -> 1 -> 2 over common positions: neither is done, whichever comes first; a third job goes on."""
    for jobs in ([(0, 1, 0, 90), (1, 2, 60, 120)], [(1, 2, 60, 120), (0, 1, 0, 90)]):
        a = Arena(cuda, 2, 64, 6, 4, seed=14)
        want = a.host()
        for p in range(64):
            for x in want:
                x[:, a.at(5, p)] = x[:, a.at(0, p)]
        ec.kv_copy(a.k, a.v, a.dev(a.table), *(a.dev(c) for c in zip(*(jobs + [(0, 5, 0, 64)]))))
        assert ec.device_error_take() == 2
        for x, y in zip(a.host(), want):
            assert (x == y).all()
