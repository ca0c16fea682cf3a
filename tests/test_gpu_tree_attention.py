"""Attention of drafted-token trees over a paged arena (ec_tree_attention) against the formula in 64 bits.

The bound of a value, from the arithmetic the operator documents (scores, weights and sums in 32 bits, q of 16 bits exact,
fp32 q in two 16-bit parts or exact, with 16-bit q the weights rounded to the cache's type):
  a score is a sum of hd products in 32 bits, off by at most (hd + 8) 2^-23 of the sum of their magnitudes (twice the
  rounding bound, since a tensor-core sum may truncate) and 2^-20 of it for the two parts of an fp32 q; its distance to
  the maximum is rounded once more, 2^-23 of it; a weight is off by that much of itself plus 2^-21 for exp, and both the
  numerator and the denominator of out = sum w v / sum w move by it: twice the largest, times sum w |v| / sum w;
  a weight rounded to 16 bits moves by half a step, 2^-11 or 2^-8 of itself (fp32 q: in two parts, 2^-20), and an fp16
  weight below 2^-14 by at most 2^-25, a part that the largest weight 1 bounds by n 2^-25 max |v|;
  sums over n keys in 32 bits: n 2^-24 at worst, taken as 2^-20 + n 2^-24 / 8 (tree and tile order);
  the result is rounded to its type once, half a step."""
from __future__ import annotations

import math

import numpy as np
import pytest

import edgecore_b200 as ec

pytestmark = pytest.mark.gpu

HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def _types(torch):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


class Case:
    """A batch of trees over a shuffled arena whose unused rows hold NaN."""

    def __init__(self, torch, q="f16", kv="f16", heads=4, kv_heads=2, hd=64, sizes=(5,), bases=(100,), window=0, seed=0, mask=None,
                 words=None, spare_pages=2, q_gain=1.0):
        rs = np.random.RandomState(seed)
        ty = _types(torch)
        self.torch, self.qt, self.kt, self.heads, self.kvh, self.hd, self.window = torch, q, kv, heads, kv_heads, hd, window
        self.sizes, self.bases = list(sizes), list(bases)
        n = len(self.sizes)
        self.start = np.cumsum([0] + self.sizes).astype(np.int32)
        rows = int(self.start[-1])
        per = max(1, max(-(-(b + t) // 64) for b, t in zip(self.bases, self.sizes))) + 1
        pages = n * per + spare_pages
        self.table = rs.permutation(pages)[: n * per].reshape(n, per).astype(np.int32)
        self.slots = rs.permutation(n).astype(np.int32)
        self.w = words or max(1, -(-max(self.sizes + [1]) // 64))
        if mask is None:
            mask = np.zeros((rows, self.w), np.uint64)
            for b, t in enumerate(self.sizes):
                if t:
                    parents = [-1] + [int(rs.randint(max(0, i - 6), i)) for i in range(1, t)]
                    m = ec.tree_mask(parents).view(np.uint64)
                    mask[self.start[b]:self.start[b + 1], : m.shape[1]] = m
        self.mask = mask
        k = torch.full((pages, 64, kv_heads, hd), math.nan, dtype=ty[kv])
        v = torch.full((pages, 64, kv_heads, hd), math.nan, dtype=ty[kv])
        for b in range(n):
            for p in range(self.bases[b] + self.sizes[b]):
                at = (self.table[self.slots[b], p // 64], p % 64)
                k[at] = torch.from_numpy(rs.randn(kv_heads, hd)).to(ty[kv])
                v[at] = torch.from_numpy(rs.randn(kv_heads, hd)).to(ty[kv])
        self.k, self.v = k.cuda(), v.cuda()
        self.q = (torch.from_numpy(rs.randn(rows, heads * hd)) * q_gain).to(ty[q]).cuda()
        self.out = torch.full_like(self.q, 7.0)

    def dev(self, a):
        return self.torch.from_numpy(np.ascontiguousarray(a)).cuda()

    def run(self, work_bytes=1 << 26, scale=0.0, max_len=None, **kw):
        work = self.torch.empty(work_bytes, dtype=self.torch.uint8, device="cuda") if work_bytes else None
        ec.tree_attention(kw.pop("out", self.out), kw.pop("q", self.q), kw.pop("k", self.k), kw.pop("v", self.v), self.dev(self.table),
                          self.dev(self.start), self.dev(np.array(self.bases, np.int32)), self.dev(self.mask.view(np.int64)),
                          slots=self.dev(self.slots), window=self.window, scale=scale, workspace=work,
                          max_len=max_len or max(b + t for b, t in zip(self.bases, self.sizes)), **kw)
        self.torch.cuda.synchronize()
        assert ec.device_error_take() == 0
        return kw.get("out", self.out)

    def expect(self, scale=0.0):
        """The result in 64 bits and the bound of every value."""
        hd, heads = self.hd, self.heads
        scale = scale or hd ** -0.5
        rows = int(self.start[-1])
        want, tol = np.zeros((rows, heads, hd)), np.zeros((rows, heads, hd))
        q = self.q.double().cpu().numpy().reshape(rows, heads, hd)
        r_w = 2.0 ** -20 if self.qt == "f32" else HALF_STEP[self.kt]
        for b, (t, base) in enumerate(zip(self.sizes, self.bases)):
            pages = self.table[self.slots[b]]
            k, v = (x.double().cpu().numpy()[pages].reshape(-1, self.kvh, hd)[: base + t] for x in (self.k, self.v))
            bits = [[bool(int(self.mask[self.start[b] + i, j // 64]) >> (j % 64) & 1) if j // 64 < self.w else False for j in range(t)]
                    for i in range(t)]
            full = [sum(bin(int(x)).count("1") for x in self.mask[self.start[b] + i]) - 1 for i in range(t)]
            for i in range(t):
                seen = np.concatenate([np.ones(base, bool), np.array(bits[i], bool)])
                if self.window:
                    where = np.concatenate([np.arange(base), base + np.array(full)])
                    seen &= where > base + full[i] - self.window
                if not seen.any():
                    continue
                for h in range(heads):
                    kk, vv, qq = k[seen, h * self.kvh // heads], v[seen, h * self.kvh // heads], q[self.start[b] + i, h]
                    s = kk @ qq * scale
                    mag = (np.abs(kk) @ np.abs(qq) * scale).max()
                    w = np.exp(s - s.max())
                    n = len(s)
                    row = self.start[b] + i
                    want[row, h] = w @ vv / w.sum()
                    move = ((hd + 8) * 2.0 ** -23 + (2.0 ** -20 if self.qt == "f32" else 0)) * mag + (s.max() - s.min()) * 2.0 ** -23 + 2.0 ** -21
                    tol[row, h] = (2 * move + r_w + 2.0 ** -20 + n * 2.0 ** -27) * (w @ np.abs(vv) / w.sum()) * 1.02 + HALF_STEP[self.qt] * np.abs(want[row, h])
                    if self.qt == "f16":
                        tol[row, h] += n * 2.0 ** -25 * np.abs(vv).max() + 2.0 ** -25
        return want.reshape(rows, -1), tol.reshape(rows, -1)

    def check(self, got=None, **kw):
        got = self.out if got is None else got
        want, tol = self.expect(**kw)
        got = got.double().cpu().numpy().reshape(want.shape)
        assert np.isfinite(got).all()
        worst = (np.abs(got - want) - tol).max() if got.size else -1.0
        assert worst <= 0, f"{worst:.3g} over the bound (error {np.abs(got - want).max():.3g})"


@pytest.mark.parametrize("q,kv", [("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "bf16")])
@pytest.mark.parametrize("heads,kv_heads,hd", [(14, 2, 64), (12, 2, 128), (4, 4, 64), (3, 1, 80), (2, 2, 8), (4, 2, 256), (5, 5, 40)])
def test_types_and_heads(cuda, q, kv, heads, kv_heads, hd):
    c = Case(cuda, q, kv, heads, kv_heads, hd, sizes=(7, 1, 20), bases=(130, 63, 0), seed=hd + heads)
    c.run()
    c.check()


@pytest.mark.parametrize("size,base", [(1, 0), (1, 1), (1, 63), (1, 64), (1, 65), (2, 127), (17, 47), (64, 0), (64, 1000), (65, 191), (130, 300)])
@pytest.mark.parametrize("q,kv", [("f16", "f16"), ("f32", "f16"), ("bf16", "bf16")])
def test_lengths_around_pages_and_words(cuda, size, base, q, kv):
    c = Case(cuda, q, kv, 6, 2, 64, sizes=(size,), bases=(base,), seed=size + base)
    c.run()
    c.check()


@pytest.mark.parametrize("work_bytes", [0, 256, 1 << 14, 1 << 24])
@pytest.mark.parametrize("q,kv,hd", [("f16", "f16", 64), ("f32", "f16", 128), ("bf16", "bf16", 128)])
def test_long_cache_split_over_ctas(cuda, work_bytes, q, kv, hd):
    c = Case(cuda, q, kv, 7, 1, hd, sizes=(3, 9), bases=(5000, 777), seed=5)
    c.run(work_bytes)
    c.check()


@pytest.mark.parametrize("window", [1, 2, 7, 64, 100, 1000])
@pytest.mark.parametrize("q,kv", [("f16", "f16"), ("f32", "bf16")])
def test_window(cuda, window, q, kv):
    c = Case(cuda, q, kv, 4, 2, 64, sizes=(12, 1, 70), bases=(200, 5, 64), window=window, seed=window)
    c.run()
    c.check()


@pytest.mark.parametrize("q,kv", [("f16", "f16"), ("f32", "f16")])
def test_rows_that_see_nothing_and_any_mask(cuda, q, kv):
    rs = np.random.RandomState(3)
    sizes, bases = (9, 4, 6), (0, 0, 30)
    mask = (rs.randint(0, 1 << 9, (19, 1))).astype(np.uint64)     # any sets; bits behind a tree's end mean nothing
    mask[[0, 4, 9, 12]] = 0                                       # sequence 0 and 1 have nothing cached: empty rows
    mask[9:13] &= np.uint64(15)
    mask[13:] &= np.uint64(63)
    c = Case(cuda, q, kv, 4, 2, 64, sizes=sizes, bases=bases, mask=mask, seed=4)
    c.run()
    c.check()
    out = c.out.cpu()
    assert (out[[0, 4, 9, 12]] == 0).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("q,kv", [("f16", "f16"), ("f32", "f16"), ("bf16", "bf16")])
def test_what_a_row_does_not_see_does_not_reach_it(cuda, bad, q, kv):
    """Two branches; the second one's node holds `bad` in K and V: only the rows that see it may change."""
    parents = [-1, 0, 0, 1, 2, 3]
    c = Case(cuda, q, kv, 4, 2, 64, sizes=(6,), bases=(70,), mask=ec.tree_mask(parents).view(np.uint64), seed=6)
    want, tol = c.expect()
    page, off = c.table[c.slots[0], (70 + 2) // 64], (70 + 2) % 64
    c.k[page, off] = bad
    c.v[page, off] = bad
    c.run()
    got = c.out.double().cpu().numpy()
    clean = [0, 1, 3, 5]
    assert (np.abs(got - want) <= tol)[clean].all()
    assert not np.isfinite(got[[2, 4]]).all()


def test_window_hides_infinities(cuda):
    c = Case(cuda, "f16", "f16", 4, 2, 64, sizes=(4,), bases=(200,), mask=ec.tree_mask([-1, 0, 1, 2]).view(np.uint64), window=50, seed=8)
    want, tol = c.expect()
    for p in range(0, 152):       # row i sees positions above 150 + i; row 0 still sees 151, the others do not
        c.v[c.table[c.slots[0], p // 64], p % 64] = math.inf
        c.k[c.table[c.slots[0], p // 64], p % 64] = math.nan if p < 151 else 0.0
    c.run()
    got = c.out.double().cpu().numpy()
    assert (np.abs(got - want) <= tol)[1:].all()
    assert not np.isfinite(got[0]).all()


# max_len only steers how the work is laid out: FAR makes short caches take the path of long ones (equal pieces of the
# pages, and tiles of 128 rows on tcgen05 from 65 rows on a KV head).
FAR = 1 << 20


@pytest.mark.parametrize("q,kv", [("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "bf16")])
@pytest.mark.parametrize("heads,kv_heads,hd", [(14, 2, 64), (12, 2, 128), (6, 6, 64), (8, 1, 128), (3, 1, 80), (4, 2, 256)])
@pytest.mark.parametrize("sizes,bases", [((64,), (1000,)), ((130, 70), (300, 64)), ((1, 40, 0, 9), (0, 63, 5, 128)), ((100,) * 3, (1, 0, 65))])
def test_pieces(cuda, q, kv, heads, kv_heads, hd, sizes, bases):
    c = Case(cuda, q, kv, heads, kv_heads, hd, sizes=sizes, bases=bases, seed=hd + len(sizes))
    c.run(max_len=FAR)
    c.check()


@pytest.mark.parametrize("window", [1, 2, 7, 64, 100, 1000])
@pytest.mark.parametrize("q,kv", [("f16", "f16"), ("bf16", "bf16"), ("f32", "f16")])
def test_pieces_window(cuda, window, q, kv):
    c = Case(cuda, q, kv, 8, 1, 64, sizes=(12, 1, 70), bases=(200, 5, 64), window=window, seed=window)
    c.run(max_len=FAR)
    c.check()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("q,kv", [("f16", "f16"), ("bf16", "bf16"), ("f32", "f16")])
def test_pieces_hidden_infinities(cuda, bad, q, kv, hd):
    """A branch that holds `bad` in K and V, in the first page of its tile and in a later one."""
    for base in (0, 70, 200):
        parents = [-1, 0, 0, 1, 2, 3] + [3] * 20
        c = Case(cuda, q, kv, 8, 1, hd, sizes=(26,), bases=(base,), mask=ec.tree_mask(parents).view(np.uint64), seed=6)
        want, tol = c.expect()
        page, off = c.table[c.slots[0], (base + 2) // 64], (base + 2) % 64
        c.k[page, off] = bad
        c.v[page, off] = bad
        c.run(max_len=FAR)
        got = c.out.double().cpu().numpy()
        clean = [i for i in range(26) if i not in (2, 4)]
        assert (np.abs(got - want) <= tol)[clean].all()
        assert not np.isfinite(got[[2, 4]]).all()


@pytest.mark.parametrize("hd", [64, 128])
def test_infinity_in_v_reaches_the_rows_that_see_it(cuda, hd):
    """+inf in one element of V: that element of the rows that see it is +inf, everything else as before."""
    for max_len in (None, FAR):
        c = Case(cuda, "f16", "f16", 8, 1, hd, sizes=(20,), bases=(100,), mask=ec.tree_mask([-1] + [0] * 19).view(np.uint64), seed=7)
        want, tol = c.expect()
        c.v[c.table[c.slots[0], 107 // 64], 107 % 64, 0, 5] = math.inf      # node 7 is seen by itself alone
        c.run(max_len=max_len)
        got = c.out.double().cpu().numpy().reshape(20, 8, hd)
        assert (got[7, :, 5] == math.inf).all()
        got[7, :, 5] = want.reshape(20, 8, hd)[7, :, 5]
        assert (np.abs(got.reshape(20, -1) - want) <= tol).all()


def test_pieces_many_sequences_and_growing_maxima(cuda):
    """70 ragged sequences; keys that grow along the cache, so that a row's maximum rises page by page."""
    rs = np.random.RandomState(15)
    sizes, bases = rs.randint(0, 25, 70), rs.randint(0, 260, 70)
    for q, kv in (("f16", "f16"), ("bf16", "bf16"), ("f32", "f16")):
        c = Case(cuda, q, kv, 8, 1, 64, sizes=sizes.tolist(), bases=bases.tolist(), seed=16)
        pos = cuda.arange(64, device="cuda")[None, :, None, None]
        c.k.mul_((1 + pos / 8).to(c.k.dtype))
        c.run(max_len=FAR)
        c.check()
        c.run()
        c.check()


@pytest.mark.parametrize("q,kv,hd", [("f16", "f16", 64), ("bf16", "bf16", 128), ("f32", "f16", 64), ("f32", "bf16", 128), ("f16", "f16", 256)])
@pytest.mark.parametrize("seqs,window", [(4, 0), (12, 90), (40, 0)])
def test_short_contexts_of_every_cluster_size(cuda, seqs, window, q, kv, hd):
    """6 KV heads and up to 5 pages: tiles for clusters of 4 CTAs, of 2 and of one, and for more of them than fit at once."""
    rs = np.random.RandomState(seqs)
    sizes, bases = rs.randint(1, 40, seqs), rs.randint(0, 270, seqs)
    c = Case(cuda, q, kv, 6, 6, hd, sizes=sizes.tolist(), bases=bases.tolist(), window=window, seed=hd + seqs)
    c.run(max_len=310)
    c.check()


@pytest.mark.parametrize("window", [1, 3, 20, 128])
@pytest.mark.parametrize("q,kv", [("f32", "bf16"), ("f16", "f16")])
def test_window_within_large_trees(cuda, window, q, kv):
    """Trees of more levels than the window: it hides nodes from their descendants, across pages and mask words."""
    chain = np.maximum(np.arange(150) - 1 - np.arange(150) % 3 % 2, -1)
    chain[1:] = np.maximum(chain[1:], 0)
    mask = ec.tree_mask(chain).view(np.uint64)
    for base in (0, 40, 130):
        c = Case(cuda, q, kv, 6, 3, 64, sizes=(150,), bases=(base,), window=window, mask=mask, seed=window)
        for far in (None, FAR):
            c.run(**({} if far is None else {"max_len": far}))
            c.check()


def test_pieces_little_work_and_small_workspaces(cuda):
    for bytes_ in (1 << 17, 1 << 19, 1 << 21, 1 << 26):
        c = Case(cuda, "bf16", "bf16", 12, 2, 128, sizes=(30, 7), bases=(700, 90), seed=17)
        c.run(bytes_, max_len=FAR)
        c.check()
    c = Case(cuda, "f16", "f16", 8, 1, 64, sizes=(9,), bases=(3,), seed=18)
    c.run(max_len=FAR)
    c.check()


def test_strides_three_dimensions_and_rows_behind_the_last_sequence(cuda):
    c = Case(cuda, "f16", "f16", 6, 2, 64, sizes=(3, 8), bases=(90, 10), seed=9)
    rows, wide = c.q.shape
    big_q = cuda.full((rows + 5, wide + 13), 3.0, dtype=cuda.float16, device="cuda")
    big_o = cuda.full((rows + 5, wide + 21), 5.0, dtype=cuda.float16, device="cuda")
    big_q[:rows, 1:wide + 1] = c.q
    c.mask = np.concatenate([c.mask, np.zeros((5, c.w), np.uint64)])
    q, out = big_q[:, 1:wide + 1], big_o[:, 3:wide + 3]
    ec.tree_attention(out, q, c.k, c.v, c.dev(c.table), c.dev(c.start), c.dev(np.array(c.bases, np.int32)), c.dev(c.mask.view(np.int64)),
                      slots=c.dev(c.slots))
    cuda.cuda.synchronize()
    assert ec.device_error_take() == 0
    c.mask = c.mask[:rows]
    c.check(out[:rows])
    rest = big_o.clone()
    rest[:rows, 3:wide + 3] = 5.0
    assert (rest == 5.0).all()
    # the heads as a dimension of their own, K and V interleaved in one pool
    both = cuda.stack([c.k, c.v], dim=2)
    out3 = cuda.empty((rows, 6, 64), dtype=cuda.float16, device="cuda")
    c.run(out=out3, q=c.q.view(rows, 6, 64), k=both[:, :, 0], v=both[:, :, 1])
    c.check(out3)


def test_scale_large_scores_and_many_words(cuda):
    c = Case(cuda, "f32", "f16", 4, 2, 64, sizes=(5,), bases=(300,), seed=10, words=3, q_gain=40.0)
    c.run()
    c.check()
    c.run(scale=0.01)
    c.check(scale=0.01)


def test_empty_trees_between_others(cuda):
    c = Case(cuda, "f16", "f16", 4, 4, 64, sizes=(0, 3, 0, 0, 2, 0), bases=(10, 64, 0, 70, 128, 3), seed=11)
    c.run()
    c.check()


def test_bad_indices_are_reported(cuda):
    c = Case(cuda, "f16", "f16", 4, 2, 64, sizes=(3, 2), bases=(90, 10), seed=12)
    good = c.table.copy()
    for spoil in ("page", "slot", "base", "rows"):
        table, slots, bases, start = good.copy(), c.slots.copy(), list(c.bases), c.start.copy()
        if spoil == "page":
            table[slots[1], 0] = 10 ** 6
        elif spoil == "slot":
            slots[1] = 2
        elif spoil == "base":
            bases[1] = 64 * table.shape[1] - 1
        else:
            start[2] = 9
        ec.tree_attention(c.out, c.q, c.k, c.v, c.dev(table), c.dev(start), c.dev(np.array(bases, np.int32)), c.dev(c.mask.view(np.int64)),
                          slots=c.dev(slots))
        assert ec.device_error_take() == 2, spoil
        assert ec.device_error_take() == 0
        want, tol = c.expect()
        got = c.out.double().cpu().numpy()
        assert (np.abs(got - want) <= tol)[:3].all(), spoil     # the first sequence is untouched by it


def test_captured_graph_replays_on_new_data_and_other_stream(cuda):
    c = Case(cuda, "bf16", "bf16", 7, 1, 128, sizes=(4, 1), bases=(2000, 65), seed=13)
    c.run()
    args = (c.dev(c.table), c.dev(c.start), c.dev(np.array(c.bases, np.int32)), c.dev(c.mask.view(np.int64)))
    slots = c.dev(c.slots)
    work = cuda.empty(1 << 22, dtype=cuda.uint8, device="cuda")
    g = cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(g):
        ec.tree_attention(c.out, c.q, c.k, c.v, *args, slots=slots, workspace=work, max_len=2004,
                          stream=cuda.cuda.current_stream().cuda_stream)
    for gain in (1.0, 0.5):
        c.q.mul_(gain)
        c.out.fill_(9.0)
        g.replay()
        cuda.cuda.synchronize()
        c.check()
    first = c.out.clone()
    s = cuda.cuda.Stream()
    c.out.fill_(9.0)
    s.wait_stream(cuda.cuda.current_stream())
    ec.tree_attention(c.out, c.q, c.k, c.v, *args, slots=slots, workspace=work, max_len=2004, stream=s.cuda_stream)
    s.synchronize()
    assert cuda.equal(c.out, first)      # the same result, bit for bit


@pytest.mark.parametrize("window", [63, 64, 65, 127, 128, 129])
@pytest.mark.parametrize("far", [None, FAR])
@pytest.mark.parametrize("q,kv", [("f16", "f16"), ("bf16", "bf16"), ("f32", "f16")])
def test_window_as_long_as_a_mask_has_bits(cuda, window, far, q, kv):
    """Rows of all bits (depth 64 words - 1) and of none (depth -1): the furthest apart that two nodes of a mask can stand.
    A window of 64 words still hides the one from the other, one more no longer does."""
    words = 1 if window < 100 else 2
    mask = np.random.RandomState(5).randint(0, 1 << 62, (20, words)).astype(np.uint64)
    mask[[0, 7]] = 2 ** 64 - 1
    mask[[1, 9]] = 0
    mask[2] = 1
    mask[3] = 2 ** 64 - 2
    for base in (0, 70):
        c = Case(cuda, q, kv, 8, 1, 64, sizes=(20,), bases=(base,), window=window, mask=mask, words=words, seed=window)
        c.run(max_len=far)
        c.check()


@pytest.mark.parametrize("q,kv,heads,kv_heads,hd,seqs,nodes,lens", [
    ("f32", "f16", 12, 2, 128, 32, 24, (450, 900)), ("f32", "bf16", 4, 2, 256, 32, 24, (560, 900)), ("f32", "f16", 14, 2, 64, 12, 9, (65, 1900)),
    ("f16", "f16", 14, 2, 64, 3, 5, (1100, 1500)), ("bf16", "bf16", 12, 2, 128, 5, 40, (100, 1300)), ("f16", "f16", 8, 8, 80, 4, 3, (1030, 1200))])
@pytest.mark.parametrize("said", [True, False])
def test_the_documented_workspace_is_all_that_a_call_uses(cuda, q, kv, heads, kv_heads, hd, seqs, nodes, lens, said):
    """With the bytes of tree_attention_work a call splits as far as with any more: the same result, bit for bit.  `said`:
    with max_len given, or left out of both calls."""
    rs = np.random.RandomState(seqs)
    c = Case(cuda, q, kv, heads, kv_heads, hd, sizes=[nodes] * seqs, bases=rs.randint(lens[0], lens[1] - nodes, seqs).tolist(), seed=hd)
    c.table = np.concatenate([c.table, np.full((seqs, max(0, 20 - c.table.shape[1])), -1, np.int32)], axis=1)   # behind the sequences: no page
    most = lens[1] if said else 0
    bytes_ = ec.tree_attention_work(seqs, seqs * nodes, heads, kv_heads, hd, most)
    assert bytes_ > 0
    outs = []
    for n in (bytes_, bytes_ + (64 << 20)):
        out = cuda.full_like(c.q, 7.0)
        ec.tree_attention(out, c.q, c.k, c.v, c.dev(c.table), c.dev(c.start), c.dev(np.array(c.bases, np.int32)), c.dev(c.mask.view(np.int64)),
                          slots=c.dev(c.slots), max_len=most, workspace=cuda.empty(n, dtype=cuda.uint8, device="cuda"))
        cuda.cuda.synchronize()
        assert ec.device_error_take() == 0
        outs.append(out)
    c.check(outs[0])
    assert cuda.equal(outs[0], outs[1])


@pytest.mark.parametrize("q,kv,hd,bytes_", [("bf16", "bf16", 128, 600 << 10), ("f16", "f16", 64, 400 << 10), ("f32", "f16", 128, 200 << 10), ("f16", "f16", 128, 2 << 20)])
def test_a_workspace_of_a_few_pieces_is_not_taken(cuda, q, kv, hd, bytes_):
    """Two or three CTAs that walk all pages would take far longer than the clusters of a call without a workspace: it runs as
    that one, bit for bit."""
    c = Case(cuda, q, kv, 12, 2, hd, sizes=[40, 55, 48, 60] * 2, bases=[900, 1200, 1100, 1050] * 2, seed=19)
    plain = c.run(0).clone()
    c.out.fill_(7.0)
    c.run(bytes_)
    c.check()
    assert cuda.equal(c.out, plain)


def test_many_tiles_in_a_piece(cuda):
    """More tiles than CTAs on the tcgen05 path: a CTA goes from tile to tile, with full halves, lone halves and odd pages."""
    rs = np.random.RandomState(23)
    seqs = 120
    c = Case(cuda, "f16", "f16", 16, 2, 64, sizes=rs.randint(1, 40, seqs).tolist(), bases=rs.randint(0, 300, seqs).tolist(), seed=24)
    c.run(max_len=FAR)
    c.check()


@pytest.mark.parametrize("q,kv,hd", [("f16", "f16", 64), ("bf16", "bf16", 128)])
@pytest.mark.parametrize("layout", ["rows", "interleaved", "padded", "position outermost"])
def test_strides_of_queries_outputs_and_caches_on_tcgen05(cuda, q, kv, hd, layout):
    """Tiles of 128 rows with queries and outputs of any alignment and row stride, and caches whose pages, positions or K and
    V lie otherwise than in one run."""
    c = Case(cuda, q, kv, 16, 2, hd, sizes=(30, 3, 17), bases=(90, 200, 0), seed=31)
    rows, wide = c.q.shape
    if layout == "rows":
        for lead, gap, tail in ((1, 13, 3), (4, 12, 4), (2, 14, 6)):      # odd; 8-byte and 4-byte aligned
            big_q = cuda.full((rows, wide + gap), 3.0, dtype=c.q.dtype, device="cuda")
            big_o = cuda.full((rows + 5, wide + gap + 8), 5.0, dtype=c.q.dtype, device="cuda")
            big_q[:, lead:lead + wide] = c.q
            out = big_o[:rows, tail:tail + wide]
            c.run(out=out, q=big_q[:, lead:lead + wide], max_len=FAR)
            c.check(out)
            c.run(out=out.fill_(7.0), q=big_q[:, lead:lead + wide])
            c.check(out)
            out.fill_(5.0)
            assert (big_o == 5.0).all()
        return
    pages = c.k.shape[0]
    if layout == "interleaved":
        pool = cuda.stack([c.k, c.v], dim=2)
        k, v = pool[:, :, 0], pool[:, :, 1]
    elif layout == "padded":
        pool = cuda.full((2, pages + 1, 64, 2 * hd + 24), math.nan, dtype=c.k.dtype, device="cuda")
        pool[0, :pages, :, : 2 * hd], pool[1, :pages, :, : 2 * hd] = c.k.flatten(2), c.v.flatten(2)
        k, v = (pool[i, :pages, :, : 2 * hd].unflatten(2, (2, hd)) for i in (0, 1))
    else:
        pool = cuda.stack([c.k.transpose(0, 1), c.v.transpose(0, 1)]).contiguous()
        k, v = pool[0].transpose(0, 1), pool[1].transpose(0, 1)
    assert cuda.equal(k.isnan(), c.k.isnan()) and (k.stride() != c.k.stride())
    for far in (FAR, None):
        c.out.fill_(7.0)
        c.run(k=k, v=v, max_len=far)
        c.check()


@pytest.mark.parametrize("kv", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,hd", [(6, 2, 64), (4, 2, 80), (3, 1, 256)])
@pytest.mark.parametrize("lead,gap", [(1, 3), (2, 6), (0, 1)])
def test_fp32_rows_of_any_alignment(cuda, kv, heads, kv_heads, hd, lead, gap):
    c = Case(cuda, "f32", kv, heads, kv_heads, hd, sizes=(9, 2), bases=(70, 129), seed=33)
    rows, wide = c.q.shape
    big = cuda.full((rows, wide + gap), 3.0, device="cuda")
    out = cuda.full((rows, wide + gap), 5.0, device="cuda")
    big[:, lead:lead + wide] = c.q
    for far in (None, FAR):
        c.run(q=big[:, lead:lead + wide], out=out[:, lead:lead + wide], max_len=far)
        c.check(out[:, lead:lead + wide])
    out[:, lead:lead + wide] = 5.0
    assert (out == 5.0).all()


@pytest.mark.parametrize("q,kv,hd", [("f16", "f16", 64), ("bf16", "bf16", 128), ("f32", "f16", 64), ("f32", "bf16", 128), ("f16", "f16", 256)])
@pytest.mark.parametrize("seqs,window", [(1, 0), (1, 90), (4, 90), (12, 0), (30, 0), (30, 90), (40, 90)])
def test_short_contexts_with_and_without_a_window(cuda, seqs, window, q, kv, hd):
    """6 KV heads and up to 5 pages, every number of sequences with both kinds of mask."""
    rs = np.random.RandomState(seqs)
    sizes, bases = rs.randint(1, 40, seqs), rs.randint(0, 270, seqs)
    c = Case(cuda, q, kv, 6, 6, hd, sizes=sizes.tolist(), bases=bases.tolist(), window=window, seed=hd + seqs)
    c.run(max_len=310)
    c.check()


@pytest.mark.parametrize("q,heads", [("f16", 1), ("f16", 8), ("f32", 1)])
def test_row_start_that_falls_and_rises_is_reported(cuda, q, heads):
    """Thousands of sequences that all claim the same rows: more places than the line of pages can count.  Nothing is written
    and the call reports a bad index."""
    rows, n, hd = 100000, 3000, 64
    start = np.zeros(n + 1, np.int32)
    start[1::2] = rows
    k = cuda.zeros(3, 64, 1, hd, dtype=cuda.float16, device="cuda")
    dev = lambda x: cuda.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
    qs = cuda.zeros(rows, heads * hd, dtype=_types(cuda)[q], device="cuda")
    out = cuda.full_like(qs, 7.0)
    ec.tree_attention(out, qs, k, k.clone(), dev(np.arange(1600, dtype=np.int32)[None] % 3), dev(start), dev(np.zeros(n, np.int32)), cuda.zeros(rows, 1, dtype=cuda.int64, device="cuda"),
                      slots=dev(np.zeros(n, np.int32)), workspace=cuda.empty(64 << 20, dtype=cuda.uint8, device="cuda"))
    cuda.cuda.synchronize()
    assert ec.device_error_take() == 2 and ec.device_error_take() == 0
    assert (out == 7.0).all()
