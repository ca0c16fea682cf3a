"""Drawing tokens (ec_sample) against the definition in 64 bits.  The token is a whole number: it has to be the definition's,
except where u times the total lies within the rounding of the weights (a few parts in 2^44 of the sum for the vocabularies
here) of a border; the seeded cases below have none, which each test asserts before it compares.  prob is one exp and one
division away from the exact share and rounded to fp32 once: 2^-24, plus 2^-40 for the rounded sum."""
from __future__ import annotations

import math

import numpy as np
import pytest

import edgecore_b200 as ec

pytestmark = pytest.mark.gpu


def definition(row, t, k, p, least, u):
    """(token, prob, distance of u's point to the nearest border as a share of the total)."""
    row = np.where(np.isnan(row), -np.inf, row.astype(np.float64))
    n, top = len(row), row.max()
    if top == -np.inf:
        return -1, 0.0, 1.0
    order = np.argsort(-row, kind="stable")
    if not t > 0:
        return int(order[0]), 1.0, 1.0
    with np.errstate(invalid="ignore"):
        w = (row == np.inf).astype(float) if top == np.inf else np.where(row == -np.inf, 0.0, np.exp((row - top) / t))
    if 0 < k < n:
        order = order[:k]
    gap = 1.0
    if p < 1:
        mass = np.cumsum(w[order])
        want = p * mass[-1]
        at = int(np.searchsorted(mass, want))
        gap = min(gap, *(abs(mass[j] - want) / mass[-1] for j in (at - 1, at) if 0 <= j < len(mass)), 1.0) if want > 0 else gap
        order = order[: at + 1]
    if least > 0:
        order = np.array([i for i in order if w[i] >= least or i == order[0]])
    kept = np.zeros(n)
    kept[order] = w[order]
    mass = np.cumsum(kept)
    point = max(u, 0.0) * mass[-1] if u == u else 0.0
    at = min(int(np.searchsorted(mass, point, side="right")), int(np.flatnonzero(kept)[-1]))
    if 0 < u < 1:
        gap = min(gap, np.abs(mass[kept > 0] - point).min() / mass[-1])
    return at, kept[at] / mass[-1], gap


def run(torch, logits, u, **kw):
    rows = logits.shape[0]
    ids = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    prob = torch.full((rows,), -7.0, device="cuda")
    ec.sample(ids, logits, torch.tensor(u, dtype=torch.float32, device="cuda"), prob=prob,
              **{k: None if v is None else torch.tensor(v, dtype=torch.int32 if k == "top_k" else torch.float32, device="cuda") for k, v in kw.items()})
    torch.cuda.synchronize()
    return ids.cpu().numpy(), prob.cpu().numpy()


def check(torch, logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    ids, prob = run(torch, logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    host = logits.float().cpu().numpy()
    f = lambda v, r, none: none if v is None else float(np.float32(v[r]))  # noqa: E731
    for r in range(len(host)):
        at, share, gap = definition(host[r], f(temperature, r, 1.0), 0 if top_k is None else top_k[r], f(top_p, r, 1.0), f(min_p, r, 0.0), float(np.float32(u[r])))
        assert gap > 1e-12, "a case on a border compares nothing"
        assert ids[r] == at, f"row {r}: {ids[r]} for {at} (gap {gap:.3g})"
        assert abs(prob[r] - share) <= (2.0 ** -24 + 2.0 ** -40) * share, f"row {r}: prob {prob[r]!r} for {share!r}"


def _logits(torch, rows, vocab, kind, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * spread
    x[:, torch.randperm(vocab, generator=g)[: min(30, vocab)]] += torch.rand(min(30, vocab), generator=g) * 10
    return x.to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kind]).cuda()


SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=50), dict(top_p=0.9), dict(min_p=0.05), dict(temperature=1.5, top_k=200, top_p=0.95, min_p=0.001),
            dict(temperature=0.3, top_p=0.5), dict(top_k=3, top_p=0.99), dict(top_p=0.999), dict(temperature=3.0, top_k=20000, top_p=0.97)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 1025, 50257, 151936])
@pytest.mark.parametrize("setting", range(len(SETTINGS)))
def test_settings(cuda, kind, vocab, setting):
    rows = 5
    s = SETTINGS[setting]
    rs = np.random.RandomState(vocab + setting)
    x = _logits(cuda, rows, vocab, kind, vocab + setting)     # 16-bit logits: many equal ones
    check(cuda, x, rs.rand(rows).astype(np.float32), **{k: [v] * rows for k, v in s.items()})


@pytest.mark.parametrize("vocab", [999, 50257])
def test_every_row_its_own_settings(cuda, vocab):
    rs = np.random.RandomState(vocab)
    rows = 200
    x = _logits(cuda, rows, vocab, "f32", vocab)
    check(cuda, x, rs.rand(rows).astype(np.float32), temperature=rs.choice([0.0, -1.0, math.nan, 0.5, 1.0, 2.0], rows), top_k=rs.choice([-3, 0, 1, 2, 40, 900, 10 ** 6], rows),
          top_p=rs.choice([0.0, 0.1, 0.8, 0.95, 1.0, 1.7], rows), min_p=rs.choice([0.0, 0.01, 0.5, 1.0, 1.5], rows))


@pytest.mark.parametrize("vocab", [300, 4097, 151936])
def test_all_equal_and_two_values(cuda, vocab):
    """Ties everywhere: they are kept lowest index first."""
    x = cuda.zeros(6, vocab, device="cuda")
    x[3:] = (cuda.arange(vocab, device="cuda") % 3 == 1).float()
    x[1] = -0.0
    x[1, ::2] = 0.0                       # the zeros are equal
    u = [0.13, 0.77, 0.5001, 0.31, 0.9, 0.62]
    check(cuda, x, u, top_k=[0, 77, 100, 0, 90, 299])
    check(cuda, x, u, top_p=[0.3, 0.51, 0.99, 0.2, 0.7, 0.95])
    check(cuda, x, u, top_k=[0, 200, 100, 10, 150, 299], top_p=[0.3, 0.51, 0.999, 0.2, 0.7, 0.95])


def test_close_logits_of_both_signs(cuda):
    """Thousands of values within a hair of zero and of each other: the selection has to tell them apart."""
    g = cuda.Generator().manual_seed(1)
    x = cuda.randn(8, 30000, generator=g) * cuda.tensor([1e-30, 1e-9, 1e-6, 1e-4, 1e-3, 1e-2, 1e-40, 5e-5])[:, None]
    x[4:, :100] += 3.0
    x = x.cuda()
    rs = np.random.RandomState(2)
    check(cuda, x, rs.rand(8).astype(np.float32), top_k=[7, 12345, 29999, 5000, 40, 3000, 15000, 101])
    check(cuda, x, rs.rand(8).astype(np.float32), top_p=[0.1, 0.5, 0.9, 0.99, 0.6, 0.7, 0.8, 0.95])


def test_infinities_and_nan(cuda):
    inf, nan = math.inf, math.nan
    rows = [[1.0, nan, 2.0, -inf, 0.5], [-inf] * 5, [nan] * 5, [inf, 1.0, inf, nan, -inf], [-inf, -inf, 3.0, nan, -inf], [3e38, -3e38, 3e38, 0.0, 1.0],
            [nan, -inf, -1e30, -1e30, nan]]
    x = cuda.tensor(rows, device="cuda")
    for u in (0.01, 0.4, 0.7, 0.99):
        check(cuda, x, [u] * len(rows))
        check(cuda, x, [u] * len(rows), temperature=[0.0] * len(rows))
        check(cuda, x, [u] * len(rows), top_k=[2] * len(rows), top_p=[0.9] * len(rows))
    check(cuda, x, [0.6] * len(rows), temperature=[inf] * len(rows))
    check(cuda, x, [0.6] * len(rows), temperature=[1e-30] * len(rows))


def test_u_at_and_outside_its_range(cuda):
    x = cuda.tensor([[0.0, 1.0, -inf_, 2.0, -inf_] for inf_ in [math.inf] * 6], device="cuda")
    ids, _ = run(cuda, x, [0.0, -1.0, math.nan, 1.0, 2.0, math.inf])
    assert ids.tolist() == [0, 0, 0, 3, 3, 3]
    x = cuda.tensor([[-math.inf, 1.0, 1.0]] * 2, device="cuda")
    ids, prob = run(cuda, x, [0.0, np.nextafter(np.float32(1), np.float32(0))])
    assert ids.tolist() == [1, 2] and prob.tolist() == [0.5, 0.5]


def test_strided_rows_and_no_prob(cuda):
    big = cuda.full((9, 5003), 50.0, device="cuda")
    x = _logits(cuda, 9, 5000, "f32", 3)
    big[:, 1:5001] = x
    rs = np.random.RandomState(3)
    u = rs.rand(9).astype(np.float32)
    check(cuda, big[:, 1:5001], u, top_k=[100] * 9, top_p=[0.9] * 9)
    ids, want = cuda.empty(9, dtype=cuda.int32, device="cuda"), run(cuda, x, u)[0]
    ec.sample(ids, big[:, 1:5001], cuda.from_numpy(u).cuda())
    assert ids.cpu().numpy().tolist() == want.tolist()
    half = cuda.zeros(4, 1001, dtype=cuda.bfloat16, device="cuda")
    y = _logits(cuda, 4, 1000, "bf16", 4)
    half[:, 1:] = y
    assert (run(cuda, half[:, 1:], u[:4])[0] == run(cuda, y, u[:4])[0]).all()


def test_a_row_depends_on_itself_alone(cuda):
    """The same row alone, among others and replayed from a graph: the same token and the same probability, bit for bit."""
    x = _logits(cuda, 300, 30011, "f32", 5)
    rs = np.random.RandomState(5)
    u = rs.rand(300).astype(np.float32)
    s = dict(temperature=[0.9] * 300, top_p=[0.95] * 300)
    ids, prob = run(cuda, x, u, **s)
    for r in (0, 17, 299):
        i, p = run(cuda, x[r:r + 1], u[r:r + 1], temperature=[0.9], top_p=[0.95])
        assert i[0] == ids[r] and p[0] == prob[r]
    dev = {k: cuda.tensor(v, device="cuda") for k, v in s.items()}
    du, out, pr = cuda.from_numpy(u).cuda(), cuda.empty(300, dtype=cuda.int32, device="cuda"), cuda.empty(300, device="cuda")
    ec.sample(out, x, du, prob=pr, **dev)
    g = cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(g):
        ec.sample(out, x, du, prob=pr, **dev, stream=cuda.cuda.current_stream().cuda_stream)
    for _ in range(3):
        out.fill_(-1)
        g.replay()
        cuda.cuda.synchronize()
        assert (out.cpu().numpy() == ids).all() and (pr.cpu().numpy() == prob).all()


def test_frequencies(cuda):
    """20000 draws of one row: each token's count within 6 standard deviations of its share."""
    n = 20000
    row = cuda.tensor([0.0, 1.0, 2.0, -1.0, 0.5, 1.5], device="cuda")
    x = row.expand(n, 6).contiguous()
    u = np.random.RandomState(7).rand(n).astype(np.float32)
    ids, _ = run(cuda, x, u, top_k=[5] * n)
    w = np.exp(row.double().cpu().numpy())
    w[3] = 0
    w /= w.sum()
    count = np.bincount(ids, minlength=6)
    assert count[3] == 0
    assert (np.abs(count - n * w) <= 6 * np.sqrt(n * w * (1 - w)) + 1e-9).all()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab,pad", [(1001, 6), (16384, 0), (16391, 6), (20011, 3), (50257, 1)])
def test_many_rows(cuda, kind, vocab, pad):
    """Enough rows for one CTA each, without top-k and top-p: the definition's tokens, and bit for bit those of the kernel that
    a call with (idle) top-k takes; rows of every alignment, with infinities and NaN among them."""
    rows = 180
    rs = np.random.RandomState(vocab)
    x = _logits(cuda, rows, vocab + pad, kind, vocab)[:, pad // 2: pad // 2 + vocab]
    if vocab > 2:
        for r, v in ((5, math.inf), (6, math.nan), (7, -math.inf)):
            x[r::40, :: 2 + r % 2] = v
        x[8] = -math.inf
        x[9] = math.nan
    u = rs.rand(rows).astype(np.float32)
    temperature, min_p = rs.choice([0.0, -1.0, math.nan, 0.02, 0.7, 1.0, 3.0], rows), rs.choice([0.0, 0.0, 0.003, 0.4, 1.0, 1.5], rows)
    check(cuda, x, u, temperature=temperature, min_p=min_p)
    for kw in (dict(), dict(temperature=temperature), dict(min_p=min_p), dict(temperature=temperature, min_p=min_p)):
        a, b = run(cuda, x, u, **kw), run(cuda, x, u, top_k=np.zeros(rows), **kw)
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1].view(np.int32), b[1].view(np.int32))


@pytest.mark.parametrize("kind,vocab,pad", [("f32", 262144, 0), ("f32", 400001, 3), ("f32", 750000, 1), ("bf16", 400001, 5), ("f16", 750000, 0)])
def test_vocabularies_up_to_the_largest(cuda, kind, vocab, pad):
    """A row fills the shared memory of 16 CTAs: one CTA on an SM, clusters of 16."""
    rows = 3
    x = _logits(cuda, rows, vocab + pad, kind, vocab % 1000)[:, pad:]
    rs = np.random.RandomState(vocab % 1000)
    for kw in (dict(temperature=[0.7] * rows), dict(top_k=[50] * rows, top_p=[0.95] * rows), dict(top_p=[0.9] * rows, min_p=[0.0001] * rows),
               dict(temperature=[3.0] * rows, top_k=[30000] * rows, top_p=[0.97] * rows), dict(temperature=[0.0, 1.0, 0.5])):
        check(cuda, x, rs.rand(rows).astype(np.float32), **kw)
