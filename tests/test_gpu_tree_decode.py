"""The serving operators inside the model calls: forks of a prompt (kv_fork), verified steps of drafted trees with greedy and
drawn choices (forward_tree), sampled batched decode (decode_sample), alone and one after the other, against the CPU oracle
stepped along the tokens that were accepted.

The oracle's and the model's logits differ by at most d = TOL x the largest logit (the bound of the batched steps).  A greedy
choice is then within 2 d of the oracle's largest logit.  A weight exp(logit / T) is off by a factor within exp(+-d / T), so a
share of the total, and any sum of shares, by at most exp(2 d / T) - 1."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

import edgecore_b200 as ec
from edgecore_b200 import synth

pytestmark = pytest.mark.gpu

TOL = 1e-3


def open_oracle(spec, path, slots):
    from oracle.oracle import Restatement
    return Restatement().open(path, batch_cap=slots, max_ctx=spec.n_ctx)


def feed(model, tokens, at, slot):
    n = len(tokens)
    return model.forward(np.asarray(tokens, np.int32), np.arange(at, at + n, dtype=np.int32), np.full(n, slot, np.int32))


def check_choice(logits, token, t=0.0, u=None, prob=None):
    logits = logits.astype(np.float64)
    d = TOL * np.abs(logits).max()
    if not t > 0:
        assert logits[token] >= logits.max() - 2 * d
        if prob is not None:
            assert prob == 1.0
        return
    w = np.exp((logits - logits.max()) / t)
    sums = np.cumsum(w) / w.sum()
    off = np.expm1(2 * d / t)
    assert (sums[token - 1] if token else 0.0) <= u + off and u <= sums[token] + off
    if prob is not None:
        assert abs(prob - w[token] / w.sum()) <= off


def draft(rs, root, truth, width, nodes, vocab):
    """A tree under `root`: `truth` is one of its paths, the other nodes hang anywhere."""
    tokens, parents, tip = [root], [-1], 0
    truth = list(truth)
    while len(tokens) < nodes:
        on = truth and rs.rand() < 0.6
        tokens.append(truth.pop(0) if on else int(rs.randint(vocab)))
        parents.append(tip if on else int(rs.randint(max(0, len(tokens) - 1 - width), len(tokens) - 1)))
        if on:
            tip = len(tokens) - 1
    return np.array(tokens, np.int32), np.array(parents, np.int32)


def walk(tokens, parents, picked):
    node, out = 0, []
    while True:
        out.append(int(picked[node]))
        node = next((c for c in range(node + 1, len(tokens)) if parents[c] == node and tokens[c] == picked[node]), None)
        if node is None:
            return out


def check_tree(oracle, tree, base, slot, picked, **kw):
    """Every node's choice against the oracle run along its path."""
    tokens, parents = tree
    for i in range(len(tokens)):
        path, j = [], i
        while j >= 0:
            path.append(tokens[j])
            j = parents[j]
        check_choice(feed(oracle, path[::-1], base, slot)[-1], int(picked[i]), **{k: v[i] for k, v in kw.items()})


def guess(model, slot, base, root, n):
    """What a good draft holds: the model's own greedy tokens, computed in a slot of another model."""
    out = []
    for i in range(n):
        root = int(np.argmax(feed(model, [root], base + i, slot)[0]))
        out.append(root)
    return out


KEYS = ["gpt2_int8", "gpt2_fp16", "qwen2_int8", "qwen2_fp16", "qwen2_bf16", "qwen2_yarn_sw_int8"]


@pytest.mark.parametrize("key", KEYS)
def test_greedy_tree_steps(tiny_models, cuda, key):
    spec, path = tiny_models[key]
    rs = np.random.RandomState(3)
    slots, lens = [4, 0, 2], [9, 3, 14]
    with ec.Model(path, batch_cap=6) as m:
        oracle = open_oracle(spec, path, 8)
        base, root = [], []
        for s, n in zip(slots, lens):
            prompt = synth.prompt_ids(spec.vocab, n, seed=s)
            for x in (m, oracle):
                feed(x, prompt[:-1], 0, s)
            base.append(n - 1)
            root.append(int(prompt[-1]))
        taken = 0
        for step in range(4):
            trees = [draft(rs, root[i], guess(oracle, slots[i], base[i], root[i], 4)[: 1 + step], 4, [7, 1, 12][(i + step) % 3], spec.vocab) for i in range(3)]
            out = m.forward_tree(trees, base, slots)
            at = 0
            for i, (tokens, parents) in enumerate(trees):
                picked = out["picked"][at:at + len(tokens)]
                at += len(tokens)
                check_tree(oracle, (tokens, parents), base[i], slots[i], picked)
                assert out["accepted"][i] == walk(tokens, parents, picked)
                feed(oracle, [root[i]] + out["accepted"][i][:-1], base[i], slots[i])
                base[i] += len(out["accepted"][i])
                root[i] = out["accepted"][i][-1]
                taken += len(out["accepted"][i])
        assert taken > 12                      # more than a token a step: drafts were accepted and their rows moved
        # and the plain step goes on from the committed rows
        for i in range(3):
            got, want = feed(m, [root[i]], base[i], slots[i]), feed(oracle, [root[i]], base[i], slots[i])
            assert np.abs(got - want).max() <= TOL * np.abs(want).max()
        oracle.close()


@pytest.mark.parametrize("key", ["gpt2_int8", "qwen2_fp16"])
def test_fork_trees_and_sampled_decode_together(tiny_models, cuda, key):
    """One prompt forked to all slots, trees with drawn choices, then sampled and greedy batched decode."""
    torch = cuda
    spec, path = tiny_models[key]
    rs = np.random.RandomState(5)
    B = 9
    with ec.Model(path, batch_cap=B) as m:
        oracle = open_oracle(spec, path, B)
        prompt = synth.prompt_ids(spec.vocab, 12, seed=1)
        feed(m, prompt[:-1], 0, 7)
        for s in range(B):
            feed(oracle, prompt[:-1], 0, s)
        m.kv_fork(7, [s for s in range(B) if s != 7], 11)
        root, base = [int(prompt[-1])] * B, [11] * B
        for step in range(3):
            trees = [draft(rs, root[s], guess(oracle, s, base[s], root[s], 3), 3, 1 + s, spec.vocab) for s in range(B)]
            rows = sum(len(t) for t, _ in trees)
            u = rs.rand(rows).astype(np.float32)
            temp = rs.choice([0.0, 0.05, 0.5, 1.0], rows).astype(np.float32)
            out = m.forward_tree(trees, base, u=u, temperature=temp)
            at = 0
            for s, (tokens, parents) in enumerate(trees):
                mine = slice(at, at + len(tokens))
                at += len(tokens)
                picked = out["picked"][mine]
                check_tree(oracle, (tokens, parents), base[s], s, picked, t=temp[mine], u=u[mine], prob=out["prob"][mine])
                assert out["accepted"][s] == walk(tokens, parents, picked)
                feed(oracle, [root[s]] + out["accepted"][s][:-1], base[s], s)
                base[s] += len(out["accepted"][s])
                root[s] = out["accepted"][s][-1]
        tok, pos = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (root, base))
        steps = 4
        u = rs.rand(steps, B).astype(np.float32)
        temp = np.array([0.0, 0.3, 1.0] * 3, np.float32)
        ids, prob = torch.full((steps, B), -7, dtype=torch.int32, device="cuda"), torch.full((steps, B), -7.0, device="cuda")
        m.decode_sample(tok, pos, steps, torch.from_numpy(u).cuda(), temperature=torch.from_numpy(temp).cuda(), d_out_ids=ids, d_out_prob=prob)
        torch.cuda.synchronize()
        assert ec.device_error_take() == 0 and m.batch_graph_kernels(2) > 0
        ids, prob = ids.cpu().numpy(), prob.cpu().numpy()
        for i in range(steps):
            for s in range(B):
                check_choice(feed(oracle, [root[s]], base[s], s)[0], int(ids[i, s]), t=temp[s], u=u[i, s], prob=prob[i, s])
                root[s], base[s] = int(ids[i, s]), base[s] + 1
        assert tok.cpu().tolist() == root and pos.cpu().tolist() == base
        greedy = torch.zeros((2, B), dtype=torch.int32, device="cuda")
        m.decode_batch(tok, pos, 2, greedy)
        torch.cuda.synchronize()
        for i in range(2):
            for s in range(B):
                check_choice(feed(oracle, [root[s]], base[s], s)[0], int(greedy[i, s]))
                root[s], base[s] = int(greedy[i, s]), base[s] + 1
        assert ec.device_error_take() == 0
        oracle.close()


@pytest.mark.parametrize("B", [3, 40])
def test_decode_sample_without_settings_and_repeated(tiny_models, cuda, B):
    """temperature 0 is decode_batch; the same u gives the same tokens, whatever call they are split over; settings of a slot
    that keep one token make it the greedy one."""
    torch = cuda
    spec, path = tiny_models["qwen2_int8"]
    prompts = [synth.prompt_ids(spec.vocab, 3 + b % 5, seed=b) for b in range(B)]
    rs = np.random.RandomState(B)
    u = torch.from_numpy(rs.rand(6, B).astype(np.float32)).cuda()

    def decode(call):
        with ec.Model(path, batch_cap=B) as m:
            for b, p in enumerate(prompts):
                feed(m, p[:-1], 0, b)
            tok = torch.tensor([int(p[-1]) for p in prompts], dtype=torch.int32, device="cuda")
            pos = torch.tensor([len(p) - 1 for p in prompts], dtype=torch.int32, device="cuda")
            ids = torch.zeros((6, B), dtype=torch.int32, device="cuda")
            call(m, tok, pos, ids)
            torch.cuda.synchronize()
            assert ec.device_error_take() == 0
            return ids.cpu().numpy()

    zeros, ones = torch.zeros(B, device="cuda"), torch.ones(B, device="cuda")
    cold = decode(lambda m, t, p, o: m.decode_sample(t, p, 6, u, temperature=zeros, d_out_ids=o))
    for kw in (dict(top_k=ones.int()), dict(top_p=zeros), dict(min_p=ones), dict(temperature=zeros, top_p=ones)):
        assert np.array_equal(decode(lambda m, t, p, o: m.decode_sample(t, p, 6, u, d_out_ids=o, **kw)), cold)
    whole = decode(lambda m, t, p, o: m.decode_sample(t, p, 6, u, d_out_ids=o))
    assert not np.array_equal(whole, cold)

    def split(m, t, p, o):
        m.decode_sample(t, p, 2, u, d_out_ids=o)
        m.decode_sample(t, p, 0, u)
        m.decode_sample(t, p, 4, u[2:], d_out_ids=o[2:])
    assert np.array_equal(decode(split), whole)
    if B >= 8:      # both on the per-layer graph, one set of logits
        assert np.array_equal(decode(lambda m, t, p, o: m.decode_batch(t, p, 6, o)), cold)


def test_fork_equals_its_source(tiny_models, cuda):
    spec, path = tiny_models["gpt2_fp16"]
    with ec.Model(path, batch_cap=5) as m:
        prompt = synth.prompt_ids(spec.vocab, 40, seed=2)
        feed(m, prompt, 0, 1)
        free = m.kv_info()["free"]
        m.kv_fork(1, [], 40)
        m.kv_fork(1, [0, 4], 0)
        assert m.kv_info()["free"] == free
        m.kv_fork(1, [0, 4], 40)
        want = feed(m, [5, 6], 40, 1)
        for s in (0, 4):
            assert np.array_equal(feed(m, [5, 6], 40, s), want)
        # the target's rows are its own
        feed(m, prompt[::-1], 0, 0)
        assert np.array_equal(feed(m, [5, 6], 40, 1), want) and np.array_equal(feed(m, [5, 6], 40, 4), want)


def test_refusals_change_nothing(tiny_models, cuda):
    torch = cuda
    spec, path = tiny_models["qwen2_fp16"]
    with ec.Model(path, batch_cap=3) as m:
        prompt = synth.prompt_ids(spec.vocab, 8, seed=2)
        feed(m, prompt, 0, 1)
        free = m.kv_info()["free"]
        one = (np.array([5]), np.array([-1]))
        last = (np.array([5, 6, 7]), np.array([-1, 0, 0]))
        for args, says in ((([one], [8], [3]), "slot 3"), (([one], [8], [-1]), "slot -1"), (([one, one], [8, 8], [1, 1]), "two trees"),
                           (([one], [-1], [1]), "exceed"), (([last], [spec.n_ctx - 2], [1]), "exceed"), (([one], [200], [1]), "eff_ctx|holds fewer"),
                           (([one], [1], [0]), "holds fewer"), (([(np.array([spec.vocab]), np.array([-1]))], [8], [1]), "token id"),
                           (([(np.array([-1]), np.array([-1]))], [8], [1]), "token id"), (([(np.array([1, 2]), np.array([-1, -1]))], [8], [1]), "parent -1"),
                           (([(np.array([1, 2]), np.array([-1, 1]))], [8], [1]), "parent 1"), (([(np.array([1]), np.array([0]))], [8], [1]), "parent 0"),
                           (([one] * 4, [8] * 4, [0, 1, 2, 3]), "n_seq")):
            with pytest.raises(RuntimeError, match=says):
                m.forward_tree(*args)
        with pytest.raises(RuntimeError, match="need u"):
            m.forward_tree([one], [8], [1], temperature=0.5)
        with pytest.raises(RuntimeError, match="max_path"):
            m.forward_tree([one], [8], [1], max_path=0)
        for bad in (dict(u=[0.5, 0.5]), dict(u=0.5, top_k=[1, 2])):
            with pytest.raises(ValueError):
                m.forward_tree([one], [8], [1], **bad)
        with pytest.raises(ValueError):
            m.forward_tree([(np.array([1, 2]), np.array([-1]))], [8], [1])
        with pytest.raises(ValueError):
            m.forward_tree([one], [8, 9], [1])
        for args, says in (((3, [0], 4), "slot 3"), ((-1, [0], 4), "slot -1"), ((1, [3], 4), "slot 3"), ((1, [1], 4), "its own"), ((1, [0, 0], 4), "twice"),
                           ((1, [0], -1), "length"), ((1, [0], spec.n_ctx + 1), "length"), ((0, [1], 1), "holds fewer"), ((1, [0] * 4, 4), "4 slots")):
            with pytest.raises(RuntimeError, match=says):
                m.kv_fork(*args)
        i, f = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(3, device="cuda")
        for args, says in (((i, i, 1, None), "must not be NULL"), ((None, i, 1, f), "must not be NULL"), ((i, i, -1, f), "n_steps"), ((i, i, spec.n_ctx + 1, f), "exceed")):
            with pytest.raises(RuntimeError, match=says):
                m.decode_sample(*args)
        m.set_vocab_shard(0, spec.vocab // 2)
        for call in (lambda: m.forward_tree([one], [8], [1]), lambda: m.forward_tree([one], [8], [1], u=[0.5]), lambda: m.decode_sample(i, i, 1, f)):
            with pytest.raises(RuntimeError, match="shard"):
                call()
        m.set_vocab_shard(0, spec.vocab)
        assert m.kv_info()["free"] == free
        # an empty tree, next to one that is not, and alone
        out = m.forward_tree([(np.zeros(0), np.zeros(0)), last], [0, 8], [2, 1])
        assert out["accepted"][0] == [] and 1 <= len(out["accepted"][1]) <= 2 and len(out["picked"]) == 3
        assert m.forward_tree([(np.zeros(0), np.zeros(0))], [8], [1])["accepted"] == [[]]
        # a shorter path than the tree would give
        best = int(m.forward_tree([one], [8], [1])["picked"][0])
        deep = (np.array([5, best]), np.array([-1, 0]))
        assert len(m.forward_tree([deep], [8], [1])["accepted"][0]) == 2
        assert m.forward_tree([deep], [8], [1], max_path=1)["accepted"] == [[best]]
        with ec.Model(path, batch_cap=3) as other:
            feed(other, prompt, 0, 1)
            want = feed(other, [5], 8, 1)
        assert np.abs(feed(m, [5], 8, 1) - want).max() <= TOL * np.abs(want).max()


@pytest.mark.parametrize("first,then", [(9, 30), (13, 20), (20, 200)])
def test_rows_that_grow_between_calls(tiny_models, cuda, first, then):
    """The argmax workspaces follow a later call of more rows: nothing behind them is written."""
    spec, path = tiny_models["qwen2_fp16"]
    with ec.Model(path, batch_cap=8) as m:
        for rows in (first, then):
            tokens = synth.prompt_ids(spec.vocab, rows, seed=rows)
            args = tokens, np.arange(rows, dtype=np.int32) % 25, np.arange(rows, dtype=np.int32) // 25
            assert np.array_equal(m.forward_argmax(*args)[0], np.argmax(m.forward(*args), axis=1))
        root, flat = (np.array([5]), np.array([-1])), (np.arange(then), np.maximum(np.arange(then) - 1 - np.arange(then) % 3, 0) - (np.arange(then) == 0))
        if then < spec.n_ctx - 25:
            out = m.forward_tree([flat], [min(25, then)], [0])
            assert out["accepted"] == [walk(flat[0], flat[1], out["picked"])]
        assert len(m.forward_tree([root], [min(25, then)], [0])["accepted"][0]) == 1


def test_a_step_does_not_depend_on_earlier_ones(cuda, tmp_path):
    """The same trees on the same caches before and after a step at a longer context: the same choices and probabilities, bit
    for bit, whatever workspace the longer step left behind."""
    spec = synth.TINY_QWEN2.with_(n_embd=512, n_head=4, n_kv_head=2, n_ctx=2048)
    path = synth.ensure_model(spec, tmp_path)
    rs = np.random.RandomState(9)
    B = 17
    with ec.Model(path, batch_cap=B) as m:
        base = [600 + int(rs.randint(0, 250)) for _ in range(B - 1)]
        for s in range(B - 1):
            feed(m, synth.prompt_ids(spec.vocab, base[s], seed=s), 0, s)
        feed(m, synth.prompt_ids(spec.vocab, 1500, seed=99), 0, B - 1)
        trees = [draft(rs, 3 + s, [], 4, 24, spec.vocab) for s in range(B - 1)]
        u, temp = rs.rand(24 * (B - 1)).astype(np.float32), np.full(24 * (B - 1), 0.7, np.float32)
        step = lambda: m.forward_tree(trees, base, u=u, temperature=temp)  # noqa: E731
        first = step()
        m.forward_tree([(np.array([5]), np.array([-1]))], [1500], [B - 1])
        again = step()
        assert np.array_equal(first["picked"], again["picked"]) and first["accepted"] == again["accepted"]
        assert np.array_equal(first["prob"].view(np.int32), again["prob"].view(np.int32))


KERNELS = """
import sys
import numpy as np, torch
from torch.profiler import ProfilerActivity, profile
import edgecore_b200 as ec
B = 160
with ec.Model(sys.argv[1], batch_cap=B) as m:
    m.forward(np.full(B, 5, np.int32), np.zeros(B, np.int32), np.arange(B, dtype=np.int32))
    u = torch.rand(1, B, device="cuda")
    def decode(**kw):
        tok, pos = torch.full((B,), 7, dtype=torch.int32, device="cuda"), torch.ones(B, dtype=torch.int32, device="cuda")
        m.decode_sample(tok, pos, 1, u, **kw)
        torch.cuda.synchronize()
    def step(**kw):
        m.forward_tree([(np.array([7]), np.array([-1]))] * B, np.ones(B, np.int32), u=u[0].cpu().numpy(), temperature=0.7, **kw)
    warm = torch.full((B,), 0.7, device="cuda")
    for call, name in ((lambda: decode(temperature=warm), "decode"), (lambda: decode(temperature=warm, top_p=warm), "decode-cut"),
                       (step, "step"), (lambda: step(top_k=50), "step-cut")):
        call()
        with profile(activities=[ProfilerActivity.CUDA]) as p:
            call()
        print(name, " ".join(sorted({k for e in p.key_averages() for k in ("k_sample_rows", "k_sample<") if k in e.key})) or "-")
"""


def test_many_rows_without_cuts_are_drawn_by_the_row_kernel(cuda, tmp_path):
    """What a caller leaves out reaches the sampler as left out: a batch with a temperature alone takes k_sample_rows, in the
    captured step and in tree steps, and one with top-k or top-p does not.  Kernel names come from the profiler, in a process
    of its own."""
    spec = synth.TINY_QWEN2.with_(vocab=20011)
    path = synth.ensure_model(spec, tmp_path)
    root = str(Path(ec.__file__).resolve().parents[1])
    r = subprocess.run([sys.executable, "-c", KERNELS, str(path)], capture_output=True, text=True, cwd=root, timeout=300)
    assert r.returncode == 0, r.stderr
    said = dict(line.split(" ", 1) for line in r.stdout.splitlines() if line.count(" ") == 1)
    if set(said.values()) == {"-"}:
        pytest.skip("the profiler names no kernels here")
    assert said == {"decode": "k_sample_rows", "decode-cut": "k_sample<", "step": "k_sample_rows", "step-cut": "k_sample<"}


def test_settings_left_out_and_settings_that_are_off(tiny_models, cuda):
    """The same draws, bit for bit, one after the other in one model: a temperature alone, and with top-k and top-p off."""
    torch = cuda
    spec = synth.TINY_QWEN2.with_(vocab=16400)
    B = 150
    rs = np.random.RandomState(12)
    u = torch.from_numpy(rs.rand(3, B).astype(np.float32)).cuda()
    temp = torch.from_numpy(rs.choice([0.0, 0.3, 1.0], B).astype(np.float32)).cuda()
    off = dict(top_k=torch.zeros(B, dtype=torch.int32, device="cuda"), top_p=torch.ones(B, device="cuda"))
    with ec.Model(synth.ensure_model(spec, Path(tiny_models["qwen2_int8"][1]).parent), batch_cap=B) as m:
        feed(m, np.full(60, 5), 0, 0)
        got = []
        for kw in (dict(), off, dict(), dict(top_p=off["top_p"]), off):
            tok = torch.arange(B, dtype=torch.int32, device="cuda")
            pos = torch.zeros(B, dtype=torch.int32, device="cuda")
            ids, prob = torch.zeros((3, B), dtype=torch.int32, device="cuda"), torch.zeros((3, B), device="cuda")
            m.decode_sample(tok, pos, 3, u, temperature=temp, d_out_ids=ids, d_out_prob=prob, **kw)
            torch.cuda.synchronize()
            assert ec.device_error_take() == 0 and m.batch_graph_kernels(2) > 0
            got.append((ids.cpu().numpy(), prob.cpu().numpy().view(np.int32)))
        for ids, prob in got[1:]:
            assert np.array_equal(ids, got[0][0]) and np.array_equal(prob, got[0][1])
        trees = [(np.array([3 + i]), np.array([-1])) for i in range(B)]
        a, b = (m.forward_tree(trees, np.zeros(B), u=u[0].cpu().numpy(), temperature=temp.cpu().numpy(), **kw) for kw in (dict(), dict(top_k=0, top_p=1.0)))
        assert np.array_equal(a["picked"], b["picked"]) and np.array_equal(a["prob"].view(np.int32), b["prob"].view(np.int32))


FEW_ROWS = """
import sys
import numpy as np, torch
from torch.profiler import ProfilerActivity, profile
import edgecore_b200 as ec
with ec.Model(sys.argv[1], batch_cap=3) as m:
    m.forward(np.full(3, 5, np.int32), np.zeros(3, np.int32), np.arange(3, dtype=np.int32))
    u = torch.rand(1, 3, device="cuda")
    def decode():
        tok, pos = torch.full((3,), 7, dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
        m.decode_sample(tok, pos, 1, u)
        torch.cuda.synchronize()
    def step(n, **kw):
        m.forward_tree([(np.arange(n), np.arange(n) - 1)], [1], [1], **kw)
    for name, call in (("decode", decode), ("one", lambda: step(1)), ("seven", lambda: step(7)), ("drawn", lambda: step(3, u=np.full(3, 0.5)))):
        call()
        with profile(activities=[ProfilerActivity.CUDA]) as p:
            call()
        print(name, ",".join(sorted({k for e in p.key_averages() for k in ("k_gemv", "k_gemm_i8", "k_gemm_f", "k_gemm_tc") if k in e.key})) or "-")
"""


@pytest.mark.parametrize("key", ["qwen2_int8", "qwen2_bf16", "gpt2_fp16"])
def test_steps_of_few_rows_stream_their_weights(tiny_models, cuda, key):
    """Below 8 rows the linears and the lm_head of a tree step and of a sampled step are GEMVs, not the tiles for operands
    that the tensor cores do not take."""
    root = str(Path(ec.__file__).resolve().parents[1])
    r = subprocess.run([sys.executable, "-c", FEW_ROWS, str(tiny_models[key][1])], capture_output=True, text=True, cwd=root, timeout=300)
    assert r.returncode == 0, r.stderr
    said = dict(line.split(" ") for line in r.stdout.splitlines() if line.count(" ") == 1)
    if set(said.values()) == {"-"}:
        pytest.skip("the profiler names no kernels here")
    assert said == {k: "k_gemv" for k in ("decode", "one", "seven", "drawn")}
