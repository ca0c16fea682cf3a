"""What the serving operators refuse before anything is launched: every bad argument that the host can see, by its message.
No GPU is needed: the checks of arguments come before the first CUDA call, and a good call on a machine without a device
(or with host memory on one with a device) is refused too."""
from __future__ import annotations

import re
import struct
import subprocess
from pathlib import Path

import numpy as np
import pytest

import edgecore_b200 as ec

torch = pytest.importorskip("torch")


def tree(**kw):
    rows, n, heads, kvh, hd, pages, words = 6, 2, 4, 2, 64, 5, 1
    t = dict(q=torch.zeros(rows, heads * hd, dtype=torch.float16), k=torch.zeros(pages, 64, kvh, hd, dtype=torch.float16),
             v=torch.zeros(pages, 64, kvh, hd, dtype=torch.float16), page_table=torch.zeros(n, 2, dtype=torch.int32),
             row_start=torch.zeros(n + 1, dtype=torch.int32), base=torch.zeros(n, dtype=torch.int32), mask=torch.zeros(rows, words, dtype=torch.int64))
    t["out"] = torch.zeros_like(kw.get("q", t["q"]))
    t.update(kw)
    return ec.tree_attention(**t)


@pytest.mark.parametrize("kw,error,says", [
    (dict(k=torch.zeros(5, 32, 2, 64, dtype=torch.float16)), ValueError, "k and v"),
    (dict(v=torch.zeros(4, 64, 2, 64, dtype=torch.float16)), ValueError, "k and v"),
    (dict(v=torch.zeros(5, 64, 2, 64, dtype=torch.bfloat16)), ValueError, "alike"),
    (dict(out=torch.zeros(6, 256)), ValueError, "q and out"),
    (dict(q=torch.zeros(6, 250, dtype=torch.float16)), ValueError, "250"),
    (dict(q=torch.zeros(6, 2, 128, dtype=torch.float16)), ValueError, "heads of 64"),
    (dict(q=torch.zeros(256, 6, dtype=torch.float16).T), ValueError, "contiguous"),
    (dict(q=torch.zeros(6, 192, dtype=torch.float16)), RuntimeError, "3 query heads over 2"),
    (dict(q=torch.zeros(6, 256, dtype=torch.bfloat16)), RuntimeError, "cache's type"),
    (dict(q=torch.zeros(6, 256, dtype=torch.float64)), RuntimeError, "cache's type"),
    (dict(k=torch.zeros(5, 64, 2, 64), v=torch.zeros(5, 64, 2, 64)), RuntimeError, "fp16 or bf16"),
    (dict(mask=torch.zeros(5, 1, dtype=torch.int64)), ValueError, "mask"),
    (dict(mask=torch.zeros(6, 1, dtype=torch.int32)), ValueError, "mask"),
    (dict(mask=torch.zeros(6, 0, dtype=torch.int64)), RuntimeError, "mask_words"),
    (dict(row_start=torch.zeros(2, dtype=torch.int32)), ValueError, "row_start"),
    (dict(base=torch.zeros(2, dtype=torch.int64)), ValueError, "base"),
    (dict(slots=torch.zeros(3, dtype=torch.int32)), ValueError, "slots"),
    (dict(page_table=torch.zeros(2, 2, dtype=torch.int64)), ValueError, "page_table"),
    (dict(page_table=torch.zeros(2, 4, dtype=torch.int32)[:, :2]), ValueError, "page_table"),
    (dict(window=-1), RuntimeError, "window"),
    (dict(scale=-0.5), RuntimeError, "scale"),
    (dict(scale=float("nan")), RuntimeError, "scale"),
    (dict(workspace=torch.zeros(64, 64)[:, :3]), ValueError, "workspace"),
    (dict(), RuntimeError, "device"),
])
def test_tree_attention(built, kw, error, says):
    with pytest.raises(error, match=says):
        tree(**kw)


@pytest.mark.parametrize("hd", [4, 12, 264])
def test_head_dim(built, hd):
    with pytest.raises(RuntimeError, match="head_dim|aligned"):
        tree(q=torch.zeros(6, 2 * hd, dtype=torch.float16), k=torch.zeros(5, 64, 2, hd, dtype=torch.float16), v=torch.zeros(5, 64, 2, hd, dtype=torch.float16))


def test_nothing_to_do_is_no_error(built):
    e = torch.zeros(0, dtype=torch.int32)
    tree(base=e, row_start=torch.zeros(1, dtype=torch.int32))
    tree(q=torch.zeros(0, 256, dtype=torch.float16), mask=torch.zeros(0, 1, dtype=torch.int64))
    ec.sample(e, torch.zeros(0, 7), torch.zeros(0))
    k = torch.zeros(2, 5, 64, 128, dtype=torch.float16)
    ec.kv_copy(k, k.clone(), torch.zeros(1, 2, dtype=torch.int32), e, e, e, e)


def commit(**kw):
    n, rows = 2, 6
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    k = torch.zeros(3, 5, 64, 128, dtype=torch.float16)
    t = dict(k=k, v=k.clone(), page_table=i(n, 2), row_start=i(n + 1), base=i(n), mask=torch.zeros(rows, 1, dtype=torch.int64), tokens=i(rows), picked=i(rows),
             accepted=i(n, 4), n_accepted=i(n), new_base=i(n))
    t.update(kw)
    ec.tree_commit(**t)


@pytest.mark.parametrize("kw,error,says", [
    (dict(k=torch.zeros(3, 5, 64, 128)), ValueError, "alike"),
    (dict(k=torch.zeros(3, 5, 64, 128), v=torch.zeros(3, 5, 64, 128)), RuntimeError, "fp16 or bf16"),
    (dict(k=torch.zeros(3, 5, 64, 100, dtype=torch.float16), v=torch.zeros(3, 5, 64, 100, dtype=torch.float16)), RuntimeError, "aligned"),
    (dict(picked=torch.zeros(5, dtype=torch.int32)), ValueError, "picked"),
    (dict(accepted=torch.zeros(3, 4, dtype=torch.int32)), ValueError, "accepted"),
    (dict(accepted=torch.zeros(2, 0, dtype=torch.int32)), RuntimeError, "max_path"),
    (dict(n_accepted=torch.zeros(1, dtype=torch.int32)), ValueError, "n_accepted"),
    (dict(new_base=torch.zeros(2)), ValueError, "new_base"),
    (dict(), RuntimeError, "device"),
])
def test_tree_commit(built, kw, error, says):
    with pytest.raises(error, match=says):
        commit(**kw)


@pytest.mark.parametrize("kw,error,says", [
    (dict(dst=torch.zeros(3, dtype=torch.int32)), ValueError, "dst"),
    (dict(start=torch.zeros(2)), ValueError, "start"),
    (dict(end=torch.zeros(4, dtype=torch.int32)[::2]), ValueError, "end"),
    (dict(zip(("src", "dst", "start", "end"), [torch.zeros(4097, dtype=torch.int32)] * 4)), RuntimeError, "4096"),
    (dict(), RuntimeError, "device"),
])
def test_kv_copy(built, kw, error, says):
    i = torch.zeros(2, dtype=torch.int32)
    k = torch.zeros(3, 5, 64, 128, dtype=torch.float16)
    with pytest.raises(error, match=says):
        ec.kv_copy(**(dict(k=k, v=k.clone(), page_table=torch.zeros(2, 2, dtype=torch.int32), src=i, dst=i, start=i, end=i) | kw))


@pytest.mark.parametrize("kw,error,says", [
    (dict(ids=torch.zeros(3, dtype=torch.int64)), ValueError, "ids"),
    (dict(u=torch.zeros(2)), ValueError, "u has"),
    (dict(u=torch.zeros(3, dtype=torch.float64)), ValueError, "u must"),
    (dict(top_k=torch.zeros(3)), ValueError, "top_k"),
    (dict(top_p=torch.zeros(1)), ValueError, "top_p"),
    (dict(min_p=torch.zeros(3, dtype=torch.float16)), ValueError, "min_p"),
    (dict(temperature=torch.zeros(6)[::2]), ValueError, "temperature"),
    (dict(prob=torch.zeros(4)), ValueError, "prob"),
    (dict(logits=torch.zeros(3, 9, dtype=torch.float64)), RuntimeError, "type"),
    (dict(logits=torch.zeros(9, 3).T), ValueError, "logits"),
    (dict(logits=torch.zeros(3, 0)), RuntimeError, "vocab"),
    (dict(logits=torch.zeros(1, 9).expand(3, 9)), RuntimeError, "stride"),
    (dict(), RuntimeError, "device"),
])
def test_sample(built, kw, error, says):
    with pytest.raises(error, match=says):
        ec.sample(**(dict(ids=torch.zeros(3, dtype=torch.int32), logits=torch.zeros(3, 9), u=torch.zeros(3)) | kw))


def test_c_entries_refuse_null(built):
    lib = ec.load_library()
    assert lib.ec_tree_attention(None, None, None) == -1 and "arena" in ec.last_error()
    assert lib.ec_tree_commit(None, None, None) == -1
    assert lib.ec_kv_copy(None, 1, None, None, None, None, None) == -1
    assert lib.ec_sample(None, None, None, 0, 1, 1, 1, None, None, None, None, None, None) == -1
    assert lib.ec_model_kv(None, None) == -1
    k = torch.zeros(1, 5, 64, 128, dtype=torch.float16)
    v, table = k.clone(), torch.zeros(1, 2, dtype=torch.int32)
    kv = ec._layers(k, v, table)
    assert lib.ec_tree_attention(kv, None, None) == -1 and "no arguments" in ec.last_error()
    names = ("k", "v", "ld_layer", "ld_page", "ld_pos", "page_table", "type", "n_layers", "n_pages", "n_slots", "pages_per_slot", "dim")
    path = ec._TREE_PATH.pack(1, 0, 1, 1, *[0] * 9)
    for field, value in (("n_pages", 0), ("pages_per_slot", 1 << 26), ("ld_pos", 120), ("ld_pos", 132), ("k", k.data_ptr() + 2), ("type", 0)):
        bad = list(ec._KV_PAGES.unpack(kv))
        bad[names.index(field)] = value
        assert lib.ec_tree_commit(ec._KV_PAGES.pack(*bad), path, None) == -1, field


def test_packed_structs_are_the_headers(built, tmp_path):
    """The struct formats of the binding against the compiler's layout of the header."""
    fields = {"ec_kv_pages": (ec._KV_PAGES, "k v ld_layer ld_page ld_pos page_table type n_layers n_pages n_slots pages_per_slot dim"),
              "ec_tree_attn": (ec._TREE_ATTN, "q out ldq ldo type n_seq rows n_head n_kv_head head_dim window max_len mask_words scale slots row_start base mask work work_bytes"),
              "ec_tree_path": (ec._TREE_PATH, "n_seq rows mask_words max_path slots row_start base mask tokens picked accepted n_accepted new_base")}
    src = ["#include <stddef.h>", "#include <stdio.h>", '#include "edgecore_b200.h"', "int main(void) {"]
    for name, (_, f) in fields.items():
        src += [f'printf("{name} {k} %zu\\n", offsetof({name}, {k}));' for k in f.split()] + [f'printf("{name} . %zu\\n", sizeof({name}));']
    (tmp_path / "p.c").write_text("\n".join(src + ["return 0; }"]))
    include = Path(ec.__file__).resolve().parents[1] / "include"
    subprocess.run(["gcc", "-I", str(include), "-o", str(tmp_path / "p"), str(tmp_path / "p.c")], check=True)
    said = [line.split() for line in subprocess.run([str(tmp_path / "p")], check=True, capture_output=True, text=True).stdout.splitlines()]
    for name, (fmt, f) in fields.items():
        codes = re.sub(r"(\d+)(.)", lambda m: m[2] * int(m[1]), fmt.format)
        at = {k: struct.calcsize(codes[:i] + "0" + c) for i, (k, c) in enumerate(zip(f.split(), codes))}
        assert len(codes) == len(f.split())
        assert {k: int(v) for n, k, v in said if n == name} == at | {".": fmt.size}


def test_tree_mask():
    m = ec.tree_mask([-1, 0, 0, 1, 3, -1])
    assert m.dtype == np.int64 and m[:, 0].tolist() == [1, 3, 5, 11, 27, 32]
    deep = ec.tree_mask([-1] + list(range(129))).view(np.uint64)
    assert deep.shape == (130, 3) and deep[129].tolist() == [2 ** 64 - 1, 2 ** 64 - 1, 3]
    assert ec.tree_mask([]).shape == (0, 1)
    for bad in ([0], [-2], [-1, 1], [-1, 0, 5]):
        with pytest.raises(ValueError):
            ec.tree_mask(bad)


def test_sample_refuses_a_vocabulary_beyond_shared_memory(built):
    with pytest.raises(RuntimeError, match="750000"):
        ec.sample(torch.zeros(1, dtype=torch.int32), torch.zeros(1, 750001), torch.zeros(1))


def test_model_entries_refuse_a_model_that_is_not_loaded(built):
    lib = ec.load_library()
    assert lib.ec_forward_tree(None, None, None, None, None, None) == -1 and "not loaded" in ec.last_error()
    assert lib.ec_kv_fork(None, 0, None, 0, 0) == -1 and "not loaded" in ec.last_error()
    assert lib.ec_decode_sample(None, None, None, 1, None, None, None, None, None, None, None) == -1 and "not loaded" in ec.last_error()


def test_misaligned_operands_are_refused(built):
    """A pointer that is not aligned to its element would fault in a kernel: refused by name, before anything asks for a device."""
    lib = ec.load_library()
    at = 1 << 20                                  # addresses that are looked at, never read
    i = torch.zeros(1, 2, dtype=torch.int32)
    k = torch.zeros(1, 5, 64, 128, dtype=torch.float16)
    kv = ec._layers(k, k.clone(), i)
    pages = list(ec._KV_PAGES.unpack(kv))
    attn = [at, at, 256, 256, 1, 2, 6, 4, 2, 64, 0, 0, 1, 0.0, at, at, at, at, 0, 0]
    path = [2, 6, 1, 4] + [at] * 9

    def said(call, name):
        assert call() == -1
        assert f": {name} must be aligned" in ec.last_error(), (name, ec.last_error())

    bad_kv = pages.copy()
    bad_kv[5] += 2
    bad_kv = ec._KV_PAGES.pack(*bad_kv)
    said(lambda: lib.ec_tree_attention(bad_kv, ec._TREE_ATTN.pack(*attn), None), "page_table")
    said(lambda: lib.ec_tree_commit(bad_kv, ec._TREE_PATH.pack(*path), None), "page_table")
    said(lambda: lib.ec_kv_copy(bad_kv, 1, at, at, at, at, None), "page_table")
    for n, name in ((14, "slots"), (15, "row_start"), (16, "base"), (17, "mask")):
        for off in ((2, 4) if name == "mask" else (1, 2)):
            args = attn.copy()
            args[n] += off
            said(lambda: lib.ec_tree_attention(kv, ec._TREE_ATTN.pack(*args), None), name)
    for n, name in ((0, "q"), (1, "out")):
        for ty, off in ((1, 1), (0, 2)):
            args = attn.copy()
            args[n] += off
            args[4] = ty
            said(lambda: lib.ec_tree_attention(kv, ec._TREE_ATTN.pack(*args), None), name)
    for n, name in enumerate(("slots", "row_start", "base", "mask", "tokens", "picked", "accepted", "n_accepted", "new_base")):
        args = path.copy()
        args[4 + n] += 4 if name == "mask" else 2
        said(lambda: lib.ec_tree_commit(kv, ec._TREE_PATH.pack(*args), None), name)
    for n, name in enumerate(("src", "dst", "start", "end")):
        args = [at] * 4
        args[n] += 2
        said(lambda: lib.ec_kv_copy(kv, 1, *args, None), name)
    for n, name in enumerate(("ids", "prob", "logits", "temperature", "top_k", "top_p", "min_p", "u")):
        args = {x: at for x in ("ids", "prob", "logits", "temperature", "top_k", "top_p", "min_p", "u")}
        args[name] += 2
        call = lambda ty=0: lib.ec_sample(args["ids"], args["prob"], args["logits"], ty, 9, 3, 9, args["temperature"], args["top_k"], args["top_p"], args["min_p"], args["u"], None)  # noqa: E731
        said(call, name)
    args = {x: at for x in args}
    args["logits"] += 1
    said(lambda: call(2), "logits")
