"""CPU checks of the 4-bit cache: its entry points' refusals before any device
work, the seeded rotation against the oracle's, the plain forms of the measured
operators against their 64-bit definitions, and the tests' own model."""
from __future__ import annotations

import ctypes as C
import sys
from pathlib import Path

import numpy as np
import pytest

import kv_model as M

REPO = Path(__file__).resolve().parents[1]


def desc(uv, **kw):
    from ultravec_ann_b200.kv import uv_kv

    a = dict(device=0, head_dim=128, kv_heads=8, layers=2, page_tokens=64, n_pages=10, max_seqs=4,
             max_pages=5, rounds=1)
    a.update(kw)
    return uv_kv(*a.values())


def test_sizes(uv):
    n = C.c_int64()
    d = desc(uv)
    assert uv.lib().uv_kv_pool_bytes(C.byref(d), C.byref(n)) == 0
    assert n.value == 2 * 10 * 8 * 64 * (64 + 4) * 2  # keys and values: d / 2 bytes and a scale
    assert uv.lib().uv_kv_work_words(C.byref(d), C.byref(n)) == 0
    assert n.value >= 3 * 10 + 2 * 4
    # a table of 2^30 entries is more than 32 bits of bytes
    d = desc(uv, max_seqs=1 << 15, max_pages=1 << 15, n_pages=1 << 20, page_tokens=32)
    assert uv.lib().uv_kv_pool_bytes(C.byref(d), C.byref(n)) == 0
    assert n.value == 2 * (1 << 20) * 8 * 32 * 136


@pytest.mark.parametrize("bad,code", [
    (dict(head_dim=96), 5), (dict(head_dim=0), 5), (dict(page_tokens=48), 5), (dict(page_tokens=0), 5),
    (dict(kv_heads=0), 1), (dict(layers=0), 1), (dict(n_pages=0), 1), (dict(max_seqs=0), 1),
    (dict(max_pages=-1), 1), (dict(rounds=0), 1), (dict(rounds=4), 1),
    (dict(max_seqs=1 << 20, max_pages=1 << 12), 1), (dict(max_pages=1 << 26), 1),
])
def test_unusable_shapes_are_refused(uv, bad, code):
    n = C.c_int64()
    d = desc(uv, **bad)
    L = uv.lib()
    assert L.uv_kv_pool_bytes(C.byref(d), C.byref(n)) == code
    assert L.uv_last_error()
    assert L.uv_kv_seed(C.byref(d), 1) == code
    assert L.uv_kv_extend(C.byref(d), None, None, 0, None) == code
    assert L.uv_kv_attend_bytes(C.byref(d), 1, 1, 1, 8, C.byref(n)) == code


def test_calls_without_buffers_are_refused(uv):
    L, d, n = uv.lib(), desc(uv), C.c_int64()
    assert L.uv_kv_pool_bytes(C.byref(d), None) == 1
    assert L.uv_kv_extend(C.byref(d), None, None, 1, None) == 1
    assert b"null" in L.uv_last_error()
    assert L.uv_kv_reset(C.byref(d), None) == 1
    assert L.uv_kv_check(C.byref(d), None, None) == 1
    assert L.uv_kv_attend_bytes(C.byref(d), 1, 1, 1, 7, C.byref(n)) == 1  # 7 heads over 8
    assert L.uv_kv_attend_bytes(C.byref(d), 1, 1, 0, 8, C.byref(n)) == 1
    p = L.uv_prompt_attention
    none = [None, 0, 0] * 3 + [None, None, None]
    assert p(0, None, None, 1, 5, 5, 4, 2, 96, 1, 0.1, 1, *none) == 5
    assert p(0, None, None, 1, 5, 5, 4, 3, 64, 1, 0.1, 1, *none) == 1
    assert p(0, None, None, 1, 5, 5, 4, 2, 64, 1, 0.1, 9, *none) == 5
    assert p(0, None, None, -1, 5, 5, 4, 2, 64, 1, 0.1, 1, *none) == 1
    assert p(0, None, None, 1, 5, 5, 4, 2, 64, 1, 0.1, 1, *none) == 1
    assert p(0, None, None, 1, 5, 5, 4, 2, 64, 1, -0.1, 1, *none) == 1
    assert p(0, None, None, 0, 0, 0, 4, 2, 64, 1, 0.1, 1, *none) == 0


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_seeded_signs_are_the_codecs(uv, oracle, dim):
    """uv_kv_seed is the codec's rotation (src/lib.rs:428-463)."""
    d = desc(uv, head_dim=dim, rounds=3)
    assert uv.lib().uv_kv_seed(C.byref(d), 42) == 0
    got = [[-1.0 if d.signs[r][i // 32] >> (i % 32) & 1 else 1.0 for i in range(dim)] for r in range(3)]
    want = np.asarray(oracle.Codec(dim, 2, 8).signs()).reshape(-1, dim)[:3]
    np.testing.assert_array_equal(np.array(got), np.sign(want))


def test_the_held_rows_keep_the_estimators_identity():
    """<y, s l> = |y|^2, an orthogonal rotation, and the error of 16 levels."""
    rng = np.random.default_rng(0)
    signs = rng.choice([-1.0, 1.0], (2, 128))
    r = M.rotation(signs)
    np.testing.assert_allclose(r @ r.T, np.eye(128), atol=1e-12)
    x = rng.standard_normal((500, 128))
    level, scale, _ = M.quantise(x, r)
    y = x @ r.T
    np.testing.assert_allclose((level * scale[:, None] * y).sum(1), (y * y).sum(1))
    err = np.square(level * scale[:, None] - y).sum() / np.square(y).sum()
    assert 0.0105 < err < 0.013  # 0.01154 / (1 - 0.01154), over 64000 values
    level, scale, _ = M.quantise(np.zeros((1, 128)), r)
    assert scale[0] == 0


def _operators():
    sys.path.insert(0, str(REPO))
    import perf.operators as ops

    return ops


@pytest.mark.parametrize("seed", range(4))
def test_plain_forms_match_their_definitions(seed):
    """Each kind at a small size: the plain form against exact(), within what the
    output's type and f32 sums allow (a code that flips on an f32 rounding moves a
    value by a step, 0.34 of its row's deviation: few, so the norm tells)."""
    import random

    import torch

    ops = _operators()
    rng = random.Random(seed)
    done = set()
    while len(done) < 4:
        c = ops.draw(rng)
        if c["kind"] in done:
            continue
        done.add(c["kind"])
        c = dict(c, hi=min(c["hi"], 120), seqs=min(c["seqs"], 4))
        c["lo"] = min(c["lo"], c["hi"])
        if c.get("prefix"):
            c["prefix"] = min(c["prefix"], 60)
        if c["kind"] == "append":
            c["q"] = min(c["q"], c["hi"])
        s = ops.prepare(c, seed)
        out = ops.run(s)
        out = [out] if isinstance(out, torch.Tensor) else list(out)
        first = [x.clone() for x in out]
        again = ops.run(s)
        for a, b in zip(first, [again] if isinstance(again, torch.Tensor) else again):
            assert torch.equal(a, b), c
        want = ops.exact(c, seed)
        if want is None:
            continue
        for a, b in zip(first, [want] if isinstance(want, torch.Tensor) else want):
            unit = 2.0 ** -8 if a.dtype == torch.bfloat16 else 2.0 ** -11
            assert float((a.double() - b).norm() / b.norm()) < unit, c


def test_listed_cases_are_named_apart_and_counted():
    ops = _operators()
    cases = ops.listed()
    assert len({c["name"] for c in cases}) == len(cases) <= 12
    assert {c["kind"] for c in cases} == {"attend", "append", "pages", "prompt"}
    for c in cases:
        w = ops.work(c)
        assert w["bytes"] > 0 and w["flops"] >= 0


def test_model_pages_by_hand():
    m = M.Pages(6, 3, 3, 32)
    assert m.extend([1], [40])
    m.fork([1], [0])
    assert m.extend([0, 1], [1, 1]) and m.moves == [(1, 2), (1, 3)] and m.refs.tolist() == [2, 0, 1, 1, 0, 0]
    m.truncate([1], [32])
    assert m.refs.tolist() == [2, 0, 1, 0, 0, 0]
    m.compact()
    assert m.moves == [(2, 1)] and m.table[0].tolist() == [0, 1, -1]
    assert not m.extend([2], [200])
