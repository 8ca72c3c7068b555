"""Rows into and out of the 4-bit cache, and attention over it, against 64-bit
models.  Tolerances follow from the roundings that the kernels document:
queries and weights in 11 bits, outputs in the type's."""
from __future__ import annotations

import math

import numpy as np
import pytest

import kv_model as M

pytestmark = pytest.mark.gpu

UNIT = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}  # half an ulp, relative


def ints(x):
    import torch

    return torch.tensor(np.asarray(x, np.int32), device="cuda")


def starts(counts):
    return ints(np.concatenate([[0], np.cumsum(counts)]))


def cache(uv, d, heads, lens, *, page=64, rounds=1, layers=1, extra=3, seed=7):
    """A cache whose sequences have these lengths, pages in no order, garbage
    (all bits) in every byte that no row has been written to."""
    import torch

    need = sum(-(-n // page) for n in lens) + extra
    c = uv.KvCache(d, heads, need, len(lens) + 1, max(max(lens), 1) + 2 * page, layers=layers,
                   page_tokens=page, rounds=rounds, seed=seed)
    c.pool.fill_(255)  # scales of NaN
    order = np.random.default_rng(seed).permutation(len(lens))
    c.extend(ints(order), ints([lens[i] for i in order]))
    c.check()
    return c, np.array([[-1.0 if c._desc.signs[r][i // 32] >> (i % 32) & 1 else 1.0
                         for i in range(d)] for r in range(rounds)])


def rows_of(rng, n, heads, d, typ, loud=True):
    import torch

    x = rng.standard_normal((n, heads, d))
    if loud:
        x = x * np.exp(0.7 * rng.standard_normal((1, heads, d))) + rng.standard_normal((1, heads, d))
    return torch.tensor(x, dtype=torch.float32, device="cuda").to(getattr(torch, typ))


def f64(x):
    return x.double().cpu().numpy()


def check_rows(c, m_rows, r, seq, first, d):
    """Codes and scales of tokens first .. of a sequence against the model."""
    n = int(c.lens[seq])
    pool, table = c.pool[0].cpu().numpy(), c.table[seq].cpu().numpy()
    for (level, scale), x in zip(M.held(pool, table, n, d), m_rows):
        want, ws, edge = M.quantise(f64(x), r)
        got = level[:, first:].transpose(1, 0, 2)
        # f32 sums of d exact products err by less than d 2^-24 of their sizes
        near = edge < 1e-4
        assert (np.abs(got - want)[~near] == 0).all()
        assert (np.abs(got - want)[near] <= 1).all()
        exact = (got == want).all(-1)
        np.testing.assert_allclose(scale[:, first:].T[exact], ws[exact], rtol=3e-5)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("typ", ["float16", "bfloat16"])
@pytest.mark.parametrize("rounds,page", [(1, 64), (3, 32), (2, 128)])
def test_append_and_read(uv, d, typ, rounds, page):
    import torch

    rng = np.random.default_rng(d + rounds)
    lens, new = [1, 2, 31, 33, 64, 65, 130, 300], [1, 1, 31, 5, 64, 64, 17, 300]
    c, signs = cache(uv, d, 3, lens, page=page, rounds=rounds)
    r = M.rotation(signs)
    order = [3, 0, 7, 2, 1, 6, 5, 4]
    n = [new[i] for i in order]
    k, v = (rows_of(rng, sum(n), 3, d, typ, x) for x in (True, False))
    c.append(ints(order), k, v, starts(n))
    before = c.pool.clone()
    kb, vb = c.read(ints(order), starts(n), sum(n), dtype=k.dtype)
    c.check()
    assert torch.equal(before, c.pool)
    at = 0
    for i, m in zip(order, n):
        check_rows(c, (k[at:at + m], v[at:at + m]), r, i, lens[i] - m, d)
        for (level, scale), got in zip(M.held(c.pool[0].cpu().numpy(), c.table[i].cpu().numpy(),
                                              lens[i], d), (kb, vb)):
            y = (level * scale[..., None])[:, lens[i] - m:].transpose(1, 0, 2)
            want = y @ r
            # f32 arithmetic: d 2^-24 of the row's norm; then the type's rounding
            tol = UNIT[typ] * np.abs(want) + d * 2.0 ** -23 * np.linalg.norm(y, axis=-1, keepdims=True)
            assert (np.abs(f64(got[at:at + m]) - want) <= tol).all()
        at += m


def test_append_writes_its_rows_and_no_other_byte(uv):
    """Tokens at odd places next to others', in pages that end inside a block."""
    import torch

    rng = np.random.default_rng(5)
    lens = [45, 64, 96]
    c, _ = cache(uv, 128, 2, lens, page=32)
    for n in ([45, 64, 96], [1, 1, 1], [3, 2, 33], [7, 64, 1]):
        k, v = (rows_of(rng, sum(n), 2, 128, "bfloat16") for _ in range(2))
        held = [M.held(c.pool[0].cpu().numpy(), c.table[i].cpu().numpy(), lens[i], 128) for i in range(3)]
        c.append(ints([0, 1, 2]), k, v, starts(n))
        for i in range(3):
            now = M.held(c.pool[0].cpu().numpy(), c.table[i].cpu().numpy(), lens[i], 128)
            for (a, s), (b, t) in zip(held[i], now):
                keep = lens[i] - n[i]
                np.testing.assert_array_equal(a[:, :keep], b[:, :keep])
                np.testing.assert_array_equal(s[:, :keep], t[:, :keep])
                assert np.isfinite(t).all()
    # bytes of no token are as they were
    pool = c.pool[0].cpu().numpy()
    (_, ks), (_, vs) = M.unpack(pool[c.table[0, 1].item()][:, 0], 128)
    assert np.isnan(ks[:, 13:]).all() and np.isnan(vs[:, 13:]).all()
    free = np.flatnonzero(c.refs.cpu().numpy() == 0)
    assert (pool[free] == 255).all()


def test_rows_of_zeros_extremes_and_numbers_that_are_none(uv):
    import torch

    c, signs = cache(uv, 128, 1, [8])
    r = M.rotation(signs)
    k = torch.zeros(8, 1, 128, device="cuda")
    k[1, 0, 5] = 1.0
    k[2] = 3.0e38
    k[3] = torch.randn(128, device="cuda") * 1e-30
    k[4] = torch.randn(128, device="cuda") * 1e30
    k[5, 0, 3] = float("inf")
    k[6, 0, 7] = float("nan")
    k[7] = torch.randn(128, device="cuda")
    k = k.bfloat16()
    c.append(ints([0]), k, k, starts([8]))
    kb, vb = c.read(ints([0]), starts([8]), 8)
    for got in (kb, vb):
        x = f64(got)[:, 0]
        assert (x[0] == 0).all()
        assert np.isnan(x[5]).all() and np.isnan(x[6]).all()
        for i in (1, 3, 4, 7):
            want = f64(k)[i, 0]
            # <x, held> = |x|^2 by the scale's definition, to the rounding of the values read
            assert abs(x[i] @ want / (want @ want) - 1) < 1e-2
    check_rows(c, (k[7:], k[7:]), r, 0, 7, 128)


def test_entries_without_rows_in_an_append(uv):
    """A forked sequence that idles in a step: its last page stays shared, and the
    other entries' rows are written."""
    import torch

    rng = np.random.default_rng(21)
    for n in (69, 70, 79, 81):
        c, signs = cache(uv, 64, 2, [n, 40], extra=9)
        c.fork(ints([0]), ints([2]))
        k, v = (rows_of(rng, 3, 2, 64, "float16") for _ in range(2))
        for order, counts, at in (([1, 2], [3, 0], [0, 3, 3]), ([2, 1], [0, 3], [0, 0, 3])):
            c.extend(ints(order), ints(counts))
            c.append(ints(order), k, v, ints(at))
            c.check()
            check_rows(c, (k, v), M.rotation(signs), 1, int(c.lens[1]) - 3, 64)
        before = c.pool.clone()
        c.append(ints([0, 2]), k[:0], v[:0], ints([0, 0, 0]))
        c.check()
        assert torch.equal(before, c.pool)


@pytest.mark.parametrize("bad,counts,status", [
    ([0, 9, 1], [40, 5, 70], 2),       # out of range
    ([0, -1, 1], [40, 5, 70], 2),
    ([0, 1, 0], [40, 70, 40], 2),      # listed twice
    ([1, 0, 1], [70, 1, 0], 2),
    ([0, 2, 1], [40, 6, 70], 16),      # its last page is shared
    ([0, 3, 1], [40, 1, 70], 16),
    ([2, 9, 2], [6, 5, 6], 2 | 16),
    ([0, 1, 2], [40, 70, 100], 16),    # a page before the last
])
def test_an_append_with_a_bad_entry_writes_nothing(uv, bad, counts, status):
    import torch

    rng = np.random.default_rng(22)
    c, signs = cache(uv, 128, 2, [40, 70, 100, 0, 0], extra=9)
    c.fork(ints([2]), ints([3]))
    k, v = (rows_of(rng, sum(counts), 2, 128, "bfloat16") for _ in range(2))
    before = c.pool.clone()
    for _ in range(3):
        c.append(ints(bad), k, v, starts(counts))
        c.append(ints([0]), k[:1], v[:1])  # stopped by the status
    assert torch.equal(before, c.pool)
    with pytest.raises(uv.KvError) as e:
        c.check()
    assert e.value.status == status
    k, v = (rows_of(rng, 74, 2, 128, "bfloat16") for _ in range(2))
    c.append(ints([1, 0]), k, v, starts([70, 4]))
    c.check()
    check_rows(c, (k[:70], v[:70]), M.rotation(signs), 1, 0, 128)


def test_an_append_looks_over_more_entries_than_threads(uv):
    import torch

    rng = np.random.default_rng(23)
    m = 2100
    c = uv.KvCache(64, 1, 2 * m + 10, m + 1, 96, page_tokens=32)
    n = [int(x) for x in rng.integers(0, 70, m)]
    order = [int(x) for x in rng.permutation(m)]
    c.extend(ints(order), ints([n[i] for i in order]))
    some = [min(n[i], int(x)) for i, x in zip(order, rng.integers(0, 70, m))]
    k, v = (rows_of(rng, sum(some), 1, 64, "float16") for _ in range(2))
    c.append(ints(order), k, v, starts(some))
    c.check()
    kb, vb = c.read(ints(order), starts(some), sum(some))
    for x, y in ((k, kb), (v, vb)):
        assert float((x.double() - y.double()).norm() / x.double().norm()) < 0.13  # 4 bits: 0.107
    before = c.pool.clone()
    c.append(ints(order[:-1] + order[5:6]), k, v, starts(some))
    with pytest.raises(uv.KvError) as e:
        c.check()
    assert e.value.status == 2 and torch.equal(before, c.pool)


@pytest.mark.parametrize("d,rounds", [(64, 1), (128, 1), (256, 1), (128, 2), (256, 3)])
def test_rows_near_the_largest_number(uv, d, rounds):
    """Rows whose transform would pass the largest float before it is scaled."""
    import torch

    rng = np.random.default_rng(24)
    sizes = [1e30, 1e34, 1e36, 1e37, 3e38, 1.0, 1e-30, 1e37, 3.3e38]
    c, signs = cache(uv, d, 1, [len(sizes)], rounds=rounds)
    r = M.rotation(signs)
    k = rows_of(rng, len(sizes), 1, d, "float32", False).double()
    k = k / k.abs().amax(-1, keepdim=True) * torch.tensor(sizes, device="cuda", dtype=torch.float64)[:, None, None]
    k[4] = 3e38  # as large in every dimension: one entry of the transform is sqrt(d) times that
    k[7, 0, 1:] = 0
    k = k.float().bfloat16()
    v = k.flip(0).contiguous()
    c.append(ints([0]), k, v, starts([len(sizes)]))
    c.check()
    check_rows(c, (k, v), r, 0, 0, d)
    assert bool(torch.isfinite(held_scales(c, d)).all())


def held_scales(c, d):
    """The scales of a cache's first sequence, keys and values."""
    import torch

    n = int(c.lens[0])
    (_, ks), (_, vs) = M.held(c.pool[0].cpu().numpy(), c.table[0].cpu().numpy(), n, d)
    return torch.tensor(np.stack([ks, vs]))


def test_strided_rows_and_other_orders(uv):
    """Heads before rows, rows of a wider tensor, a misaligned view."""
    import torch

    rng = np.random.default_rng(11)
    a, _ = cache(uv, 64, 4, [50, 20])
    b, _ = cache(uv, 64, 4, [50, 20])
    k, v = (rows_of(rng, 70, 4, 64, "float16") for _ in range(2))
    n = starts([50, 20])
    a.append(ints([0, 1]), k, v, n)
    wide = torch.zeros(70, 4, 200, dtype=torch.float16, device="cuda")
    wide[:, :, 8:72] = k
    turned = v.transpose(0, 1).contiguous().transpose(0, 1)
    b.append(ints([0, 1]), wide[:, :, 8:72], turned, n)
    assert torch.equal(a.pool, b.pool)
    b.pool.fill_(255)
    wide[:, :, 3:67] = k
    b.append(ints([0, 1]), wide[:, :, 3:67], turned, n)
    assert torch.equal(a.pool, b.pool)
    q = rows_of(rng, 70, 8, 64, "float16", False)
    want = a.attend(ints([0, 1]), q, n, 50)
    wide = torch.zeros(8, 70, 136, dtype=torch.float16, device="cuda")
    wide[:, :, 64:128] = q.transpose(0, 1)
    assert torch.equal(want, a.attend(ints([0, 1]), wide[:, :, 64:128].transpose(0, 1), n, 50))


def fill(c, lens, d, heads, typ, rng):
    for i, n in enumerate(lens):
        if n:
            k, v = (rows_of(rng, n, heads, d, typ) for _ in range(2))
            c.append(ints([i]), k, v, starts([n]))
    c.check()


def attend_tolerance(out, size, reach, typ):
    """Scores err by 2^-11 of sum |q_i k_i| (the rounded query; f32 sums and the
    exponential add less than a sixteenth of that), weights by 2^-11 more; each
    weight's error counts once in the numerator and once in the sum.  The way
    back through two bfloats a value adds 2^-16 of the norm."""
    eps = 2 * (1.07 * 2.0 ** -11 * reach + 2.0 ** -11 + 2.0 ** -16)
    return np.maximum(eps * size, 2.0 ** -24)[..., None] + (UNIT[typ] + 2.0 ** -16) * np.abs(out) * 1.01


CASES = [  # d, kv heads, group, lens, rows of each, page, rounds, type
    (64, 2, 4, [300], [1], 64, 1, "float16"),
    (128, 2, 8, [1, 31, 32, 33, 700, 64], [1] * 6, 64, 1, "bfloat16"),
    (128, 1, 1, [5, 129], [5, 3], 32, 1, "float16"),
    (128, 2, 5, [40, 200, 90, 7], [4, 1, 9, 7], 128, 3, "bfloat16"),
    (256, 1, 3, [33, 260], [2, 4], 64, 1, "float16"),
    (64, 1, 16, [100, 65, 2], [3, 8, 1], 32, 2, "bfloat16"),
    (64, 3, 40, [90], [1], 64, 1, "float16"),
    (128, 1, 6, [150], [70], 64, 1, "float16"),
]


@pytest.mark.parametrize("d,heads,group,lens,rows,page,rounds,typ", CASES)
def test_attend(uv, d, heads, group, lens, rows, page, rounds, typ):
    rng = np.random.default_rng(len(lens) + d)
    c, signs = cache(uv, d, heads, lens, page=page, rounds=rounds)
    fill(c, lens, d, heads, typ, rng)
    r = M.rotation(signs)
    order = list(rng.permutation(len(lens)))
    n = [rows[i] for i in order]
    q = rows_of(rng, sum(n), heads * group, d, typ, False)
    one = all(x == 1 for x in n)
    out, lse = c.attend(ints(order), q, None if one else starts(n), max(n), lse=True)
    scale, at = 1 / math.sqrt(d), 0
    pool = c.pool[0].cpu().numpy()
    for i, m in zip(order, n):
        want, wl, size, reach = M.attend(f64(q[at:at + m]),
                                         M.held(pool, c.table[i].cpu().numpy(), lens[i], d), r, scale)
        got = f64(out[at:at + m])
        tol = attend_tolerance(want, size, reach, typ)
        assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())
        seen = np.isfinite(wl)
        assert (np.abs(f64(lse[at:at + m]) - wl)[seen] <= (1.07 * 2.0 ** -11 * reach + 1e-5)[seen]).all()
        at += m
    c.check()


def test_attend_rows_that_see_nothing(uv):
    """More rows than tokens, an empty sequence, a sequence out of range."""
    rng = np.random.default_rng(2)
    c, signs = cache(uv, 128, 2, [0, 3, 70])
    fill(c, [0, 3, 70], 128, 2, "bfloat16", rng)
    q = rows_of(rng, 12, 4, 128, "bfloat16", False)
    out, lse = c.attend(ints([0, 1, 99, 2]), q, starts([2, 5, 3, 2]), 5, lse=True)
    assert (f64(out)[[0, 1, 2, 3, 7, 8, 9]] == 0).all()
    assert np.isneginf(f64(lse)[[0, 1, 2, 3, 7, 8, 9]]).all()
    r = M.rotation(signs)
    for at, m, s, n in ((4, 3, 1, 3), (10, 2, 2, 70)):
        want, _, size, reach = M.attend(f64(q[at:at + m]), M.held(
            c.pool[0].cpu().numpy(), c.table[s].cpu().numpy(), n, 128), r, 1 / math.sqrt(128))
        assert (np.abs(f64(out[at:at + m]) - want) <= attend_tolerance(want, size, reach, "bfloat16")).all()


def test_what_a_row_does_not_see_does_not_reach_it(uv):
    """Later rows' keys and values of infinity and NaN, and very large ones."""
    import torch

    rng = np.random.default_rng(3)
    lens = [80]
    q = rows_of(rng, 6, 4, 128, "bfloat16", False)
    k, v = (rows_of(rng, 80, 2, 128, "bfloat16") for _ in range(2))
    c, _ = cache(uv, 128, 2, lens)
    c.append(ints([0]), k, v, starts([80]))
    want = c.attend(ints([0]), q, starts([6]), 6)
    for bad in (float("inf"), float("nan"), 3e38, -3e38):
        for x in (0, 1):
            kk, vv = k.clone(), v.clone()
            (kk, vv)[x][77:, :, 9] = bad
            c.append(ints([0]), kk, vv, starts([80]))
            got = c.attend(ints([0]), q, starts([6]), 6)
            assert torch.equal(got[:3], want[:3])
            if not math.isfinite(bad):
                assert bool(got[3:].isnan().any())


def test_scores_and_values_of_every_size(uv):
    """Scores of +-thousands, and value scales that grow by 2^60 along the sequence."""
    import torch

    rng = np.random.default_rng(4)
    c, signs = cache(uv, 64, 1, [500])
    r = M.rotation(signs)
    k, v = (rows_of(rng, 500, 1, 64, "bfloat16") for _ in range(2))
    k = (k.float() * torch.linspace(0.01, 300, 500, device="cuda")[:, None, None]).bfloat16()
    v = (v.float() * torch.exp2(torch.linspace(-30, 30, 500, device="cuda"))[:, None, None]).bfloat16()
    c.append(ints([0]), k, v, starts([500]))
    q = rows_of(rng, 500, 2, 64, "bfloat16", False)
    out = c.attend(ints([0]), q, starts([500]), 500)
    want, _, size, reach = M.attend(f64(q), M.held(c.pool[0].cpu().numpy(), c.table[0].cpu().numpy(),
                                                   500, 64), r, 0.125)
    # a weight below 2^-24 of the largest scaled one is lost: 500 of them at most
    eps = np.expm1(np.minimum(2 * 1.07 * 2.0 ** -11 * reach, 50)) + 2.0 ** -9
    tol = eps[..., None] * size[..., None] + 2.0 ** -8 * np.abs(want) * 1.01
    assert np.isfinite(f64(out)).all()
    assert (np.abs(f64(out) - want) <= tol).all()


def test_one_long_sequence_and_many_ragged_ones_split_alike(uv):
    """The same rows give the same bits, whoever shares the call (one part), and
    the split's sums stay within the tolerance of the other order."""
    import torch

    rng = np.random.default_rng(8)
    lens = [20_000, 1, 900, 4000, 33]
    c, signs = cache(uv, 128, 2, lens)
    fill(c, lens, 128, 2, "bfloat16", rng)
    q = rows_of(rng, 5, 16, 128, "bfloat16", False)
    every = ints([0, 1, 2, 3, 4])
    out = c.attend(every, q)
    for _ in range(3):
        assert torch.equal(out, c.attend(every, q))  # no atomics: no order
    r, pool = M.rotation(signs), c.pool[0].cpu().numpy()
    for i, n in enumerate(lens):
        want, _, size, reach = M.attend(f64(q[i:i + 1]), M.held(pool, c.table[i].cpu().numpy(), n, 128),
                                        r, 1 / math.sqrt(128))
        assert (np.abs(f64(out[i:i + 1]) - want) <= attend_tolerance(want, size, reach, "bfloat16")).all()
        alone = c.attend(ints([i]), q[i:i + 1].contiguous())
        assert (np.abs(f64(alone) - want) <= attend_tolerance(want, size, reach, "bfloat16")).all()


@pytest.mark.parametrize("n,rounds", [(40, 1), (5000, 1), (5000, 3)])
def test_values_near_the_largest_number(uv, n, rounds):
    """Sums of thousands of them are beyond a float; their means are not."""
    import torch

    rng = np.random.default_rng(26)
    d = 128
    c, signs = cache(uv, d, 1, [n], rounds=rounds)
    k, v = (rows_of(rng, n, 1, d, "float32", False) for _ in range(2))
    v = (v.clamp(-3, 3) + 0.5) * 1e37
    c.append(ints([0]), k.bfloat16(), v.bfloat16(), starts([n]))
    q = rows_of(rng, 2, 4, d, "bfloat16", False) * 0.5
    out = c.attend(ints([0]), q, starts([2]), 2)
    want, _, size, reach = M.attend(f64(q), M.held(c.pool[0].cpu().numpy(), c.table[0].cpu().numpy(), n, d),
                                    M.rotation(signs), 1 / math.sqrt(d))
    assert (np.abs(f64(out) - want) <= attend_tolerance(want, size, reach, "bfloat16")).all()


@pytest.mark.parametrize("lens", [[1], [40], [6000], [20_000, 3]])
def test_queries_and_keys_that_are_no_numbers(uv, lens):
    """NaN in a query makes its own row NaN and no other, however its job is split;
    so does a key of NaN for the rows that see it."""
    import torch

    rng = np.random.default_rng(27)
    c, _ = cache(uv, 128, 1, lens)
    fill(c, lens, 128, 1, "bfloat16", rng)
    n, seqs = len(lens), ints(range(len(lens)))
    q = rows_of(rng, n, 8, 128, "bfloat16", False)
    want, sums = c.attend(seqs, q, lse=True)
    for bad in (math.nan, math.inf):
        x = q.clone()
        x[0, 2, 5] = bad
        got, lse = c.attend(seqs, x, lse=True)
        assert bool(got[0, 2].isnan().all()) and bool(lse[0, 2].isnan())
        for a, b in ((got, want), (lse, sums)):
            a[0, 2] = b[0, 2]
            assert torch.equal(a, b)
    k = rows_of(rng, 1, 1, 128, "bfloat16")
    for bad in (math.nan, math.inf):
        k[0, 0, 9] = bad
        c.append(ints([0]), k, torch.zeros_like(k))
        got, lse = c.attend(seqs, q, lse=True)
        assert bool(got[0].isnan().all()) and bool(lse[0].isnan().all())
        assert torch.equal(got[1:], want[1:]) and torch.equal(lse[1:], sums[1:])
    c.check()


def crowd(uv, d, n, many):
    """A cache of one head whose first sequence has n tokens; `many` in all share its
    pages, so that a warp goes through many tiles of a job."""
    c = uv.KvCache(d, 1, -(-n // 64) + 2, many, n + 64, seed=7)
    c.extend(ints([0]), ints([n]))
    c.check()
    signs = np.array([[-1.0 if c._desc.signs[0][i // 32] >> (i % 32) & 1 else 1.0 for i in range(d)]])
    return Shared(c, many), signs


class Shared:
    """Appends while the first sequence is alone, attends with everyone."""

    def __init__(self, c, many):
        self.c, self.rest = c, ints(range(1, many))
        self.pool, self.table = c.pool, c.table

    def append(self, *a):
        self.c.free(self.rest)
        self.c.append(*a)
        self.c.fork(ints([0] * len(self.rest)), self.rest)

    def attend(self, *a):
        return self.c.attend(*a)

    def check(self):
        self.c.check()


@pytest.mark.parametrize("d,group", [(64, 2), (128, 1), (128, 4), (256, 2)])
@pytest.mark.parametrize("typ", ["float16", "bfloat16"])
def test_values_beside_larger_ones_of_no_weight(uv, typ, d, group):
    """A token of negligible weight whose values are 2^12 to 2^40 times the others'
    takes nothing from them: the bound is that of the roundings, which is of the
    weighted values' size."""
    import torch

    rng = np.random.default_rng(d + group)
    n = 300
    c, signs = crowd(uv, d, n, 400)
    r = M.rotation(signs)
    for at, size in ((0, 2.0 ** 12), (17, 2.0 ** 14), (40, 2.0 ** 15), (150, 2.0 ** 20), (290, 2.0 ** 24), (31, 2.0 ** 40)):
        k, v = (rows_of(rng, n, 1, d, "bfloat16", False) * 0.3 for _ in range(2))
        k[:, :, 0] = 0
        k[at, :, 0] = -90 * math.sqrt(d) / 4
        v[at] = v[at] * size
        c.append(ints([0]), k, v, starts([n]))
        q = rows_of(rng, 3, group, d, typ, False) * 0.3
        q[:, :, 0] = 4
        out = c.attend(ints(range(400)), q.repeat(400, 1, 1), starts([3] * 400), 3)
        want, _, big, reach = M.attend(f64(q), M.held(c.pool[0].cpu().numpy(), c.table[0].cpu().numpy(), n, d),
                                       r, 1 / math.sqrt(d))
        # the scores that count are those of keys that weigh: reach without the odd one
        near = M.held(c.pool[0].cpu().numpy(), c.table[0].cpu().numpy(), n, d)
        near[0][1][:, at] = 0
        reach = M.attend(f64(q), near, r, 1 / math.sqrt(d))[3]
        err = np.abs(f64(out).reshape(400, *want.shape) - want)
        assert (err <= attend_tolerance(want, big, reach, typ)).all(), (at, size)
    c.check()


@pytest.mark.parametrize("typ", ["float16", "bfloat16"])
@pytest.mark.parametrize("up", [True, False])
def test_weights_and_values_that_run_against_each_other(uv, typ, up):
    """Scores rise by 40 nats along 500 tokens while the values shrink as much (or
    the reverse), so that every token adds as much to the output."""
    import torch

    rng = np.random.default_rng(25)
    n, d = 500, 64
    c, signs = crowd(uv, d, n, 400)
    r = M.rotation(signs)
    climb = torch.linspace(-20, 20, n, device="cuda") * (1 if up else -1)
    k, v = (rows_of(rng, n, 1, d, "float32", False) for _ in range(2))
    q = rows_of(rng, 4, 2, d, "float32", False) * 0.1
    q[:, :, 0] = 4
    k *= 0.05
    k[:, 0, 0] = climb * math.sqrt(d) / 4
    q, k = q.to(getattr(torch, typ)), k.bfloat16()
    c.append(ints([0]), k, k, starts([n]))
    (kl, ks), _ = M.held(c.pool[0].cpu().numpy(), c.table[0].cpu().numpy(), n, d)
    e = (kl[0] * ks[0][:, None]) @ (f64(q)[0, 0] @ r.T) / math.sqrt(d)  # what the held keys score
    v = ((1 + 0.3 * v.double()) * torch.tensor(1e7 * np.exp(-e), device="cuda")[:, None, None]).bfloat16()
    c.append(ints([0]), k, v, starts([n]))
    out = c.attend(ints(range(400)), q.repeat(400, 1, 1), starts([4] * 400), 4)
    held = M.held(c.pool[0].cpu().numpy(), c.table[0].cpu().numpy(), n, d)
    want, _, size, reach = M.attend(f64(q), held, r, 1 / math.sqrt(d))
    err = np.abs(f64(out).reshape(400, *want.shape) - want)
    assert (err <= attend_tolerance(want, size, reach, typ)).all()
    c.check()


@pytest.mark.parametrize("lens", [[20_000], [9000, 40, 7000, 300], [2500] * 24])
def test_every_split_job_is_joined_every_time(uv, lens):
    """Outputs that hold NaN before the call have the same bits after each of many
    calls: of the blocks that share a job (one to two hundred, finishing
    together), some one joins it, every time."""
    import torch

    rng = np.random.default_rng(len(lens))
    heads, d = 2, 128
    c, _ = cache(uv, d, heads, lens)
    fill(c, lens, d, heads, "bfloat16", rng)
    n = len(lens)
    q = rows_of(rng, n, 4 * heads, d, "bfloat16", False)
    seqs, L, st = ints(range(n)), uv.lib(), torch.cuda.current_stream().cuda_stream
    want, sums = c.attend(seqs, q, lse=True)
    out, lse, missed = torch.empty_like(want), torch.empty_like(sums), torch.zeros((), device="cuda")
    scratch = torch.zeros(1 << 24, dtype=torch.uint8, device="cuda")
    for _ in range(1500):
        out.fill_(math.nan)
        lse.fill_(math.nan)
        assert L.uv_kv_attend(c._p, 0, seqs.data_ptr(), None, n, n, 1, 1, q.data_ptr(), 4 * heads * d, d, 4 * heads,
                              1 / math.sqrt(d), out.data_ptr(), lse.data_ptr(), scratch.data_ptr(),
                              scratch.numel(), st) == 0
        missed += (out != want).any() | (lse != sums).any()
    assert int(missed) == 0
    c.check()


@pytest.mark.parametrize("typ", ["float16", "bfloat16"])
def test_a_long_flat_sequence(uv, typ):
    """150,001 tokens of nearly equal weight: the outputs are 1 / 80 of a value,
    so what the sums lose of codes that all are positive would show."""
    import torch

    n, d = 150_001, 128
    c = uv.KvCache(d, 1, 2400, 2, n, page_tokens=64)
    c.extend(ints([1]), ints([n]))
    c.check()
    g = torch.Generator(device="cuda").manual_seed(3)
    tiles = c.pool[0]
    half = 32 * d // 2
    for at, size in ((0, 0.05), (half + 128, 1.0)):
        code = (torch.randn(*tiles.shape[:-1], 32 * d, generator=g, device="cuda") / 0.3352).floor().add(8)
        code = code.clamp(0, 15).to(torch.uint8)
        tiles[..., at:at + half] = code[..., 0::2] | (code[..., 1::2] << 4)
        scale = size * 0.3352 * torch.exp(0.2 * torch.randn(*tiles.shape[:-1], 32, generator=g, device="cuda"))
        tiles[..., at + half:at + half + 128] = scale.view(torch.uint8)
    signs = np.array([[-1.0 if c._desc.signs[0][i // 32] >> (i % 32) & 1 else 1.0 for i in range(d)]])
    q = rows_of(np.random.default_rng(0), 2, 4, d, typ, False)
    out = c.attend(ints([1]), q, starts([2]), 2)
    want, _, size, reach = M.attend(f64(q), M.held(tiles.cpu().numpy(), c.table[1].cpu().numpy(), n, d),
                                    M.rotation(signs), 1 / math.sqrt(d))
    err = np.abs(f64(out) - want)
    assert (err <= attend_tolerance(want, size, reach, typ)).all()
    # the roundings of 150,000 weights are independent, so their sum is far below
    # the bound: a tenth of the output's size would be a lost sum
    assert np.linalg.norm(err) < 0.1 * np.linalg.norm(want)
    c.check()


def test_pools_beyond_32_bits_of_bytes_and_other_layers(uv):
    import torch

    heads, d, page = 8, 128, 64
    n_pages = 70_000  # 69632 bytes each: 4.9 GB
    c = uv.KvCache(d, heads, n_pages, 4, 2000, layers=1, page_tokens=page)
    c.refs[: n_pages - 40] = 1  # somebody else's
    c2 = uv.KvCache.over(c.pool, c.table, c.lens, c.refs, head_dim=d, page_tokens=page,
                         signs=torch.ones(1, d))
    c2.extend(ints([1]), ints([900]))
    c2.check()
    assert int(c2.table[1, 0]) == n_pages - 40
    rng = np.random.default_rng(1)
    k, v = (rows_of(rng, 900, heads, d, "bfloat16") for _ in range(2))
    c2.append(ints([1]), k, v, starts([900]))
    kb, vb = c2.read(ints([1]), starts([900]), 900)
    for x, y in ((k, kb), (v, vb)):
        assert float(((x.double() - y.double()).norm() / x.double().norm())) < 0.13  # 4 bits: 0.107
    q = rows_of(rng, 1, 16, d, "bfloat16", False)
    out = c2.attend(ints([1]), q)
    small, _ = uv.KvCache(d, heads, 20, 4, 2000, layers=3, page_tokens=page), None
    small.extend(ints([2]), ints([900]))
    for r in range(3):
        for w in range(8):
            small._desc.signs[r][w] = 0
    small.pool.fill_(255)
    small.append(ints([2]), k, v, starts([900]), layer=1)
    small.check()
    assert torch.equal(out, small.attend(ints([2]), q, layer=1))
    assert bool((small.pool[0] == 255).all()) and bool((small.pool[2] == 255).all())
    del c, c2


def test_append_refuses_shared_pages_and_unknown_sequences(uv):
    rng = np.random.default_rng(6)
    c, _ = cache(uv, 64, 1, [70])
    k = rows_of(rng, 1, 1, 64, "float16")
    c.fork(ints([0]), ints([1]))
    before = c.pool.clone()
    c.append(ints([1]), k, k)
    with pytest.raises(uv.KvError) as e:
        c.check()
    assert e.value.status == 16 and bool((before == c.pool).all())
    c.append(ints([9]), k, k)
    with pytest.raises(uv.KvError) as e:
        c.check()
    assert e.value.status == 2 and bool((before == c.pool).all())
    # an extend that found no page stops the rows that were meant for it
    c.extend(ints([1]), ints([100_000]))
    c.append(ints([0]), k, k)
    with pytest.raises(uv.KvError) as e:
        c.check()
    assert e.value.status == 4 and bool((before == c.pool).all())


def test_other_streams_and_graphs(uv):
    import torch

    rng = np.random.default_rng(12)
    lens = [100, 40]
    c, _ = cache(uv, 128, 2, lens)
    fill(c, lens, 128, 2, "bfloat16", rng)
    q = rows_of(rng, 2, 8, 128, "bfloat16", False)
    k = rows_of(rng, 2, 2, 128, "bfloat16")
    s, one = ints([0, 1]), ints([1, 1])
    twin, _ = cache(uv, 128, 2, lens)
    twin.pool.copy_(c.pool)
    want = []
    for _ in range(4):
        twin.extend(s, one)
        twin.append(s, k, k)
        want.append(twin.attend(s, q))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.extend(s, one)
        c.append(s, k, k)
        assert torch.equal(c.attend(s, q), want[0])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.extend(s, one)
        c.append(s, k, k)
        out = c.attend(s, q)
    for i in range(1, 4):
        graph.replay()
        assert torch.equal(out, want[i])
    c.check()


def test_scratch_of_the_library_and_refused_arguments(uv):
    import ctypes as C

    import torch

    rng = np.random.default_rng(13)
    c, _ = cache(uv, 128, 2, [50])
    fill(c, [50], 128, 2, "bfloat16", rng)
    q = rows_of(rng, 1, 4, 128, "bfloat16", False)
    want, seqs = c.attend(ints([0]), q), ints([0])
    out = torch.zeros_like(q)
    st = torch.cuda.current_stream().cuda_stream

    def call(**kw):
        a = dict(kv=c._p, layer=0, seqs=seqs.data_ptr(), starts=None, n=1, rows=1, most=1, dtype=1,
                 q=q.data_ptr(), qr=512, qh=128, heads=4, scale=1 / math.sqrt(128), out=out.data_ptr(),
                 lse=None, scratch=None, size=0, stream=st)
        a.update(kw)
        return uv.lib().uv_kv_attend(*a.values())

    assert call() == 0
    assert torch.equal(out, want)
    for bad in (dict(layer=1), dict(layer=-1), dict(n=-1), dict(n=9), dict(rows=2), dict(dtype=7),
                dict(q=None), dict(q=q.data_ptr() + 2), dict(qr=3), dict(heads=3), dict(heads=0),
                dict(out=None), dict(most=0), dict(seqs=None), dict(scratch=out.data_ptr(), size=4),
                dict(q=np.zeros(512, np.int16).ctypes.data)):
        assert call(**bad) in (1, 5), bad
    assert call(n=0, rows=0) == 0
    for bad in (q.float(), q[0], q[:, :, :64], q[:, :3]):
        with pytest.raises((ValueError, uv.UVError)):
            c.attend(ints([0]), bad)
    with pytest.raises(ValueError):
        c.append(ints([0]), q, q)
    with pytest.raises(uv.UVError):
        uv.KvCache(96, 2, 4, 4, 100)
    with pytest.raises(uv.UVError):
        uv.KvCache(128, 2, 4, 4, 100, page_tokens=48)
    with pytest.raises(uv.UVError):
        uv.KvCache(128, 2, 4, 4, 100, rounds=4)
    with pytest.raises(ValueError):
        uv.KvCache.over(c.pool, c.table, c.lens, c.refs, signs=torch.zeros(1, 128), head_dim=128,
                        page_tokens=64)
    assert isinstance(C.c_void_p(c._p), C.c_void_p)
