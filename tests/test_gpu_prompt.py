"""Attention over packed prompts against a 64-bit model."""
from __future__ import annotations

import math

import numpy as np
import pytest

import kv_model as M

pytestmark = pytest.mark.gpu

UNIT = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}  # half an ulp, relative


def starts(counts):
    import torch

    return torch.tensor(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32), device="cuda")


def rows(rng, n, heads, d, typ, size=1.0):
    import torch

    return torch.tensor(size * rng.standard_normal((n, heads, d)), dtype=torch.float32,
                        device="cuda").to(getattr(torch, typ))


def f64(x):
    return x.double().cpu().numpy()


def tolerance(out, size, reach, typ):
    """Products of the inputs are exact and add up in f32: scores err by less
    than 2^-17 of sum |q_i k_i| and the exponential, with its argument, by less
    than 2^-14; a weight rounds to the type, the sum takes it unrounded; the
    output rounds."""
    eps = UNIT[typ] + 2 * (2.0 ** -17 * reach + 2.0 ** -14)
    return eps[..., None] * size * 1.02 + UNIT[typ] * np.abs(out) * 1.01 + 2.0 ** -24


def compare(out, lse, q, k, v, nq, nk, causal, typ, scale):
    a = b = 0
    for n, m in zip(nq, nk):
        want, wl, size, reach = M.prompt(f64(q[a:a + n]), f64(k[b:b + m]), f64(v[b:b + m]), causal, scale)
        err, tol = np.abs(f64(out[a:a + n]) - want), tolerance(want, size, reach, typ)
        assert (err <= tol).all(), float((err / tol).max())
        got, seen = f64(lse[a:a + n]), np.isfinite(wl)
        assert (np.isneginf(got) == ~seen).all()
        assert (np.abs(got - wl)[seen] <= (2.0 ** -17 * reach + 2.0 ** -13)[seen]).all()
        a, b = a + n, b + m


CASES = [  # d, q heads, kv heads, queries, keys, causal, type
    (64, 8, 2, [77], [77], True, "float16"),
    (128, 4, 4, [1, 2, 63, 64, 65], [1, 2, 63, 64, 65], True, "bfloat16"),
    (128, 4, 1, [127, 128, 129, 1], [127, 128, 129, 1], True, "float16"),
    (64, 3, 3, [255, 256, 257], [255, 256, 257], False, "bfloat16"),
    (128, 2, 2, [33, 5, 200], [333, 5, 201], True, "bfloat16"),
    (64, 6, 2, [10, 130], [300, 131], False, "float16"),
    (128, 3, 1, [300], [300], True, "bfloat16"),
    (128, 6, 3, [0, 40, 0, 0, 9, 0], [0, 40, 0, 7, 9, 0], True, "float16"),
    (64, 2, 1, [513], [600], True, "float16"),
]


@pytest.mark.parametrize("d,hq,hk,nq,nk,causal,typ", CASES)
def test_prompt(uv, d, hq, hk, nq, nk, causal, typ):
    rng = np.random.default_rng(d + hq + len(nq))
    q, k, v = rows(rng, sum(nq), hq, d, typ, 1.5), rows(rng, sum(nk), hk, d, typ), rows(rng, sum(nk), hk, d, typ)
    out, lse = uv.prompt_attention(q, k, v, starts(nq), starts(nk), causal=causal, lse=True)
    compare(out, lse, q, k, v, nq, nk, causal, typ, 1 / math.sqrt(d))


def test_more_queries_than_keys_leaves_rows_empty(uv):
    rng = np.random.default_rng(1)
    for d in (64, 128):
        q, k, v = (rows(rng, n, 2, d, "bfloat16") for n in (200, 70, 70))
        out, lse = uv.prompt_attention(q, k, v, starts([150, 50]), starts([70, 0]), lse=True)
        compare(out, lse, q, k, v, [150, 50], [70, 0], True, "bfloat16", 1 / math.sqrt(d))
        assert (f64(out)[:80] == 0).all() and (f64(out)[150:] == 0).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan"), 3e38])
def test_what_a_row_does_not_see_does_not_reach_it(uv, d, bad):
    """Infinities and NaN in the keys and values of later tokens and of the next
    sequence leave a row's bits as they are; rows that see a NaN have one."""
    import torch

    rng = np.random.default_rng(2)
    n = [150, 90, 64]
    for hk in (1, 2):
        q, k, v = (rows(rng, sum(n), h, d, "bfloat16") for h in (2, hk, hk))
        want = uv.prompt_attention(q, k, v, starts(n))
        for which in (0, 1):
            kv = [k.clone(), v.clone()]
            kv[which][100:150, :, 3] = bad   # rows 100.. of the first sequence see it
            kv[which][150 + 90:, :, 5] = bad  # the third sequence
            got = uv.prompt_attention(q, *kv, starts(n))
            assert torch.equal(got[:100], want[:100])
            assert torch.equal(got[150:240], want[150:240])
            if math.isnan(bad):
                where = slice(None) if which == 0 else 3
                assert bool(got[100:150, :, where].isnan().all())
            elif which == 1 and math.isinf(bad):
                assert bool((got[100:150, :, 3] == bad).all())
                assert torch.isfinite(got[100:150, :, :3]).all()


def test_large_scores_and_a_scale(uv):
    rng = np.random.default_rng(3)
    for d in (64, 128):
        q, k, v = rows(rng, 300, 2, d, "bfloat16", 30.0), rows(rng, 300, 2, d, "bfloat16", 5.0), \
            rows(rng, 300, 2, d, "bfloat16")
        out, lse = uv.prompt_attention(q, k, v, starts([300]), scale=0.3, lse=True)
        a, wl, size, reach = M.prompt(f64(q), f64(k), f64(v), True, 0.3)
        eps = np.expm1(2 * (2.0 ** -17 * reach + 2.0 ** -14)) + UNIT["bfloat16"]
        assert (np.abs(f64(out) - a) <= eps[..., None] * size * 1.02 + 2.0 ** -8 * np.abs(a) * 1.01).all()
        assert (np.abs(f64(lse) - wl) <= 2.0 ** -17 * reach + 2.0 ** -13).all()


def test_strides_streams_and_repeats(uv):
    import torch

    rng = np.random.default_rng(4)
    n = starts([200, 57])
    q, k, v = rows(rng, 257, 4, 128, "bfloat16"), rows(rng, 257, 2, 128, "bfloat16"), rows(rng, 257, 2, 128, "bfloat16")
    want = uv.prompt_attention(q, k, v, n)
    assert torch.equal(want, uv.prompt_attention(q, k, v, n))
    one = torch.cat([q, k, v], 1)  # as a fused projection gives them
    assert torch.equal(want, uv.prompt_attention(one[:, :4], one[:, 4:6], one[:, 6:], n))
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    off = torch.zeros(257 * 2 * 128 + 3, dtype=torch.bfloat16, device="cuda")[3:].view(257, 2, 128)
    off.copy_(v)
    assert torch.equal(want, uv.prompt_attention(qt, k, off, n))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = uv.prompt_attention(q, k, v, n)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want, got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = uv.prompt_attention(q, k, v, n)
    got.zero_()
    graph.replay()
    assert torch.equal(want, got)


def test_one_row_one_head_and_broadcast_heads(uv):
    import torch

    rng = np.random.default_rng(9)
    q, k, v = (rows(rng, n, 1, 64, "float16") for n in (1, 300, 300))
    out, lse = uv.prompt_attention(q, k, v, starts([1]), starts([300]), lse=True)
    compare(out, lse, q, k, v, [1], [300], True, "float16", 0.125)
    q = rows(rng, 40, 4, 64, "float16")
    k, v = (rows(rng, 40, 1, 64, "float16") for _ in range(2))
    wide = uv.prompt_attention(q, k.expand(-1, 2, -1), v.expand(-1, 2, -1), starts([40]))
    assert torch.equal(wide, uv.prompt_attention(q, k, v, starts([40])))
    st = torch.cuda.current_stream().cuda_stream
    n = starts([40]).data_ptr()
    out = torch.empty_like(q)
    for strides in ((0, 64), (256, 0), (3, 64), (-256, 64)):
        rc = uv.lib().uv_prompt_attention(0, n, None, 1, 40, 40, 4, 4, 64, 1, 0.125, 0, q.data_ptr(), *strides,
                                          q.data_ptr(), 256, 64, q.data_ptr(), 256, 64, out.data_ptr(), None, st)
        assert rc == 1, strides


@pytest.mark.parametrize("d,causal", [(64, True), (128, True), (128, False)])
def test_a_few_rows_behind_many_keys(uv, d, causal):
    """The last rows of 70,001 tokens, whose scores climb along the sequence, so
    that the references move again and again from the last keys to the first."""
    import torch

    rng = np.random.default_rng(d)
    q, k, v = rows(rng, 3, 2, d, "bfloat16"), rows(rng, 70_001, 1, d, "bfloat16"), rows(rng, 70_001, 1, d, "bfloat16")
    slope = torch.linspace(60, 0, 70_001, device="cuda")[:, None, None]
    k = (k.float() + slope * q.float().mean(1, keepdim=True)[:1] / d).bfloat16()
    out, lse = uv.prompt_attention(q, k, v, starts([3]), starts([70_001]), causal=causal, lse=True)
    compare(out, lse, q, k, v, [3], [70_001], causal, "bfloat16", 1 / math.sqrt(d))


@pytest.mark.parametrize("typ", ["float16", "bfloat16"])
@pytest.mark.parametrize("d,hq,hk", [(64, 2, 1), (128, 4, 2), (128, 3, 1)])
@pytest.mark.parametrize("excess", [15, 100])
def test_a_reference_of_few_keys_is_left_where_it_is_too_low(uv, typ, d, hq, hk, excess):
    """Keys ahead of the queries by no multiple of 128: some rows of a warp see
    their first keys in a block whose other rows have references already, of a
    key or a few.  Keys of that block stand above those references by `excess`
    nats."""
    rng = np.random.default_rng(excess)
    nq, nk = [200, 64, 40], [1200, 64, 90]
    for at in (900, 960, 1023):
        q, k, v = rows(rng, sum(nq), hq, d, typ, 0.3), rows(rng, sum(nk), hk, d, typ), rows(rng, sum(nk), hk, d, typ)
        q[:, :, 0] = 4
        k[:, :, 0] = 0
        for key in (at, 1200 + 3, 1264 + 45):
            k[key, :, 0] = excess * math.sqrt(d) / 4
        out, lse = uv.prompt_attention(q, k, v, starts(nq), starts(nk), lse=True)
        compare(out, lse, q, k, v, nq, nk, True, typ, 1 / math.sqrt(d))


@pytest.mark.parametrize("typ", ["float16", "bfloat16"])
@pytest.mark.parametrize("d,key", [(64, 290), (64, 7), (128, 290), (128, 7)])
def test_small_weights_beside_a_large_one(uv, typ, d, key):
    """A key that stands 16 nats above the others and has values of zero: what is
    left is weights of 1e-7, in as many bits as any others."""
    rng = np.random.default_rng(d + key)
    n = 300
    q, k, v = rows(rng, n, 2, d, typ, 0.3), rows(rng, n, 2, d, typ), rows(rng, n, 2, d, typ, 1000.0)
    q[:, :, 0] = 4
    k[:, :, 0] = 0
    k[key, :, 0] = 16 * math.sqrt(d) / 4
    v[key] = 0
    out, lse = uv.prompt_attention(q, k, v, starts([n]), causal=False, lse=True)
    compare(out, lse, q, k, v, [n], [n], False, typ, 1 / math.sqrt(d))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_one_score_that_is_no_number(uv, d, causal):
    """One key that gives NaN or +inf makes every row that sees it NaN, wherever in
    a block it lies; one that gives -inf weighs nothing."""
    import torch

    rng = np.random.default_rng(d)
    n = 300
    q, k, v = rows(rng, n, 2, d, "bfloat16"), rows(rng, n, 1, d, "bfloat16"), rows(rng, n, 1, d, "bfloat16")
    q[:, :, 3] = 1
    k[:, :, 3] = 0
    want = uv.prompt_attention(q, k, v, starts([n]), causal=causal)
    for key in (1, 2, 3, 4, 5, 6, 7, 8, 64, 127, 128, 129, 200, 299):
        first = key if causal else 0
        for bad in (math.nan, math.inf):
            kk = k.clone()
            kk[key, :, 3] = bad
            got, lse = uv.prompt_attention(q, kk, v, starts([n]), causal=causal, lse=True)
            assert bool(got[first:].isnan().all()), (key, bad)
            assert bool(lse[first:].isnan().all()), (key, bad)
            assert torch.equal(got[:first], want[:first])
        kk[key, :, 3] = -math.inf
        got, lse = uv.prompt_attention(q, kk, v, starts([n]), causal=causal, lse=True)
        kk[key, :, 3] = -1e6  # a score of -88,000 at the least: a weight of zero
        a, wl, size, reach = M.prompt(f64(q), f64(kk), f64(v), causal, 1 / math.sqrt(d))
        kk[key] = 0
        reach = M.prompt(f64(q), f64(kk), f64(v), causal, 1 / math.sqrt(d))[3]
        assert (np.abs(f64(got) - a) <= tolerance(a, size, reach, "bfloat16")).all(), key
        assert (np.abs(f64(lse) - wl) <= 2.0 ** -17 * reach + 2.0 ** -13).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,size", [(300, 1e37), (3000, 1e38), (300, 1e-30)])
def test_values_near_the_largest_number(uv, d, n, size):
    """Sums of many of them are beyond a float; their means are not.  Small ones
    keep their bits too."""
    rng = np.random.default_rng(n)
    q, k, v = rows(rng, 200, 2, d, "bfloat16", 0.5), rows(rng, n, 1, d, "bfloat16"), rows(rng, n, 1, d, "bfloat16")
    v = ((v.float().clamp(-2, 2) + 0.5) * size).bfloat16()
    out, lse = uv.prompt_attention(q, k, v, starts([200]), starts([n]), lse=True)
    want, wl, big, reach = M.prompt(f64(q), f64(k), f64(v), True, 1 / math.sqrt(d))
    err, tol = np.abs(f64(out) - want) / size, tolerance(want / size, big / size, reach, "bfloat16")
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("d", [64, 128])
def test_a_row_whose_scores_are_all_minus_infinity(uv, d):
    """It has no softmax (NaN, and a sum of zero), other than a row that sees nothing."""
    rng = np.random.default_rng(d)
    q, k, v = rows(rng, 200, 2, d, "float16"), rows(rng, 160, 1, d, "float16"), rows(rng, 160, 1, d, "float16")
    q[:, :, 0] = 1
    k[:150, :, 0] = -math.inf  # rows 40 .. 189 see those alone, rows 0 .. 39 none at all
    out, lse = uv.prompt_attention(q, k[:160], v, starts([0, 200]), starts([0, 160]), lse=True)
    assert bool((out[:40] == 0).all()) and bool((lse[:40] == -math.inf).all())
    assert bool(out[40:190].isnan().all()) and bool((lse[40:190] == -math.inf).all())
    want, wl, size, reach = M.prompt(f64(q[190:]), f64(k[150:]), f64(v[150:]), True, 1 / math.sqrt(d))
    assert (np.abs(f64(out[190:]) - want) <= tolerance(want, size, reach, "float16")).all()


@pytest.mark.parametrize("n", [1, 33, 150])
def test_many_sequences_of_every_length(uv, n):
    """Entries over all lanes, and more than the ordered search takes."""
    rng = np.random.default_rng(n)
    nq = [int(x) for x in rng.integers(0, 200, n)]
    nk = [x + int(y) for x, y in zip(nq, rng.integers(0, 150, n))]
    nq[0], nk[0] = 130, 400
    q, k, v = rows(rng, sum(nq), 2, 64, "bfloat16"), rows(rng, sum(nk), 1, 64, "bfloat16"), rows(rng, sum(nk), 1, 64, "bfloat16")
    for causal in (True, False):
        out, lse = uv.prompt_attention(q, k, v, starts(nq), starts(nk), causal=causal, lse=True)
        a = np.concatenate([[0], np.cumsum(nq)])
        b = np.concatenate([[0], np.cumsum(nk)])
        for i in list(range(min(n, 4))) + [n // 2, n - 1]:
            x, y = slice(a[i], a[i + 1]), slice(b[i], b[i + 1])
            compare(out[x], lse[x], q[x], k[y], v[y], [nq[i]], [nk[i]], causal, "bfloat16", 0.125)
        assert np.isfinite(f64(out)).all()


@pytest.mark.parametrize("d,hq,causal", [(64, 16, True), (128, 16, True), (128, 18, True), (128, 16, False)])
def test_more_work_than_blocks(uv, d, hq, causal):
    """Every block takes several pieces of work, some with values that are no
    numbers: what one piece has met does not reach the next."""
    import torch

    rng = np.random.default_rng(d + hq)
    nq = [int(x) for x in rng.integers(1, 300, 48)]
    nk = [x + 70 * (i % 3) for i, x in enumerate(nq)]
    q, k = rows(rng, sum(nq), hq, d, "bfloat16"), rows(rng, sum(nk), 2, d, "bfloat16")
    v = rows(rng, sum(nk), 2, d, "bfloat16")
    bad, clean = v.clone(), v.clone()
    b = np.concatenate([[0], np.cumsum(nk)])
    a = np.concatenate([[0], np.cumsum(nq)])
    where = {}
    for i in range(0, 48, 3):
        key, head, col = int(rng.integers(0, nk[i])), int(rng.integers(0, 2)), int(rng.integers(0, d))
        what = (math.inf, -math.inf, math.nan)[i // 3 % 3]
        bad[b[i] + key, head, col] = what
        clean[b[i] + key, head, col] = 0
        where[i] = key, head, col, what
    out, lse = uv.prompt_attention(q, k, bad, starts(nq), starts(nk), causal=causal, lse=True)
    for i, (key, head, col, what) in where.items():
        first = max(0, key - (nk[i] - nq[i])) if causal else 0  # row that sees the key
        part = out[a[i] + first:a[i + 1], head * (hq // 2):(head + 1) * (hq // 2), col]
        assert bool((part.isnan() if math.isnan(what) else part == what).all())
        mine = f64(clean[b[i]:b[i + 1]])
        want = M.prompt(f64(q[a[i]:a[i + 1]]), f64(k[b[i]:b[i + 1]]), mine, causal, 1 / math.sqrt(d))[0]
        part.copy_(torch.tensor(want[first:, head * (hq // 2):(head + 1) * (hq // 2), col]))
    compare(out, lse, q, k, clean, nq, nk, causal, "bfloat16", 1 / math.sqrt(d))


@pytest.mark.parametrize("d,causal", [(64, True), (128, True), (128, False)])
def test_marks_of_every_piece(uv, d, causal):
    """Infinities in nearly every piece of work, in columns of their own: each
    piece's marks stay until its rows are out, call after call."""
    import torch

    rng = np.random.default_rng(d)
    nq = [int(x) for x in rng.integers(1, 140, 150)]
    q, k, v = (rows(rng, sum(nq), h, d, "bfloat16") for h in (8, 2, 2))
    a = np.concatenate([[0], np.cumsum(nq)])
    where = []
    for i in range(150):
        key, col = a[i] + int(rng.integers(0, nq[i])), int(rng.integers(0, d))
        where.append((i, key, col))
        v[key, :, col] = math.inf
    want = uv.prompt_attention(q, k, v, starts(nq), causal=causal)
    inf = torch.zeros_like(want, dtype=torch.bool)
    for i, key, col in where:
        inf[key if causal else a[i]:a[i + 1], :, col] = True
    assert torch.equal(want == math.inf, inf) and not bool(want.isnan().any())
    differ = torch.zeros((), device="cuda")
    for _ in range(300):
        differ += (uv.prompt_attention(q, k, v, starts(nq), causal=causal) != want).any()
    assert int(differ) == 0


def test_refused_arguments(uv):
    import torch

    rng = np.random.default_rng(5)
    q = rows(rng, 10, 4, 128, "bfloat16")
    n = starts([10])
    for a in ((q, q[:, :3], q[:, :3]), (q, q, q[:, :2]), (q, q.half(), q), (q.float(), q.float(), q.float()),
              (q[:, :, :96], q[:, :, :96], q[:, :, :96]), (q, q, q[:5]), (q.cpu(), q.cpu(), q.cpu())):
        with pytest.raises((ValueError, uv.UVError)):
            uv.prompt_attention(*a, n)
    with pytest.raises(ValueError):
        uv.prompt_attention(q, q, q, n.long())
    with pytest.raises(ValueError):
        uv.prompt_attention(q, q, q, n, torch.cat([n, n]))
    with pytest.raises(uv.UVError):
        uv.prompt_attention(q, q[:5], q[:5], n)
    none = uv.prompt_attention(q[:0], q[:0], q[:0], starts([0]))
    assert none.shape == (0, 4, 128)
