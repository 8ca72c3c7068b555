"""Page operations of the 4-bit cache against a Python model: every table,
length, count and byte, over random call sequences, and the refusals that the
device makes."""
from __future__ import annotations

import numpy as np
import pytest

import kv_model as M

pytestmark = pytest.mark.gpu


def ints(x):
    import torch

    return torch.tensor(np.asarray(x, np.int32), device="cuda")


def make(uv, n_pages=40, max_seqs=9, max_len=500, layers=2, page=64, heads=3, d=64):
    import torch

    c = uv.KvCache(d, heads, n_pages, max_seqs, max_len, layers=layers, page_tokens=page)
    g = torch.Generator(device="cuda").manual_seed(n_pages)
    c.pool.copy_(torch.randint(0, 256, c.pool.shape, generator=g, device="cuda", dtype=torch.uint8))
    return c, M.Pages(n_pages, max_seqs, c.table.shape[1], page)


def same(c, m, pool):
    np.testing.assert_array_equal(c.table.cpu().numpy(), m.table)
    np.testing.assert_array_equal(c.lens.cpu().numpy(), m.lens)
    np.testing.assert_array_equal(c.refs.cpu().numpy(), m.refs)
    got = c.pool.cpu().numpy()
    for a, b in m.moves:
        pool[:, b] = pool[:, a]
    m.moves = []
    np.testing.assert_array_equal(got, pool)
    assert int(c.work[2]) == int((m.refs > 0).sum())


@pytest.mark.parametrize("page,n_pages,seed", [(32, 64, 0), (64, 40, 1), (128, 23, 2), (64, 5000, 3),
                                               (256, 12, 4)])
def test_random_calls(uv, page, n_pages, seed):
    rng = np.random.default_rng(seed)
    seqs = 9 if n_pages < 1000 else 40
    c, m = make(uv, n_pages, seqs, 7 * page + 3, 2, page)
    pool = c.pool.cpu().numpy().copy()
    for step in range(60):
        op = rng.choice(["extend", "extend", "extend", "fork", "copy", "truncate", "free", "compact"])
        empty, live = np.flatnonzero(m.lens == 0), np.flatnonzero(m.lens > 0)
        if op == "extend":
            s = rng.permutation(seqs)[:rng.integers(1, seqs + 1)]
            n = [int(min(rng.choice([0, 1, 1, page, rng.integers(0, 3 * page)]),
                         m.table.shape[1] * page - m.lens[x])) for x in s]
            c.extend(ints(s), ints(n))
            if not m.extend(s, n):
                with pytest.raises(uv.KvError) as e:
                    c.check()
                assert e.value.status == 1
        elif op in ("fork", "copy") and len(empty) and len(live):
            k = int(rng.integers(1, len(empty) + 1))
            src, dst = rng.choice(live, k), rng.permutation(empty)[:k]
            if op == "fork":
                lens = None if rng.random() < 0.5 else [int(rng.integers(0, m.lens[x] + 9)) for x in src]
                c.fork(ints(src), ints(dst), None if lens is None else ints(lens))
                m.fork(src, dst, lens)
            elif sum(m.pages(m.lens[x]) for x in src) <= (m.refs == 0).sum():
                c.copy(ints(src), ints(dst))
                m.copy(src, dst)
        elif op in ("truncate", "free") and len(live):
            s = rng.permutation(live)[:rng.integers(1, len(live) + 1)]
            if op == "free":
                c.free(ints(s))
                m.truncate(s)
            else:
                lens = [int(rng.integers(0, m.lens[x] + 5)) for x in s]
                c.truncate(ints(s), ints(lens))
                m.truncate(s, lens)
        elif op == "compact":
            c.compact()
            m.compact()
        same(c, m, pool)
    c.check()


def test_more_entries_than_threads(uv):
    """Over 1024 sequences in a call: shared last pages, long and short growth."""
    c, m = make(uv, 9000, 2600, 300, 1, 32, heads=1)
    pool = c.pool.cpu().numpy().copy()
    rng = np.random.default_rng(1)
    a, b = np.arange(1300), np.arange(1300, 2600)
    for step, most in enumerate((50, 2, 180)):
        n = rng.integers(0, most, 1300)
        c.extend(ints(a), ints(n))
        assert m.extend(a, n)
        same(c, m, pool)
        if step == 0:
            c.fork(ints(a), ints(b))
            m.fork(a, b)
    both = rng.permutation(2600)
    n = rng.integers(0, 3, 2600)
    c.extend(ints(both), ints(n))
    assert m.extend(both, n)
    same(c, m, pool)
    c.truncate(ints(both), ints(m.lens[both] // 2))
    m.truncate(both, m.lens[both] // 2)
    same(c, m, pool)
    c.check()


def test_beams_copy_a_shared_last_page_and_nothing_else(uv):
    c, m = make(uv)
    pool = c.pool.cpu().numpy().copy()
    for do, model in (((c.extend), m.extend),):
        do(ints([0, 1]), ints([70, 128]))
        model([0, 1], [70, 128])
    c.fork(ints([0, 0, 0, 1]), ints([3, 4, 5, 6]))
    m.fork([0, 0, 0, 1], [3, 4, 5, 6])
    c.extend(ints([3, 4, 5, 6]), ints([1, 1, 0, 1]))
    assert m.extend([3, 4, 5, 6], [1, 1, 0, 1])
    assert len(m.moves) == 2  # sequence 5 takes nothing, 6's last page is full
    same(c, m, pool)


@pytest.mark.parametrize("call,bit", [
    (lambda c: c.extend(ints([0, 0]), ints([1, 1])), 2),
    (lambda c: c.extend(ints([9]), ints([1])), 2),
    (lambda c: c.extend(ints([-1]), ints([1])), 2),
    (lambda c: c.extend(ints([2]), ints([-4])), 2),
    (lambda c: c.extend(ints([2, 0]), ints([5, 600])), 4),
    (lambda c: c.extend(ints([2, 3, 4, 5, 6, 7, 8]), ints([500] * 7)), 1),
    (lambda c: c.fork(ints([0, 0]), ints([1, 2])), 8),
    (lambda c: c.fork(ints([0, 0]), ints([2, 2])), 2),
    (lambda c: c.fork(ints([2]), ints([2])), 2),
    (lambda c: c.fork(ints([0]), ints([2]), ints([-1])), 2),
    (lambda c: c.copy(ints([0, 1]), ints([2, 1])), 2 | 8),
    (lambda c: c.copy(ints([0]), ints([77])), 2),
    (lambda c: c.truncate(ints([0, 0]), ints([1, 1])), 2),
    (lambda c: c.truncate(ints([0]), ints([-1])), 2),
    (lambda c: c.free(ints([1 << 20])), 2),
])
def test_refused_calls_change_nothing_until_checked(uv, call, bit):
    c, m = make(uv)
    pool = c.pool.cpu().numpy().copy()
    c.extend(ints([0, 1]), ints([70, 128]))
    m.extend([0, 1], [70, 128])
    call(c)
    same(c, m, pool)
    c.extend(ints([3]), ints([1]))  # stopped by the status
    c.free(ints([0]))
    c.fork(ints([0]), ints([4]))
    c.copy(ints([0]), ints([4]))
    c.compact()
    same(c, m, pool)
    with pytest.raises(uv.KvError) as e:
        c.check()
    assert e.value.status == bit
    c.check()
    c.extend(ints([3]), ints([1]))
    m.extend([3], [1])
    same(c, m, pool)


def test_reset_and_the_last_free_page(uv):
    c, m = make(uv, n_pages=4)
    pool = c.pool.cpu().numpy().copy()
    c.extend(ints([2, 1]), ints([64, 192]))
    m.extend([2, 1], [64, 192])
    same(c, m, pool)
    c.reset()
    assert int(c.refs.abs().sum()) == 0 and int(c.lens.sum()) == 0 and bool((c.table == -1).all())
    c.extend(ints([0]), ints([256]))
    c.check()
    assert c.table[0].tolist()[:4] == [0, 1, 2, 3]


def test_no_entries_and_host_buffers(uv):
    import torch

    c, _ = make(uv)
    none = ints([])
    c.extend(none, none)
    c.fork(none, none)
    c.copy(none, none)
    c.free(none)
    c.check()
    with pytest.raises(ValueError):
        c.extend(torch.zeros(1, dtype=torch.int32), ints([1]))
    with pytest.raises(ValueError):
        c.extend(ints([1]).long(), ints([1]))
    with pytest.raises(ValueError):
        c.extend(ints([1, 2]), ints([1]))
    host = np.zeros(4, np.int32)
    rc = uv.lib().uv_kv_extend(c._p, host.ctypes.data, host.ctypes.data, 1, None)
    assert rc == 1 and b"device memory" in uv.lib().uv_last_error()
    rc = uv.lib().uv_kv_extend(c._p, ints([0] * 10).data_ptr(), ints([0] * 10).data_ptr(), 10, None)
    assert rc == 1


def test_a_step_runs_in_a_graph(uv):
    """Extending, forking and freeing replay on the device's own state."""
    import torch

    c, m = make(uv)
    pool = c.pool.cpu().numpy().copy()
    s, one = ints([0, 1, 2]), ints([33, 1, 64])
    src, dst = ints([0]), ints([5])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        c.extend(s, one)
    torch.cuda.current_stream().wait_stream(stream)
    m.extend([0, 1, 2], [33, 1, 64])
    same(c, m, pool)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.fork(src, dst)
        c.extend(s, one)
        c.free(dst)
    for _ in range(3):
        graph.replay()
        m.fork([0], [5])
        m.extend([0, 1, 2], [33, 1, 64])
        m.truncate([5])
        same(c, m, pool)
    c.check()
