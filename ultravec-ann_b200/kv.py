"""A cache held in 4 bits, and attention over it and over whole prompts.

`KvCache` is the paged cache of a model's keys and values in the codec's
manner: rotated rows as 4-bit levels with one rescaled factor each (the
estimator of src/trellis.rs:1483-1536), attended to without being decoded.
`prompt_attention` attends over packed prompts.  Arrays are CUDA torch
tensors; every call is ordered on torch's current stream of their device, and
none but `check` waits for it, so a serving step can be captured in a graph.
They infer only: outputs carry no gradient, also where an input asks for one.

A step for sequences that already have tokens:

    cache.extend(seqs, counts)                       # room, once for all layers
    for each layer:
        cache.append(seqs, k, v, starts, layer=i)    # the new rows
        out = cache.attend(seqs, q, starts, most, layer=i)
"""
from __future__ import annotations

import ctypes as C
import math

from .binding import UVError, check, lib

TILE = 32


class uv_kv(C.Structure):
    _fields_ = [("device", C.c_int32), ("head_dim", C.c_int32), ("kv_heads", C.c_int32),
                ("layers", C.c_int32), ("page_tokens", C.c_int32), ("n_pages", C.c_int32),
                ("max_seqs", C.c_int32), ("max_pages", C.c_int32), ("rounds", C.c_int32),
                ("reserved", C.c_int32), ("signs", (C.c_uint32 * 8) * 3),
                ("pool", C.c_void_p), ("table", C.c_void_p), ("lens", C.c_void_p),
                ("refs", C.c_void_p), ("work", C.c_void_p)]


class KvError(UVError):
    """What `check` found: `status` holds the UV_KV_* bits."""

    WHAT = {1: "no free page", 2: "a sequence out of range or listed twice, or a negative count",
            4: "more tokens than a sequence's table row holds", 8: "the target has tokens",
            16: "rows appended to a shared page", 32: "a bounded device wait gave up"}

    def __init__(self, status: int):
        super().__init__(1, "; ".join(w for b, w in self.WHAT.items() if status & b))
        self.status = status


torch = None
_raw_stream = None


def _load():
    """torch and the library, on first use (the rest of the package works
    without torch); the library's functions by name."""
    global torch, _raw_stream
    if torch is None:
        import torch as t

        # the current stream's handle without a Stream object around it
        _raw_stream = getattr(t._C, "_cuda_getCurrentRawStream", None) or (
            lambda i: t.cuda.current_stream(i).cuda_stream)
        torch = t
    return lib()


def _dtype(x) -> int:
    d = x.dtype
    if d is torch.bfloat16:
        return 1
    if d is torch.float16:
        return 0
    raise ValueError("rows must be float16 or bfloat16")


def _operand(x, heads, dim, index, name):
    """Tensor and element strides of rows x heads x dim; laid out anew when a
    row is not dense or not aligned."""
    shape = x.shape
    if len(shape) != 3 or (heads is not None and shape[1] != heads) or shape[2] != dim:
        raise ValueError(f"{name} must be rows x {heads or 'heads'} x {dim}, got {tuple(shape)}")
    if x.get_device() != index:
        raise ValueError(f"{name} must be on cuda:{index}")
    row, head, one = x.stride()
    if one != 1 or row % 8 or head % 8 or row <= 0 or head <= 0 or x.data_ptr() % 16:
        # (contiguous() would give a dense but misaligned view back as it is)
        x = torch.empty(shape, dtype=x.dtype, device=x.device).copy_(x)
        row, head, one = x.stride()
    return x, row, head


def _ints(x, n, index, name):
    if (x.dtype is not torch.int32 or x.get_device() != index or x.dim() != 1
            or not x.is_contiguous()):
        raise ValueError(f"{name} must be a dense int32 vector on cuda:{index}")
    if n is not None and x.shape[0] != n:
        raise ValueError(f"{name} must have {n} entries, got {x.shape[0]}")
    return x.data_ptr()


class KvCache:
    """Pages of 4-bit keys and values for up to `max_seqs` sequences."""

    def __init__(self, head_dim: int, kv_heads: int, n_pages: int, max_seqs: int, max_len: int, *,
                 layers: int = 1, page_tokens: int = 64, seed: int = 42, rounds: int = 1,
                 device: int = 0):
        _load()
        dev = torch.device("cuda", device)
        max_pages = -(-max_len // page_tokens)
        desc = uv_kv(device, head_dim, kv_heads, layers, page_tokens, n_pages, max_seqs, max_pages,
                     rounds)
        check(lib().uv_kv_seed(C.byref(desc), seed))
        size = C.c_int64()
        check(lib().uv_kv_pool_bytes(C.byref(desc), C.byref(size)))
        pool = torch.empty((layers, n_pages, kv_heads, page_tokens // TILE, TILE * (head_dim + 8)),
                           dtype=torch.uint8, device=dev)
        assert pool.numel() == size.value
        i32 = dict(dtype=torch.int32, device=dev)
        self._attach(desc, pool, torch.empty((max_seqs, max_pages), **i32),
                     torch.empty(max_seqs, **i32), torch.empty(n_pages, **i32))
        self.reset()

    @classmethod
    def over(cls, pool, table, lens, refs, *, signs, head_dim: int, page_tokens: int) -> "KvCache":
        """A cache over the caller's own buffers, in use as they are: pool
        uint8 [layers, pages, heads, page_tokens / 32, 32 (head_dim + 8)], table
        int32 [sequences, columns], lens and refs int32; signs [rounds,
        head_dim] of +-1."""
        _load()
        layers, pages, heads, tiles, width = pool.shape
        if tiles * TILE != page_tokens or width != TILE * (head_dim + 8):
            raise ValueError(f"the pool's pages do not have the shape of {page_tokens} tokens of "
                             f"{head_dim} dimensions")
        import numpy as np

        s = signs.cpu().numpy() if hasattr(signs, "cpu") else np.asarray(signs)
        if s.ndim != 2 or not 1 <= s.shape[0] <= 3 or s.shape[1] != head_dim:
            raise ValueError("signs must be 1 to 3 rounds of head_dim values")
        if not (np.abs(s) == 1).all():
            raise ValueError("signs must be +1 or -1")
        desc = uv_kv(pool.device.index or 0, head_dim, heads, layers, page_tokens, pages,
                     table.shape[0], table.shape[1], s.shape[0])
        bits = np.packbits(s < 0, axis=1, bitorder="little").view(np.uint32)
        for r, row in enumerate(bits):
            desc.signs[r][:len(row)] = row.tolist()
        self = cls.__new__(cls)
        self._attach(desc, pool, table, lens, refs)
        check(self._lib.uv_kv_recount(self._p, _raw_stream(self._index)))
        return self

    def _attach(self, desc, pool, table, lens, refs):
        for x, t, shape, name in (
                (pool, torch.uint8, None, "pool"),
                (table, torch.int32, (desc.max_seqs, desc.max_pages), "table"),
                (lens, torch.int32, (desc.max_seqs,), "lens"),
                (refs, torch.int32, (desc.n_pages,), "refs")):
            if x.dtype != t or not x.is_contiguous() or x.device != pool.device or not x.is_cuda:
                raise ValueError(f"{name} must be a dense {t} tensor on the pool's GPU")
            if shape is not None and tuple(x.shape) != shape:
                raise ValueError(f"{name} must have the shape {shape}, got {tuple(x.shape)}")
        words = C.c_int64()
        check(lib().uv_kv_work_words(C.byref(desc), C.byref(words)))
        self.pool, self.table, self.lens, self.refs = pool, table, lens, refs
        self.work = torch.empty(words.value, dtype=torch.int32, device=pool.device)
        desc.pool, desc.table, desc.lens = pool.data_ptr(), table.data_ptr(), lens.data_ptr()
        desc.refs, desc.work = refs.data_ptr(), self.work.data_ptr()
        self._desc, self._p, self.device = desc, C.addressof(desc), pool.device
        self.head_dim, self.kv_heads, self.layers = desc.head_dim, desc.kv_heads, desc.layers
        self.page_tokens, self.n_pages, self.max_seqs = desc.page_tokens, desc.n_pages, desc.max_seqs
        self._lib, self._index = lib(), pool.device.index
        self._scale = 1.0 / math.sqrt(desc.head_dim)
        self._scratch_bytes = {}

    def reset(self) -> None:
        """Empty: no sequence has tokens, every page is free."""
        check(self._lib.uv_kv_reset(self._p, _raw_stream(self._index)))

    def check(self) -> None:
        """Waits for the stream and raises KvError if a call since the last
        check could not be done; until then calls that change the cache do
        nothing."""
        status = C.c_int32()
        check(self._lib.uv_kv_check(self._p, C.byref(status), _raw_stream(self._index)))
        if status.value:
            raise KvError(status.value)

    # -- pages --
    def extend(self, seqs, counts) -> None:
        """Room for counts[i] more tokens of seqs[i], which its length then
        includes.  The lowest free pages are taken, in the list's order; a
        shared last page is copied first.  All or nothing."""
        n, i = seqs.shape[0], self._index
        check(self._lib.uv_kv_extend(self._p, _ints(seqs, None, i, "seqs"),
                                     _ints(counts, n, i, "counts"), n, _raw_stream(i)))

    def fork(self, src, dst, lens=None) -> None:
        """The empty sequence dst[i] shares the pages of src[i]'s first
        lens[i] tokens (all of them by default)."""
        n, i = dst.shape[0], self._index
        check(self._lib.uv_kv_fork(self._p, _ints(src, n, i, "src"), _ints(dst, None, i, "dst"),
                                   None if lens is None else _ints(lens, n, i, "lens"), n,
                                   _raw_stream(i)))

    def copy(self, src, dst) -> None:
        """The empty sequence dst[i] gets a copy of src[i] in pages of its own."""
        n, i = dst.shape[0], self._index
        check(self._lib.uv_kv_copy(self._p, _ints(src, n, i, "src"), _ints(dst, None, i, "dst"), n,
                                   _raw_stream(i)))

    def truncate(self, seqs, lens) -> None:
        """Sequence seqs[i] keeps its first lens[i] tokens."""
        n, i = seqs.shape[0], self._index
        check(self._lib.uv_kv_truncate(self._p, _ints(seqs, None, i, "seqs"),
                                       _ints(lens, n, i, "lens"), n, _raw_stream(i)))

    def free(self, seqs) -> None:
        """Sequences keep nothing; pages that no sequence holds are free."""
        i = self._index
        check(self._lib.uv_kv_truncate(self._p, _ints(seqs, None, i, "seqs"), None, seqs.shape[0],
                                       _raw_stream(i)))

    def compact(self) -> None:
        """Moves the used pages to the lowest numbers."""
        check(self._lib.uv_kv_compact(self._p, _raw_stream(self._index)))

    # -- rows --
    def append(self, seqs, k, v, starts=None, *, layer: int = 0) -> None:
        """Quantises k and v (rows x kv_heads x head_dim) into the last tokens
        of the sequences: rows [starts[b], starts[b + 1]) are the last of
        seqs[b] (one row each without starts).  All or nothing: a sequence out
        of range or listed twice, or a shared page, is left to `check`."""
        i, n, dtype = self._index, seqs.shape[0], _dtype(k)
        if v.dtype is not k.dtype or v.shape != k.shape:
            raise ValueError("k and v must have one type and one shape")
        k, kr, kh = _operand(k, self.kv_heads, self.head_dim, i, "k")
        v, vr, vh = _operand(v, self.kv_heads, self.head_dim, i, "v")
        check(self._lib.uv_kv_append(
            self._p, layer, _ints(seqs, None, i, "seqs"),
            None if starts is None else _ints(starts, n + 1, i, "starts"), n, k.shape[0], dtype,
            k.data_ptr(), kr, kh, v.data_ptr(), vr, vh, _raw_stream(i)))

    def read(self, seqs, starts, rows: int, *, dtype=None, layer: int = 0):
        """The last starts[b + 1] - starts[b] tokens of seqs[b] as they are
        held: (k, v), rows x kv_heads x head_dim of dtype (bfloat16)."""
        i, n = self._index, seqs.shape[0]
        k = torch.empty((rows, self.kv_heads, self.head_dim), dtype=dtype or torch.bfloat16,
                        device=self.device)
        v = torch.empty_like(k)
        check(self._lib.uv_kv_read(
            self._p, layer, _ints(seqs, None, i, "seqs"),
            None if starts is None else _ints(starts, n + 1, i, "starts"), n, rows, _dtype(k),
            k.data_ptr(), v.data_ptr(), _raw_stream(i)))
        return k, v

    # -- attention --
    def attend(self, seqs, q, starts=None, most: int = 1, *, scale: float | None = None,
               layer: int = 0, lse: bool = False):
        """Attention of q (rows x q_heads x head_dim, packed like append's
        rows) over the cache; row i of n sees the tokens up to its own.  most:
        the longest entry's rows.  Returns out, or (out, lse) with lse=True."""
        i, n, dim, dtype = self._index, seqs.shape[0], self.head_dim, _dtype(q)
        q, qr, qh = _operand(q, None, dim, i, "q")
        rows, heads = q.shape[0], q.shape[1]
        key = (n, rows, most if starts is not None else 1, heads)
        size = self._scratch_bytes.get(key)
        if size is None:
            b = C.c_int64()
            check(self._lib.uv_kv_attend_bytes(self._p, *key, C.byref(b)))
            if len(self._scratch_bytes) > 1000:
                self._scratch_bytes.clear()
            size = self._scratch_bytes[key] = -(-b.value // 4)  # int32 words
        out = (torch.empty_like(q) if qh == dim and qr == heads * dim else
               torch.empty((rows, heads, dim), dtype=q.dtype, device=self.device))
        sums = (torch.empty((rows, heads), dtype=torch.float32, device=self.device) if lse
                else None)
        scratch = self.work.new_empty(size)
        check(self._lib.uv_kv_attend(
            self._p, layer, _ints(seqs, None, i, "seqs"),
            None if starts is None else _ints(starts, n + 1, i, "starts"), n, rows, key[2], dtype,
            q.data_ptr(), qr, qh, heads, self._scale if scale is None else scale, out.data_ptr(),
            None if sums is None else sums.data_ptr(), scratch.data_ptr(), 4 * size,
            _raw_stream(i)))
        return (out, sums) if lse else out


def prompt_attention(q, k, v, starts, starts_k=None, *, causal: bool = True,
                     scale: float | None = None, lse: bool = False):
    """Attention over packed prompts: q rows x q_heads x head_dim, k and v rows
    x kv_heads x head_dim; sequence b has query rows [starts[b], starts[b + 1])
    and key rows [starts_k[b], starts_k[b + 1]) (the same by default), its
    queries being the last of its keys.  Returns out, or (out, lse)."""
    L = _load()
    i, dim, dtype = q.get_device(), q.shape[-1], _dtype(q)
    if i < 0:
        raise ValueError("q must be a CUDA tensor")
    if k.dtype is not q.dtype or v.dtype is not q.dtype or v.shape != k.shape:
        raise ValueError("q, k and v must have one type, k and v one shape")
    q, qr, qh = _operand(q, None, dim, i, "q")
    k, kr, kh = _operand(k, None, dim, i, "k")
    v, vr, vh = _operand(v, None, dim, i, "v")
    rows, heads = q.shape[0], q.shape[1]
    n = starts.shape[0] - 1
    out = (torch.empty_like(q) if qh == dim and qr == heads * dim else
           torch.empty((rows, heads, dim), dtype=q.dtype, device=q.device))
    sums = torch.empty((rows, heads), dtype=torch.float32, device=q.device) if lse else None
    check(L.uv_prompt_attention(
        i, _ints(starts, None, i, "starts"),
        None if starts_k is None else _ints(starts_k, n + 1, i, "starts_k"), n, rows, k.shape[0],
        heads, k.shape[1], dim, int(causal), 1.0 / math.sqrt(dim) if scale is None else scale,
        dtype, q.data_ptr(), qr, qh, k.data_ptr(), kr, kh, v.data_ptr(), vr, vh, out.data_ptr(),
        None if sums is None else sums.data_ptr(), _raw_stream(i)))
    return (out, sums) if lse else out
