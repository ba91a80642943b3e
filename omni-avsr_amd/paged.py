"""The paged key / value cache and its operators on tensors (C ABI: include/omni_avsr.h, oavsr_op_qk_norm_rope and oavsr_op_paged_*).

A decoder layer with its cache in pages runs, per step,

    q   = paged.append(kv, batch, qkv, inv_freq)      # norm + rotation of the fused [q | k | v] rows, k and v into the pages
    out = paged.attention(kv, batch, q)               # the new tokens over their sequences' context

with one `PagedKV` per layer (its pool of pages) and one `PagedBatch` per step (row offsets, lengths and page table of the sequences, shared by all layers).
Everything is queued on the current stream of the tensors' device; nothing is synchronised, and every call can be captured into a graph.  An argument that
does not fit raises ValueError before anything is queued.  Lengths and page numbers are device data: a bad one never reaches memory outside the given
tensors, and sets its bit in `PagedKV.status` (`PagedKV.check()` raises)."""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import lib as L

_DT = {torch.float32: L.DT_F32, torch.bfloat16: L.DT_BF16}
_E4M3 = torch.float8_e4m3fn


def _need(ok, what):
    if not ok:
        raise ValueError("paged: " + what)


def _on_gpu(t, name, dtype, device=None):
    _need(isinstance(t, torch.Tensor) and t.is_cuda, f"{name} has to be a tensor on a GPU")
    _need(t.dtype == dtype, f"{name} is {t.dtype}, {dtype} is wanted")
    _need(device is None or t.device == device, f"{name} is on {t.device}, the others on {device}")


def _rows_of(t, name, width, dtype, device):
    """Row stride of [rows][width] or [rows][heads][head_dim] rows, each of them one piece of memory."""
    _on_gpu(t, name, dtype, device)
    _need(t.dim() in (2, 3), f"{name} has {t.dim()} dimensions")
    _need(t.shape[1] * (t.shape[2] if t.dim() == 3 else 1) == width, f"{name} has rows of shape {tuple(t.shape[1:])}, {width} values are wanted")
    if t.shape[0] == 0:
        return width
    _need(t.stride(-1) == 1 and (t.dim() == 2 or t.shape[1] == 1 or t.stride(1) == t.shape[2]), f"a row of {name} has to be one piece of memory (strides {t.stride()})")
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), width)


def _apart(rows, stride, name):
    """Output rows must not share memory."""
    _need(rows.shape[0] <= 1 or stride >= rows.shape[1] * (rows.shape[2] if rows.dim() == 3 else 1), f"rows of {name} overlap (strides {rows.stride()})")


class _on:
    """The device of the tensors, where it is not the current one."""
    __slots__ = ("guard",)

    def __init__(self, device):
        self.guard = None if torch.cuda.current_device() == device.index else torch.cuda.device(device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        return C.c_void_p(torch.cuda.current_stream().cuda_stream)

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


class PagedKV:
    """A layer's pool of pages: k and v [n_pages][n_kv_heads][page_size][head_dim] in float32, bfloat16, or float8_e4m3fn with k_scale and v_scale
    [n_pages][n_kv_heads][page_size] (float32).  Pages may be further apart than they are large (a view of a larger pool), k's and v's by the same stride.
    Keeps the tensors; `status` is one int32 of device memory."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        _need(isinstance(k, torch.Tensor) and k.is_cuda, "k has to be a tensor on a GPU")
        _need(k.dim() == 4, f"k has {k.dim()} dimensions, [n_pages][n_kv_heads][page_size][head_dim] is wanted")
        self.device, self.is_8bit = k.device, k.dtype == _E4M3
        _need(self.is_8bit or k.dtype in _DT, f"a cache of {k.dtype} is not supported")
        _on_gpu(v, "v", k.dtype, k.device)
        _need(v.shape == k.shape, f"k is {tuple(k.shape)}, v {tuple(v.shape)}")
        n, heads, page, dim = k.shape
        inner = (page * dim, dim, 1)
        for t, name in ((k, "k"), (v, "v")):
            _need(n == 0 or t.stride()[1:] == inner, f"a page of {name} has to be one piece of memory (strides {t.stride()})")
        stride = k.stride(0) if n > 1 else heads * page * dim
        _need(n <= 1 or v.stride(0) == stride, f"k's pages are {k.stride(0)} apart, v's {v.stride(0)}")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.status = torch.zeros(1, dtype=torch.int32, device=k.device)
        d = self.desc = L.PagedKvDesc()
        d.format = L.KV_E4M3 if self.is_8bit else L.KV_SAME
        d.dtype = L.DT_BF16 if self.is_8bit else _DT[k.dtype]
        d.n_kv_heads, d.head_dim, d.page_size, d.n_pages = heads, dim, page, n
        d.K, d.V, d.page_stride, d.status = k.data_ptr(), v.data_ptr(), stride, self.status.data_ptr()
        _need(self.is_8bit == (k_scale is not None) and self.is_8bit == (v_scale is not None), "k_scale and v_scale belong to an 8-bit cache, and only to one")
        if self.is_8bit:
            for t, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
                _on_gpu(t, name, torch.float32, k.device)
                _need(t.shape == k.shape[:3], f"{name} is {tuple(t.shape)}, {tuple(k.shape[:3])} is wanted")
                _need(n == 0 or t.stride()[1:] == (page, 1), f"a page of {name} has to be one piece of memory (strides {t.stride()})")
            d.scale_stride = k_scale.stride(0) if n > 1 else heads * page
            _need(n <= 1 or v_scale.stride(0) == d.scale_stride, f"k_scale's pages are {k_scale.stride(0)} apart, v_scale's {v_scale.stride(0)}")
            d.k_scale, d.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
        else:
            d.scale_stride = 0
        self._other = None

    @classmethod
    def empty(cls, n_pages, page_size, n_kv_heads, head_dim, dtype=torch.bfloat16, device="cuda"):
        """A pool of its own; dtype float8_e4m3fn: with scales."""
        shape = (n_pages, n_kv_heads, page_size, head_dim)
        kv = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(2)]
        scales = [torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2)] if dtype == _E4M3 else []
        return cls(*kv, *scales)

    def _for(self, dtype):
        """The description for rows of `dtype` (an 8-bit cache serves both)."""
        _need(dtype in _DT, f"rows of {dtype} are not supported")
        code = _DT[dtype]
        if self.desc.dtype == code:
            return self.desc
        _need(self.is_8bit, f"rows are {dtype}, the cache is {self.k.dtype}")
        if self._other is None:
            self._other = type(self.desc).from_buffer_copy(self.desc)
            self._other.dtype = code
        return self._other

    def check(self):
        """Raises RuntimeError if a call has met a bad page number or length since the last check (waits for the device; clears the word)."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            what = [s for b, s in ((L.PAGED_BAD_PAGE, "a page number outside the pool"), (L.PAGED_BAD_LENGTH, "a length outside the batch's bounds")) if bits & b]
            raise RuntimeError("paged: " + " and ".join(what) + " was met")


class PagedBatch:
    """The sequences of a step: cu_q [n_seqs + 1] (row offsets of their new tokens), ctx_len [n_seqs] (tokens in the cache, the new ones among them), table
    [n_seqs][pages], all int32 on the device.  max_q and max_ctx bound a sequence's new tokens and context.  Keeps the tensors: refilled in place, the
    same batch serves the next step."""

    def __init__(self, cu_q, ctx_len, table, *, max_q, max_ctx):
        for t, name, dim in ((cu_q, "cu_q", 1), (ctx_len, "ctx_len", 1), (table, "table", 2)):
            _on_gpu(t, name, torch.int32, getattr(cu_q, "device", None))
            _need(t.dim() == dim, f"{name} has {t.dim()} dimensions")
            _need(t.numel() == 0 or t.stride(-1) == 1 or t.shape[-1] == 1, f"{name} has to be one piece of memory (strides {t.stride()})")
        n = ctx_len.shape[0]
        _need(cu_q.shape[0] == n + 1 and table.shape[0] == n, f"{n} sequences by ctx_len, {cu_q.shape[0] - 1} by cu_q, {table.shape[0]} by table")
        _need(0 <= max_q < 2 ** 31 and 0 <= max_ctx < 2 ** 31, f"max_q {max_q}, max_ctx {max_ctx}")
        self.device, self.cu_q, self.ctx_len, self.table = cu_q.device, cu_q, ctx_len, table
        d = self.desc = L.PagedBatchDesc()
        d.n_seqs, d.max_q, d.max_ctx = n, max_q, max_ctx
        d.cu_q, d.ctx_len, d.table = cu_q.data_ptr(), ctx_len.data_ptr(), table.data_ptr()
        d.ld_table = table.stride(0) if n > 1 else table.shape[1]
        _need(n <= 1 or d.ld_table >= table.shape[1], "rows of table overlap")
        _need(table.shape[1] <= d.ld_table, "table")
        self.width = table.shape[1]

    def _for(self, rows, kv):
        _need(self.device == kv.device, f"the batch is on {self.device}, the cache on {kv.device}")
        _need(self.desc.max_ctx <= self.width * kv.desc.page_size, f"a table of {self.width} pages of {kv.desc.page_size} does not hold max_ctx {self.desc.max_ctx}")
        d = L.PagedBatchDesc.from_buffer_copy(self.desc)      # two threads may use one batch
        d.rows = rows
        return d


def _rope_desc(qkv, n_heads, n_kv_heads, head_dim, pos, inv_freq, q_gain, k_gain, eps, interleaved, rot_scale):
    d = L.QkRopeDesc()
    rows, dev = qkv.shape[0], qkv.device
    d.dtype, d.rows, d.n_heads, d.n_kv_heads, d.head_dim = _DT[qkv.dtype], rows, n_heads, n_kv_heads, head_dim
    d.qkv, d.rot_scale, d.eps, d.interleaved = qkv.data_ptr(), rot_scale, eps, bool(interleaved)
    if pos is not None:
        _on_gpu(pos, "pos", torch.int32, dev)
        _need(pos.dim() == 1 and pos.shape[0] == rows and (rows <= 1 or pos.stride(0) == 1), f"pos is {tuple(pos.shape)}, one number per row is wanted")
        d.pos = pos.data_ptr()
    if inv_freq is not None:
        _on_gpu(inv_freq, "inv_freq", torch.float32, dev)
        _need(inv_freq.dim() == 1 and inv_freq.is_contiguous() and inv_freq.numel() > 0, f"inv_freq is {tuple(inv_freq.shape)}, one piece of memory is wanted")
        d.inv_freq, d.rot_dim = inv_freq.data_ptr(), 2 * inv_freq.shape[0]
    _need((q_gain is None) == (k_gain is None), "gains for both queries and keys, or for neither")
    if q_gain is not None:
        for t, name in ((q_gain, "q_gain"), (k_gain, "k_gain")):
            _on_gpu(t, name, torch.float32, dev)
            _need(t.shape == (head_dim,) and t.is_contiguous(), f"{name} is {tuple(t.shape)}, ({head_dim},) is wanted")
        d.q_gain, d.k_gain = q_gain.data_ptr(), k_gain.data_ptr()
    return d


def _checked(rc):
    """An argument that the library refuses is a ValueError here; a device error stays one."""
    if rc == -1:
        raise ValueError("paged: " + L.last_error())
    L.check(rc)


def qk_norm_rope(qkv, n_heads, n_kv_heads, pos, inv_freq, *, q_gain=None, k_gain=None, eps=1e-6, interleaved=False, rot_scale=1.0, out=None):
    """Norm (with q_gain, k_gain) and rotation (by pos * inv_freq; None: none) of the query and key heads of fused rows [rows][(n_heads + 2 n_kv_heads) *
    head_dim].  Returns q [rows][n_heads][head_dim] and k [rows][n_kv_heads][head_dim]; `out` = (q, k) to write into, which may be qkv's own parts.
    inv_freq [rot_dim / 2]: the first rot_dim dimensions of a head turn, halves against each other, or neighbours when interleaved."""
    _need(isinstance(qkv, torch.Tensor) and qkv.is_cuda and qkv.dim() == 2 and qkv.dtype in _DT, "qkv has to be rows of float32 or bfloat16 on a GPU")
    _need(n_heads > 0 and n_kv_heads > 0 and qkv.shape[1] % (n_heads + 2 * n_kv_heads) == 0, f"rows of {qkv.shape[1]} values do not hold {n_heads} + 2 x {n_kv_heads} heads")
    head_dim, rows, dev = qkv.shape[1] // (n_heads + 2 * n_kv_heads), qkv.shape[0], qkv.device
    with _on(dev) as stream:
        d = _rope_desc(qkv, n_heads, n_kv_heads, head_dim, pos, inv_freq, q_gain, k_gain, eps, interleaved, rot_scale)
        d.ld = _rows_of(qkv, "qkv", qkv.shape[1], qkv.dtype, dev)
        if out is None:
            q, k = (torch.empty(rows, h, head_dim, dtype=qkv.dtype, device=dev) for h in (n_heads, n_kv_heads))
            d.ldq, d.ldk = n_heads * head_dim, n_kv_heads * head_dim
        else:
            q, k = out
            _need(q.shape[0] == rows and k.shape[0] == rows, f"out has {q.shape[0]} and {k.shape[0]} rows, qkv {rows}")
            d.ldq = _rows_of(q, "out[0]", n_heads * head_dim, qkv.dtype, dev)
            d.ldk = _rows_of(k, "out[1]", n_kv_heads * head_dim, qkv.dtype, dev)
            _apart(q, d.ldq, "out[0]")
            _apart(k, d.ldk, "out[1]")
        d.q_out, d.k_out = q.data_ptr(), k.data_ptr()
        _checked(L.load().oavsr_op_qk_norm_rope(C.byref(d), stream))
    return q, k


def append(kv, batch, qkv, inv_freq=None, *, pos=None, q_gain=None, k_gain=None, eps=1e-6, interleaved=False, rot_scale=1.0, out=None):
    """qk_norm_rope of the batch's rows, the keys and values going into their sequences' pages.  Returns q [rows][n_heads][head_dim] (`out`: where to, which
    may be qkv's own part).  pos [rows]: positions to turn by where they are not the tokens' places in their sequences.  Rows of no sequence are left."""
    heads, head_dim = kv.desc.n_kv_heads, kv.desc.head_dim
    _need(isinstance(qkv, torch.Tensor) and qkv.is_cuda and qkv.dim() == 2, "qkv has to be rows on a GPU")
    desc, rows, dev = kv._for(qkv.dtype), qkv.shape[0], qkv.device
    n_heads = qkv.shape[1] // head_dim - 2 * heads
    _need(n_heads > 0 and qkv.shape[1] % head_dim == 0, f"rows of {qkv.shape[1]} values do not hold query heads beside 2 x {heads} heads of {head_dim}")
    with _on(dev) as stream:
        b = batch._for(rows, kv)
        d = _rope_desc(qkv, n_heads, heads, head_dim, pos, inv_freq, q_gain, k_gain, eps, interleaved, rot_scale)
        d.ld = _rows_of(qkv, "qkv", qkv.shape[1], qkv.dtype, kv.device)
        if out is None:
            q = torch.empty(rows, n_heads, head_dim, dtype=qkv.dtype, device=dev)
            d.ldq = n_heads * head_dim
        else:
            q = out
            _need(q.shape[0] == rows, f"out has {q.shape[0]} rows, qkv {rows}")
            d.ldq = _rows_of(q, "out", n_heads * head_dim, qkv.dtype, dev)
            _apart(q, d.ldq, "out")
        d.q_out = q.data_ptr()
        _checked(L.load().oavsr_op_paged_append(C.byref(desc), C.byref(b), C.byref(d), stream))
    return q


def read(kv, batch, rows=None, *, dtype=None, out=None):
    """The cached keys and values of the batch's `rows` rows (cu_q[-1]; more are left out), as (k, v) [rows][n_kv_heads][head_dim] in `dtype` (default: the
    cache's; bfloat16 of an 8-bit one).  `out` = (k, v) to write into, either may be None; rows of no sequence are left as they were."""
    heads, head_dim = kv.desc.n_kv_heads, kv.desc.head_dim
    given = [t for t in out or () if t is not None]
    _need(out is None or (len(out) == 2 and given), "out is (k, v), one of them at least a tensor")
    _need(out is not None or rows is not None, "rows or out is needed")
    if dtype is None:
        dtype = given[0].dtype if given else torch.bfloat16 if kv.is_8bit else kv.k.dtype
    desc = kv._for(dtype)
    with _on(kv.device) as stream:
        if out is None:
            k, v = (torch.empty(rows, heads, head_dim, dtype=dtype, device=kv.device) for _ in range(2))
        else:
            k, v = out
            rows = given[0].shape[0] if rows is None else rows
            _need(all(t.shape[0] == rows for t in given), f"out has {[t.shape[0] for t in given]} rows, {rows} are wanted")
        ld = []
        for t, name in ((k, "out[0]"), (v, "out[1]")):
            ld.append(heads * head_dim if t is None else _rows_of(t, name, heads * head_dim, dtype, kv.device))
            if t is not None:
                _apart(t, ld[-1], name)
        b = batch._for(rows, kv)
        _checked(L.load().oavsr_op_paged_read(C.byref(desc), C.byref(b), None if k is None else k.data_ptr(), ld[0], None if v is None else v.data_ptr(), ld[1], stream))
    return k, v


def attention(kv, batch, q, scale=None, *, out=None, lse=None, split_keys=0):
    """Causal attention of the batch's new tokens q [rows][n_heads][head_dim] (or [rows][n_heads * head_dim]) over their sequences' cached context.  Returns
    out, shaped like q.  scale: default head_dim ** -0.5.  lse: float32 [rows][n_heads] to fill.  split_keys: keys per workgroup (a multiple of 256; 0: the
    library's rule), for results whose last bits do not follow the batch a row is in."""
    heads, head_dim = kv.desc.n_kv_heads, kv.desc.head_dim
    _need(isinstance(q, torch.Tensor) and q.is_cuda and q.dim() in (2, 3), "q has to be rows on a GPU")
    desc, rows, dev = kv._for(q.dtype), q.shape[0], q.device
    width = q.shape[1] * (q.shape[2] if q.dim() == 3 else 1)
    _need(width % head_dim == 0 and (q.dim() == 2 or q.shape[2] == head_dim), f"q is {tuple(q.shape)}, the cache's heads have {head_dim} dimensions")
    d = L.PagedAttnDesc()
    d.n_heads, d.scale, d.split_keys = width // head_dim, head_dim ** -0.5 if scale is None else scale, split_keys
    _need(math.isfinite(d.scale), f"scale {scale}")
    with _on(dev) as stream:
        d.Q, d.ldq = q.data_ptr(), _rows_of(q, "q", width, q.dtype, kv.device)
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=dev)
            d.ldo = width
        else:
            _need(out.shape[0] == rows, f"out has {out.shape[0]} rows, q {rows}")
            d.ldo = _rows_of(out, "out", width, q.dtype, dev)
            _apart(out, d.ldo, "out")
        d.O = out.data_ptr()
        if lse is not None:
            _on_gpu(lse, "lse", torch.float32, dev)
            _need(lse.shape == (rows, d.n_heads) and lse.is_contiguous(), f"lse is {tuple(lse.shape)}, ({rows}, {d.n_heads}) in one piece is wanted")
            d.lse = lse.data_ptr()
        b, lib = batch._for(rows, kv), L.load()
        need = lib.oavsr_paged_attention_workspace(C.byref(desc), C.byref(b), C.byref(d))
        if need < 0:
            _checked(-1)
        work = torch.empty(need, dtype=torch.uint8, device=dev) if need else None      # of this call alone; the allocator reuses it in stream order
        if need:
            d.workspace, d.workspace_bytes = work.data_ptr(), need
        _checked(lib.oavsr_op_paged_attention(C.byref(desc), C.byref(b), C.byref(d), stream))
    return out
