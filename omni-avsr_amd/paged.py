"""The paged key / value cache and its operators on tensors (C ABI: include/omni_avsr.h, oavsr_op_qk_norm_rope and oavsr_op_paged_*).

A decoder layer with its cache in pages runs, per step,

    q   = paged.append(kv, batch, qkv, inv_freq)      # norm + rotation of the fused [q | k | v] rows, k and v into the pages
    out = paged.attention(kv, batch, q)               # the new tokens over their sequences' context

with one `PagedKV` per layer (its pool of pages) and one `PagedBatch` per step (row offsets, lengths and page table of the sequences, shared by all layers).
Everything is queued on the current stream of the tensors' device; nothing is synchronised, and every call can be captured into a graph.  An argument that
does not fit raises ValueError before anything is queued, and so does one that asks for gradients (an input, an output or a pool that requires grad or
carries a tangent of forward mode): these are forward passes.  Lengths and page numbers are device data: a bad one never reaches memory outside the given
tensors, and sets its bit in `PagedKV.status` (`PagedKV.check()` raises)."""
from __future__ import annotations

import ctypes as C
import functools

import torch
import torch.autograd.forward_ad as _forward_ad

from . import lib as L

_DT = {torch.float32: L.DT_F32, torch.bfloat16: L.DT_BF16}
_E4M3 = torch.float8_e4m3fn


def _need(ok, what):
    if not ok:
        raise ValueError("paged: " + what)


def _no_gradient(t, name):
    _need(not (t.requires_grad and torch.is_grad_enabled()), f"{name} asks for gradients, and none are formed here: call under torch.no_grad(), or detach it")


def _no_tangents(*tensors):
    """For calls inside a level of forward mode, which no_grad leaves on."""
    for t in tensors:
        _need(not isinstance(t, torch.Tensor) or _forward_ad.unpack_dual(t).tangent is None, "a tensor carries a tangent, and no gradients are formed here: detach it")


def _on_gpu(t, name, dtype, index=None):
    """The device's index of a tensor on a GPU (that of `index`)."""
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() >= 0 and (index is None or t.get_device() == index)):
        _need(isinstance(t, torch.Tensor) and t.is_cuda, f"{name} has to be a tensor on a GPU")
        _need(t.dtype == dtype, f"{name} is {t.dtype}, {dtype} is wanted")
        _need(False, f"{name} is on {t.device}, the others on cuda:{index}")
    return t.get_device()


def _rows_of(t, name, width, dtype, index, rows=None, written=False):
    """Row stride of [rows][width] or [rows][heads][head_dim] rows, each of them one piece of memory; rows that are written must not overlap."""
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == index and t.is_contiguous():      # the common case
        n = t.shape[0] if t.dim() in (2, 3) else -1
        if n == rows if rows is not None else n >= 0:
            if t.numel() == n * width and n > 0:
                return width
    _on_gpu(t, name, dtype, index)
    shape, stride = t.shape, t.stride()
    n = shape[0] if len(shape) > 1 else -1
    _need(len(shape) in (2, 3), f"{name} has {len(shape)} dimensions")
    _need(shape[1] * (shape[2] if len(shape) == 3 else 1) == width, f"{name} has rows of shape {tuple(shape[1:])}, {width} values are wanted")
    _need(rows is None or n == rows, f"{name} has {n} rows, {rows} are wanted")
    if n == 0:
        return width
    _need(stride[-1] == 1 and (len(shape) == 2 or shape[1] == 1 or stride[1] == shape[2]), f"a row of {name} has to be one piece of memory (strides {stride})")
    if n == 1:
        return width
    _need(not written or stride[0] >= width, f"rows of {name} overlap (strides {stride})")
    _need(stride[0] >= width, f"row strides of {name} are shorter than the rows (strides {stride})")
    return stride[0]


def _apart(a, lda, wa, b, ldb, wb, rows, names):
    """Rows of a (lda apart, wa long, from that byte on) and of b share no memory: behind each other, or columns of the same rows.  All in bytes."""
    if rows == 0 or a + (rows - 1) * lda + wa <= b or b + (rows - 1) * ldb + wb <= a:
        return
    off = (b - a) % lda
    _need(lda == ldb and wa <= off and off + wb <= lda, f"{names} overlap")


_lib = functools.lru_cache(None)(L.load)
_stream = torch._C._cuda_getCurrentRawStream      # of a device's index


_device = torch._C._cuda_getDevice               # the current one's index
_written = torch._C._increment_version           # tensors of the caller's that a call writes: a backward pass that has saved one is refused, as after torch's own writes


class _Keeps:
    """An object whose tensors' addresses were taken when it was made: others in their place would not be seen, so they are not accepted."""

    def __setattr__(self, name, value):
        if name in self._kept and self.__dict__.get(name, value) is not value:
            _need(False, f"{name} is kept as it was given: write into it, or make another {type(self).__name__}")
        self.__dict__[name] = value


class PagedKV(_Keeps):
    """A layer's pool of pages: k and v [n_pages][n_kv_heads][page_size][head_dim] in float32, bfloat16, or float8_e4m3fn with k_scale and v_scale
    [n_pages][n_kv_heads][page_size] (float32).  Pages may be further apart than they are large (a view of a larger pool), k's and v's by the same stride.
    Keeps the tensors; `status` is one int32 of device memory, cleared when the constructor returns (which waits for the current stream for that)."""

    _kept = ("k", "v", "k_scale", "v_scale", "status")

    def __init__(self, k, v, k_scale=None, v_scale=None):
        _need(isinstance(k, torch.Tensor) and k.is_cuda, "k has to be a tensor on a GPU")
        _need(k.dim() == 4, f"k has {k.dim()} dimensions, [n_pages][n_kv_heads][page_size][head_dim] is wanted")
        self.device, self.index, self.is_8bit = k.device, k.get_device(), k.dtype == _E4M3
        _need(self.is_8bit or k.dtype in _DT, f"a cache of {k.dtype} is not supported")
        _on_gpu(v, "v", k.dtype, self.index)
        _need(v.shape == k.shape, f"k is {tuple(k.shape)}, v {tuple(v.shape)}")
        n, heads, page, dim = k.shape
        inner = (page * dim, dim, 1)
        for t, name in ((k, "k"), (v, "v")):
            _need(n == 0 or t.stride()[1:] == inner, f"a page of {name} has to be one piece of memory (strides {t.stride()})")
        stride = k.stride(0) if n > 1 else heads * page * dim
        _need(n <= 1 or v.stride(0) == stride, f"k's pages are {k.stride(0)} apart, v's {v.stride(0)}")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self._pools = tuple(t for t in (k, v, k_scale, v_scale) if t is not None)
        self.status = torch.zeros(1, dtype=torch.int32, device=k.device)
        if not torch.cuda.is_current_stream_capturing():      # the word is clear for calls on any stream from here on
            torch.cuda.current_stream(self.index).synchronize()
        d = self.desc = L.PagedKvDesc()
        d.format = L.KV_E4M3 if self.is_8bit else L.KV_SAME
        d.dtype = L.DT_BF16 if self.is_8bit else _DT[k.dtype]
        d.n_kv_heads, d.head_dim, d.page_size, d.n_pages = heads, dim, page, n
        d.K, d.V, d.page_stride, d.status = k.data_ptr(), v.data_ptr(), stride, self.status.data_ptr()
        _need(self.is_8bit == (k_scale is not None) and self.is_8bit == (v_scale is not None), "k_scale and v_scale belong to an 8-bit cache, and only to one")
        if self.is_8bit:
            for t, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
                _on_gpu(t, name, torch.float32, self.index)
                _need(t.shape == k.shape[:3], f"{name} is {tuple(t.shape)}, {tuple(k.shape[:3])} is wanted")
                _need(n == 0 or t.stride()[1:] == (page, 1), f"a page of {name} has to be one piece of memory (strides {t.stride()})")
            d.scale_stride = k_scale.stride(0) if n > 1 else heads * page
            _need(n <= 1 or v_scale.stride(0) == d.scale_stride, f"k_scale's pages are {k_scale.stride(0)} apart, v_scale's {v_scale.stride(0)}")
            d.k_scale, d.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
        # the same for rows of either type, of an 8-bit cache
        self.descs = {t: d for t, code in _DT.items() if code == d.dtype}
        if self.is_8bit:
            self.descs[torch.float32] = type(d).from_buffer_copy(d)
            self.descs[torch.float32].dtype = L.DT_F32
        self.heads, self.head_dim, self.page, self.shape = heads, dim, page, (heads, dim, page, d.format)

    @classmethod
    def empty(cls, n_pages, page_size, n_kv_heads, head_dim, dtype=torch.bfloat16, device="cuda"):
        """A pool of its own; dtype float8_e4m3fn: with scales."""
        shape = (n_pages, n_kv_heads, page_size, head_dim)
        kv = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(2)]
        scales = [torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2)] if dtype == _E4M3 else []
        return cls(*kv, *scales)

    def _for(self, dtype):
        """The description for rows of `dtype`, of pools that ask for no gradients."""
        for t in self._pools:
            if t.requires_grad:
                _no_gradient(t, "a pool of the cache")
        d = self.descs.get(dtype)
        if d is None:
            _need(dtype in _DT, f"rows of {dtype} are not supported")
            _need(False, f"rows are {dtype}, the cache is {self.k.dtype}")
        return d

    def check(self):
        """Raises RuntimeError if a call has met a bad page number or length since the last check.  Waits for the device, so that calls queued before, on any
        stream, are covered, and takes the bits off the word in one step: what others set meanwhile is the next check's.  Not while a graph is captured."""
        with torch.cuda.device(self.index):
            torch.cuda.synchronize()
            taken = torch.empty_like(self.status)
            _checked(_lib().oavsr_paged_take_status(C.byref(self.desc), taken.data_ptr(), _stream(self.index)))
            bits = int(taken.item())
        if bits:
            what = [s for b, s in ((L.PAGED_BAD_PAGE, "a page number outside the pool"), (L.PAGED_BAD_LENGTH, "a length outside the batch's bounds")) if bits & b]
            raise RuntimeError("paged: " + " and ".join(what) + " was met")


class PagedBatch(_Keeps):
    """The sequences of a step: cu_q [n_seqs + 1] (row offsets of their new tokens), ctx_len [n_seqs] (tokens in the cache, the new ones among them), table
    [n_seqs][pages], all int32 on the device.  max_q and max_ctx bound a sequence's new tokens and context.  Keeps the tensors: refilled in place, the
    same batch serves the next step."""

    _kept = ("cu_q", "ctx_len", "table")

    def __init__(self, cu_q, ctx_len, table, *, max_q, max_ctx):
        self.index = _on_gpu(cu_q, "cu_q", torch.int32)
        for t, name, dim in ((cu_q, "cu_q", 1), (ctx_len, "ctx_len", 1), (table, "table", 2)):
            _on_gpu(t, name, torch.int32, self.index)
            _need(t.dim() == dim, f"{name} has {t.dim()} dimensions")
            _need(t.numel() == 0 or t.stride(-1) == 1 or t.shape[-1] == 1, f"{name} has to be one piece of memory (strides {t.stride()})")
        n = ctx_len.shape[0]
        _need(cu_q.shape[0] == n + 1 and table.shape[0] == n, f"{n} sequences by ctx_len, {cu_q.shape[0] - 1} by cu_q, {table.shape[0]} by table")
        _need(0 <= max_q < 2 ** 31 and 0 <= max_ctx < 2 ** 31, f"max_q {max_q}, max_ctx {max_ctx}")
        self.cu_q, self.ctx_len, self.table, self.width = cu_q, ctx_len, table, table.shape[1]
        d = self.desc = L.PagedBatchDesc()
        d.n_seqs, d.max_q, d.max_ctx = n, max_q, max_ctx
        d.cu_q, d.ctx_len, d.table = cu_q.data_ptr(), ctx_len.data_ptr(), table.data_ptr()
        d.ld_table = table.stride(0) if n > 1 else self.width
        _need(n <= 1 or d.ld_table >= self.width, f"rows of table overlap (strides {table.stride()})")
        self._descs, self._work = {}, {}

    def _for(self, rows, kv):
        """The description for so many rows."""
        if self.index != kv.index or self.desc.max_ctx > self.width * kv.page:
            _need(self.index == kv.index, f"the batch is on cuda:{self.index}, the cache on cuda:{kv.index}")
            _need(False, f"a table of {self.width} pages of {kv.page} does not hold max_ctx {self.desc.max_ctx}")
        d = self._descs.get(rows)
        if d is None:
            d = L.PagedBatchDesc.from_buffer_copy(self.desc)
            d.rows = rows
            if len(self._descs) >= 64:
                self._descs.clear()
            self._descs[rows] = d
        return d

    def _workspace(self, d, kv, dtype, n_heads, split_keys):
        """Bytes that attention needs: they follow from bounds that do not change, so they are kept."""
        key = (d.rows, kv.shape, dtype, n_heads, split_keys)
        need = self._work.get(key)
        if need is None:
            _need(0 <= split_keys < 2 ** 31, f"split_keys {split_keys} (a multiple of 256)")
            a = L.PagedAttnDesc(n_heads, 1.0)
            a.split_keys = split_keys
            need = _lib().oavsr_paged_attention_workspace(C.byref(kv._for(dtype)), C.byref(d), C.byref(a))
            if need < 0:
                _checked(-1)
            if len(self._work) >= 64:
                self._work.clear()
            self._work[key] = need
        return need


def _vector(t, name, dtype, index, n=None):
    """Address of a vector (of n) in one piece."""
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == index and t.dim() == 1 and (n is None or t.numel() == n) and t.is_contiguous()):
        _on_gpu(t, name, dtype, index)
        _need(False, f"{name} is {tuple(t.shape)} (strides {t.stride()}), a vector{'' if n is None else f' of {n}'} in one piece is wanted")
    if t.requires_grad:
        _no_gradient(t, name)
    return t.data_ptr()


def _gains(q_gain, k_gain, index, head_dim):
    if q_gain is None and k_gain is None:
        return None, None
    _need(q_gain is not None and k_gain is not None, "gains for both queries and keys, or for neither")
    return _vector(q_gain, "q_gain", torch.float32, index, head_dim), _vector(k_gain, "k_gain", torch.float32, index, head_dim)


def _checked(rc):
    """An argument that the library refuses is a ValueError here; a device error stays one."""
    if rc == -1:
        raise ValueError("paged: " + L.last_error())
    L.check(rc)


def qk_norm_rope(qkv, n_heads, n_kv_heads, pos, inv_freq, *, q_gain=None, k_gain=None, eps=1e-6, interleaved=False, rot_scale=1.0, out=None):
    """Norm (with q_gain, k_gain) and rotation (by pos * inv_freq; None: none) of the query and key heads of fused rows [rows][(n_heads + 2 n_kv_heads) *
    head_dim].  Returns q [rows][n_heads][head_dim] and k [rows][n_kv_heads][head_dim]; `out` = (q, k) to write into: qkv's own parts, or memory apart from
    it.  inv_freq [rot_dim / 2]: the first rot_dim dimensions of a head turn, halves against each other, or neighbours when interleaved."""
    if not (isinstance(qkv, torch.Tensor) and qkv.dim() == 2 and qkv.dtype in _DT and qkv.is_cuda):
        _need(False, "qkv has to be rows of float32 or bfloat16 on a GPU")
    if _forward_ad._current_level >= 0:
        _no_tangents(qkv, inv_freq, q_gain, k_gain, *(out or ()))
    if qkv.requires_grad:
        _no_gradient(qkv, "qkv")
    rows, width = qkv.shape
    dtype, index, all_heads = qkv.dtype, qkv.get_device(), n_heads + 2 * n_kv_heads
    if _device() != index:
        with torch.cuda.device(index):
            return qk_norm_rope(qkv, n_heads, n_kv_heads, pos, inv_freq, q_gain=q_gain, k_gain=k_gain, eps=eps, interleaved=interleaved, rot_scale=rot_scale, out=out)
    if not (n_heads > 0 and n_kv_heads > 0 and width % all_heads == 0):
        _need(False, f"rows of {width} values do not hold {n_heads} + 2 x {n_kv_heads} heads")
    head_dim = width // all_heads
    at_freq, rot = (None, 0) if inv_freq is None else (_vector(inv_freq, "inv_freq", torch.float32, index), 2 * inv_freq.numel())
    at_pos = None if pos is None else _vector(pos, "pos", torch.int32, index, rows)
    at_q, at_k = _gains(q_gain, k_gain, index, head_dim)
    ld = width if rows and qkv.is_contiguous() else _rows_of(qkv, "qkv", width, dtype, index)
    ldq, ldk = n_heads * head_dim, n_kv_heads * head_dim
    if out is None:
        q, k = qkv.new_empty((rows, n_heads, head_dim)), qkv.new_empty((rows, n_kv_heads, head_dim))
    else:
        q, k = out
        ldq, ldk = _rows_of(q, "out[0]", ldq, dtype, index, rows, True), _rows_of(k, "out[1]", ldk, dtype, index, rows, True)
        _no_gradient(q, "out[0]")
        _no_gradient(k, "out[1]")
        e, at, to_q, to_k, q_wide, k_wide = qkv.element_size(), qkv.data_ptr(), q.data_ptr(), k.data_ptr(), n_heads * head_dim, n_kv_heads * head_dim
        if to_q != at or (ldq != ld and rows > 1):                      # else: the rows' own queries
            _apart(at, ld * e, width * e, to_q, ldq * e, q_wide * e, rows, "qkv and out[0]")
        if to_k != at + q_wide * e or (ldk != ld and rows > 1):         # else: their own keys
            _apart(at, ld * e, width * e, to_k, ldk * e, k_wide * e, rows, "qkv and out[1]")
        _apart(to_q, ldq * e, q_wide * e, to_k, ldk * e, k_wide * e, rows, "out[0] and out[1]")
    d = L.QkRopeDesc(_DT[dtype], rows, n_heads, n_kv_heads, head_dim, qkv.data_ptr(), ld, q.data_ptr(), ldq, k.data_ptr(), ldk, at_pos, at_freq, rot,
                     bool(interleaved), rot_scale, at_q, at_k, eps)
    _checked(_lib().oavsr_op_qk_norm_rope(C.byref(d), _stream(index)))
    if out is not None:
        _written((q, k))
    return q, k


def append(kv, batch, qkv, inv_freq=None, *, pos=None, q_gain=None, k_gain=None, eps=1e-6, interleaved=False, rot_scale=1.0, out=None):
    """qk_norm_rope of the batch's rows, the keys and values going into their sequences' pages.  Returns q [rows][n_heads][head_dim] (`out`: where to, qkv's own
    part or memory apart from it).  pos [rows]: positions to turn by where they are not the tokens' places in their sequences.  Rows of no sequence, and those
    before their sequence's first place (where ctx_len counts fewer tokens than are new), are left as they were: in a q made here, undefined."""
    if not (isinstance(qkv, torch.Tensor) and qkv.dim() == 2 and qkv.is_cuda):
        _need(False, "qkv has to be rows on a GPU")
    heads, head_dim, index = kv.heads, kv.head_dim, kv.index
    if _device() != index:
        with torch.cuda.device(index):
            return append(kv, batch, qkv, inv_freq, pos=pos, q_gain=q_gain, k_gain=k_gain, eps=eps, interleaved=interleaved, rot_scale=rot_scale, out=out)
    if _forward_ad._current_level >= 0:
        _no_tangents(qkv, inv_freq, q_gain, k_gain, out, *kv._pools)
    if qkv.requires_grad:
        _no_gradient(qkv, "qkv")
    rows, width = qkv.shape
    dtype = qkv.dtype
    desc = kv._for(dtype)
    n_heads = width // head_dim - 2 * heads
    if not (n_heads > 0 and width % head_dim == 0):
        _need(False, f"rows of {width} values do not hold query heads beside 2 x {heads} heads of {head_dim}")
    ld = width if rows and qkv.is_contiguous() and qkv.get_device() == index else _rows_of(qkv, "qkv", width, dtype, index)
    at_freq, rot = (None, 0) if inv_freq is None else (_vector(inv_freq, "inv_freq", torch.float32, index), 2 * inv_freq.numel())
    at_pos = None if pos is None else _vector(pos, "pos", torch.int32, index, rows)
    at_q, at_k = _gains(q_gain, k_gain, index, head_dim)
    b = batch._for(rows, kv)
    ldq = n_heads * head_dim
    written = kv._pools
    if out is None:
        out = qkv.new_empty((rows, n_heads, head_dim))
    else:
        ldq = _rows_of(out, "out", ldq, dtype, index, rows, True)
        _no_gradient(out, "out")
        if out.data_ptr() != qkv.data_ptr() or (ldq != ld and rows > 1):      # else: the rows' own queries
            e = qkv.element_size()
            _apart(qkv.data_ptr(), ld * e, width * e, out.data_ptr(), ldq * e, n_heads * head_dim * e, rows, "qkv and out")
        written += (out,)
    d = L.QkRopeDesc(_DT[dtype], rows, n_heads, heads, head_dim, qkv.data_ptr(), ld, out.data_ptr(), ldq, None, 0, at_pos, at_freq, rot, bool(interleaved), rot_scale,
                     at_q, at_k, eps)
    _checked(_lib().oavsr_op_paged_append(C.byref(desc), C.byref(b), C.byref(d), _stream(index)))
    _written(written)
    return out


def read(kv, batch, rows=None, *, dtype=None, out=None):
    """The cached keys and values of the batch's `rows` rows (cu_q[-1]; more are left out), as (k, v) [rows][n_kv_heads][head_dim] in `dtype` (default: the
    cache's; bfloat16 of an 8-bit one).  `out` = (k, v) to write into, either may be None; rows of no sequence are left as they were."""
    heads, head_dim, index = kv.heads, kv.head_dim, kv.index
    if _device() != index:
        with torch.cuda.device(index):
            return read(kv, batch, rows, dtype=dtype, out=out)
    if _forward_ad._current_level >= 0:
        _no_tangents(*(out or ()), *kv._pools)
    ldk = ldv = width = heads * head_dim
    if out is None:
        if not (rows is not None):
            _need(False, "rows or out is needed")
        if dtype is None:
            dtype = torch.bfloat16 if kv.is_8bit else kv.k.dtype
        desc = kv._for(dtype)
        k = torch.empty((rows, heads, head_dim), dtype=dtype, device=kv.device)
        v = torch.empty_like(k)
        at_k, at_v = k.data_ptr(), v.data_ptr()
    else:
        given = [t for t in out if t is not None]
        if not (len(out) == 2 and given and all(isinstance(t, torch.Tensor) for t in given)):
            _need(False, "out is (k, v), one of them at least a tensor")
        k, v = out
        dtype = given[0].dtype if dtype is None else dtype
        rows = given[0].shape[0] if rows is None else rows
        desc = kv._for(dtype)
        at_k = at_v = None
        if k is not None:
            ldk, at_k = _rows_of(k, "out[0]", width, dtype, index, rows, True), k.data_ptr()
            _no_gradient(k, "out[0]")
        if v is not None:
            ldv, at_v = _rows_of(v, "out[1]", width, dtype, index, rows, True), v.data_ptr()
            _no_gradient(v, "out[1]")
        if len(given) == 2:
            e = k.element_size()
            _apart(at_k, ldk * e, width * e, at_v, ldv * e, width * e, rows, "out[0] and out[1]")
    b = batch._for(rows, kv)
    _checked(_lib().oavsr_op_paged_read(C.byref(desc), C.byref(b), at_k, ldk, at_v, ldv, _stream(index)))
    if out is not None:
        _written(given)
    return k, v


def attention(kv, batch, q, scale=None, *, out=None, lse=None, split_keys=0):
    """Causal attention of the batch's new tokens q [rows][n_heads][head_dim] (or [rows][n_heads * head_dim]) over their sequences' cached context.  Returns
    out, shaped like q (which it may be).  scale: default head_dim ** -0.5.  lse: float32 [rows][n_heads] to fill.  split_keys: keys per workgroup
    (a multiple of 256; 0: the library's rule): a row then has the same bits in any batch of the same max_q.  max_q chooses the kernel: up to 16 rows per kv
    head (max_q * n_heads / n_kv_heads) weigh bf16 values by two bf16 numbers each, more by one, a rounding more."""
    index, head_dim = kv.index, kv.head_dim
    if not (isinstance(q, torch.Tensor) and q.dim() in (2, 3) and q.is_cuda):
        _need(False, "q has to be rows on a GPU")
    if _device() != index:
        with torch.cuda.device(index):
            return attention(kv, batch, q, scale, out=out, lse=lse, split_keys=split_keys)
    if _forward_ad._current_level >= 0:
        _no_tangents(q, out, lse, *kv._pools)
    if q.requires_grad:
        _no_gradient(q, "q")
    dtype, shape = q.dtype, q.shape
    desc, rows = kv._for(dtype), shape[0]
    width = shape[1] * shape[2] if len(shape) == 3 else shape[1]
    n_heads = width // head_dim
    if not (width % head_dim == 0 and (len(shape) == 2 or shape[2] == head_dim)):
        _need(False, f"q is {tuple(shape)}, the cache's heads have {head_dim} dimensions")
    scale = head_dim ** -0.5 if scale is None else scale
    ldq = width if rows and q.is_contiguous() and q.get_device() == index else _rows_of(q, "q", width, dtype, index)
    b = batch._for(rows, kv)
    need = batch._workspace(b, kv, dtype, n_heads, split_keys)
    ldo = width
    given = None if out is None and lse is None else [t for t in (out, lse) if t is not None]
    if out is None:
        out = torch.empty_like(q) if ldq == width else q.new_empty(shape)
    else:
        ldo = _rows_of(out, "out", width, dtype, index, rows, True)
        _no_gradient(out, "out")
        if out.data_ptr() != q.data_ptr() or (ldo != ldq and rows > 1):
            e = q.element_size()
            _apart(q.data_ptr(), ldq * e, width * e, out.data_ptr(), ldo * e, width * e, rows, "q and out")
    at_lse = None
    if lse is not None:
        _on_gpu(lse, "lse", torch.float32, index)
        if not (lse.shape == (rows, n_heads) and lse.is_contiguous()):
            _need(False, f"lse is {tuple(lse.shape)}, ({rows}, {n_heads}) in one piece is wanted")
        _no_gradient(lse, "lse")
        at_lse = lse.data_ptr()
    work = torch.empty(need, dtype=torch.uint8, device=kv.device) if need else None      # of this call alone; the allocator reuses it in stream order
    d = L.PagedAttnDesc(n_heads, scale, q.data_ptr(), ldq, out.data_ptr(), ldo, at_lse, split_keys, None if work is None else work.data_ptr(), need)
    _checked(_lib().oavsr_op_paged_attention(C.byref(desc), C.byref(b), C.byref(d), _stream(index)))
    if given:
        _written(given)
    return out
