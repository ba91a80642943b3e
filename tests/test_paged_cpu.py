"""CPU: what the paged-cache entry points refuse (before any device call), the workspace rule, and the checks of lengths and page numbers."""
import ctypes as C

import pytest
import torch

from omni_avsr_amd import lib as L, paged

A = 1 << 20          # stands for a device address, 16-byte aligned; never followed


def kv_desc(**over):
    d = L.PagedKvDesc()
    d.dtype, d.format, d.n_kv_heads, d.head_dim, d.page_size, d.n_pages, d.K, d.V = L.DT_BF16, L.KV_SAME, 2, 64, 16, 10, A, A
    for k, v in over.items():
        setattr(d, k, v)
    if "page_stride" not in over:
        d.page_stride = d.n_kv_heads * d.page_size * d.head_dim
    if "scale_stride" not in over:
        d.scale_stride = d.n_kv_heads * d.page_size
    return d


def batch_desc(**over):
    d = L.PagedBatchDesc()
    d.n_seqs, d.rows, d.max_q, d.max_ctx, d.cu_q, d.ctx_len, d.table, d.ld_table = 2, 5, 4, 40, A, A, A, 3
    for k, v in over.items():
        setattr(d, k, v)
    return d


def rope_desc(**over):
    d = L.QkRopeDesc()
    d.dtype, d.rows, d.n_heads, d.n_kv_heads, d.head_dim, d.qkv, d.ld, d.q_out, d.ldq, d.k_out, d.ldk = L.DT_BF16, 5, 4, 2, 64, A, 512, A, 256, A, 128
    d.pos, d.inv_freq, d.rot_dim, d.rot_scale = A, A, 64, 1.0
    for k, v in over.items():
        setattr(d, k, v)
    return d


def attn_desc(**over):
    d = L.PagedAttnDesc()
    d.n_heads, d.scale, d.Q, d.ldq, d.O, d.ldo = 4, 0.125, A, 256, A, 256
    for k, v in over.items():
        setattr(d, k, v)
    return d


def refused(rc, word):
    assert rc == -1 and word in L.last_error(), (rc, L.last_error())


BAD_KV = [(dict(dtype=7), "dtype"), (dict(format=2), "format"), (dict(head_dim=96), "head_dim"), (dict(page_size=24), "page_size"), (dict(page_size=8), "page_size"),
          (dict(page_size=512, page_stride=1 << 20), "page_size"), (dict(n_kv_heads=0), "sizes"), (dict(n_pages=-1), "sizes"), (dict(page_stride=2040), "stride"),
          (dict(page_stride=2052), "stride"), (dict(K=None), "null"), (dict(V=A + 8), "aligned"), (dict(format=1), "scales"),
          (dict(format=1, k_scale=A, v_scale=A, scale_stride=31), "scale stride"), (dict(format=1, k_scale=A, v_scale=A, scale_stride=34), "scale stride")]
BAD_BATCH = [(dict(n_seqs=-1), "sizes"), (dict(rows=-1), "sizes"), (dict(max_q=-1), "sizes"), (dict(max_ctx=49), "table"), (dict(cu_q=None), "null"),
             (dict(table=None), "null"), (dict(ctx_len=None), "null"), (dict(ld_table=-1), "table"), (dict(ld_table=1 << 33, max_ctx=(1 << 30) + 1), "max_ctx")]


@pytest.mark.parametrize("kv,batch,word", [(k, {}, w) for k, w in BAD_KV] + [({}, b, w) for b, w in BAD_BATCH])
def test_cache_and_batch_refusals(kv, batch, word):
    lib, k, b = L.load(), kv_desc(**kv), batch_desc(**batch)
    r = rope_desc(rows=b.rows)
    refused(lib.oavsr_op_paged_attention(C.byref(k), C.byref(b), C.byref(attn_desc()), None), word)
    refused(lib.oavsr_paged_attention_workspace(C.byref(k), C.byref(b), C.byref(attn_desc())), word)
    refused(lib.oavsr_op_paged_append(C.byref(k), C.byref(b), C.byref(r), None), word)
    refused(lib.oavsr_op_paged_read(C.byref(k), C.byref(b), A, 128, A, 128, None), word)
    refused(lib.oavsr_paged_check_host(C.byref(k), C.byref(b)), word)


@pytest.mark.parametrize("over,word", [
    (dict(dtype=3), "dtype"), (dict(rows=-1), "sizes"), (dict(n_heads=0), "sizes"), (dict(head_dim=32), "head_dim"), (dict(ld=504), "shorter"), (dict(ldq=248), "shorter"),
    (dict(ld=516), "aligned"), (dict(qkv=A + 2), "aligned"), (dict(q_gain=A), "gains"), (dict(q_gain=A, k_gain=A + 4), "aligned"), (dict(q_gain=A, k_gain=A, eps=-1.0), "eps"),
    (dict(rot_dim=24), "rotated"), (dict(rot_dim=0), "rotated"), (dict(rot_dim=80), "rotated"), (dict(q_out=None), "null")])
def test_rope_refusals(over, word):
    lib = L.load()
    refused(lib.oavsr_op_qk_norm_rope(C.byref(rope_desc(**over)), None), word)
    refused(lib.oavsr_op_paged_append(C.byref(kv_desc()), C.byref(batch_desc()), C.byref(rope_desc(**over)), None), word)


def test_rope_alone_needs_keys_and_positions():
    lib = L.load()
    refused(lib.oavsr_op_qk_norm_rope(C.byref(rope_desc(k_out=None)), None), "null")
    refused(lib.oavsr_op_qk_norm_rope(C.byref(rope_desc(pos=None)), None), "null")
    refused(lib.oavsr_op_qk_norm_rope(C.byref(rope_desc(ldk=120)), None), "shorter")
    assert lib.oavsr_op_qk_norm_rope(C.byref(rope_desc(rows=0)), None) == 0


@pytest.mark.parametrize("over", [dict(rows=4), dict(dtype=L.DT_F32), dict(n_kv_heads=1), dict(head_dim=128, ld=1024, ldq=512)])
def test_append_rows_have_to_fit_the_cache_and_the_batch(over):
    refused(L.load().oavsr_op_paged_append(C.byref(kv_desc()), C.byref(batch_desc()), C.byref(rope_desc(**over)), None), "not the batch's")


@pytest.mark.parametrize("over,word", [
    (dict(n_heads=3), "multiple"), (dict(n_heads=0), "multiple"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(split_keys=100), "split_keys"), (dict(split_keys=-256), "split_keys"), (dict(ldq=248), "strides"), (dict(ldo=260), "strides"),
    (dict(Q=None), "null"), (dict(O=A + 8), "aligned"), (dict(n_heads=1 << 29, ldq=1 << 35, ldo=1 << 35), "too many")])
def test_attention_refusals(over, word):
    refused(L.load().oavsr_op_paged_attention(C.byref(kv_desc()), C.byref(batch_desc()), C.byref(attn_desc(**over)), None), word)


def test_attention_workspace():
    """(head_dim + 2) floats per split, row and head; too small a workspace is refused; nothing without splits or rows."""
    lib, kv = L.load(), kv_desc()
    b = batch_desc(max_ctx=5000, ld_table=400)
    need = lib.oavsr_paged_attention_workspace(C.byref(kv), C.byref(b), C.byref(attn_desc(split_keys=1024)))
    assert need == 5 * 5 * 4 * 66 * 4
    refused(lib.oavsr_op_paged_attention(C.byref(kv), C.byref(b), C.byref(attn_desc(split_keys=1024, workspace=A, workspace_bytes=need - 1)), None), "workspace")
    refused(lib.oavsr_op_paged_attention(C.byref(kv), C.byref(b), C.byref(attn_desc(split_keys=1024, workspace_bytes=need)), None), "workspace")
    assert lib.oavsr_paged_attention_workspace(C.byref(kv), C.byref(b), C.byref(attn_desc(split_keys=5120))) == 0
    assert lib.oavsr_op_paged_attention(C.byref(kv), C.byref(batch_desc(rows=0)), C.byref(attn_desc()), None) == 0
    assert lib.oavsr_op_paged_attention(C.byref(kv), C.byref(batch_desc(n_seqs=0)), C.byref(attn_desc()), None) == 0
    assert lib.oavsr_op_paged_read(C.byref(kv), C.byref(b), None, 0, None, 0, None) == 0


def test_null_descriptors():
    lib = L.load()
    for rc in (lib.oavsr_op_qk_norm_rope(None, None), lib.oavsr_op_paged_append(None, None, None, None), lib.oavsr_op_paged_read(None, None, None, 0, None, 0, None),
               lib.oavsr_op_paged_attention(None, None, None, None), lib.oavsr_paged_attention_workspace(None, None, None), lib.oavsr_paged_check_host(None, None)):
        refused(rc, "null desc")


PAGE, LENGTH = L.PAGED_BAD_PAGE, L.PAGED_BAD_LENGTH


@pytest.mark.parametrize("cu,ctx,table,bits", [
    ([0, 2, 5], [20, 33], [[1, 2, -1], [3, 4, 5]], 0),               # a place behind the context is not looked at
    ([0, 2, 5], [0, 2], [[-1, -1, -1], [9, -1, -1]], 0),             # an empty context; rows before their sequence's first place
    ([0, 0, 5], [16, 17], [[0, -9, 99], [0, 1, 99]], LENGTH),        # five new tokens, max_q 4
    ([0, 2, 5], [17, 33], [[1, 10, 0], [3, 4, 5]], PAGE),            # one behind the pool
    ([0, 2, 5], [17, 33], [[1, -1, 0], [3, 4, 5]], PAGE),
    ([0, 2, 5], [17, 33], [[1, -2 ** 31, 0], [3, 2 ** 31 - 1, 5]], PAGE),
    ([0, 2, 5], [41, 1], [[1, 2, 3], [3, 4, 5]], LENGTH),            # longer than max_ctx; its pages up to there are sound
    ([0, 2, 5], [2 ** 31 - 1, -1], [[1, 2, 3], [3, 4, 5]], LENGTH),
    ([0, 3, 2], [3, 3], [[1, 2, 3], [3, 4, 5]], LENGTH),             # falls
    ([0, 2, 6], [3, 4], [[1, 2, 3], [3, 4, 5]], LENGTH),             # passes the rows
    ([-1, 2, 5], [3, 4], [[1, 2, 3], [3, 4, 5]], LENGTH),
    ([-2 ** 31, 2 ** 31 - 1, 5], [3, 4], [[1, 2, 3], [3, 4, 5]], LENGTH),
    ([0, 2, 5], [41, 33], [[1, 2, 30], [3, 4, 5]], PAGE | LENGTH)])
def test_lengths_and_page_numbers(cu, ctx, table, bits):
    """The functions the kernels look sequences and pages up with, on host arrays."""
    t = [torch.tensor(x, dtype=torch.int32) for x in (cu, ctx, table)]
    b = batch_desc(cu_q=t[0].data_ptr(), ctx_len=t[1].data_ptr(), table=t[2].data_ptr())
    assert L.load().oavsr_paged_check_host(C.byref(kv_desc()), C.byref(b)) == bits


def test_tensors_of_the_host_are_refused():
    k, i = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: paged.PagedKV(k, k), lambda: paged.PagedBatch(i, i[:1], i[None], max_q=1, max_ctx=1),
                 lambda: paged.qk_norm_rope(torch.zeros(2, 512), 4, 2, i, torch.zeros(32))):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_status_is_taken_from_one_word_into_another():
    lib = L.load()
    refused(lib.oavsr_paged_take_status(None, A, None), "null desc")
    refused(lib.oavsr_paged_take_status(C.byref(kv_desc()), A, None), "null status")
    refused(lib.oavsr_paged_take_status(C.byref(kv_desc(status=A)), None, None), "null status")


@pytest.mark.parametrize("cu,ctx,table,bits", [
    ([0, 0, 4], [33, 33], [[-1, -1, -1], [3, 4, 5]], 0),             # an idle slot: its old length, its pages given back
    ([0, 4, 4], [33, 40], [[3, 4, 5], [1, 99, 99]], 0),
    ([0, 0, 4], [41, 33], [[-1, -1, -1], [3, 4, 5]], LENGTH),        # its length is looked at
    ([0, 5, 5], [33, 0], [[-1, -1, -1], [3, 4, 5]], LENGTH),         # skipped for its five new tokens
    ([0, 6, 5], [33, 0], [[-1, -1, -1], [3, 4, 5]], LENGTH),
    ([0, 1, 1], [33, 33], [[3, -1, 5], [3, 4, 5]], PAGE)])
def test_pages_of_sequences_that_bring_no_rows_are_not_looked_at(cu, ctx, table, bits):
    test_lengths_and_page_numbers(cu, ctx, table, bits)


@pytest.mark.parametrize("call", [
    lambda lib: lib.oavsr_op_qk_norm_rope(C.byref(rope_desc(rows=1 << 26)), None),                                                   # a wave per row: 2^32 threads
    lambda lib: lib.oavsr_op_paged_append(C.byref(kv_desc()), C.byref(batch_desc(rows=1 << 26)), C.byref(rope_desc(rows=1 << 26)), None),
    lambda lib: lib.oavsr_op_paged_read(C.byref(kv_desc()), C.byref(batch_desc(rows=1 << 26)), A, 128, A, 128, None),
    lambda lib: lib.oavsr_op_paged_read(C.byref(kv_desc()), C.byref(batch_desc(rows=2 ** 31 - 1)), A, 128, A, 128, None),
    lambda lib: lib.oavsr_op_paged_attention(C.byref(kv_desc()), C.byref(batch_desc(n_seqs=1 << 23)), C.byref(attn_desc()), None),     # single tokens: 256 threads a sequence and kv head
    lambda lib: lib.oavsr_op_paged_attention(C.byref(kv_desc()), C.byref(batch_desc(rows=1 << 22, max_q=1 << 22, max_ctx=5000, ld_table=400)),
                                             C.byref(attn_desc(split_keys=256, workspace=A, workspace_bytes=1 << 60)), None)])          # the join: 256 threads a row and head
def test_launches_of_more_threads_than_a_grid_holds_are_refused(call):
    """2^32 threads and more in one launch: refused before anything is queued."""
    refused(call(L.load()), "too many")
