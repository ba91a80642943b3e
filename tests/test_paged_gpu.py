"""-m gpu: the paged key / value cache -- norm + rotation, append, read back, attention -- against plain 64-bit forms on the same (rounded) inputs.

Tolerances count roundings.  u(t) = eps(t) / 2 is the largest relative error of one rounding to t (bf16 2^-8, f32 2^-24, e4m3 2^-4).
  rotation   one rounding of the result, u(t) |y|; before it f32 work on the pair (a, b): the norm's sum of head_dim squares (half its relative error), the
             angle to 2^-24, sine and cosine to 4 u(f32), two products and a sum: (head_dim / 2 + 16) u(f32) (|a| + |b|)
  8 bits     u(e4m3) |x| or half the smallest step, 2^-10 scale; then x's own error as above and the rounding of what is read
  attention  with P the exact probabilities and S = max_j sum_d |q_d k_jd| scale:  a score is off by (head_dim + 4) u(f32) S, so a probability by twice
             that and 4 u(f32) for the exponential; sums over n keys by n u(f32); bf16 rounds the unnormalised P once, u(bf16).  All of it times
             A = sum_j P_j |v_j|, then u(t) |y|."""
import math

import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu

from omni_avsr_amd import paged  # noqa: E402
from omni_avsr_amd.weights import rope_inv_freq  # noqa: E402
from gpu_util import DEV, tdt  # noqa: E402

E4M3 = torch.float8_e4m3fn
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
U32 = 2.0 ** -24


def rnd(*shape, seed=0, scale=1.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def within(got, want, tol, what):
    """|got - want| <= tol everywhere, element by element (64 bits, on the CPU)."""
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} / {bad.numel()} off, worst {float(((got - want).abs() / (tol + 1e-300))[bad].max()):.3g} x the bound"


class Pool:
    """A cache on the GPU whose every byte is NaN until written, its pages shuffled, and the batch's tables; a 64-bit copy of what was written."""

    def __init__(self, kv_heads, head_dim, page, dtype, fmt, lens, seed=0, spare=2, gap=0):
        self.kvh, self.d, self.page, self.fmt, self.dtype = kv_heads, head_dim, page, fmt, tdt(dtype)
        need = [-(-max(n, 0) // page) for n in lens]
        self.n = sum(need) + spare
        stored = E4M3 if fmt == "e4m3" else self.dtype
        def pool(*shape, dt):
            size = math.prod(shape[1:]) + gap                    # pages further apart than they are large
            flat = torch.full((self.n, size), 0x7f if dt == E4M3 else float("nan"), dtype=torch.uint8 if dt == E4M3 else dt, device=DEV)
            flat = flat.view(dt) if dt == E4M3 else flat
            return flat.as_strided((self.n, *shape[1:]), (size, *torch.empty(shape[1:], device="meta").stride()))
        shape = (self.n, kv_heads, page, head_dim)
        t = [pool(*shape, dt=stored) for _ in range(2)]
        if fmt == "e4m3":
            t += [pool(*shape[:3], dt=torch.float32) for _ in range(2)]
        self.kv = paged.PagedKV(*t)
        order = torch.randperm(self.n, generator=torch.Generator().manual_seed(seed + 99)).tolist()
        width = max(max(need), 1)
        self.table = torch.full((len(lens), width), -7, dtype=torch.int32)
        for s, m in enumerate(need):
            for j in range(m):
                self.table[s, j] = order.pop()

    def batch(self, new, ctx, max_q=None, max_ctx=None):
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
        return paged.PagedBatch(i32(cu), i32(ctx), self.table.to(DEV), max_q=max(new) if max_q is None else max_q, max_ctx=max(max(ctx), 0) if max_ctx is None else max_ctx)

    def fill(self, lens, seed=1, scale=1.0):
        """Random keys and values for every sequence, written through append (no rotation); returns them as 64-bit lists, as the cache holds them."""
        rows = sum(lens)
        qkv = rnd(rows, 3 * self.kvh * self.d, seed=seed, scale=scale).to(self.dtype).to(DEV)
        b = self.batch(lens, lens)
        paged.append(self.kv, b, qkv)
        k, v = paged.read(self.kv, b, rows, dtype=torch.float32 if self.fmt == "e4m3" else self.dtype)
        self.kv.check()
        return [list(x.cpu().double().split(lens)) for x in (k, v)]


# ---- norm and rotation ------------------------------------------------------------------------------------------------------------------------
def rotated(x, pos, inv, gain, eps, rot, interleaved, m):
    """(result, error bound before the last rounding) of heads x [rows][heads][head_dim] in 64 bits."""
    x = x.double()
    d = x.shape[-1]
    if gain is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * gain.double()
    y, size = x.clone(), x.abs()
    if rot:
        t = pos.double()[:, None, None] * inv.double()
        a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
        u, v, s = m * (a * t.cos() - b * t.sin()), m * (b * t.cos() + a * t.sin()), m * (a.abs() + b.abs())
        if interleaved:
            y[..., 0:rot:2], y[..., 1:rot:2], size[..., 0:rot:2], size[..., 1:rot:2] = u, v, s, s
        else:
            y[..., :rot // 2], y[..., rot // 2:rot], size[..., :rot // 2], size[..., rot // 2:rot] = u, v, s, s
    return y, (d / 2 + 16) * U32 * size


def freqs(rot):
    return rope_inv_freq(rot, 500000.0, dict(factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=8192)) if rot else None


ROPE = [("f32", 4, 2, 64, 64, False, True, 7), ("bf16", 4, 2, 64, 64, False, True, 7), ("bf16", 28, 4, 128, 128, False, False, 33), ("bf16", 5, 1, 128, 128, True, True, 1),
        ("f32", 7, 7, 128, 32, True, False, 3), ("bf16", 14, 2, 64, 16, False, True, 65), ("bf16", 40, 8, 128, 96, False, True, 2049), ("f32", 9, 3, 64, 48, False, True, 2100),
        ("bf16", 3, 1, 64, 0, False, True, 5), ("f32", 16, 4, 64, 0, False, False, 4)]


@pytest.mark.parametrize("dtype,H,KV,d,rot,inter,norm,rows", ROPE)
def test_qk_norm_rope(dtype, H, KV, d, rot, inter, norm, rows):
    dt = tdt(dtype)
    qkv = rnd(rows, (H + 2 * KV) * d, seed=rows, dtype=dt)
    qkv[0, :d] = 0                                                    # a head of zeros
    pos = torch.randint(0, 200000, (rows,), generator=torch.Generator().manual_seed(2), dtype=torch.int32)
    pos[-1] = 2 ** 20 + 1
    inv, m = freqs(rot), 1.25 if rot else 1.0
    gains = [rnd(d, seed=s) for s in (5, 6)] if norm else [None, None]
    dev = [None if t is None else t.to(DEV) for t in (inv, *gains)]
    # rows further apart than they are long
    wide = torch.full((rows, qkv.shape[1] + 8), float("nan"), dtype=dt, device=DEV)
    wide[:, :qkv.shape[1]] = qkv.to(DEV)
    q, k = paged.qk_norm_rope(wide[:, :qkv.shape[1]], H, KV, pos.to(DEV), dev[0], q_gain=dev[1], k_gain=dev[2], eps=1e-5, interleaved=inter, rot_scale=m)
    x = qkv.view(rows, H + 2 * KV, d)
    for got, part, gain, what in ((q, x[:, :H], gains[0], "q"), (k, x[:, H:H + KV], gains[1], "k")):
        y, err = rotated(part, pos, inv, gain, 1e-5, rot, inter, m)
        within(got, y, err + U[dt] * (y.abs() + err), what)
    # in place, on the rows' own parts: the same bits, the values untouched
    row = wide[:, :qkv.shape[1]]
    parts = (row[:, :H * d], row[:, H * d:(H + KV) * d])
    paged.qk_norm_rope(row, H, KV, pos.to(DEV), dev[0], q_gain=dev[1], k_gain=dev[2], eps=1e-5, interleaved=inter, rot_scale=m, out=parts)
    assert torch.equal(parts[0].reshape(q.shape), q) and torch.equal(parts[1].reshape(k.shape), k)
    assert torch.equal(row[:, (H + KV) * d:].cpu(), qkv[:, (H + KV) * d:]) and wide[:, qkv.shape[1]:].isnan().all()


# ---- append and read ----------------------------------------------------------------------------------------------------------------------------
def e4m3(x, scale):
    """The e4m3 value nearest to x / scale (64 bits; ties to even), times scale."""
    y = x / scale
    step = torch.exp2((torch.frexp(y)[1] - 1).clamp_min(-6).double() - 3)
    return (torch.round(y / step) * step).clamp(-448, 448) * scale


APPEND = [("bf16", "same", 28, 4, 128, 16, False, [1, 1, 1], [1, 16, 17]), ("f32", "same", 4, 2, 64, 32, True, [5, 0, 40], [5, 0, 77]),
          ("bf16", "e4m3", 14, 2, 64, 16, True, [3, 1, 31], [3, 900, 31]), ("bf16", "e4m3", 8, 1, 128, 128, False, [130], [130]),
          ("f32", "e4m3", 6, 3, 128, 64, True, [1, 65], [64, 65]), ("bf16", "same", 12, 2, 128, 256, True, [300, 1], [300, 257]),
          ("bf16", "e4m3", 40, 8, 128, 64, True, [2051], [2060]), ("bf16", "same", 16, 16, 64, 64, False, [1] * 70, list(range(1, 71))),
          ("bf16", "same", 4, 4, 64, 16, False, [0, 2, 0, 0, 3, 0], [4, 2, 0, 9, 30, 0])]


@pytest.mark.parametrize("dtype,fmt,H,KV,d,page,norm,new,ctx", APPEND)
def test_append_and_read(dtype, fmt, H, KV, d, page, norm, new, ctx):
    dt, rows = tdt(dtype), sum(new)
    pool = Pool(KV, d, page, dtype, fmt, ctx, gap=64)
    before = [t.clone() for t in (pool.kv.k, pool.kv.v)]
    pad = 3                                                           # rows behind the last sequence
    qkv = rnd(rows + pad, (H + 2 * KV) * d, seed=4, dtype=dt)
    inv, gains = freqs(d), [rnd(d, seed=s) for s in (5, 6)] if norm else [None, None]
    dev = [None if t is None else t.to(DEV) for t in (inv, *gains)]
    b = pool.batch(new, ctx)
    q = torch.full((rows + pad, H, d), 7.0, dtype=dt, device=DEV)
    paged.append(pool.kv, b, qkv.to(DEV), dev[0], q_gain=dev[1], k_gain=dev[2], out=q)
    rd = torch.float32 if fmt == "e4m3" else dt
    k, v = (torch.full((rows + pad, KV, d), 7.0, dtype=rd, device=DEV) for _ in range(2))
    paged.read(pool.kv, b, out=(k, v))
    pool.kv.check()
    for t in (q, k, v):
        assert (t[rows:] == 7).all(), "rows of no sequence were written"
    pos = torch.cat([torch.arange(c - n, c) for n, c in zip(new, ctx)])
    x = qkv[:rows].view(rows, H + 2 * KV, d)
    y, err = rotated(x[:, :H], pos, inv, gains[0], 1e-6, d, False, 1.0)
    within(q[:rows], y, err + U[dt] * (y.abs() + err), "q")
    y, err = rotated(x[:, H:H + KV], pos, inv, gains[1], 1e-6, d, False, 1.0)
    val = x[:, H + KV:].double()
    if fmt == "e4m3":
        scale = (val.abs().amax(-1, keepdim=True) / 448).float().clamp_min(2.0 ** -126).double()
        assert torch.equal(v[:rows].cpu(), e4m3(val, scale).float()), "values in 8 bits"
        s = y.abs().amax(-1, keepdim=True) / 448
        within(k[:rows], y, 2.0 ** -4 * (y.abs() + err) + 2.0 ** -10 * s + err + U32 * y.abs() * 4, "keys in 8 bits")
    else:
        assert torch.equal(v[:rows].cpu(), x[:, H + KV:])
        within(k[:rows], y, err + U[dt] * (y.abs() + err), "k")
    # nothing but the new tokens' places changed
    for t, old in zip((pool.kv.k, pool.kv.v), before):
        same = t.view(torch.uint8) == old.view(torch.uint8)
        for s, (n, c) in enumerate(zip(new, ctx)):
            for p in range(c - n, c):
                same[int(pool.table[s, p // page]), :, p % page] = True
        assert same.all(), "other places of the pool were written"


def test_append_positions_of_its_own_and_rows_before_the_first_place():
    """pos turns the keys by other positions than their places; of more new tokens than context only the last have a place, and the others are left."""
    H, KV, d, rows = 2, 1, 64, 6
    pool = Pool(KV, d, 16, "f32", "same", [4])
    qkv, pos, inv = rnd(rows, 4 * d, seed=1), torch.tensor([9, 8, 7, 100, 3, 5], dtype=torch.int32), freqs(d)
    q = torch.full((rows, H, d), 7.0, device=DEV)
    b = pool.batch([rows], [4])
    paged.append(pool.kv, b, qkv.to(DEV), inv.to(DEV), pos=pos.to(DEV), out=q)
    assert (q[:2] == 7).all()
    k, _ = paged.read(pool.kv, pool.batch([4], [4]), 4)
    x = qkv[2:].view(4, 4, d)
    y, err = rotated(x[:, :2], pos[2:], inv, None, 0, d, False, 1.0)
    within(q[2:], y, err + U32 * y.abs(), "q")
    y, err = rotated(x[:, 2:3], pos[2:], inv, None, 0, d, False, 1.0)
    within(k, y, err + U32 * y.abs(), "k")


def test_8bit_rows_at_their_borders():
    """Zeros, one value, ties (448 x small fractions), the smallest and the largest numbers, an infinity and a NaN: exactly the e4m3 value that 64 bits give."""
    d, rows = 64, 10
    x = torch.zeros(rows, 3 * d)
    v = x[:, 2 * d:]
    v[1, 5] = -3.0
    v[2] = torch.arange(d) / 64.0 * 448 * 7                              # amax times multiples of 1 / 63: many quotients next to ties
    v[3] = torch.tensor([448.0] + [2.0 ** -6 * (1 + j / 16.0) for j in range(d - 1)])      # middles between neighbours, ties to even
    v[4] = torch.tensor([448.0] + [2.0 ** -10 * j for j in range(d - 1)])                # below the smallest normal
    v[5] = torch.tensor([1e-37 * (j + 1) for j in range(d)])
    v[6] = torch.tensor([1e-42 * (j - 30) for j in range(d)])
    v[7] = torch.tensor([3e38 / (j + 1) for j in range(d)])
    v[8, 3], v[9, 60] = float("inf"), float("nan")
    pool = Pool(1, d, 16, "f32", "e4m3", [rows])
    b = pool.batch([rows], [rows])
    paged.append(pool.kv, b, x.to(DEV))
    _, got = paged.read(pool.kv, b, rows, dtype=torch.float32)
    got = got.cpu()[:, 0]
    want = v[:8].double()
    scale = (want.abs().amax(-1, keepdim=True) / 448).float().clamp_min(2.0 ** -126).double()
    assert torch.equal(got[:8], e4m3(want, scale).float())
    assert got[8:].isnan().all()


# ---- attention ----------------------------------------------------------------------------------------------------------------------------------
def attended(q, k, v, new, ctx, scale, bf16, seen=None):
    """Exact output, its error bound (before the last rounding) and lse; q [rows][H][d], k and v lists of [ctx][KV][d]."""
    H, d = q.shape[1:]
    out, err, lse = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64), torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    row = 0
    for s, (n, c) in enumerate(zip(new, ctx)):
        K, V = k[s], v[s]
        if n and len(K):
            G = H // K.shape[1]
            Q = q[row:row + n].double().transpose(0, 1)                                            # [H][n][d]
            Kh, Vh = (t.transpose(0, 1).repeat_interleave(G, 0) for t in (K, V))                   # [H][c][d]
            far = torch.arange(len(K))[None] > torch.arange(c - n, c)[:, None]
            S = (Q @ Kh.transpose(1, 2) * scale).masked_fill(far, -math.inf)
            top = (Q.abs() @ Kh.abs().transpose(1, 2) * scale).masked_fill(far, 0).amax(-1, keepdim=True)
            some = (~far).any(-1)
            P = torch.softmax(S, -1).masked_fill(~some[:, None], 0)
            A = P @ Vh.abs()
            rel = 2 * (d + 4) * U32 * top + 4 * U32 + 2 * (len(K) + 8) * U32 + (U[torch.bfloat16] * 1.01 if bf16 else 0)
            out[row:row + n] = (P @ Vh).transpose(0, 1)
            err[row:row + n] = (A * rel).transpose(0, 1)
            lse[row:row + n] = torch.logsumexp(S, -1).transpose(0, 1)
        row += n
    return out, err, lse


ATT = [  # dtype, format, H, KV, d, page, new, ctx
    ("bf16", "same", 32, 8, 64, 16, [1], [313]), ("bf16", "same", 28, 4, 128, 64, [1] * 9, [1, 2, 63, 64, 65, 700, 128, 127, 1500]),
    ("bf16", "e4m3", 32, 8, 128, 128, [1, 1], [2000, 33]), ("bf16", "e4m3", 14, 2, 64, 16, [70, 1, 33, 1, 1], [500, 400, 33, 1, 77]),
    ("f32", "same", 16, 2, 128, 32, [30, 70, 1], [150, 70, 90]), ("f32", "e4m3", 4, 4, 64, 64, [1, 40], [300, 40]),
    ("bf16", "same", 32, 8, 128, 256, [200], [1100]), ("bf16", "same", 8, 8, 64, 32, [129, 64, 1, 5], [129, 300, 65, 6]),
    ("bf16", "same", 40, 8, 128, 16, [3, 2, 4], [30, 2, 700]), ("bf16", "same", 8, 1, 64, 64, [0, 5, 0, 1, 0], [10, 5, 0, 200, 0]),
    ("f32", "same", 3, 1, 64, 16, [1, 2], [1, 400]), ("bf16", "same", 6, 2, 128, 16, [1] * 70, list(range(1, 71))), ("bf16", "e4m3", 24, 1, 128, 32, [2, 1], [90, 64]),
    ("bf16", "same", 4, 2, 64, 16, [10, 3], [4, 3])]


@pytest.mark.parametrize("split", [0, 256])
@pytest.mark.parametrize("dtype,fmt,H,KV,d,page,new,ctx", ATT)
def test_attention(dtype, fmt, H, KV, d, page, new, ctx, split):
    dt, rows, pad = tdt(dtype), sum(new), 2
    pool = Pool(KV, d, page, dtype, fmt, ctx, seed=len(ctx))
    k, v = pool.fill(ctx)
    q = rnd(rows + pad, H, d, seed=8, scale=1.5, dtype=dt)
    out, lse = torch.full((rows + pad, H, d), 7.0, dtype=dt, device=DEV), torch.full((rows + pad, H), 7.0, device=DEV)
    b = pool.batch(new, ctx)
    paged.attention(pool.kv, b, q.to(DEV), out=out, lse=lse, split_keys=split)
    pool.kv.check()
    y, err, z = attended(q[:rows], k, v, new, ctx, d ** -0.5, dtype == "bf16")
    within(out[:rows], y, err + U[dt] * (y.abs() + err), "attention")
    assert (out[rows:] == 7).all() and (lse[rows:] == 7).all(), "rows of no sequence were written"
    empty = z == -math.inf
    assert torch.equal(lse[:rows].cpu() == -math.inf, empty) and (out[:rows].cpu()[empty] == 0).all()
    top = q[:rows].double().abs().amax() * d ** 0.5 * 6
    within(lse[:rows][~empty.to(DEV)], z[~empty], 2 * (d + 4) * U32 * top + 4e-6, "lse")
    again = torch.empty_like(out)
    paged.attention(pool.kv, b, q.to(DEV), out=again, split_keys=split)
    assert torch.equal(again[:rows], out[:rows])


@pytest.mark.parametrize("dtype,fmt", [("bf16", "same"), ("f32", "same"), ("bf16", "e4m3")])
def test_attention_one_key_dominates_late(dtype, fmt):
    """The running maximum jumps in a late tile, by more than an exponential holds."""
    pool = Pool(2, 64, 16, dtype, fmt, [900])
    k, v = pool.fill([900])
    q = rnd(3, 4, 64, seed=2, dtype=tdt(dtype))
    q[2, 0] = (k[0][850, 0] * 40).to(q.dtype)
    out = paged.attention(pool.kv, pool.batch([3], [900]), q.to(DEV))
    y, err, _ = attended(q, k, v, [3], [900], 0.125, dtype == "bf16")
    within(out, y, err + U[tdt(dtype)] * (y.abs() + err), "attention")


@pytest.mark.parametrize("dtype,fmt,H,KV,d", [("bf16", "same", 8, 2, 64), ("bf16", "same", 4, 1, 128), ("f32", "same", 4, 2, 64), ("bf16", "e4m3", 8, 2, 128)])
@pytest.mark.parametrize("new", [3, 80, 200])
def test_attention_keys_a_row_does_not_see_do_not_count(dtype, fmt, H, KV, d, new):
    """Infinities and NaN in later tokens' keys and values leave the rows before them exactly as they are."""
    ctx, dt = new + 37, tdt(dtype)
    pool = Pool(KV, d, 16, dtype, fmt, [ctx])
    pool.fill([ctx])
    b, q = pool.batch([new], [ctx]), rnd(new, H, d, seed=3, dtype=dt).to(DEV)
    good = paged.attention(pool.kv, b, q)
    bad = {ctx - 1: float("nan"), ctx - new // 2: float("inf")}
    for p, value in bad.items():
        page, off = int(pool.table[0, p // 16]), p % 16
        for t, s in ((pool.kv.k, pool.kv.k_scale), (pool.kv.v, pool.kv.v_scale)):
            (t if s is None else s)[page, :, off] = value
    out = paged.attention(pool.kv, b, q)
    first = min(bad) - (ctx - new)                                  # the first row that sees a bad token
    assert torch.equal(out[:first], good[:first]) and not out[first:].isfinite().all(-1).any()


def test_attention_reads_strided_rows_and_a_shared_prefix():
    """q inside fused rows, out inside wider rows, pages of a larger pool, and two sequences whose tables begin with the same pages."""
    H, KV, d, page = 8, 2, 64, 16
    pool = Pool(KV, d, page, "bf16", "same", [64, 40], gap=128)
    k, v = pool.fill([64, 40])
    pool.table[1, :2] = pool.table[0, :2]
    k[1][:32], v[1][:32] = k[0][:32], v[0][:32]
    wide = rnd(5, (H + 2 * KV) * d + 8, seed=5, dtype=torch.bfloat16)
    q = wide.to(DEV)[:, :H * d]
    hold = torch.full((5, H * d + 64), 7.0, dtype=torch.bfloat16, device=DEV)
    out = paged.attention(pool.kv, pool.batch([2, 3], [64, 40]), q, out=hold[:, 32:32 + H * d])
    y, err, _ = attended(wide[:, :H * d].reshape(5, H, d), k, v, [2, 3], [64, 40], d ** -0.5, True)
    within(out.reshape(5, H, d), y, err + U[torch.bfloat16] * (y.abs() + err), "attention")
    assert (hold[:, :32] == 7).all() and (hold[:, 32 + H * d:] == 7).all()


@pytest.mark.parametrize("fmt", ["same", "e4m3"])
@pytest.mark.parametrize("new", [1, 2, 40])
def test_attention_split_by_the_caller_is_the_same_in_any_batch(fmt, new):
    """split_keys given: a sequence's rows have the same bits alone, among a few and among many others (the same max_q), where the library's own rule takes
    other splits and workgroups."""
    lens = [1200, 300, 2049, 70] + [130 + 9 * i for i in range(76)]
    pool = Pool(2, 128, 64, "bf16", fmt, lens)
    pool.fill(lens)
    q = rnd(len(lens) * new, 8, 128, seed=1, dtype=torch.bfloat16).to(DEV)

    def some(which):
        rows = torch.cat([q[s * new:(s + 1) * new] for s in which])
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
        b = paged.PagedBatch(i32([new * i for i in range(len(which) + 1)]), i32([lens[s] for s in which]), pool.table[which].to(DEV), max_q=new, max_ctx=max(lens[s] for s in which))
        return paged.attention(pool.kv, b, rows, split_keys=512).split(new)

    every = some(list(range(len(lens))))
    for s in range(4):
        assert torch.equal(some([s])[0], every[s])
    assert all(torch.equal(x, every[s]) for s, x in enumerate(some([0, 1, 2, 3])))


@pytest.mark.parametrize("dtype,fmt", [("bf16", "same"), ("bf16", "e4m3"), ("f32", "same")])
def test_attention_of_chunks_among_single_tokens_is_that_of_chunks_alone(dtype, fmt):
    """split_keys given and the same max_q: chunks of one batch have the same bits beside ten single tokens, where workgroups hold fewer rows."""
    new, lens = [90, 77, 41] + [1] * 10, [700, 1300, 41] + [60 + 150 * i for i in range(10)]
    pool = Pool(2, 128, 32, dtype, fmt, lens)
    pool.fill(lens)
    q = rnd(sum(new), 8, 128, seed=2, dtype=tdt(dtype)).to(DEV)
    every = pool.batch(new, lens)
    few = paged.PagedBatch(every.cu_q[:4].clone(), every.ctx_len[:3].clone(), every.table[:3], max_q=90, max_ctx=1300)
    alone = paged.attention(pool.kv, few, q[:sum(new[:3])], split_keys=512)
    assert torch.equal(paged.attention(pool.kv, every, q, split_keys=512)[:sum(new[:3])], alone)


@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("bf16", 128), ("f32", 128)])
@pytest.mark.parametrize("new", [1, 40])
def test_attention_split_by_the_caller_is_the_same_beside_a_longer_context(dtype, d, new):
    """split_keys given: the row's splits are joined alike where another sequence has many more of them."""
    lens = [1900, 700, 6000]
    pool = Pool(2, d, 64, dtype, "same", lens)
    pool.fill(lens)
    q = rnd(3 * new, 8, d, seed=4, dtype=tdt(dtype)).to(DEV)
    every = pool.batch([new] * 3, lens)
    few = paged.PagedBatch(every.cu_q[:3].clone(), every.ctx_len[:2].clone(), every.table[:2], max_q=new, max_ctx=1900)
    assert torch.equal(paged.attention(pool.kv, few, q[:2 * new], split_keys=256), paged.attention(pool.kv, every, q, split_keys=256)[:2 * new])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("new", [[1, 2], [90, 3, 40]])
def test_attention_into_its_queries(dtype, new):
    ctx = [700 + 13 * n for n in new]
    pool = Pool(2, 128, 16, dtype, "same", ctx)
    pool.fill(ctx)
    q, b = rnd(sum(new), 4, 128, seed=5, dtype=tdt(dtype)).to(DEV), pool.batch(new, ctx)
    for split in (0, 256, 1024):
        want, buf = paged.attention(pool.kv, b, q, split_keys=split), q.clone()
        assert paged.attention(pool.kv, b, buf, out=buf, split_keys=split) is buf and torch.equal(buf, want)


@pytest.mark.parametrize("dtype,H,KV,d", [("bf16", 8, 2, 128), ("f32", 4, 2, 64)])
@pytest.mark.parametrize("new", [1, 60])
def test_attention_infinite_values_that_are_seen(dtype, H, KV, d, new):
    """A seen value that is infinite makes its dimension infinite, and leaves the others."""
    ctx, dt = 150, tdt(dtype)
    pool = Pool(KV, d, 16, dtype, "same", [ctx])
    pool.fill([ctx])
    q, b = rnd(new, H, d, seed=3, dtype=dt).to(DEV), pool.batch([new], [ctx])
    good = paged.attention(pool.kv, b, q)
    pool.kv.v[int(pool.table[0, 1]), 0, 3, 7] = float("-inf")
    out = paged.attention(pool.kv, b, q)
    assert (out[:, :H // KV, 7] == -math.inf).all()
    out[:, :H // KV, 7] = good[:, :H // KV, 7]
    within(out, good.cpu().double(), 4 * U[dt] * good.cpu().double().abs() + 4 * U[dt] * good.cpu().double().abs().amax(), "the other dimensions")


# ---- together -----------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,fmt,H,KV,d", [("bf16", "same", 8, 2, 64), ("f32", "same", 4, 2, 128), ("bf16", "e4m3", 7, 1, 128)])
def test_prompts_in_chunks_then_single_tokens(dtype, fmt, H, KV, d):
    """Two sequences as a server runs them: prompts in chunks of uneven size, one sequence already decoding while the other's prompt goes on, then single tokens.
    Every step's rows equal whole-sequence attention in 64 bits on what the cache holds."""
    dt, total, page = tdt(dtype), [90, 41], 16
    steps = [(33, 40), (50, 1), (5, 0), (1, 0), (1, 0)]
    pool = Pool(KV, d, page, dtype, fmt, total)
    qkv = [rnd(n, (H + 2 * KV) * d, seed=s, dtype=dt) for s, n in enumerate(total)]
    inv, gain = freqs(d).to(DEV), [(1 + 0.1 * rnd(d, seed=9)).to(DEV), (1 + 0.1 * rnd(d, seed=10)).to(DEV)]
    done, outs, qs = [0, 0], [[], []], [[], []]
    for new in steps:
        ctx = [a + n for a, n in zip(done, new)]
        rows = torch.cat([x[a:c] for x, a, c in zip(qkv, done, ctx)]).to(DEV)
        b = pool.batch(list(new), ctx)
        q = paged.append(pool.kv, b, rows, inv, q_gain=gain[0], k_gain=gain[1])
        o = paged.attention(pool.kv, b, q)
        for s, (x, y) in enumerate(zip(q.cpu().split(new), o.cpu().split(new))):
            qs[s].append(x)
            outs[s].append(y)
        done = ctx
    pool.kv.check()
    assert done == total
    k, v = (list(t.cpu().double().split(total)) for t in paged.read(pool.kv, pool.batch(total, total), sum(total), dtype=torch.float32 if fmt == "e4m3" else dt))
    y, err, _ = attended(torch.cat([torch.cat(x) for x in qs]), k, v, total, total, d ** -0.5, dtype == "bf16")
    within(torch.cat([torch.cat(x) for x in outs]), y, err + U[dt] * (y.abs() + err), "attention over the cache")


@pytest.mark.parametrize("fmt,top", [("same", 600), ("same", 5000), ("e4m3", 5000)])
def test_a_step_captured_into_a_graph(fmt, top):
    """append + attention of a decode step in a graph (one launch of attention, and split ones with their workspace), its lengths and tables refilled in place
    between replays, eager work between them: the eager results."""
    H, KV, d, page, n = 8, 2, 64, 16, 5
    pool = Pool(KV, d, page, "bf16", fmt, [top] * n)
    start = [37, top - 88, 1, 255, 300]
    pool.fill([top] * n)
    b = pool.batch([1] * n, start, max_ctx=top)
    rows, inv = torch.zeros(n, (H + 2 * KV) * d, dtype=torch.bfloat16, device=DEV), freqs(d).to(DEV)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(2):
            paged.attention(pool.kv, b, paged.append(pool.kv, b, rows, inv))
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged.attention(pool.kv, b, paged.append(pool.kv, b, rows, inv))
    for step in range(4):
        rows.copy_(rnd(n, rows.shape[1], seed=step, dtype=torch.bfloat16))
        b.ctx_len.copy_(torch.tensor([s + step for s in start], dtype=torch.int32))
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, paged.attention(pool.kv, b, paged.append(pool.kv, b, rows, inv)))
    pool.kv.check()


def test_two_streams_at_once():
    """The same cache read on two streams at the same time, split attention with a workspace for each call."""
    lens = [3000, 2000]
    pool = Pool(2, 128, 64, "bf16", "same", lens)
    pool.fill(lens)
    b, q = pool.batch([1, 1], lens), rnd(2, 8, 128, seed=1, dtype=torch.bfloat16).to(DEV)
    want = paged.attention(pool.kv, b, q)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for s, o in zip(streams, got):
            with torch.cuda.stream(s):
                o.append(paged.attention(pool.kv, b, q))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for o in got for x in o)


def test_many_sequences():
    """More sequences than a wave looks through at once: single tokens of 5000, and ragged chunks of 150 with empty ones among them."""
    d, page = 64, 16
    for new, ctx in (([1] * 5000, [1 + i % 40 for i in range(5000)]), ([(i * 7) % 23 for i in range(150)], [(i * 7) % 23 + (i * 5) % 60 for i in range(150)])):
        pool = Pool(1, d, page, "bf16", "same", ctx)
        k, v = pool.fill(ctx)
        q = rnd(sum(new), 4, d, seed=1, dtype=torch.bfloat16)
        out = paged.attention(pool.kv, pool.batch(new, ctx), q.to(DEV))
        pool.kv.check()
        y, err, _ = attended(q, k, v, new, ctx, d ** -0.5, True)
        within(out, y, err + U[torch.bfloat16] * (y.abs() + err), "attention")


@pytest.mark.parametrize("fmt,new", [("same", 1), ("same", 50), ("e4m3", 1), ("e4m3", 50)])
def test_pages_behind_four_gigabytes(fmt, new):
    """Page numbers whose bytes lie behind 2^32 (and their elements behind 2^31): written, read and attended there."""
    KV, d, page, ctx = 4, 128, 128, 300
    bytes_per_page = KV * page * d * (1 if fmt == "e4m3" else 2)
    n = (5 << 30) // bytes_per_page
    dt = E4M3 if fmt == "e4m3" else torch.bfloat16
    t = [torch.empty(n, KV, page, d, dtype=dt, device=DEV) for _ in range(2)]
    if fmt == "e4m3":
        t += [torch.empty(n, KV, page, device=DEV) for _ in range(2)]
    pool = Pool(KV, d, page, "bf16", fmt, [ctx])
    pool.kv, pool.table = paged.PagedKV(*t), torch.tensor([[n - 1, n - 7, n - 2]], dtype=torch.int32)
    k, v = pool.fill([ctx])
    q = rnd(new, 8, d, seed=1, dtype=torch.bfloat16)
    out = paged.attention(pool.kv, pool.batch([new], [ctx]), q.to(DEV))
    y, err, _ = attended(q, k, v, [new], [ctx], d ** -0.5, True)
    within(out, y, err + U[torch.bfloat16] * (y.abs() + err), "attention")


@pytest.mark.parametrize("dtype,fmt,H,KV,d,page,new,ctx", [
    ("bf16", "same", 8, 2, 64, 16, [64, 64], [5000, 5000]), ("bf16", "same", 4, 1, 128, 64, [300], [4000]), ("bf16", "e4m3", 32, 8, 128, 32, [40], [2500]),
    ("f32", "same", 8, 2, 64, 16, [100, 9], [900, 2100]), ("f32", "e4m3", 4, 2, 128, 16, [33], [1300]), ("bf16", "same", 14, 2, 64, 256, [5, 400], [3000, 410])])
def test_attention_long_contexts(dtype, fmt, H, KV, d, page, new, ctx):
    """Chunks over contexts that the library's own rule splits, and does not split, in every kernel's several tiles."""
    dt = tdt(dtype)
    pool = Pool(KV, d, page, dtype, fmt, ctx)
    k, v = pool.fill(ctx)
    q = rnd(sum(new), H, d, seed=8, scale=1.5, dtype=dt)
    lse = torch.empty(sum(new), H, device=DEV)
    out = paged.attention(pool.kv, pool.batch(new, ctx), q.to(DEV), lse=lse)
    y, err, z = attended(q, k, v, new, ctx, d ** -0.5, dtype == "bf16")
    within(out, y, err + U[dt] * (y.abs() + err), "attention")
    top = q.double().abs().amax() * d ** 0.5 * 6
    within(lse, z, 2 * (d + 4) * U32 * top + 2 * (max(ctx) + 8) * U32 + 4e-6, "lse")


# ---- bad lengths and page numbers (the host-side twin of these checks runs on the CPU) -----------------------------------------------------------------
def test_bad_pages_and_lengths_are_reported_and_harmless():
    H, KV, d, page = 4, 2, 64, 16
    lens = [64, 64, 64]
    pool = Pool(KV, d, page, "bf16", "same", lens)
    k, v = pool.fill(lens)
    q = rnd(6, H, d, seed=1, dtype=torch.bfloat16)
    rows = rnd(6, (H + 2 * KV) * d, seed=2, dtype=torch.bfloat16).to(DEV)

    def zeroed(x, s, lo, hi):
        x = [t.clone() for t in x]
        x[s][lo:hi] = 0
        return x

    table = pool.table.clone()
    pool.table[1, 1] = pool.n                                        # one behind the pool
    b = pool.batch([2, 2, 2], lens)
    out = paged.attention(pool.kv, b, q.to(DEV))
    with pytest.raises(RuntimeError, match="page number"):
        pool.kv.check()
    y, err, _ = attended(q, zeroed(k, 1, 16, 32), zeroed(v, 1, 16, 32), [2, 2, 2], lens, d ** -0.5, True)
    within(out, y, err + U[torch.bfloat16] * (y.abs() + err), "a page that is none attends as zeros")
    pool.table[1] = table[1]
    pool.table[2, 3] = -5                                            # the page of the new tokens
    b = pool.batch([2, 2, 2], lens)
    before = pool.kv.k.clone()
    paged.append(pool.kv, b, rows)
    with pytest.raises(RuntimeError, match="page number"):
        pool.kv.check()
    changed = (pool.kv.k.view(torch.int16) != before.view(torch.int16)).any(-1).any(1).nonzero().tolist()
    assert sorted(changed) == sorted([int(table[s, 3]), off] for s in (0, 1) for off in (14, 15))
    kk, _ = paged.read(pool.kv, b, 6)
    with pytest.raises(RuntimeError, match="page number"):
        pool.kv.check()
    assert (kk[4:] == 0).all() and (kk[:4] != 0).any()
    # lengths: the second sequence passes the rows, the third is longer than max_ctx says; the first is answered as ever
    pool.table.copy_(table)
    pool.fill(lens)
    want = paged.attention(pool.kv, pool.batch([2, 2, 2], lens), q.to(DEV))
    b = pool.batch([2, 2, 2], lens)
    b.cu_q.copy_(torch.tensor([0, 2, 9, 6], dtype=torch.int32))
    out = torch.full((6, H, d), 7.0, dtype=torch.bfloat16, device=DEV)
    paged.attention(pool.kv, b, q.to(DEV), out=out)
    with pytest.raises(RuntimeError, match="length"):
        pool.kv.check()
    assert torch.equal(out[:2], want[:2]) and (out[2:] == 7).all()
    b = pool.batch([2, 2, 2], lens)
    b.ctx_len.copy_(torch.tensor([64, 64, 2 ** 31 - 1], dtype=torch.int32))
    out = paged.attention(pool.kv, b, q.to(DEV))
    with pytest.raises(RuntimeError, match="length"):
        pool.kv.check()
    assert torch.equal(out[:4], want[:4]) and out[4:].isfinite().all()


@pytest.mark.parametrize("cu,lens", [([0, 5, 3, 8], [64, 64, 64]), ([0, 4, 4, 8], [64, -1, 64]), ([0, 4, 4, 8], [64, 65, 64])])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_bad_sequences_without_rows_are_reported_by_every_call(dtype, cu, lens):
    H, KV, d, page = 4, 2, 64, 16
    pool = Pool(KV, d, page, dtype, "same", [64, 64, 64])
    pool.fill([64, 64, 64])
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    rows, q = rnd(8, (H + 2 * KV) * d, seed=2, dtype=tdt(dtype)).to(DEV), rnd(8, H, d, seed=1, dtype=tdt(dtype)).to(DEV)
    few, many = (paged.PagedBatch(i32(cu), i32(lens), pool.table.to(DEV), max_q=m, max_ctx=64) for m in (5, 20))
    for call in (lambda: paged.append(pool.kv, few, rows), lambda: paged.read(pool.kv, few, 8), lambda: paged.attention(pool.kv, few, q), lambda: paged.attention(pool.kv, many, q)):
        pool.kv.check()
        call()
        with pytest.raises(RuntimeError, match="length"):
            pool.kv.check()


# ---- refusals of the tensor layer ---------------------------------------------------------------------------------------------------------------
def test_refusals():
    H, KV, d = 4, 2, 64
    kv = paged.PagedKV.empty(6, 16, KV, d)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    b = paged.PagedBatch(i32(0, 2), i32(20), i32(1, 2)[None], max_q=2, max_ctx=32)
    q, bf = torch.zeros(2, H, d, dtype=torch.bfloat16, device=DEV), torch.bfloat16
    qkv = torch.zeros(2, (H + 2 * KV) * d, dtype=bf, device=DEV)
    z = lambda *s, dt=bf: torch.zeros(*s, dtype=dt, device=DEV)  # noqa: E731
    calls = {
        "float32, the cache": lambda: paged.attention(kv, b, q.float()), "float16": lambda: paged.attention(kv, b, q.half()),
        "heads have 64": lambda: paged.attention(kv, b, z(2, 4, 32)), "multiple of kv": lambda: paged.attention(kv, b, z(2, 3, d)),
        "one piece": lambda: paged.attention(kv, b, z(2, d, H).transpose(1, 2)), "aligned": lambda: paged.attention(kv, b, z(2, H * d + 8)[:, 4:-4]), "strides": lambda: paged.attention(kv, b, z(2, H * d + 4)[:, :-4]),
        "3 rows, 2 are": lambda: paged.attention(kv, b, q, out=z(3, H, d)), "scale": lambda: paged.attention(kv, b, q, scale=0.0), "scale nan": lambda: paged.attention(kv, b, q, scale=float("nan")),
        "split_keys": lambda: paged.attention(kv, b, q, split_keys=64), "lse": lambda: paged.attention(kv, b, q, lse=z(2, H)), "overlap": lambda: paged.attention(kv, b, q, out=z(1, H, d).expand(2, H, d)),
        "does not hold max_ctx": lambda: paged.attention(kv, paged.PagedBatch(i32(0, 2), i32(20), i32(1, 2)[None], max_q=2, max_ctx=33), q),
        "query heads": lambda: paged.append(kv, b, z(2, 2 * KV * d)), "gains": lambda: paged.append(kv, b, qkv, q_gain=z(d, dt=torch.float32)),
        "q_gain is": lambda: paged.append(kv, b, qkv, q_gain=z(d), k_gain=z(d)), "pos is": lambda: paged.append(kv, b, qkv, pos=i32(1)),
        "inv_freq is": lambda: paged.append(kv, b, qkv, z(32)), "rotated": lambda: paged.append(kv, b, qkv, z(12, dt=torch.float32)),
        "rows or out": lambda: paged.read(kv, b), "out\\[0\\] has 3": lambda: paged.read(kv, b, 2, out=(z(3, KV, d), None)),
        "head_dim": lambda: paged.attention(paged.PagedKV.empty(2, 16, KV, 32), b, z(2, H, 32)), "page_size": lambda: paged.attention(paged.PagedKV.empty(2, 24, KV, d), b, q),
        "positions": lambda: paged.qk_norm_rope(qkv, H, KV, None, z(32, dt=torch.float32)), "do not hold": lambda: paged.qk_norm_rope(qkv, 3, KV, None, None),
        "v \\(": lambda: paged.PagedKV(z(2, 2, 16, 64), z(2, 2, 16, 32)), "8-bit": lambda: paged.PagedKV(z(2, 2, 16, 64), z(2, 2, 16, 64), z(2, 2, 16, dt=torch.float32)),
        "sequences by": lambda: paged.PagedBatch(i32(0, 2), i32(20, 1), i32(1, 2)[None], max_q=2, max_ctx=32), "int32": lambda: paged.PagedBatch(i32(0, 2).long(), i32(20), i32(1)[None], max_q=1, max_ctx=1),
    }
    for word, call in calls.items():
        with pytest.raises(ValueError, match=word.split(" nan")[0] if word != "v \\(" else "v"):
            call()
    # no gradients are formed: asking for them is refused, and a call under no_grad is none that asks
    gain, freq = torch.ones(d, device=DEV, requires_grad=True), z(32, dt=torch.float32)
    for call in (lambda: paged.attention(kv, b, q.clone().requires_grad_()), lambda: paged.append(kv, b, qkv.clone().requires_grad_()),
                 lambda: paged.qk_norm_rope(qkv.clone().requires_grad_(), H, KV, i32(0, 1), freq), lambda: paged.append(kv, b, qkv, q_gain=gain, k_gain=gain)):
        with pytest.raises(ValueError, match="gradients"):
            call()
        with torch.no_grad():
            call()
    # empty calls are calls
    none = paged.PagedBatch(i32(0), i32(), torch.zeros(0, 0, dtype=torch.int32, device=DEV), max_q=0, max_ctx=0)
    assert paged.attention(kv, none, z(0, H, d)).shape == (0, H, d)
    assert paged.append(kv, none, z(0, (H + 2 * KV) * d)).shape == (0, H, d)
    assert paged.read(kv, none, 0)[0].shape == (0, KV, d)
    assert paged.qk_norm_rope(z(0, (H + 2 * KV) * d), H, KV, i32(), z(32, dt=torch.float32))[1].shape == (0, KV, d)


@pytest.mark.parametrize("dtype,fmt,H,KV,d", [("bf16", "same", 8, 2, 64), ("bf16", "same", 4, 1, 128), ("f32", "same", 4, 2, 64), ("bf16", "e4m3", 8, 2, 128), ("f32", "e4m3", 4, 2, 64)])
@pytest.mark.parametrize("new,split", [(1, 0), (3, 256), (80, 0), (80, 256)])
def test_attention_scores_of_minus_infinity(dtype, fmt, H, KV, d, new, split):
    """Keys that score -infinity weigh nothing; a row of which every visible key does is NaN, as its softmax is, with lse -infinity; a row that sees none is zero."""
    ctx, low, dt = new + 520, 500, tdt(dtype)
    pool = Pool(KV, d, 16, dtype, fmt, [ctx, 1])
    k, v = pool.fill([ctx, 1])
    q = rnd(new + 3, H, d, seed=3, dtype=dt)
    q[..., 0] = q[..., 0].abs() + 0.5
    b = pool.batch([new, 3], [ctx, 1], max_q=max(new, 3))

    def bad_keys(s, n):                                              # the first n keys of sequence s: their products with any q are -infinity
        p = torch.arange(n)
        page, off = pool.table[s, p // 16].long().to(DEV), (p % 16).to(DEV)
        if fmt == "e4m3":
            key = torch.zeros(d, dtype=torch.uint8, device=DEV)
            key[0] = 0xb8                                            # -1, of an infinite scale
            pool.kv.k.view(torch.uint8)[page, :, off] = key
            pool.kv.k_scale[page, :, off] = math.inf
        else:
            pool.kv.k[page, :, off, 0] = -math.inf

    def run():
        out, lse = torch.full((new + 3, H, d), 7.0, dtype=dt, device=DEV), torch.full((new + 3, H), 7.0, device=DEV)
        paged.attention(pool.kv, b, q.to(DEV), out=out, lse=lse, split_keys=split)
        return out, lse

    bad_keys(0, low)
    out, lse = run()
    y, err, z = attended(q[:new], [k[0][low:]], [v[0][low:]], [new], [ctx - low], d ** -0.5, dtype == "bf16")
    within(out[:new], y, err + U[dt] * (y.abs() + err), "beside keys that weigh nothing")
    assert lse[:new].isfinite().all()
    bad_keys(0, ctx)
    bad_keys(1, 1)
    out, lse = run()
    assert out[:new].isnan().all() and out[-1].isnan().all() and (lse[:new] == -math.inf).all() and (lse[-3:] == -math.inf).all()
    assert (out[new:new + 2] == 0).all()


def test_8bit_rows_next_to_ties_at_small_scales():
    """The f32 (bf16) numbers next to the middle between two e4m3 values, times scales from 2^-126 to 2^-96: the residual of their quotients lies below the smallest f32."""
    d = 64
    g = torch.Generator().manual_seed(3)
    steps = torch.arange(1, 128, dtype=torch.uint8)[:126].view(E4M3).double()               # the positive e4m3 values, 448 the last
    middle = (steps[1:] + steps[:-1]) / 2
    rows = []
    for e in range(-126, -95):
        for i in range(8):
            scale = (2.0 ** e * (1 + torch.rand(1, generator=g, dtype=torch.float64))).float()
            x = torch.zeros(d)
            x[0] = scale * 448
            scale = (x[0].double() / 448).float().clamp_min(2.0 ** -126).double()
            t = (middle[torch.randint(0, len(middle), (d - 1,), generator=g)] * scale).float()
            t = t.bfloat16().float() if i % 2 else torch.nextafter(t, t * (i / 2 - 1) * 2) if i in (0, 4) else t
            sign = torch.randint(0, 2, (d - 1,), generator=g).float() * 2 - 1
            x[1:] = t.clamp_max(float(x[0])) * sign
            rows.append(x)
    v = torch.stack(rows)
    n = len(v)
    pool = Pool(1, d, 16, "f32", "e4m3", [n])
    b = pool.batch([n], [n])
    paged.append(pool.kv, b, torch.cat([torch.zeros(n, 2 * d), v], 1).to(DEV))
    _, got = paged.read(pool.kv, b, n, dtype=torch.float32)
    want = v.double()
    scale = (want.abs().amax(-1, keepdim=True) / 448).float().clamp_min(2.0 ** -126).double()
    off = got.cpu()[:, 0] != e4m3(want, scale).float()
    assert not off.any(), f"{int(off.sum())} of {off.numel()}, in rows {off.any(1).nonzero()[:, 0].tolist()[:8]}"


def test_what_asks_for_gradients_is_refused_wherever_it_stands():
    """Pools, scales, outputs and lse that require grad, and tangents of forward mode (which no_grad does not switch off): refused, nothing queued."""
    H, KV, d = 4, 2, 64
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt, device=DEV)  # noqa: E731
    b = paged.PagedBatch(i32(0, 2), i32(20), i32(1, 2)[None], max_q=2, max_ctx=32)
    q, qkv, freq, gain = z(2, H, d), z(2, (H + 2 * KV) * d), z(32, dt=torch.float32), z(d, dt=torch.float32)
    pool = lambda: (z(6, KV, 16, d), z(6, KV, 16, d))  # noqa: E731
    pool8 = lambda: (z(6, KV, 16, d).to(E4M3), z(6, KV, 16, d).to(E4M3), z(6, KV, 16, dt=torch.float32), z(6, KV, 16, dt=torch.float32))  # noqa: E731
    kv = paged.PagedKV(*pool())
    uses = lambda c: (lambda: paged.attention(c, b, q), lambda: paged.append(c, b, qkv), lambda: paged.read(c, b, 2))  # noqa: E731
    calls = []
    for make, which in ((pool, 0), (pool, 1), (pool8, 2), (pool8, 3)):
        t = make()
        c = paged.PagedKV(*t)
        t[which].requires_grad_()                                     # after the cache was made, too
        calls += uses(c)
    g = lambda t: t.requires_grad_()  # noqa: E731
    calls += [lambda: paged.attention(kv, b, q, out=g(z(2, H, d))), lambda: paged.attention(kv, b, q, lse=g(z(2, H, dt=torch.float32))),
              lambda: paged.append(kv, b, qkv, out=g(z(2, H, d))), lambda: paged.read(kv, b, out=(g(z(2, KV, d)), None)), lambda: paged.read(kv, b, out=(None, g(z(2, KV, d)))),
              lambda: paged.qk_norm_rope(qkv, H, KV, i32(0, 1), freq, out=(g(z(2, H, d)), z(2, KV, d))),
              lambda: paged.qk_norm_rope(qkv, H, KV, i32(0, 1), freq, out=(z(2, H, d), g(z(2, KV, d))))]
    for call in calls:
        with pytest.raises(ValueError, match="gradients"):
            call()
        with torch.no_grad():
            call()
    kv.check()
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        duals = [lambda: paged.attention(kv, b, dual(q)), lambda: paged.append(kv, b, dual(qkv)), lambda: paged.append(kv, b, qkv, dual(freq)),
                 lambda: paged.append(kv, b, qkv, q_gain=dual(gain), k_gain=gain), lambda: paged.qk_norm_rope(dual(qkv), H, KV, i32(0, 1), freq),
                 lambda: paged.attention(kv, b, q, out=dual(z(2, H, d))), lambda: paged.attention(kv, b, q, lse=dual(z(2, H, dt=torch.float32)))]
        for c in (paged.PagedKV(dual(pool()[0]), pool()[1]), paged.PagedKV(pool()[0], dual(pool()[1])), paged.PagedKV(*pool8()[:2], dual(pool8()[2]), pool8()[3])):
            duals += uses(c)
        for call in duals:
            with pytest.raises(ValueError, match="gradients"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="gradients"):
                call()
        for call in uses(kv):                                         # plain tensors inside a level are plain
            call()


def test_what_is_written_is_known_to_autograd():
    """A tensor that a backward pass has saved and a call then writes: the backward pass is refused, as after any write in place."""
    H, KV, d = 4, 2, 64
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt, device=DEV)  # noqa: E731
    b = paged.PagedBatch(i32(0, 2), i32(20), i32(1, 2)[None], max_q=2, max_ctx=32)
    q, qkv, freq = z(2, H, d), z(2, (H + 2 * KV) * d), z(32, dt=torch.float32)
    kv, kv8 = paged.PagedKV.empty(6, 16, KV, d), paged.PagedKV.empty(6, 16, KV, d, dtype=E4M3)
    out, lse, keys, vals = z(2, H, d), z(2, H, dt=torch.float32), z(2, KV, d), z(2, KV, d)
    fused = z(2, (H + 2 * KV) * d)
    for call, written in ((lambda: paged.attention(kv, b, q, out=out, lse=lse), (out, lse)), (lambda: paged.append(kv, b, qkv), (kv.k, kv.v)),
                          (lambda: paged.append(kv8, b, qkv, out=out), (out, kv8.k, kv8.v, kv8.k_scale, kv8.v_scale)), (lambda: paged.read(kv, b, out=(keys, vals)), (keys, vals)),
                          (lambda: paged.read(kv, b, out=(keys, None)), (keys,)), (lambda: paged.qk_norm_rope(qkv, H, KV, i32(0, 1), freq, out=(out, keys)), (out, keys)),
                          (lambda: paged.append(kv, b, fused, out=fused[:, :H * d]), (fused,))):
        before = [t._version for t in written]
        call()
        assert all(t._version > n for t, n in zip(written, before))
    w = torch.ones(2, H, d, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    loss = (w * out).sum()
    paged.attention(kv, b, q, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():                                      # such tensors have no version
        paged.append(kv, b, z(2, (H + 2 * KV) * d), out=z(2, H, d))


def _one_token(page):
    """One token in `page`."""
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    return paged.PagedBatch(i32([0, 1]), i32([1]), i32([[page]]), max_q=1, max_ctx=1)


def test_check_sees_calls_on_every_stream():
    """A call that waits on another stream is waited for; each report is given once."""
    kv = paged.PagedKV.empty(6, 16, 2, 64)
    bad, side = _one_token(6), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)
        paged.read(kv, bad, 1)
    with pytest.raises(RuntimeError, match="page number"):
        kv.check()
    kv.check()


def test_a_cache_made_behind_queued_work_reports_on_another_stream():
    """The status word is clear when the constructor returns, whatever is still queued on the current stream."""
    k, v = (torch.zeros(6, 2, 16, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    bad, side = _one_token(6), torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)
    kv = paged.PagedKV(k, v)
    with torch.cuda.stream(side):
        paged.read(kv, bad, 1)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="page number"):
        kv.check()


def test_tensors_that_a_cache_or_a_batch_keeps_are_not_exchanged():
    """Their addresses were taken: another tensor in their place would not be seen.  Writing into them is how they change."""
    kv = paged.PagedKV.empty(6, 16, 2, 64, dtype=E4M3)
    b = _one_token(1)
    for owner, names in ((kv, ("k", "v", "k_scale", "v_scale", "status")), (b, ("cu_q", "ctx_len", "table"))):
        for name in names:
            old = getattr(owner, name)
            with pytest.raises(ValueError, match=name):
                setattr(owner, name, old.clone())
            assert getattr(owner, name) is old
    b.ctx_len += 0                                                    # the same tensor again
    b.table[:] = 2
    paged.read(kv, b, 1)
    kv.check()


@pytest.mark.parametrize("cu,ctx,bad", [([0, 5, 5], [5, 0], True), ([0, 0, 0], [3, 65], True), ([0, -1, 0], [3, 3], True), ([0, 0, 0], [3, 64], False)])
@pytest.mark.parametrize("max_q", [5, 90])
def test_lengths_are_checked_where_there_are_no_rows(cu, ctx, bad, max_q):
    """Calls of no rows over sequences whose lengths say otherwise."""
    kv = paged.PagedKV.empty(6, 16, 2, 64)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    b = paged.PagedBatch(i32(cu), i32(ctx), i32([[0, 1, 2, 3]] * 2), max_q=max_q, max_ctx=64)
    for call in (lambda: paged.append(kv, b, torch.zeros(0, 512, dtype=torch.bfloat16, device=DEV)), lambda: paged.read(kv, b, 0),
                 lambda: paged.attention(kv, b, torch.zeros(0, 4, 64, dtype=torch.bfloat16, device=DEV)),
                 lambda: paged.attention(kv, b, torch.zeros(0, 4, 64, dtype=torch.bfloat16, device=DEV), split_keys=256)):
        kv.check()
        call()
        if bad:
            with pytest.raises(RuntimeError, match="length"):
                kv.check()
    kv.check()


@pytest.mark.parametrize("split", [2 ** 32, 2 ** 32 + 256, -2 ** 32, 2 ** 31])
def test_split_keys_that_do_not_fit_are_refused(split):
    kv = paged.PagedKV.empty(6, 16, 2, 64)
    with pytest.raises(ValueError, match="split_keys"):
        paged.attention(kv, _one_token(1), torch.zeros(1, 4, 64, dtype=torch.bfloat16, device=DEV), split_keys=split)


def test_outputs_that_overlap_what_is_read_are_refused():
    """An output may be the part it replaces; any other share of memory is refused, columns beside each other are not."""
    H, KV, d = 4, 2, 64
    kv = paged.PagedKV.empty(6, 16, KV, d)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    b = paged.PagedBatch(i32(0, 3), i32(20), i32(1, 2)[None], max_q=3, max_ctx=32)
    wide = torch.zeros(4, (2 * H + 2 * KV) * d, dtype=torch.bfloat16, device=DEV)
    qkv, q, k, rest = wide[:3, :(H + 2 * KV) * d], wide[:3, :H * d], wide[:3, H * d:(H + KV) * d], wide[:3, (H + 2 * KV) * d:]
    flat = wide.view(-1)
    pos = i32(0, 1, 2)
    rope = lambda out: paged.qk_norm_rope(qkv, H, KV, pos, None, out=out)  # noqa: E731
    apart = torch.zeros(3, H, d, dtype=torch.bfloat16, device=DEV)
    bad = [lambda: rope((k.new_zeros(3, H * d), q[:, :KV * d])), lambda: rope((wide[1:, :H * d], k)), lambda: rope((flat[:3 * H * d].view(3, H, d), apart[:, :KV])),
           lambda: rope((apart, apart[:, :KV])), lambda: rope((rest, wide[:3, (H + 2 * KV) * d + d:(2 * KV + H) * d + d + KV * d])),
           lambda: paged.append(kv, b, qkv, out=wide[:3, d:H * d + d]), lambda: paged.append(kv, b, qkv, out=flat[:3 * H * d].view(3, H, d)),
           lambda: paged.attention(kv, b, q, out=wide[1:, :H * d]), lambda: paged.attention(kv, b, q, out=wide[:3, d:H * d + d]),
           lambda: paged.read(kv, b, out=(k, k)), lambda: paged.read(kv, b, out=(k, wide[:3, H * d + d:(H + KV) * d + d]))]
    for call in bad:
        with pytest.raises(ValueError, match="overlap|row of out"):
            call()
    rope((q, k))
    rope((rest, k))
    paged.append(kv, b, qkv, out=rest)
    paged.append(kv, b, qkv, out=q)
    paged.attention(kv, b, q, out=q)
    paged.attention(kv, b, q, out=rest)
    paged.read(kv, b, out=(k, wide[:3, (H + KV) * d:(H + 2 * KV) * d]))
    paged.attention(kv, b, q, split_keys=256)


SMALL_F32 = [("f32", "e4m3", 4, 2, 64, 16, [1, 3, 0, 8], [300, 5, 9, 8]), ("f32", "e4m3", 8, 1, 128, 32, [1, 2], [700, 64]), ("f32", "e4m3", 14, 2, 64, 64, [1] * 3, [1, 64, 1500]),
             ("f32", "e4m3", 16, 1, 128, 256, [1, 1], [257, 1]), ("f32", "e4m3", 2, 1, 64, 16, [1] * 300, [1 + 3 * i for i in range(300)]),
             ("f32", "e4m3", 8, 2, 128, 16, [1, 2] * 80, [2 + 5 * i for i in range(160)])]


@pytest.mark.parametrize("split", [0, 256])
@pytest.mark.parametrize("case", SMALL_F32, ids=lambda c: f"{c[2]}-{c[3]}-{c[4]}-{len(c[6])}")
def test_attention_of_few_f32_rows_over_8_bits(case, split):
    """Up to 16 rows per kv head and sequence, exact f32 over e4m3 bytes: workgroups of eight waves, and of four (more sequences than CUs, or a pinned split)."""
    test_attention(*case, split)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [3, 80])
def test_attention_f32_over_8_bits_keys_a_row_does_not_see_do_not_count(d, new):
    test_attention_keys_a_row_does_not_see_do_not_count("f32", "e4m3", 4, 2, d, new)


@pytest.mark.parametrize("fmt,H,KV,d,ctx", [("same", 32, 8, 64, 313), ("same", 28, 4, 128, 700), ("e4m3", 32, 8, 128, 600), ("e4m3", 14, 2, 64, 500)])
def test_attention_single_tokens_weigh_values_by_two_numbers(fmt, H, KV, d, ctx):
    """bf16, up to 16 rows: a weight is the sum of two bf16 numbers, cut off at 2^-7 of it and rounded at 2^-8 of the rest, so 2^-15 stands where one number's 2^-8 would:
    a bound that weights of one number break."""
    n = 6
    pool = Pool(KV, d, 16, "bf16", fmt, [ctx] * n)
    k, v = pool.fill([ctx] * n)
    q = rnd(n, H, d, seed=8, dtype=torch.bfloat16)
    out = paged.attention(pool.kv, pool.batch([1] * n, [ctx] * n), q.to(DEV))
    y, err, _ = attended(q, k, v, [1] * n, [ctx] * n, d ** -0.5, False)
    G = H // KV
    P = [torch.softmax(torch.einsum("hd,chd->hc", q[s].double(), k[s].repeat_interleave(G, 1)) * d ** -0.5, -1) for s in range(n)]
    size = torch.stack([torch.einsum("hc,chd->hd", p, x.abs().repeat_interleave(G, 1)) for p, x in zip(P, v)])
    tol = err + 2.0 ** -15 * size
    tol = tol + U[torch.bfloat16] * (y.abs() + tol)
    within(out, y, tol, "two numbers")
    one = torch.stack([torch.einsum("hc,chd->hd", p.bfloat16().double(), x.repeat_interleave(G, 1)) for p, x in zip(P, v)]).bfloat16().double()
    assert ((one - y).abs() > tol).any()


@pytest.mark.parametrize("dtype,fmt", [("bf16", "same"), ("f32", "same"), ("bf16", "e4m3"), ("f32", "e4m3")])
@pytest.mark.parametrize("new,split", [(1, 0), (1, 256), (40, 0), (40, 256)])
def test_attention_of_large_values(dtype, fmt, new, split):
    """Values of 2^126 whose largest weight comes late and is about 2^7 times the first tile's: a mean of equal numbers is that number, and no weight above 1 may
    carry the sum out of range."""
    ctx, d, dt = 300, 64, tdt(dtype)
    pool = Pool(1, d, 16, dtype, fmt, [ctx])
    rows = torch.zeros(ctx, 3 * d)
    rows[:, d] = -200.0                                              # q . k / 8 of all keys but two
    rows[0, d], rows[256, d] = 0.0, 4.84375
    rows[:, 2 * d:] = 2.0 ** 126
    paged.append(pool.kv, pool.batch([ctx], [ctx]), rows.to(dt).to(DEV))
    _, v = paged.read(pool.kv, pool.batch([ctx], [ctx]), ctx, dtype=torch.float32 if fmt == "e4m3" else dt)
    q = torch.zeros(new, 4, d, dtype=dt, device=DEV)
    q[..., 0] = 8.0
    out = paged.attention(pool.kv, pool.batch([new], [ctx]), q, split_keys=split)
    want = v[:1].double().cpu().expand(new, 4, d)
    within(out, want, (U[dt] + (U[torch.bfloat16] if dtype == "bf16" else 0) + 16 * U32) * want, "a mean of equal numbers")
