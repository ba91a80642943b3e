"""The operators of a paged key / value cache, as cases to be timed and checked.

Four operators, which a decoder layer calls one after the other when its cache lies in pages:

  rope       norms of queries and keys per head and the position rotation, in one pass over fused [q | k | v] rows
  append     the same pass, with the rotated keys and the values written into the pages of their sequences
  cache      append into an 8-bit cache (e4m3 bytes, one f32 scale per token and kv head), and the written rows read back
  attention  the new tokens of a batch against their cached context: causal, grouped heads, single tokens and chunks mixed

A cache is a pool of pages [n_pages][kv heads][page][head_dim].  A batch is cu_q (row offsets of every sequence's new tokens), ctx (its cached tokens,
the new ones among them) and a page table [sequences][pages]; a new token's place is ctx - new + its index.  `own` says which side runs: the plain
form in elementary torch operations, or the calls into the framework."""
import math
import random

import torch

own = False

DEV = "cuda"
E4M3 = torch.float8_e4m3fn
TINY = 2.0 ** -126                          # the smallest scale of an 8-bit row: rows of zeros keep one too
ROPE = dict(theta=500000.0, factor=8.0, low=1.0, high=4.0, old=8192)      # base and long-context scaling of the rotation's frequencies


# ---- cases ---------------------------------------------------------------------------------------------------------------------------------
def _attention(name, dtype, kv, heads, kv_heads, head_dim, page, seqs, chunks, new, ctx, ragged):
    return dict(name=name, op="attention", dtype=dtype, kv=kv, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page, seqs=seqs, chunks=chunks, new=new,
                ctx=ctx, ragged=ragged)


def _rows(name, op, dtype, kv, heads, kv_heads, head_dim, page, seqs, new, ctx, ragged, norm, interleaved, rot):
    return dict(name=name, op=op, dtype=dtype, kv=kv, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page, seqs=seqs, chunks=seqs, new=new, ctx=ctx,
                ragged=ragged, norm=norm, interleaved=interleaved, rot=rot)


def listed():
    return [
        # one utterance alone, one token, the prompt of a 16 s clip behind it: launch latency
        _attention("decode_1_row", "bf16", "same", 32, 8, 64, 16, 1, 0, 1, 313, False),
        # a full decode step of many utterances of different lengths: the cache read once
        _attention("decode_97_rows", "bf16", "same", 28, 4, 128, 64, 97, 0, 1, 6000, True),
        # few long contexts in 8 bits: the long axis is all the parallelism there is
        _attention("decode_long_8bit", "bf16", "e4m3", 32, 8, 128, 128, 3, 0, 1, 131072, False),
        # one chunk of a long prompt over what is cached of it: products
        _attention("chunk_over_16k", "bf16", "same", 32, 8, 128, 64, 1, 1, 2048, 16384, False),
        # a serving step: some prompts' chunks and the single tokens of running sequences in one call, odd lengths
        _attention("mixed_8bit", "bf16", "e4m3", 14, 2, 64, 16, 24, 5, 701, 4999, True),
        # the exact-f32 mode
        _attention("chunk_f32", "f32", "same", 16, 2, 128, 32, 4, 4, 301, 1503, True),
        # one decode step's new tokens into the cache
        _rows("append_decode", "append", "bf16", "same", 28, 4, 128, 16, 64, 1, 900, True, False, False, 128),
        # whole prompts into the cache, with norms of queries and keys
        _rows("append_prompts", "append", "bf16", "same", 40, 8, 128, 64, 9, 1500, 1500, True, True, False, 128),
        # few rows, adjacent pairs, half of the head rotated, f32
        _rows("rope_few_f32", "rope", "f32", "same", 16, 2, 64, 16, 7, 1, 100000, False, False, True, 32),
        # the rows of a large prefill
        _rows("rope_prefill", "rope", "bf16", "same", 32, 8, 128, 16, 1, 16384, 131072, False, True, False, 128),
        # a decode step into an 8-bit cache and back
        _rows("cache_decode_8bit", "cache", "bf16", "e4m3", 14, 2, 64, 16, 96, 1, 700, True, False, False, 64),
        # prompts into an 8-bit cache and back, as a prefix is handed on
        _rows("cache_prompts_8bit", "cache", "bf16", "e4m3", 32, 8, 128, 64, 6, 2100, 4000, True, True, False, 128),
    ]


# head layouts of the configurations the framework knows, and generic ones: (heads, kv heads, head_dim)
_LAYOUTS = [(32, 8, 128), (28, 4, 128), (40, 8, 128), (14, 2, 64), (12, 2, 128), (16, 2, 128), (16, 16, 64), (8, 1, 64), (6, 2, 128)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c):
    w = work(c)
    pad = c["seqs"] * c["heads"] * c["new"] * c["ctx"] if c["op"] == "attention" else 0
    pool = 0 if c["op"] == "rope" else c["seqs"] * c["ctx"] * c["kv_heads"] * c["head_dim"]
    return w["bytes"], w["flops"], pad, pool


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "rope", "append", "cache"])
    top = [max(v) for v in zip(*(_cost(c) for c in listed() if c["op"] == op))]
    while True:
        heads, kv_heads, head_dim = rng.choice(_LAYOUTS)
        dtype = "f32" if rng.random() < 0.2 and op != "cache" else "bf16"
        kv = "e4m3" if op == "cache" or (op == "attention" and rng.random() < 0.4) else "same"
        page = rng.choice([16, 32, 64, 128, 256])
        if op == "attention":
            seqs, ctx = _log(rng, 1, 200), _log(rng, 1, 131072)
            one = rng.random() < 0.4                                   # a decode step; else chunks, some of them beside single tokens
            new = 1 if one else min(ctx, _log(rng, 2, 2048))
            c = _attention("", dtype, kv, heads, kv_heads, head_dim, page, seqs, 0 if one else rng.randint(1, seqs), new, ctx, rng.random() < 0.7)
        else:
            seqs, new = _log(rng, 1, 128), 1 if rng.random() < 0.3 else _log(rng, 2, 8192)
            ctx = new + (0 if rng.random() < 0.3 else _log(rng, 1, 131072 if op == "rope" else 8192))
            rot = rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4])
            c = _rows("", op, dtype, kv, heads, kv_heads, head_dim, page, seqs, new, ctx, rng.random() < 0.7, rng.random() < 0.5, rng.random() < 0.3, rot)
        del c["name"]
        if all(a <= b for a, b in zip(_cost(c), top)):
            return c


def lengths(case):
    """(new tokens, cached tokens) of every sequence: a property of the case."""
    r = random.Random(case["seqs"] * 1000003 + case["ctx"] * 131 + case["new"])
    new, ctx = [], []
    for i in range(case["seqs"]):
        n = case["new"] if i < case["chunks"] else 1
        t = case["ctx"]
        if case["ragged"] and i:
            n = r.randint(max(1, n // 4), n)
            t = r.randint(max(n, t // 8), t)
        new.append(n)
        ctx.append(t)
    return new, ctx


def work(case):
    new, ctx = lengths(case)
    e = 4 if case["dtype"] == "f32" else 2
    h, g, d = case["heads"], case["kv_heads"], case["head_dim"]
    rows = sum(new)
    token = 2 * g * (d + 4 if case["kv"] == "e4m3" else d * e)          # one cached token: its keys and values, with their scales
    if case["op"] == "attention":
        pairs = sum(n * t - n * (n - 1) // 2 for n, t in zip(new, ctx))
        return {"bytes": 2 * rows * h * d * e + sum(ctx) * token, "flops": 4 * d * h * pairs}
    if case["op"] == "rope":
        return {"bytes": 2 * rows * (h + g) * d * e, "flops": 6 * rows * (h + g) * d}
    written = rows * ((2 * h + 2 * g) * d * e + token)
    return {"bytes": written + (rows * (token + 2 * g * d * e) if case["op"] == "cache" else 0), "flops": 6 * rows * (h + g) * d}


# ---- inputs --------------------------------------------------------------------------------------------------------------------------------
def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _inv_freq(rot):
    """Frequencies of `rot` rotated dimensions with the long-context scaling: low ones divided by `factor`, high ones kept, a ramp between."""
    f = ROPE["theta"] ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    turns = ROPE["old"] * f / (2 * math.pi)
    keep = ((turns - ROPE["low"]) / (ROPE["high"] - ROPE["low"])).clamp(0, 1)
    return (f * (keep + (1 - keep) / ROPE["factor"])).float()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt, e4m3 = _dtype(case), case["kv"] == "e4m3"
    h, kvh, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    new, ctx = lengths(case)
    rows = sum(new)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    s = {"case": case, "rows": rows, "max_q": max(new), "max_ctx": max(ctx),
         "cu_q": torch.tensor(cu, dtype=torch.int32, device=DEV), "ctx": torch.tensor(ctx, dtype=torch.int32, device=DEV)}
    if case["op"] != "rope":                                           # pages in any order, a few of the pool unused; places behind a sequence's last page hold -1
        width = -(-max(ctx) // page)
        need = [-(-t // page) for t in ctx]
        n_pages = sum(need) + 3
        order = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
        first = torch.tensor([sum(need[:i]) for i in range(len(need))], device=DEV)
        col = torch.arange(width, device=DEV)
        used = col[None] < torch.tensor(need, device=DEV)[:, None]
        s["table"] = torch.where(used, order[(first[:, None] + col).clamp_max(n_pages - 1)], -1).to(torch.int32)
        for name in ("k", "v"):
            x = torch.randn(n_pages, kvh, page, d, generator=g, device=DEV, dtype=torch.bfloat16 if e4m3 else dt)
            if e4m3:
                scale = (x.float().abs().amax(-1) / 448).clamp_min(TINY)
                s[name + "_scale"] = scale
                x = (x.float() / scale[..., None]).to(E4M3)
            s[name] = x
    if case["op"] == "attention":
        s["q"] = (1.5 * torch.randn(rows, h, d, generator=g, device=DEV)).to(dt)
        return s
    s["qkv"] = torch.randn(rows, (h + 2 * kvh) * d, generator=g, device=DEV).to(dt)
    s["inv_freq"] = _inv_freq(case["rot"]).to(DEV)
    if case["norm"]:
        s["q_gain"] = 1 + 0.2 * torch.randn(d, generator=g, device=DEV)
        s["k_gain"] = 1 + 0.2 * torch.randn(d, generator=g, device=DEV)
    if case["op"] == "rope":
        s["pos"] = torch.cat([torch.arange(t - n, t, dtype=torch.int32) for n, t in zip(new, ctx)]).to(DEV)
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------------------------------
EPS = 1e-6


def run(s):
    if own:
        return _own(s)
    op = s["case"]["op"]
    if op == "attention":
        return _plain_attention(s)
    if op == "rope":
        return _plain_rotated(s, s["pos"])[:2]
    return _plain_append(s)


def _own(s):
    from omni_avsr_amd import paged
    case = s["case"]
    kw = dict(q_gain=s.get("q_gain"), k_gain=s.get("k_gain"), eps=EPS, interleaved=case.get("interleaved"))
    if case["op"] == "rope":
        return paged.qk_norm_rope(s["qkv"], case["heads"], case["kv_heads"], s["pos"], s["inv_freq"], **kw)
    if "handles" not in s:                                              # a program keeps them as long as the pool and the step's tables
        s["handles"] = (paged.PagedKV(s["k"], s["v"], s.get("k_scale"), s.get("v_scale")),
                        paged.PagedBatch(s["cu_q"], s["ctx"], s["table"], max_q=s["max_q"], max_ctx=s["max_ctx"]))
    kv, batch = s["handles"]
    if case["op"] == "attention":
        return paged.attention(kv, batch, s["q"])
    q = paged.append(kv, batch, s["qkv"], s["inv_freq"], **kw)
    if case["op"] == "append":
        return q, s["k"], s["v"]
    return (q,) + paged.read(kv, batch, s["rows"], dtype=s["qkv"].dtype)


def _plain_places(s):
    """Sequence, position, page and offset of every new token."""
    row = torch.arange(s["rows"], device=DEV)
    cu, ctx, page = s["cu_q"].long(), s["ctx"].long(), s["case"]["page"]
    seq = torch.bucketize(row, cu, right=True) - 1
    pos = ctx[seq] - (cu[seq + 1] - row)
    return pos, s["table"].long()[seq, pos // page], pos % page


def _plain_rotated(s, pos):
    """Queries and keys after norm and rotation, and the values, rounded to the rows' type (f32 before that)."""
    case = s["case"]
    h, kvh, d, rot = case["heads"], case["kv_heads"], case["head_dim"], case["rot"]
    x = s["qkv"].float().view(s["rows"], h + 2 * kvh, d)
    qk = x[:, :h + kvh]
    if case["norm"]:
        gain = torch.cat([s["q_gain"].expand(h, d), s["k_gain"].expand(kvh, d)])
        qk = qk * torch.rsqrt((qk * qk).mean(-1, keepdim=True) + EPS) * gain
    angle = pos.double()[:, None] * s["inv_freq"].double()              # far positions: 32 bits lose the angle
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    if case["interleaved"]:
        a, b = qk[..., 0:rot:2], qk[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = qk[..., :rot // 2], qk[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    qk = torch.cat([turned, qk[..., rot:]], -1)
    dt = s["qkv"].dtype
    return qk[:, :h].to(dt), qk[:, h:].to(dt), qk[:, h:], x[:, h + kvh:]


def _plain_append(s):
    pos, page, off = _plain_places(s)
    q, _, k32, v32 = _plain_rotated(s, pos)
    dt = s["qkv"].dtype
    if s["case"]["kv"] != "e4m3":
        s["k"][page, :, off] = k32.to(dt)
        s["v"][page, :, off] = v32.to(dt)
        return q, s["k"], s["v"]
    return q, _plain_8bit(s, "k", k32, page, off).to(dt), _plain_8bit(s, "v", v32, page, off).to(dt)


def _plain_8bit(s, name, x, page, off):
    scale = (x.abs().amax(-1).double() / 448).float().clamp_min(TINY)
    y = x.double() / scale[..., None].double()                          # next to a border between two steps 32 bits lose the side
    near = y.float()
    bits = near.view(torch.int32) - (near.double().abs() > y.abs()).int()
    odd = (bits | (near.double() != y).int()).view(torch.float32)       # cut off, the lowest bit set where something was: rounds as all of y's bits would
    pool, scales = s[name].view(torch.uint8), s[name + "_scale"]
    pool[page, :, off] = odd.to(E4M3).view(torch.uint8)
    scales[page, :, off] = scale
    return pool[page, :, off].view(E4M3).float() * scales[page, :, off][..., None]


def _plain_context(s, name):
    """[sequences][kv heads][max_ctx][head_dim] in f32: the pages of every sequence in a row."""
    page = s["table"].long().clamp_min(0)
    x = s[name].view(torch.uint8)[page].view(E4M3).float() if s[name].dtype == E4M3 else s[name][page].float()
    if name + "_scale" in s:
        x = x * s[name + "_scale"][page][..., None]
    n, p, kvh, size, d = x.shape
    return x.transpose(1, 2).reshape(n, kvh, p * size, d)[:, :, :s["max_ctx"]]


def _plain_attention(s):
    case = s["case"]
    h, kvh, d = case["heads"], case["kv_heads"], case["head_dim"]
    group = h // kvh
    k, v = _plain_context(s, "k"), _plain_context(s, "v")
    n, span = s["ctx"].numel(), s["max_q"]
    cu, ctx = s["cu_q"].long(), s["ctx"].long()
    index = torch.arange(span, device=DEV)
    row = (cu[:-1, None] + index).clamp_max(s["rows"] - 1)              # [sequences][span], padded at each sequence's end
    q = s["q"].float()[row].view(n, span, kvh, group, d).transpose(1, 2).reshape(n, kvh, span * group, d)
    score = torch.matmul(q, k.transpose(-1, -2).contiguous()).view(n, kvh, span, group, -1)
    pos = (ctx - cu[1:] + cu[:-1])[:, None] + index
    seen = torch.arange(s["max_ctx"], device=DEV) <= pos[..., None]
    score = (score * d ** -0.5).masked_fill_(~seen[:, None, :, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(n, kvh, span * group, -1), v).view(n, kvh, span, group, d) / total
    out = out.permute(0, 2, 1, 3, 4).reshape(n, span, h, d)
    return out[index < (cu[1:] - cu[:-1])[:, None]].to(s["q"].dtype)


# ---- 64 bits -------------------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(s)
    new, ctx = lengths(case)
    place = [(i, p) for i, (n, t) in enumerate(zip(new, ctx)) for p in range(t - n, t)]
    q, k, v = _exact_rotated(s, torch.tensor([p for _, p in place], device=DEV))
    if case["op"] == "rope":
        return q, k
    if case["op"] == "cache":
        return q, _exact_8bit(k), _exact_8bit(v)
    table, size = s["table"].tolist(), case["page"]
    slot = torch.tensor([table[i][p // size] * size + p % size for i, p in place], device=DEV)
    pools = []
    for pool, x in ((s["k"], k), (s["v"], v)):
        n, kvh, _, d = pool.shape
        flat = pool.double().transpose(1, 2).reshape(n * size, kvh, d)
        flat[slot] = x
        pools.append(flat.view(n, size, kvh, d).transpose(1, 2))
    return (q, *pools)


def _exact_rotated(s, pos):
    case = s["case"]
    h, kvh, d, half = case["heads"], case["kv_heads"], case["head_dim"], case["rot"] // 2
    q, k, v = s["qkv"].double().view(-1, h + 2 * kvh, d).split([h, kvh, kvh], 1)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), torch.outer(pos.double(), s["inv_freq"].double()))[:, None]
    done = []
    for x, gain in ((q, s.get("q_gain")), (k, s.get("k_gain"))):
        if gain is not None:
            x = x / (x.square().sum(-1, keepdim=True) / d + EPS).sqrt() * gain.double()
        x = x.clone()
        pair = x[..., :2 * half].unflatten(-1, (half, 2) if case["interleaved"] else (2, half))
        pair = pair if case["interleaved"] else pair.transpose(-1, -2)
        z = torch.view_as_real(torch.complex(pair[..., 0], pair[..., 1]) * turn)
        x[..., :2 * half] = (z if case["interleaved"] else z.transpose(-1, -2)).flatten(-2)
        done.append(x)
    return done[0], done[1], v


def _exact_8bit(x):
    """What e4m3 bytes with one f32 scale per row stand for: three bits behind the leading one, ties to even, steps of 2^-9 below 2^-6, 448 at most."""
    scale = (x.abs().amax(-1, keepdim=True) / 448).float().clamp_min(TINY).double()
    y = x / scale
    step = torch.exp2(torch.frexp(y)[1].sub(1).clamp_min(-6).double() - 3)
    return (torch.round(y / step) * step).clamp(-448, 448) * scale


def _exact_attention(s):
    case = s["case"]
    h, kvh, d = case["heads"], case["kv_heads"], case["head_dim"]
    new, ctx = lengths(case)
    out = torch.empty(s["rows"], h, d, dtype=torch.float64, device=DEV)
    row = 0
    for i, (n, t) in enumerate(zip(new, ctx)):
        pages = s["table"][i, :-(-t // case["page"])].long()
        far = torch.ones(n, t, dtype=torch.bool, device=DEV).triu(t - n + 1)
        for j in range(kvh):
            both = []
            for name in ("k", "v"):
                x = s[name][:, j][pages] if s[name].dtype != E4M3 else s[name].view(torch.uint8)[:, j][pages].view(E4M3)
                x = x.double() * s[name + "_scale"][:, j][pages][..., None].double() if name + "_scale" in s else x.double()
                both.append(x.reshape(-1, d)[:t])
            for head in range(j * h // kvh, (j + 1) * h // kvh):
                score = s["q"][row:row + n, head].double() @ both[0].T.contiguous() / math.sqrt(d)
                out[row:row + n, head] = torch.softmax(score.masked_fill(far, -math.inf), -1) @ both[1]
        row += n
    return out
