"""The work of a layer on a chunk of new tokens, as cases that can be timed: rotate and append the chunk's keys and values,
attend from the chunk over a paged cache, uncompressed or packed.

A case is a flat dict; `op` says which operator:

  rope    queries and keys rotated by their positions, keys and values appended to an uncompressed paged cache (rope_append)
  dense   causal attention of every sequence's newest tokens over such a cache (paged_chunk_attention)
  packed  the same over a cache of 4-, 3- or 2-bit codes and norms (TQPagedAttention.forward_chunk)

  d, heads, kv_heads, block, dtype   head size, query and kv heads, tokens per cache block, "bf16" or "f16"
  rope:    tokens; rotary (coordinates that turn), sections ("" or the pairs of each axis, as "16-24-24"), interleaved; span
           (positions lie below it)
  dense, packed: seqs; new_lo, new_hi and ctx_lo, ctx_hi: new tokens and context before them of a sequence, uniform in the ranges;
           lens_seed; window (0: all keys); bits and layout ("primary": K and V rows inside one byte tensor, as a serving engine
           allocates it; "split") of a packed cache

`own` chooses between the framework's operators and their plain forms.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
LARGEST = 2048 * 30720 * 32          # new tokens x context x query heads of the largest listed case


def listed():
    def rope(name, tokens, **more):
        case = dict(name=name, op="rope", d=128, heads=32, kv_heads=8, block=16, dtype="bf16", tokens=tokens, rotary=128, sections="",
                    interleaved=False, span=40960)
        case.update(more)
        return case

    def attend(name, op, seqs, new, ctx, **more):
        case = dict(name=name, op=op, d=128, heads=32, kv_heads=8, block=16, dtype="bf16", seqs=seqs, new_lo=new[0], new_hi=new[1],
                    ctx_lo=ctx[0], ctx_hi=ctx[1], lens_seed=2, window=0)
        if op == "packed":
            case.update(bits=4, layout="primary")
        case.update(more)
        return case

    return [
        # one user's next token: a launch and little else
        rope("rope_one_token", 1),
        # a batch of decode steps on one of eight ranks of a 64-head layer, half of each head turning
        rope("rope_decode_rank", 200, heads=8, kv_heads=1, rotary=64, interleaved=True, dtype="f16"),
        # an image among text: positions in time, height and width
        rope("rope_image", 4097, sections="16-24-24"),
        # a prompt chunk
        rope("rope_chunk", 8192),
        # the first chunk of a prompt: nothing before it
        attend("dense_first_chunk", "dense", 1, (2048, 2048), (0, 0)),
        # a chunk of a long prompt: the largest case
        attend("dense_long_prompt", "dense", 1, (2048, 2048), (30720, 30720)),
        # continuous batching: prompts of all lengths beside decode steps, groups of seven heads of 64
        attend("dense_mixed_batch", "dense", 24, (1, 300), (0, 4000), d=64, heads=28, kv_heads=4, dtype="f16"),
        # a few tokens a sequence, heads of 256, keys no older than 1024 tokens
        attend("dense_window_verify", "dense", 9, (3, 6), (900, 9000), d=256, heads=16, kv_heads=4, window=1024),
        # one user's draft of three tokens, a few hundred tokens in: latency
        attend("packed_draft_one_user", "packed", 1, (3, 3), (700, 700)),
        # drafts of four tokens verified over the headline benchmark's ragged contexts
        attend("packed_verify_batch", "packed", 16, (4, 4), (1024, 40000), dtype="f16", layout="split"),
        # prompt chunks continued over a packed context
        attend("packed_prompt_chunk", "packed", 2, (1000, 1024), (7000, 8192)),
        # short continued turns at 3 bits
        attend("packed_turns_3bit", "packed", 12, (1, 90), (100, 6000), bits=3, layout="split"),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choices(("rope", "dense", "packed"), (25, 38, 37))[0]
    case = dict(op=op, d=rng.choices((64, 128, 256), (22, 56, 22))[0], block=rng.choices((16, 32), (75, 25))[0],
                dtype=rng.choices(("bf16", "f16"), (60, 40))[0])
    # whole layers, and the slices of them that ranks of a sharded model keep
    case["heads"], case["kv_heads"] = rng.choices(((32, 8), (64, 8), (16, 4), (8, 2), (8, 1), (28, 4), (40, 8), (16, 16)),
                                                  (34, 12, 12, 10, 10, 8, 7, 7))[0]
    if op == "rope":
        most = 8192 * 48 * 128 // ((case["heads"] + 2 * case["kv_heads"]) * case["d"])
        case["tokens"] = log_int(1, max(1, most))
        case["rotary"] = rng.choice([r for r in (32, 64, 128, 256) if r <= case["d"]])
        case["interleaved"] = rng.random() < 0.3
        case["sections"] = ""
        if rng.random() < 0.4:
            half = case["rotary"] // 2
            a = rng.randrange(1, half // 2)
            b = rng.randrange(1, half - a)
            case["sections"] = "%d-%d-%d" % (a, b, half - a - b) if half - a - b > 0 else "%d-%d" % (a, half - a)
        case["span"] = log_int(512, 131072)
        return case
    # from a draft of a few tokens a sequence to whole prompt chunks; padded scores bounded by the largest listed case
    new = log_int(1, 8) if rng.random() < 0.4 else log_int(8, 2048)
    case["seqs"] = log_int(1, max(1, min(64, 4096 // new)))
    spread = rng.choice((0.0, 0.5, 0.95))
    case["new_lo"], case["new_hi"] = max(1, int(new * (1 - spread))), new
    most = LARGEST // (2 * case["seqs"] * new * case["heads"]) - new
    most = min(most, 40000, (1 << 30) // (case["seqs"] * case["kv_heads"] * case["d"] * 2))
    case["ctx_hi"] = log_int(1, most) if most > 1 and rng.random() < 0.9 else 0
    case["ctx_lo"] = int(case["ctx_hi"] * (1 - spread))
    case["lens_seed"] = rng.randrange(1000)
    case["window"] = log_int(16, 8192) if op == "dense" and rng.random() < 0.25 else 0
    if op == "packed":
        case["bits"] = rng.choices((4, 3, 2), (60, 20, 20))[0]
        case["layout"] = rng.choice(("primary", "split"))
    return case


def _lens(case):
    """(new tokens, tokens with them) of every sequence."""
    rng = np.random.default_rng(case["lens_seed"])
    new = rng.integers(case["new_lo"], case["new_hi"] + 1, size=case["seqs"]).astype(np.int64)
    return new, new + rng.integers(case["ctx_lo"], case["ctx_hi"] + 1, size=case["seqs"]).astype(np.int64)


def work(case):
    d, qh, kvh = case["d"], case["heads"], case["kv_heads"]
    if case["op"] == "rope":
        t, r = case["tokens"], case["rotary"]
        axes = len(case["sections"].split("-"))
        return {"bytes": t * (2 * (qh + 2 * kvh) * d * 2 + 4 * r + 8 * axes + 8), "flops": t * (qh + kvh) * 3 * r}
    new, ctx = _lens(case)
    first = ctx - new                # position of a sequence's first new token
    w = case["window"] or int(ctx.max())
    # keys that the tokens at first .. ctx - 1 see, and the oldest key that any of them sees
    seen = sum(int(np.minimum(np.arange(a, b) + 1, w).sum()) for a, b in zip(first, ctx))
    held = int((ctx - np.maximum(first + 1 - w, 0)).sum())
    row = 2 * d if case["op"] == "dense" else d * case["bits"] // 8 + 4
    turn = 0 if case["op"] == "dense" else 4 * d * d * qh * int(new.sum())
    return {"bytes": 2 * held * kvh * row + 4 * int(new.sum()) * qh * d + 4 * int((-(-ctx // case["block"])).sum()) + 8 * case["seqs"],
            "flops": 4 * d * qh * seen + turn}


# ---- inputs -------------------------------------------------------------------------------------------------

class _State:
    pass


def _vectors(gen, dtype, *shape):
    """Keys and values as a cache meets them: normal entries, the scale of a vector lognormal."""
    x = torch.randn(shape, device=DEVICE, generator=gen)
    return x.mul_(torch.exp(0.5 * torch.randn(shape[:-1], device=DEVICE, generator=gen)).unsqueeze(-1)).to(dtype)


def _levels(d, bits):
    """Levels and boundaries of least squared error for the coordinates of a random unit vector (normal, variance 1 / d)."""
    n = 1 << bits
    phi = lambda x: math.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)  # noqa: E731
    cdf = lambda x: 0.5 * math.erfc(-x / math.sqrt(2))  # noqa: E731
    c = [2.0 * (2 * i + 1 - n) / n for i in range(n)]
    for _ in range(400):
        b = [-12.0] + [(x + y) / 2 for x, y in zip(c, c[1:])] + [12.0]
        c = [(phi(x) - phi(y)) / (cdf(y) - cdf(x)) for x, y in zip(b, b[1:])]
    return [x / math.sqrt(d) for x in c], [(x + y) / 2 / math.sqrt(d) for x, y in zip(c, c[1:])]


def _rotation(d):
    g = torch.Generator().manual_seed(42)
    q, r = torch.linalg.qr(torch.randn(d, d, generator=g, dtype=torch.float64))
    return (q * torch.sign(torch.diagonal(r))).float()


def _pack(codes, bits):
    """uint8 codes [..., d] as one big-endian bit stream a row."""
    c = codes.reshape(*codes.shape[:-1], -1, 8)
    if bits == 4:
        out = c[..., 0::2] * 16 + c[..., 1::2]
    elif bits == 2:
        out = c[..., 0::4] * 64 + c[..., 1::4] * 16 + c[..., 2::4] * 4 + c[..., 3::4]
    else:
        w = c.to(torch.int32)
        w = sum(w[..., i] << (21 - 3 * i) for i in range(8))
        out = torch.stack([w >> 16, (w >> 8) & 255, w & 255], -1).to(torch.uint8)
    return out.reshape(*codes.shape[:-1], -1)


def _unpack(rows, bits, d):
    """The codes of `d` coordinates a row, as int32."""
    b = rows[..., :d * bits // 8].to(torch.int32)
    if bits == 4:
        out = torch.stack([b >> 4, b & 15], -1)
    elif bits == 2:
        out = torch.stack([b >> 6, (b >> 4) & 3, (b >> 2) & 3, b & 3], -1)
    else:
        b = b.reshape(*b.shape[:-1], -1, 3)
        w = (b[..., 0] << 16) + (b[..., 1] << 8) + b[..., 2]
        out = torch.stack([(w >> (21 - 3 * i)) & 7 for i in range(8)], -1)
    return out.reshape(*rows.shape[:-1], d)


def _codes(gen, boundaries, bits, d, *shape):
    """Packed codes of vectors in random directions."""
    out = torch.empty(*shape, d * bits // 8, dtype=torch.uint8, device=DEVICE)
    flat = out.view(-1, d * bits // 8)
    step = (64 << 20) // d
    for i in range(0, len(flat), step):
        y = torch.randn(min(step, len(flat) - i), d, device=DEVICE, generator=gen).mul_(1 / math.sqrt(d))
        flat[i:i + step] = _pack(torch.bucketize(y, boundaries, out_int32=True).to(torch.uint8), bits)
    return out


def _pool(case, seed, s):
    """Block tables over a pool in random order, with four blocks that no sequence has."""
    new, ctx = _lens(case)
    need = -(-ctx // case["block"])
    blocks = int(need.sum()) + 4
    order = np.random.default_rng(seed).permutation(blocks)
    tables = np.zeros((len(ctx), int(need.max())), dtype=np.int32)
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = order[at:at + n]
        at += int(n)
    s.tables = torch.from_numpy(tables).to(DEVICE)
    s.lens = torch.from_numpy(ctx.astype(np.int32)).to(DEVICE)
    s.starts = torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).to(DEVICE)
    s.most_new, s.most_ctx = int(new.max()), int(ctx.max())
    return blocks


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dt, qh, kvh, d, bs = DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["d"], case["block"]
    s = _State()
    s.op, s.d, s.qh, s.kvh, s.block = case["op"], d, qh, kvh, bs
    if s.op == "rope":
        t, r = case["tokens"], case["rotary"]
        blocks = -(-t // bs) + 4
        s.query = torch.randn((t, qh, d), device=DEVICE, generator=gen).to(dt)
        s.key, s.value = _vectors(gen, dt, t, kvh, d), _vectors(gen, dt, t, kvh, d)
        s.sections = tuple(int(x) for x in case["sections"].split("-")) if case["sections"] else None
        s.interleaved = case["interleaved"]
        # the table a model keeps: cosines, then sines
        angle = torch.arange(case["span"], device=DEVICE, dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(0, r, 2, device=DEVICE, dtype=torch.float64) / r)
        s.cos_sin = torch.cat([angle.cos(), angle.sin()], 1).float()
        axes = (len(s.sections), t) if s.sections else (t,)
        s.positions = torch.randint(case["span"], axes, device=DEVICE, generator=gen)
        # a prompt's tokens fill blocks in order; the blocks lie anywhere
        order = torch.from_numpy(np.random.default_rng(seed).permutation(blocks)).to(DEVICE)
        at = torch.arange(t, device=DEVICE)
        s.slots = order[at // bs] * bs + at % bs
        s.key_cache = torch.zeros(blocks, bs, kvh, d, dtype=dt, device=DEVICE)
        s.value_cache = torch.zeros_like(s.key_cache)
        return s
    blocks = _pool(case, seed, s)
    s.window = case["window"]
    s.query = torch.randn((int(s.starts[-1]), qh, d), device=DEVICE, generator=gen).to(dt)
    if s.op == "dense":
        s.key_cache, s.value_cache = _vectors(gen, dt, blocks, bs, kvh, d), _vectors(gen, dt, blocks, bs, kvh, d)
        return s
    s.bits = case["bits"]
    levels, boundaries = _levels(d, s.bits)
    s.rotation = _rotation(d).to(DEVICE)
    s.levels = torch.tensor(levels, device=DEVICE)
    boundaries = torch.tensor(boundaries, device=DEVICE)
    rows = d * s.bits // 8
    if case["layout"] == "primary":
        kv = torch.zeros(blocks, 2, bs, kvh, rows + 4, dtype=torch.uint8, device=DEVICE)
        s.k_rows, s.v_rows = kv[:, 0, :, :, :rows], kv[:, 1, :, :, :rows]
        s.k_rows.copy_(_codes(gen, boundaries, s.bits, d, blocks, bs, kvh))
        s.v_rows.copy_(_codes(gen, boundaries, s.bits, d, blocks, bs, kvh))
    else:
        s.k_rows, s.v_rows = _codes(gen, boundaries, s.bits, d, blocks, bs, kvh), _codes(gen, boundaries, s.bits, d, blocks, bs, kvh)
    norm = math.sqrt(d)
    s.k_norms = norm * torch.exp(0.5 * torch.randn((blocks, bs, kvh), device=DEVICE, generator=gen))
    s.v_norms = norm * torch.exp(0.5 * torch.randn((blocks, bs, kvh), device=DEVICE, generator=gen))
    if own:
        import aitherkvcache_amd as akv
        tq = akv.TurboQuant(head_dim=d, bits=s.bits, device=DEVICE, dtype=dt)
        tq.rotation, tq.centroids, tq.boundaries_inner = s.rotation, s.levels, boundaries
        s.attn = akv.TQPagedAttention(tq, qh)
    return s


# ---- the operators ------------------------------------------------------------------------------------------

def run(s):
    if s.op == "rope":
        return _run_rope(s)
    return _run_dense(s) if s.op == "dense" else _run_packed(s)


def _run_rope(s):
    if own:
        import aitherkvcache_amd as akv
        q = akv.rope_append(s.query, s.key, s.value, s.positions, s.cos_sin, s.slots, s.key_cache, s.value_cache,
                            sections=s.sections, interleaved=s.interleaved)
        return [q, s.key_cache, s.value_cache]
    half = s.cos_sin.shape[1] // 2
    if s.sections is None:
        row = s.cos_sin[s.positions]
        cos, sin = row[:, :half], row[:, half:]
    else:
        axis = torch.repeat_interleave(torch.arange(len(s.sections)), torch.tensor(s.sections)).to(DEVICE)
        at, pair = s.positions[axis].T, torch.arange(half, device=DEVICE)
        cos, sin = s.cos_sin[at, pair], s.cos_sin[at, half + pair]
    cos, sin = cos[:, None], sin[:, None]

    def turned(x):
        y = x.float()
        a, b = (y[..., 0:2 * half:2], y[..., 1:2 * half:2]) if s.interleaved else (y[..., :half], y[..., half:2 * half])
        u, v = a * cos - b * sin, b * cos + a * sin
        z = torch.stack([u, v], -1).flatten(-2) if s.interleaved else torch.cat([u, v], -1)
        return torch.cat([z, y[..., 2 * half:]], -1).to(x.dtype)

    block, at = s.slots // s.block, s.slots % s.block
    s.key_cache[block, at] = turned(s.key)
    s.value_cache[block, at] = s.value
    return [turned(s.query), s.key_cache, s.value_cache]


def _attend(s, k, v):
    """Plain attention over the keys and values of every sequence, float32 [seqs, tokens, kv heads, d] each."""
    seqs, most, kvh, d = k.shape
    group = s.qh // kvh
    new = s.starts[1:] - s.starts[:-1]
    j, at = torch.arange(s.most_new, device=DEVICE), torch.arange(most, device=DEVICE)
    there = j[None] < new[:, None]                                                   # [seqs, new]
    token = torch.where(there, s.starts[:-1, None] + j[None], 0)
    q = s.query.float()[token].reshape(seqs, s.most_new, kvh, group, d).permute(0, 2, 3, 1, 4).reshape(seqs, kvh, -1, d)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()).view(seqs, kvh, group, s.most_new, most).mul_(1 / math.sqrt(d))
    pos = (s.lens - new)[:, None] + j[None]
    seen = at <= pos[..., None]
    if s.window:
        seen &= at > pos[..., None] - s.window
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True).clamp_min(-1e38)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.view(seqs, kvh, -1, most), v.permute(0, 2, 1, 3).contiguous())
    out = out.view(seqs, kvh, group, s.most_new, d) / total.clamp_min(1e-38)
    return out.permute(0, 3, 1, 2, 4).reshape(seqs, s.most_new, s.qh, d)[there].to(s.query.dtype)


def _rows(s, cache):
    """What the tables name, [seqs, tokens, kv heads, ...], no further than the longest sequence."""
    x = cache[s.tables]
    return x.reshape(x.shape[0], -1, *x.shape[3:])[:, :s.most_ctx]


def _run_dense(s):
    if own:
        import aitherkvcache_amd as akv
        return akv.paged_chunk_attention(s.query, s.key_cache, s.value_cache, s.tables, s.lens, s.starts, window=s.window,
                                         max_query_len=s.most_new)
    return _attend(s, _rows(s, s.key_cache).float(), _rows(s, s.value_cache).float())


def _run_packed(s):
    if own:
        return s.attn.forward_chunk(s.query, s.k_rows, s.k_norms, s.v_rows, s.v_norms, s.tables, s.lens, s.starts, block_size=s.block,
                                    max_query_len=s.most_new)

    def vectors(rows, norms):
        y = s.levels[_unpack(_rows(s, rows), s.bits, s.d)]
        return torch.matmul(y, s.rotation).mul_(_rows(s, norms)[..., None])

    return _attend(s, vectors(s.k_rows, s.k_norms), vectors(s.v_rows, s.v_norms))


# ---- 64 bits ------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    d, bs = s.d, s.block
    if s.op == "rope":
        half = s.cos_sin.shape[1] // 2
        table = s.cos_sin.double()
        pos = s.positions if s.sections else s.positions[None]
        out = [s.query.double(), s.key.double()]
        at = 0
        for axis, pairs in enumerate(s.sections or (half,)):          # an axis turns a run of pairs
            p = torch.arange(at, at + pairs, device=DEVICE)
            turn = torch.complex(table[:, p], table[:, half + p])[pos[axis]][:, None]
            first, second = (2 * p, 2 * p + 1) if s.interleaved else (p, half + p)
            for x in out:
                z = torch.complex(x[..., first], x[..., second]) * turn
                x[..., first], x[..., second] = z.real, z.imag
            at += pairs
        k, v = s.key_cache.double(), s.value_cache.double()
        k.view(-1, *k.shape[2:])[s.slots] = out[1]
        v.view(-1, *v.shape[2:])[s.slots] = s.value.double()
        return [out[0], k, v]
    result = torch.zeros(s.query.shape, dtype=torch.float64, device=DEVICE)
    new, ctx = _lens(case)
    at = 0
    for i, (n, c) in enumerate(zip(new.tolist(), ctx.tolist())):
        blocks = s.tables[i, :-(-c // bs)].long()
        flat = lambda x: x[blocks].flatten(0, 1)[:c]  # noqa: E731
        if s.op == "dense":
            k, v = flat(s.key_cache).double(), flat(s.value_cache).double()
        else:
            k, v = (((s.levels.double()[_unpack(flat(r), s.bits, d)] * flat(m).double()[..., None]) @ s.rotation.double())
                    for r, m in ((s.k_rows, s.k_norms), (s.v_rows, s.v_norms)))
        pos = torch.arange(c - n, c, device=DEVICE)[:, None]
        key = torch.arange(c, device=DEVICE)[None]
        hidden = (key > pos) | ((key <= pos - s.window) if s.window else False)
        for h in range(s.qh):
            kv = h // (s.qh // s.kvh)
            logits = (s.query[at:at + n, h].double() @ k[:, kv].T) / math.sqrt(d)
            result[at:at + n, h] = torch.softmax(logits.masked_fill(hidden, -math.inf), 1) @ v[:, kv]
        at += n
    return result
