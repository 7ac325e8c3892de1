"""The operators of serving over a paged KV cache, as cases that can be timed and compared.

A serving step takes them one after the other: blocks and slots for the new tokens, the new tokens' queries and keys
normalised, rotated and written into the cache, their attention over the cache, the verification of drafted tokens, and
the blocks of what was refused given back.

Kinds:
  plan     block tables, slots and positions from request lengths, then the blocks behind the kept lengths given back
  qkv      per-head norm and rotation of queries and keys, keys and values into the cache
  chunk    attention of new tokens over the paged cache, from one token a sequence to a prompt's piece
  verify   drafted tokens against the target's probabilities
"""
import math
import random

import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_EPS = 1e-6
_THETA = 500000.0
_NO_KEYS = -3.402823e38


# -- the cases --------------------------------------------------------------------------------------

def listed():
    return [
        # the smallest call: a decode step of 64 users, one token each
        dict(name="plan_decode64", kind="plan", seqs=64, new=1, ragged=False, cached=3000, page=16, shape=1),
        # prompts of very different lengths admitted together, 32-token pages, a padded batch of tokens
        dict(name="plan_prompts", kind="plan", seqs=300, new=400, ragged=True, cached=700, page=32, shape=2),
        # one token of one user: latency
        dict(name="qkv_token", kind="qkv", dtype="bf16", tokens=1, pad=0, heads=32, kv=8, dim=128, rot=128, halves=True, norm=True, page=16),
        # a piece of prompts, as large as one step takes
        dict(name="qkv_prompt", kind="qkv", dtype="bf16", tokens=8192, pad=0, heads=32, kv=8, dim=128, rot=128, halves=True, norm=True, page=16),
        # f32 with adjacent pairs, part of a narrow head rotated, an odd and padded batch
        dict(name="qkv_ragged_f32", kind="qkv", dtype="f32", tokens=777, pad=23, heads=12, kv=4, dim=80, rot=40, halves=False, norm=False, page=24),
        # one token of one user over a short context: latency of attention
        dict(name="chunk_token", kind="chunk", dtype="bf16", seqs=1, q=1, big=0, ctx=300, ragged=False, pad=0, heads=32, kv=8, dim=128, page=16,
             causal=True, shape=3),
        # a decode step of 32 users of different lengths
        dict(name="chunk_decode32", kind="chunk", dtype="f16", seqs=32, q=1, big=0, ctx=8192, ragged=True, pad=0, heads=32, kv=8, dim=128, page=16,
             causal=True, shape=4),
        # five drafted tokens of each of eight users over an f32 cache
        dict(name="chunk_drafts_f32", kind="chunk", dtype="f32", seqs=8, q=5, big=0, ctx=2000, ragged=True, pad=3, heads=32, kv=8, dim=128, page=16,
             causal=True, shape=5),
        # a step that mixes 31 users' single tokens with a piece of 1000 tokens of one prompt
        dict(name="chunk_mixed", kind="chunk", dtype="bf16", seqs=32, q=1, big=1000, ctx=4096, ragged=True, pad=0, heads=32, kv=8, dim=128, page=32,
             causal=True, shape=6),
        # a piece of 2048 tokens at the end of a long prompt: the most arithmetic
        dict(name="chunk_prompt", kind="chunk", dtype="bf16", seqs=1, q=2048, big=0, ctx=8192, ragged=False, pad=0, heads=32, kv=8, dim=128, page=64,
             causal=True, shape=7),
        # one user's four drafts
        dict(name="verify_one", kind="verify", seqs=1, drafts=4, ragged=False, vocab=32000, certain=False, shape=8),
        # a batch of 64 users, up to five drafts each, a large vocabulary
        dict(name="verify_batch", kind="verify", seqs=64, drafts=5, ragged=True, vocab=128256, certain=False, shape=9),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "qkv", "qkv", "chunk", "chunk", "chunk", "chunk", "verify"])
    page = rng.choice([8, 16, 16, 16, 32, 64, 128, 24])
    shape = rng.randrange(1 << 20)
    if kind == "plan":
        seqs = _log(rng, 1, 512)
        return dict(kind=kind, seqs=seqs, new=_log(rng, 1, max(1, min(4000, 60000 // seqs))), ragged=rng.random() < 0.7,
                    cached=_log(rng, 1, 8000), page=rng.choice([page, 1]), shape=shape)
    heads, kv = rng.choice([(32, 8), (32, 8), (32, 8), (64, 8), (16, 16), (8, 1), (12, 4), (14, 2)])
    dim = rng.choice([128, 128, 128, 64, 96, 80, 256])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "qkv":
        size = (heads + 2 * kv) * dim * (4 if dtype == "f32" else 2)
        rot = rng.choice([dim, dim, dim // 2])
        return dict(kind=kind, dtype=dtype, tokens=_log(rng, 1, 8192 * 6144 * 2 // size), pad=rng.choice([0, 0, 7]), heads=heads, kv=kv, dim=dim,
                    rot=rot, halves=rng.random() < 0.6, norm=rng.random() < 0.6, page=page)
    if kind == "verify":
        return dict(kind=kind, seqs=_log(rng, 1, 64), drafts=rng.randint(1, 5), ragged=rng.random() < 0.5,
                    vocab=rng.choice([32000, 128256, 50257, _log(rng, 1000, 128256)]), certain=rng.random() < 0.3, shape=shape)
    form = rng.choice(["token", "token", "drafts", "piece", "mixed"])
    seqs = 1 if form == "piece" and rng.random() < 0.5 else _log(rng, 1, 32 if form != "piece" else 8)
    q = 1 if form in ("token", "mixed") else rng.randint(2, 8) if form == "drafts" else _log(rng, 16, 2048 // seqs)
    big = _log(rng, 64, 1024) if form == "mixed" else 0
    # the cache stays below half a gigabyte of each of K and V, and the pairs below those of the listed prompt
    keys = (1 << 29) // (kv * dim * (4 if dtype == "f32" else 2)) // seqs
    pairs = 14 * 2 ** 20 * 4096 // (heads * dim) // (8 if dtype == "f32" or dim > 128 else 1)
    ctx = _log(rng, 100, max(200, min(32768, keys, pairs // max(q * seqs, big + seqs))))
    q, big = min(q, ctx), min(big, ctx)
    return dict(kind=kind, dtype=dtype, seqs=seqs, q=q, big=big, ctx=ctx, ragged=rng.random() < 0.6, pad=rng.choice([0, 0, 5]), heads=heads, kv=kv,
                dim=dim, page=page, causal=rng.random() < 0.85, shape=shape)


def _lengths(case):
    """What the host knows of a batch: the new tokens and the context of each sequence."""
    rng = random.Random(case.get("shape", 0))
    n = case["seqs"]
    if case["kind"] == "plan":
        new = [_log(rng, 1, 2 * case["new"]) if case["ragged"] else case["new"] for _ in range(n)]
        if case["ragged"] and n > 2:
            new[1] = 0                                     # a sequence that waits
        cached = [rng.randint(0, case["cached"]) for _ in range(n)]
        return new, cached
    new = [case["q"]] * n
    if case["ragged"] and case["q"] > 1:
        new = [rng.randint(1, case["q"]) for _ in range(n)]
        new[0] = case["q"]
    if case["big"]:
        new[n // 2] = case["big"]
    ctx = [rng.randint(max(new[i], case["ctx"] // 8), max(new[i], case["ctx"])) if case["ragged"] else max(case["ctx"], new[i]) for i in range(n)]
    ctx[0] = max(ctx[0], case["ctx"])
    return new, ctx


# -- inputs -----------------------------------------------------------------------------------------

class _State:
    pass


_ctx = None


def _context():
    """One context per process, on the stream torch works on."""
    global _ctx
    from webgpu_b200 import backend as B

    if _ctx is None:
        _ctx = B.load().create_context(torch.cuda.current_device())
    _ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    return _ctx


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = _State()
    s.case = case
    kind = case["kind"]

    def normal(shape, dtype=torch.float32):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    def shuffled(n):
        return torch.randperm(n, generator=g, device="cuda").to(torch.int32)

    if kind == "plan":
        new, cached = _lengths(case)
        n, page = case["seqs"], case["page"]
        s.max_blocks = max((c + t + page - 1) // page for c, t in zip(cached, new)) + 3
        held = [(c + page - 1) // page for c in cached]
        wanted = sum((c + t + page - 1) // page for c, t in zip(cached, new)) - sum(held)
        ids = shuffled(sum(held) + wanted + 11)
        s.table = torch.full((n, s.max_blocks), -1, dtype=torch.int32, device="cuda")
        col = torch.arange(s.max_blocks, device="cuda")
        s.table[col[None, :] < _ints(held)[:, None]] = ids[:sum(held)]
        s.free = ids[sum(held):].clone()
        s.count = _ints([s.free.numel()])
        s.cached, s.new = _ints(cached), _ints(new)
        s.tokens = sum(new) + (5 if case["ragged"] else 0)
        # of the new tokens, those that are kept
        s.keep = (s.cached + (s.new * torch.rand(n, generator=g, device="cuda")).to(torch.int32)).contiguous()
        s.starts, s.lens = _ints([0] * (n + 1)), _ints([0] * n)
        s.pos, s.slots = _ints([0] * s.tokens), _ints([0] * s.tokens)
        _wrap(s, "table", "free", "count", "cached", "new", "keep", "starts", "lens", "pos", "slots")
    elif kind == "qkv":
        td, T, D, page = _DT[case["dtype"]], case["tokens"] + case["pad"], case["dim"], case["page"]
        H, KV, rot = case["heads"], case["kv"], case["rot"]
        s.qkv = normal((T, (H + 2 * KV) * D), td)
        s.wq, s.wk = 1 + 0.1 * normal((D,)), 1 + 0.1 * normal((D,))
        blocks = (case["tokens"] + page - 1) // page + 2
        s.slots = shuffled(blocks * page)[:T].contiguous()
        s.pos = torch.randint(0, 9000, (T,), generator=g, device="cuda", dtype=torch.int32)
        if case["pad"]:
            s.slots[case["tokens"]:] = -1
        angle = torch.arange(9000, device="cuda", dtype=torch.float64)[:, None] * _THETA ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
        s.cos, s.sin = angle.cos().float(), angle.sin().float()
        s.q = torch.zeros((T, H, D), device="cuda", dtype=td)
        s.kc, s.vc = (torch.zeros((blocks, KV, page, D), device="cuda", dtype=td) for _ in range(2))
        _wrap(s, "qkv", "wq", "wk", "slots", "pos", "cos", "sin", "q", "kc", "vc")
    elif kind == "chunk":
        td, D, page = _DT[case["dtype"]], case["dim"], case["page"]
        H, KV, n = case["heads"], case["kv"], case["seqs"]
        s.new, s.ctx = _lengths(case)
        s.T = sum(s.new) + case["pad"]
        held = [(c + page - 1) // page for c in s.ctx]
        s.max_blocks = max(held) + 1
        blocks = sum(held) + 2
        s.table = torch.full((n, s.max_blocks), -1, dtype=torch.int32, device="cuda")
        s.table[torch.arange(s.max_blocks, device="cuda")[None, :] < _ints(held)[:, None]] = shuffled(blocks)[:sum(held)]
        s.q = normal((s.T, H, D), td)
        s.kc, s.vc = normal((blocks, KV, page, D), td), normal((blocks, KV, page, D), td)
        starts = [0]
        for t in s.new:
            starts.append(starts[-1] + t)
        s.starts, s.lens = _ints(starts), _ints(s.ctx)
        s.out = torch.zeros((s.T, H, D), device="cuda", dtype=td)
        s.lse = torch.zeros((s.T, H), device="cuda", dtype=torch.float32)
        _wrap(s, "table", "q", "kc", "vc", "starts", "lens", "out", "lse")
        if own:
            s.code = _code(case["dtype"])
            s.work = torch.empty(max(1, _context().paged_chunk_workspace(n, s.T, H, KV, D, s.code)), dtype=torch.uint8, device="cuda")
            _wrap(s, "work")
    elif kind == "verify":
        n, V = case["seqs"], case["vocab"]
        rng = random.Random(case["shape"])
        drafts = [rng.randint(0, case["drafts"]) if case["ragged"] else case["drafts"] for _ in range(n)]
        starts = [0]
        for d in drafts:
            starts.append(starts[-1] + d + 1)
        s.R = starts[-1]
        s.n_drafts = drafts
        logits = 3 * normal((s.R, V))
        s.p = torch.softmax(logits, -1)
        if case["certain"]:
            # drafts looked up in the text rather than drawn: mostly likely tokens
            s.q = None
            s.tokens = torch.multinomial(s.p, 1, generator=g)[:, 0].to(torch.int32)
        else:
            s.q = torch.softmax(logits + 0.5 * normal((s.R, V)), -1)
            s.tokens = torch.multinomial(s.q, 1, generator=g)[:, 0].to(torch.int32)
        # row r holds the token fed in there: the draft that row r - 1 gave
        s.tokens = torch.cat([s.tokens[-1:], s.tokens[:-1]]).contiguous()
        s.u = torch.rand(s.R, generator=g, device="cuda")
        s.starts = _ints(starts)
        s.lens = _ints([1000 + 3 * i + d for i, d in enumerate(drafts)])
        s.out, s.accepted, s.kept = _ints([0] * s.R), _ints([0] * n), _ints([0] * n)
        _wrap(s, "p", "tokens", "u", "starts", "lens", "out", "accepted", "kept")
        s.b_q = None
        if s.q is not None:
            _wrap(s, "q")
    else:
        raise ValueError(kind)
    return s


def _wrap(s, *names):
    if own:
        ctx = _context()
        for name in names:
            t = getattr(s, name)
            setattr(s, "b_" + name, ctx.wrap(t.data_ptr(), t.numel() * t.element_size()))


def _code(dtype):
    from webgpu_b200 import backend as B

    return {"f32": B.F32, "f16": B.F16, "bf16": B.BF16}[dtype]


# -- one pass ---------------------------------------------------------------------------------------

def run(s):
    return {"plan": _plan, "qkv": _qkv, "chunk": _chunk, "verify": _verify}[s.case["kind"]](s)


def _plan(s):
    n, page, T = s.case["seqs"], s.case["page"], s.tokens
    if own:
        ctx = _context()
        ctx.paged_reserve(s.b_cached, s.b_new, s.b_table, s.b_free, s.b_count, s.b_starts, s.b_lens, s.b_pos, s.b_slots, n, s.max_blocks, page, T,
                          flags=1)
        ctx.paged_release(s.b_keep, s.b_table, s.b_free, s.b_count, n, s.max_blocks, page, flags=1)
        return [s.starts, s.lens, s.pos, s.slots, s.table, s.free, s.count]
    s.lens = s.cached + s.new
    s.starts = torch.cat([torch.zeros_like(s.new[:1]), torch.cumsum(s.new, 0, dtype=torch.int32)])
    col = torch.arange(s.max_blocks, device="cuda", dtype=torch.int32)[None, :]
    # blocks that the new tokens reach and the table does not hold yet, in order, from the end of the free list
    wanted = (col >= (s.cached // page)[:, None]) & (col < ((s.lens + page - 1) // page)[:, None]) & (s.table < 0) & (s.new > 0)[:, None]
    k = torch.cumsum(wanted.flatten(), 0).reshape(wanted.shape)
    s.table = torch.where(wanted, s.free[(s.count - k).clamp(0, s.free.numel() - 1)], s.table)
    s.count = s.count - k[-1, -1].to(torch.int32)
    # the place of each new token
    t = torch.arange(T, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s.starts[1:].contiguous(), t, right=True).clamp(max=n - 1)
    real = t < s.starts[-1]
    s.pos = torch.where(real, s.cached[seq] + t - s.starts[seq], 0)
    s.slots = torch.where(real, s.table[seq, s.pos // page] * page + s.pos % page, -1)
    # the blocks behind the kept tokens go back, the first of them on top
    gone = (col >= ((s.keep + page - 1) // page)[:, None]) & (s.table >= 0) & (s.keep >= 0)[:, None]
    j = torch.cumsum(gone.flatten(), 0).reshape(gone.shape)
    m = j[-1, -1]
    place = torch.where(gone, s.count + m - j, s.free.numel())
    grown = torch.cat([s.free, s.free[:1]])
    grown[place.flatten()] = s.table.flatten()
    s.free = grown[:-1]
    s.table = torch.where(gone, -1, s.table)
    s.count = s.count + m.to(torch.int32)
    return [s.starts, s.lens, s.pos, s.slots, s.table, s.free, s.count]


def _qkv(s):
    c = s.case
    H, KV, D, rot, page = c["heads"], c["kv"], c["dim"], c["rot"], c["page"]
    if own:
        from webgpu_b200 import backend as B

        _context().paged_qkv(s.b_qkv, s.b_wq if c["norm"] else None, s.b_wk if c["norm"] else None, s.b_cos, s.b_sin, s.b_pos, s.b_slots, s.b_q,
                             s.b_kc, s.b_vc, s.qkv.shape[0], H, KV, D, rot, page, _EPS, _code(c["dtype"]),
                             flags=B.FLAG_NO_SYNC | (B.FLAG_ROPE_HALVES if c["halves"] else 0))
        return [s.q, s.kc, s.vc]
    n = c["tokens"]
    x = s.qkv[:n].float().reshape(n, H + 2 * KV, D)
    cos, sin = s.cos[s.pos[:n].long()][:, None, :], s.sin[s.pos[:n].long()][:, None, :]

    def head(y, w):
        if c["norm"]:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + _EPS) * w
        r = y[..., :rot]
        if c["halves"]:
            a, b = r[..., :rot // 2], r[..., rot // 2:]
            r = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
        else:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
        return torch.cat([r, y[..., rot:]], -1)

    s.q[:n] = head(x[:, :H], s.wq).to(s.q.dtype)
    slot = s.slots[:n].long()
    s.kc[slot // page, :, slot % page] = head(x[:, H:H + KV], s.wk).to(s.q.dtype)
    s.vc[slot // page, :, slot % page] = s.qkv[:n].reshape(n, H + 2 * KV, D)[:, H + KV:]
    return [s.q, s.kc, s.vc]


def _chunk(s):
    c = s.case
    H, KV, D, page = c["heads"], c["kv"], c["dim"], c["page"]
    scale = 1.0 / math.sqrt(D)
    if own:
        from webgpu_b200 import backend as B

        _context().paged_chunk_attention(s.b_q, s.b_kc, s.b_vc, s.b_table, s.b_starts, s.b_lens, s.b_out, c["seqs"], s.T, H, KV, D, page, s.max_blocks,
                                         scale, s.code, s.b_work, lse=s.b_lse,
                                         flags=B.FLAG_NO_SYNC | (B.FLAG_ATTN_CAUSAL if c["causal"] else 0))
        return [s.out, s.lse]
    at = 0
    for i, (t, keys) in enumerate(zip(s.new, s.ctx)):
        blocks = s.table[i, :(keys + page - 1) // page].long()
        k, v = (x[blocks].float().transpose(0, 1).reshape(KV, -1, D)[:, :keys] for x in (s.kc, s.vc))
        q = s.q[at:at + t].float().reshape(t, KV, H // KV, D).permute(1, 2, 0, 3)
        seen = None
        if c["causal"] and t > 1:
            seen = torch.arange(keys, device="cuda")[None, :] <= torch.arange(keys - t, keys, device="cuda")[:, None]
        for h in range(0, KV, KV if t * keys * H <= 1 << 26 else 1):
            part = slice(h, KV if t * keys * H <= 1 << 26 else h + 1)
            x = torch.matmul(q[part], k[part, None].transpose(-1, -2)) * scale
            if seen is not None:
                x = x.masked_fill(~seen, float("-inf"))
            top = x.amax(-1, keepdim=True)
            x = torch.exp(x - top)
            total = x.sum(-1, keepdim=True)
            o = torch.matmul(x, v[part, None]) / total
            s.out.view(s.T, KV, H // KV, D)[at:at + t, part] = o.permute(2, 0, 1, 3).to(s.out.dtype)
            s.lse.view(s.T, KV, H // KV)[at:at + t, part] = (top + torch.log(total))[..., 0].permute(2, 0, 1)
        at += t
    return [s.out, s.lse]


def _verify(s):
    c = s.case
    n, V = c["seqs"], c["vocab"]
    if own:
        _context().verify_drafts(s.b_p, s.b_q, s.b_tokens, s.b_u, s.b_starts, s.b_out, s.b_accepted, n, s.R, V, context_lens=s.b_lens,
                                 kept_lens=s.b_kept, flags=1)
        return [s.out, s.accepted, s.kept]
    starts = s.starts.long()
    drafts = starts[1:] - starts[:-1] - 1
    i = torch.arange(c["drafts"], device="cuda")[None, :]
    row = (starts[:-1, None] + i).clamp(max=s.R - 1)
    token = s.tokens[(row + 1).clamp(max=s.R - 1)].long()
    p = s.p[row, token].double()
    q = torch.ones_like(p) if s.q is None else s.q[row, token].double()
    taken = torch.cumprod(((s.u[row].double() * q < p) & (i < drafts[:, None])).int(), 1)
    s.accepted = taken.sum(1, dtype=torch.int32)
    # where the sequence goes on: what the target wants more than the draft did, or the target alone behind the last draft
    last = starts[:-1] + s.accepted
    weight = s.p[last].double()
    refused = s.accepted < drafts
    if s.q is None:
        less = torch.zeros_like(weight).scatter_(1, s.tokens[(last + 1).clamp(max=s.R - 1)].long()[:, None], 1.0)
    else:
        less = s.q[last].double()
    rest = (weight - less).clamp(min=0)
    weight = torch.where((refused & (rest.sum(1) > 0))[:, None], rest, weight)
    up_to = torch.cumsum(weight, 1)
    total = up_to[:, -1:]
    drawn = (up_to <= s.u[starts[1:] - 1].double()[:, None] * total).sum(1)
    most = V - 1 - (weight > 0).flip(1).int().argmax(1)
    drawn = torch.minimum(drawn, most)
    s.out = torch.full_like(s.out, -1)
    s.out[row[taken > 0]] = s.tokens[row[taken > 0] + 1]
    s.out[last] = drawn.to(torch.int32)
    s.kept = s.lens - (drafts - s.accepted).to(torch.int32)
    return [s.out, s.accepted, s.kept]


# -- the same from the definition, in 64 bits ---------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": _exact_plan, "qkv": _exact_qkv, "chunk": _exact_chunk, "verify": _exact_verify}[case["kind"]](s)


def _exact_plan(s):
    page = s.case["page"]
    cached, new, keep, free = s.cached.tolist(), s.new.tolist(), s.keep.tolist(), s.free.tolist()
    table = s.table.tolist()
    top = len(free)
    starts, lens, pos, slots = [0], [], [], []
    for row, c, t in zip(table, cached, new):
        for p in range(c, c + t):
            if row[p // page] < 0:
                top -= 1
                row[p // page] = free[top]
            pos.append(p)
            slots.append(row[p // page] * page + p % page)
        starts.append(starts[-1] + t)
        lens.append(c + t)
    pos += [0] * (s.tokens - len(pos))
    slots += [-1] * (s.tokens - len(slots))
    back = []
    for row, k in zip(table, keep):
        for b in range((k + page - 1) // page, len(row)):
            if row[b] >= 0:
                back.append(row[b])
                row[b] = -1
    for b in reversed(back):
        free[top] = b
        top += 1
    return [_ints(x) for x in (starts, lens, pos, slots, table, free, [top])]


def _exact_qkv(s):
    c = s.case
    H, KV, D, rot, page = c["heads"], c["kv"], c["dim"], c["rot"], c["page"]
    q, kc, vc = s.q.double(), s.kc.double(), s.vc.double()
    n = c["tokens"]
    at, places = s.pos[:n].long(), s.slots[:n].long()
    z = torch.complex(s.cos.double()[at], s.sin.double()[at])[:, None]
    first = torch.arange(rot // 2, device="cuda") if c["halves"] else torch.arange(0, rot, 2, device="cuda")
    second = first + (rot // 2 if c["halves"] else 1)
    for h in range(H + KV):
        y = s.qkv[:n, h * D:(h + 1) * D].double()
        if c["norm"]:
            y = y / (y.square().sum(1, keepdim=True) / D + _EPS).sqrt() * (s.wq if h < H else s.wk).double()
        turned = torch.complex(y[:, first], y[:, second]) * z[:, 0]
        y = y.clone()
        y[:, first], y[:, second] = turned.real, turned.imag
        if h < H:
            q[:n, h] = y
        else:
            kc[places // page, h - H, places % page] = y
            vc[places // page, h - H, places % page] = s.qkv[:n, (h + KV) * D:(h + KV + 1) * D].double()
    return [q, kc, vc]


def _exact_chunk(s):
    c = s.case
    H, KV, page = c["heads"], c["kv"], c["page"]
    if sum(t * k for t, k in zip(s.new, s.ctx)) * H * c["dim"] > 1 << 40:
        return None
    out, lse = torch.zeros(s.out.shape, device="cuda", dtype=torch.float64), torch.zeros(s.lse.shape, device="cuda", dtype=torch.float64)
    row = 0
    for i, (t, keys) in enumerate(zip(s.new, s.ctx)):
        at = torch.arange(keys, device="cuda")
        block, off = s.table[i][at // page].long(), at % page
        sees = torch.arange(t, device="cuda") + (keys - t) if c["causal"] else torch.full((t,), keys - 1, device="cuda")
        for h in range(H):
            k, v = s.kc[block, h * KV // H, off].double(), s.vc[block, h * KV // H, off].double()
            for a in range(0, t, 1024):
                x = torch.einsum("td,kd->tk", s.q[row + a:row + min(t, a + 1024), h].double(), k) / math.sqrt(c["dim"])
                x[at[None, :] > sees[a:a + 1024, None]] = float("-inf")
                z = torch.logsumexp(x, 1)
                lse[row + a:row + min(t, a + 1024), h] = z
                out[row + a:row + min(t, a + 1024), h] = torch.exp(x - z[:, None]) @ v
        row += t
    return [out, lse]


def _exact_verify(s):
    tokens, u = s.tokens.tolist(), s.u.double().tolist()
    out, accepted = [-1] * s.R, []
    row = 0
    for d in s.n_drafts:
        a = 0
        while a < d:
            x = tokens[row + a + 1]
            if not u[row + a] * (1.0 if s.q is None else float(s.q[row + a, x])) < float(s.p[row + a, x]):
                break
            out[row + a] = x
            a += 1
        w = s.p[row + a].double().cpu()
        if a < d:
            if s.q is None:
                rest = w.clone()
                rest[tokens[row + a + 1]] = max(0.0, float(w[tokens[row + a + 1]]) - 1.0)
            else:
                rest = torch.relu(w - s.q[row + a].double().cpu())
            if float(rest.sum()) > 0:
                w = rest
        sums = w.numpy().cumsum()
        x = int((sums <= u[row + d] * sums[-1]).sum())
        out[row + a] = min(x, int(w.nonzero().max()))
        accepted.append(a)
        row += d + 1
    kept = [n - d + a for n, d, a in zip(s.lens.tolist(), s.n_drafts, accepted)]
    return [_ints(x) for x in (out, accepted, kept)]


# -- what a pass cannot do without ------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "plan":
        new, cached = _lengths(case)
        page = case["page"]
        taken = sum((c + t + page - 1) // page - (c + page - 1) // page for c, t in zip(cached, new))
        # lengths in, starts and lengths out, 8 bytes a token, the blocks that change hands; one division and one sum a token
        return {"bytes": 20 * len(new) + 8 * sum(new) + 12 * taken, "flops": 2 * sum(new) + 4 * len(new)}
    if kind == "qkv":
        e = 4 if case["dtype"] == "f32" else 2
        H, KV, D, n = case["heads"], case["kv"], case["dim"], case["tokens"]
        table = min(n, 9000) * case["rot"] * 4
        return {"bytes": n * (H + 2 * KV) * D * 2 * e + n * 8 + table, "flops": n * (H + KV) * (4 * D + 3 * case["rot"])}
    if kind == "chunk":
        e = 4 if case["dtype"] == "f32" else 2
        H, KV, D = case["heads"], case["kv"], case["dim"]
        new, ctx = _lengths(case)
        pairs = sum(t * k - (t * (t - 1) // 2 if case["causal"] else 0) for t, k in zip(new, ctx))
        return {"bytes": 2 * KV * D * e * sum(ctx) + sum(new) * H * (2 * D * e + 4), "flops": 4 * H * D * pairs}
    n, V = case["seqs"], case["vocab"]
    d = case["drafts"] / (2 if case["ragged"] else 1)
    return {"bytes": n * (V * 4 * (1 if case["certain"] else 2) + d * 16 + 28), "flops": n * V * 3}
