"""The operators of a paged KV cache (lux/gpu/paged_ext.h) against plain 64-bit forms, at the sizes, masks and layouts where they can
go wrong.  Whole numbers are equal; the bounds of the others count roundings (tests/paged_reference.py)."""
import math
import random

import pytest
import torch

import paged_reference as ref
from webgpu_b200 import backend as B

pytestmark = pytest.mark.gpu

CODE = {"f32": B.F32, "f16": B.F16, "bf16": B.BF16}


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Bufs:
    """Torch tensors as backend buffers."""

    def __init__(self, ctx):
        self.ctx, self.held = ctx, []

    def __call__(self, t):
        if t is None:
            return None
        torch.cuda.synchronize()
        if t.numel() == 0:
            t = torch.zeros(4, dtype=torch.int32, device="cuda")
        self.held.append(t)                                    # a temporary's memory would be the next one's
        return self.ctx.wrap(t.data_ptr(), t.numel() * t.element_size())


@pytest.fixture
def buf(ctx):
    return Bufs(ctx)


# ---- blocks and slots ---------------------------------------------------------------------------------------------------------------


class Pool:
    def __init__(self, seqs, width, page, blocks, seed=1):
        self.page, self.width = page, width
        self.table = torch.full((seqs, width), -1, dtype=torch.int32, device="cuda")
        ids = list(range(blocks))
        random.Random(seed).shuffle(ids)
        self.free, self.count = ints(ids or [0]), ints([blocks])

    def reserve(self, ctx, buf, cached, new, max_tokens, alias=False):
        n = len(cached)
        c, t = ints(cached), ints(new)
        starts, lens = torch.full((n + 1,), -7, dtype=torch.int32, device="cuda"), c if alias else torch.full((n,), -7, dtype=torch.int32, device="cuda")
        pos, slots = (torch.full((max(1, max_tokens),), -7, dtype=torch.int32, device="cuda") for _ in range(2))
        want = ref.plan(cached, new, self.table.tolist(), self.free.tolist(), int(self.count), self.page, max_tokens)
        before = self.table.tolist(), self.free.tolist(), int(self.count)
        try:
            ctx.paged_reserve(buf(c), buf(t), buf(self.table), buf(self.free), buf(self.count), buf(starts), buf(lens), buf(pos), buf(slots), n, self.width,
                              self.page, max_tokens)
            failed = False
        except B.BackendError as e:
            assert e.code == B.DEVICE_LOST and ctx.last_device_status() == 0x7C05000B
            failed = True
        assert failed == (want is None)
        if want is None:
            assert (self.table.tolist(), self.free.tolist(), int(self.count)) == before
            assert starts.tolist() == [0] * (n + 1) and lens.tolist() == list(cached)
            assert pos.tolist()[:max_tokens] == [0] * max_tokens and slots.tolist()[:max_tokens] == [-1] * max_tokens
            return None
        w_starts, w_lens, w_pos, w_slots, w_table, w_count = want
        assert starts.tolist() == w_starts and lens.tolist() == w_lens
        assert pos.tolist()[:max_tokens] == w_pos and slots.tolist()[:max_tokens] == w_slots
        assert self.table.tolist() == w_table and int(self.count) == w_count and self.free.tolist() == before[1]
        return w_lens

    def release(self, ctx, buf, keep):
        want = ref.release(keep, self.table.tolist(), self.free.tolist(), int(self.count), self.page)
        before = self.table.tolist(), self.free.tolist(), int(self.count)
        try:
            ctx.paged_release(buf(ints(keep)), buf(self.table), buf(self.free), buf(self.count), len(keep), self.width, self.page)
            failed = False
        except B.BackendError as e:
            assert e.code == B.DEVICE_LOST and ctx.last_device_status() == 0x7C05000B
            failed = True
        assert failed == (want is None)
        assert (self.table.tolist(), self.free.tolist(), int(self.count)) == (before if want is None else want)


@pytest.mark.parametrize("seqs,width,page,most,steps", [(1, 9, 16, 40, 6), (33, 5, 8, 9, 5), (70, 300, 1, 60, 5), (3, 4000, 1, 3000, 3),
                                                        (1200, 4, 16, 12, 3), (2500, 3, 24, 8, 2), (1, 1, 1, 1, 2)])
def test_plan_steps(ctx, buf, seqs, width, page, most, steps):
    """Steps of a serving host: tokens reserved, some of them given back, sequences ended, others idle."""
    rng = random.Random(seqs * width)
    pool = Pool(seqs, width, page, seqs * width)
    lens = [0] * seqs
    for step in range(steps):
        new = [0 if rng.random() < 0.2 else min(rng.randint(0, most), width * page - n) for n in lens]
        total = pool.reserve(ctx, buf, lens, new, sum(new) + rng.choice([0, 1, 37]), alias=step % 2 == 1)
        assert total is not None
        keep = [-1 if rng.random() < 0.3 else 0 if rng.random() < 0.1 else n - rng.randint(0, min(n, t)) for n, t in zip(total, new)]
        pool.release(ctx, buf, keep)
        lens = [n if k < 0 else k for n, k in zip(total, keep)]
    pool.release(ctx, buf, [0] * seqs)
    assert int(pool.count) == seqs * width and sorted(pool.free.tolist()) == list(range(seqs * width))


def test_plan_gives_the_same_blocks_again(ctx, buf):
    pool = Pool(5, 8, 4, 40)
    cached, new = [3, 0, 8, 30, 1], [5, 9, 0, 2, 4]
    pool.reserve(ctx, buf, [0] * 5, cached, 60)
    pool.reserve(ctx, buf, cached, new, 60)
    table, count = pool.table.tolist(), int(pool.count)
    pool.release(ctx, buf, cached)
    pool.reserve(ctx, buf, cached, new, 60)
    assert pool.table.tolist() == table and int(pool.count) == count


@pytest.mark.parametrize("tokens", [30, 5000])
def test_plan_hands_out_nothing_where_something_does_not_fit(ctx, buf, tokens):
    pool = Pool(4, 8, 4, 20)
    good = [3, 4, 5, 6]
    assert pool.reserve(ctx, buf, [0, 0, 0, 0], good, tokens) is not None
    for cached, new in [([3, 4, 5, -1], [1, 1, 1, 1]), (good, [1, 1, -1, 1]), (good, [0, 0, 0, 27]), (good, [25, 25, 10, 6]),
                        (good, [2 ** 31 - 1, 0, 0, 0]), ([2 ** 31 - 1, 4, 5, 6], [2 ** 31 - 1, 0, 0, 0])]:
        assert pool.reserve(ctx, buf, cached, new, tokens) is None
    assert pool.reserve(ctx, buf, good, [2, 2, 2, 2], 7) is None
    assert pool.reserve(ctx, buf, good, [2, 2, 2, 2], 8) is not None
    count = int(pool.count)
    for wrong in (-1, 21):
        pool.count.fill_(wrong)
        assert pool.reserve(ctx, buf, good, [1, 1, 1, 1], tokens) is None
        pool.release(ctx, buf, [0, 0, 0, 0])
    pool.count.fill_(20)                                       # a full list has no room
    pool.release(ctx, buf, [0, 0, 0, 0])
    pool.count.fill_(count)
    pool.release(ctx, buf, [0, 0, 0, 0])
    assert int(pool.count) == 20


def test_plan_without_sequences_or_tokens(ctx, buf):
    pool = Pool(3, 4, 4, 12)
    pool.reserve(ctx, buf, [0, 0, 0], [0, 0, 0], 0)
    pool.reserve(ctx, buf, [], [], 9)
    pool.release(ctx, buf, [])


# ---- norm, rotation and append --------------------------------------------------------------------------------------------------------


def run_qkv(ctx, buf, dtype, T, H, KV, D, rot, page, halves, norm, stride=0, shift=0, seed=3, pad=0, scale=1.0):
    dt = ref.DTYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(seed)
    row = (H + 2 * KV) * D
    flat = (scale * torch.randn(shift + T * max(stride, row), generator=g, device="cuda")).to(dt)
    qkv = flat[shift:].reshape(T, max(stride, row))
    wq, wk = (torch.randn(D, generator=g, device="cuda") for _ in range(2)) if norm else (None, None)
    cos, sin = ctx_tables(rot, 500)
    pos = torch.randint(0, 500, (T,), generator=g, device="cuda", dtype=torch.int32)
    blocks = (T + page - 1) // page + 2
    slots = torch.randperm(blocks * page, generator=g, device="cuda")[:T].to(torch.int32)
    slots[T - pad:] = -1
    q = torch.randn(T, H, D, generator=g, device="cuda").to(dt)
    kc, vc = (torch.randn(blocks, KV, page, D, generator=g, device="cuda").to(dt) for _ in range(2))
    want = ref.qkv_step(qkv, wq, wk, cos, sin, pos, slots, H, KV, D, rot, page, 1e-5, halves, q, kc, vc)
    x = ctx.wrap(qkv.data_ptr(), (flat.numel() - shift) * flat.element_size())
    torch.cuda.synchronize()
    ctx.paged_qkv(x, buf(wq), buf(wk), buf(cos) if rot else None, buf(sin) if rot else None, buf(pos) if rot else None, buf(slots), buf(q), buf(kc), buf(vc),
                  T, H, KV, D, rot, page, 1e-5, CODE[dtype], qkv_stride=stride, flags=B.FLAG_ROPE_HALVES if halves else 0)
    wq_, wkc, wvc, tq, tk = want
    assert ((q.double() - wq_).abs() <= tq).all()
    assert ((kc.double() - wkc).abs() <= tk).all()
    assert torch.equal(vc.double(), wvc)


def ctx_tables(rot, rows):
    if not rot:
        return None, None
    angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    return angle.cos().float().contiguous(), angle.sin().float().contiguous()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,H,KV,D,rot,page,halves,norm", [
    (1, 32, 8, 128, 128, 16, True, True), (5, 4, 4, 64, 64, 1, False, True), (13, 14, 2, 96, 96, 24, True, False), (3, 8, 1, 80, 40, 16, False, True),
    (4, 3, 3, 80, 20, 8, True, True), (2, 5, 1, 256, 128, 32, True, True), (2, 2, 2, 1024, 1024, 4, True, True), (3, 2, 1, 520, 6, 4, False, True),
    (3, 1, 2, 6, 4, 2, True, True), (3, 2, 2, 2, 2, 2, False, True), (4, 6, 2, 64, 0, 16, False, True), (4, 6, 2, 64, 0, 16, False, False),
    (2, 0, 3, 64, 64, 16, True, True), (70, 40, 8, 128, 64, 16, True, True)])
def test_qkv(ctx, buf, dtype, T, H, KV, D, rot, page, halves, norm):
    run_qkv(ctx, buf, dtype, T, H, KV, D, rot, page, halves, norm)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_qkv_strides_alignment_and_padding(ctx, buf, dtype):
    run_qkv(ctx, buf, dtype, 9, 4, 2, 64, 64, 16, True, True, stride=8 * 64 + 24, pad=3)
    run_qkv(ctx, buf, dtype, 9, 4, 2, 64, 64, 16, False, True, stride=8 * 64 + 3)
    run_qkv(ctx, buf, dtype, 9, 4, 2, 64, 32, 16, True, True, shift=1)
    run_qkv(ctx, buf, dtype, 9, 4, 2, 64, 32, 16, True, True, shift=2, pad=9)
    # values whose squares are small or large, but not out of range
    run_qkv(ctx, buf, dtype, 9, 4, 2, 64, 64, 16, True, True, scale=1e-3)
    run_qkv(ctx, buf, dtype, 9, 4, 2, 64, 64, 16, True, True, scale=1e4)


@pytest.mark.parametrize("dtype,H,KV,D,rot,page,halves,norm,stride,pad", [
    ("bf16", 32, 8, 128, 128, 16, True, True, 0, 0), ("f16", 4, 2, 64, 32, 16, False, True, 0, 100), ("f32", 12, 4, 80, 40, 24, False, False, 0, 7),
    ("f32", 6, 3, 256, 256, 8, True, True, 0, 0), ("bf16", 3, 1, 6, 4, 16, True, True, 0, 3), ("bf16", 4, 2, 64, 64, 16, True, True, 8 * 64 + 8, 5),
    ("f32", 90, 10, 128, 128, 16, True, True, 0, 0)])
def test_qkv_many_tokens(ctx, buf, dtype, H, KV, D, rot, page, halves, norm, stride, pad):
    run_qkv(ctx, buf, dtype, 1300, H, KV, D, rot, page, halves, norm, stride=stride, pad=pad)


def test_qkv_places_outside(ctx, buf):
    """A slot behind the cache or a position behind the tables: reported, that token left out, the others done."""
    H, KV, D, page = 4, 2, 64, 16
    cos, sin = ctx_tables(D, 10)
    qkv = torch.randn(4, (H + 2 * KV) * D, device="cuda")
    for slots, pos, status in [([0, 32, 2, 3], [1, 1, 1, 1], 0x7C050009), ([0, 2 ** 31 - 1, 2, 3], [1, 1, 1, 1], 0x7C050009),
                               ([0, 1, 2, 3], [1, 10, 1, 1], 0x7C05000A), ([0, 1, 2, 3], [1, -1, 1, 1], 0x7C05000A)]:
        q, kc, vc = torch.zeros(4, H, D, device="cuda"), torch.zeros(2, KV, page, D, device="cuda"), torch.zeros(2, KV, page, D, device="cuda")
        with pytest.raises(B.BackendError) as e:
            ctx.paged_qkv(buf(qkv), None, None, buf(cos), buf(sin), buf(ints(pos)), buf(ints(slots)), buf(q), buf(kc), buf(vc), 4, H, KV, D, D, page, 1e-5,
                          B.F32)
        assert e.value.code == B.DEVICE_LOST and ctx.last_device_status() == status
        assert q[1].abs().max() == 0 and (q[[0, 2, 3]].abs().amax((1, 2)) > 0).all()
        assert torch.equal(vc[0, :, [0, 2, 3]].transpose(0, 1), qkv[[0, 2, 3]].reshape(3, H + 2 * KV, D)[:, H + KV:])
        assert vc[0, :, 1].abs().max() == 0 and vc[1].abs().max() == 0


# ---- attention ------------------------------------------------------------------------------------------------------------------------


class Batch:
    """New tokens `new` of contexts `lens` over a paged cache whose other places hold NaN."""

    def __init__(self, dtype, H, KV, D, page, new, lens, pad=0, lead=0, seed=5, spare=2, scale=None, gain=1.0):
        self.dt, self.H, self.KV, self.D, self.page, self.new, self.lens = ref.DTYPES[dtype], H, KV, D, page, new, lens
        self.code = CODE[dtype]
        self.scale = scale if scale is not None else 1 / math.sqrt(D)
        g = torch.Generator(device="cuda").manual_seed(seed)
        held = [(max(0, n) + page - 1) // page for n in lens]
        self.width = max(held + [1]) + 1
        blocks = sum(held) + spare
        order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((len(lens), self.width), -1, dtype=torch.int32, device="cuda")
        self.kc, self.vc = (torch.full((blocks, KV, page, D), math.nan, device="cuda", dtype=self.dt) for _ in range(2))
        at = 0
        for s, n in enumerate(lens):
            n = max(0, n)
            self.table[s, :held[s]] = order[at:at + held[s]]
            at += held[s]
            k = torch.arange(n, device="cuda")
            b, off = self.table[s][k // page].long(), k % page
            for c in (self.kc, self.vc):
                c[b, :, off] = (gain * torch.randn(n, KV, D, generator=g, device="cuda")).to(self.dt)
        self.starts = [lead]
        for t in new:
            self.starts.append(self.starts[-1] + t)
        self.T = self.starts[-1] + pad
        self.q = (gain * torch.randn(self.T, H, D, generator=g, device="cuda")).to(self.dt)

    def run(self, ctx, buf, causal=True, lse=True, q=None, out=None, flags=0):
        q = self.q if q is None else q
        self.out = torch.full((self.T, self.H, self.D), 77.0, device="cuda", dtype=self.dt) if out is None else out
        self.lse = torch.full((self.T, self.H), 77.0, device="cuda") if lse else None
        need = ctx.paged_chunk_workspace(len(self.lens), self.T, self.H, self.KV, self.D, self.code)
        self.work = torch.full((need,), 255, dtype=torch.uint8, device="cuda")      # NaN wherever it is read unwritten
        self.args = [buf(q), buf(self.kc), buf(self.vc), buf(self.table), buf(ints(self.starts)), buf(ints(self.lens)), buf(self.out)]
        work, lse = buf(self.work), buf(self.lse)
        self.call = lambda f: ctx.paged_chunk_attention(*self.args, len(self.lens), self.T, self.H, self.KV, self.D, self.page, self.width, self.scale,
                                                        self.code, work, lse=lse, flags=f | (B.FLAG_ATTN_CAUSAL if causal else 0))
        self.keep = ctx, buf
        self.call(flags)

    def check(self, causal=True):
        torch.cuda.synchronize()
        out, lse, tol, ltol = ref.attention(self.q, self.kc, self.vc, self.table, self.starts, self.lens, self.scale, causal)
        mine = torch.zeros(self.T, dtype=torch.bool, device="cuda")
        mine[self.starts[0]:self.starts[-1]] = True
        assert (self.out[~mine] == 77).all()
        got, want = self.out[mine].double(), out[mine]
        assert torch.equal(got.isnan(), want.isnan())
        err = ((got - want).abs() - tol[mine]).nan_to_num(0)
        assert (err <= 0).all(), (err.max(), (err > 0).sum(), (err > 0).nonzero()[:4].tolist())
        if self.lse is not None:
            assert (self.lse[~mine] == 77).all()
            err = (self.lse[mine].double() - lse[mine]).abs() - ltol[mine]
            assert not self.lse[mine].isnan().any() and (err <= 0).all(), err.max()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,KV,D,page,new,lens", [
    (32, 8, 128, 16, [1], [300]),
    (32, 8, 128, 16, [1], [1]),
    (32, 8, 128, 16, [1, 1, 1, 1, 1], [5, 1000, 64, 65, 129]),
    (32, 8, 128, 16, [7], [7]),
    (32, 8, 128, 16, [200], [200]),
    (32, 8, 128, 32, [130, 1, 0, 33], [1000, 700, 50, 33]),
    (4, 4, 64, 16, [300, 5], [300, 400]),
    (14, 2, 64, 24, [100, 3], [500, 3]),
    (8, 1, 128, 1, [40], [90]),
    (12, 4, 96, 8, [70, 1], [130, 999]),
    (6, 2, 80, 128, [33], [257]),
    (2, 1, 256, 64, [20, 1], [150, 300]),
    (40, 1, 64, 16, [3, 9], [70, 9]),
    (128, 1, 64, 16, [5], [333]),
    (130, 1, 32, 300, [2], [310]),
    (3, 3, 37, 5, [11], [60]),
    (5, 1, 8, 4, [64, 65], [64, 165]),
])
def test_attention(ctx, buf, dtype, H, KV, D, page, new, lens):
    b = Batch(dtype, H, KV, D, page, new, lens, pad=3)
    b.run(ctx, buf)
    b.check()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention_of_long_contexts_is_cut_and_put_together(ctx, buf, dtype):
    b = Batch(dtype, 8, 2, 128, 16, [1, 70, 2], [30000, 9000, 12345])
    b.run(ctx, buf)
    b.check()
    first = b.out.clone(), b.lse.clone()
    b.run(ctx, buf)                                            # the same bits again
    assert torch.equal(b.out, first[0]) and torch.equal(b.lse, first[1])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attention_of_sequences_that_weigh_differently(ctx, buf, dtype):
    """Prompts, drafts, single tokens and sequences without new ones side by side: shares go by rows as well as by keys."""
    new = [1, 0, 5, 130, 1, 2, 0, 33, 1, 1, 64, 8, 1, 3, 257, 1]
    lens = [900, 70, 1500, 130, 64, 3, 0, 500, 1, 2000, 65, 1200, 33, 700, 400, 128]
    for H, KV in ((8, 2), (6, 6)):
        b = Batch(dtype, H, KV, 64, 16, new, lens, lead=2, pad=1)
        b.run(ctx, buf)
        b.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_of_tables_that_are_mostly_empty(ctx, buf, dtype):
    """Rows of a table that could hold 2^20 keys: the costs of such a call do not fit 32 bits, whatever the lengths are."""
    b = Batch(dtype, 32, 8, 64, 16, [1, 40, 300], [900, 40, 310])
    table = torch.full((3, 1 << 16), -1, dtype=torch.int32, device="cuda")
    table[:, :b.width] = b.table
    b.table, b.width = table, 1 << 16
    b.run(ctx, buf)
    b.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_without_causal_mask(ctx, buf, dtype):
    b = Batch(dtype, 8, 2, 64, 16, [40, 1, 7], [100, 3, 2000])
    b.run(ctx, buf, causal=False)
    b.check(causal=False)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attention_rows_without_keys(ctx, buf, dtype):
    """No context, a context below zero, and contexts shorter than the chunk: the rows that see nothing are zero."""
    b = Batch(dtype, 8, 2, 128, 16, [3, 2, 150, 20, 0, 4], [0, -5, 40, 19, 0, 4], pad=2, lead=5)
    b.run(ctx, buf)
    b.check()
    assert (b.out[5:10] == 0).all() and (b.lse[5:10] == -3.402823e38).all() and (b.out[10:120] == 0).all()
    b.run(ctx, buf, causal=False, lse=False)
    b.check(causal=False)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attention_of_what_a_row_must_not_see(ctx, buf, dtype, bad):
    """Keys and values of later tokens that are no numbers leave the earlier rows as they were; the rows that see them show it."""
    new, lens = [100, 90], [400, 90]
    b = Batch(dtype, 8, 2, 128, 16, new, lens)
    b.run(ctx, buf)
    plain = b.out.clone()
    for s, key in [(0, 350), (1, 77)]:
        blk, off = int(b.table[s, key // 16]), key % 16
        b.vc[blk, :, off, 5] = bad
        b.kc[blk, :, off, 9] = bad
    b.run(ctx, buf)
    torch.cuda.synchronize()
    for s, key in [(0, 350), (1, 77)]:
        first = b.starts[s] + key - (lens[s] - new[s])         # the first row that sees it
        rows = slice(b.starts[s], first)
        tol = ref.half_step(b.dt) * 4 if dtype != "f32" else 1e-5
        assert ((b.out[rows].float() - plain[rows].float()).abs() <= tol * (1 + plain[rows].float().abs())).all()
        after = b.out[first:b.starts[s + 1]].float()
        if math.isnan(bad):
            assert after.isnan().all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention_scores_far_apart(ctx, buf, dtype):
    """Large scores (one key takes all) and none at all (all keys alike)."""
    b = Batch(dtype, 8, 2, 128, 16, [65, 1], [600, 2000], gain=6.0)
    b.run(ctx, buf)
    b.check()
    b = Batch(dtype, 8, 2, 128, 16, [65, 1], [600, 2000], scale=0.0)
    b.run(ctx, buf)
    b.check()
    b = Batch(dtype, 8, 2, 128, 16, [65, 1], [600, 2000], scale=-0.3)
    b.run(ctx, buf)
    b.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_of_unaligned_views(ctx, buf, dtype):
    b = Batch(dtype, 8, 2, 64, 16, [20, 1], [100, 50])
    for name in ("q", "kc", "vc"):
        t = getattr(b, name)
        moved = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].reshape(t.shape)
        moved.copy_(t)
        setattr(b, name, moved)
    out = torch.full((b.T * 8 * 64 + 1,), 77.0, dtype=b.dt, device="cuda")[1:].reshape(b.T, 8, 64)
    b.run(ctx, buf, out=out)
    b.check()


def test_attention_reports_blocks_outside_the_cache(ctx, buf):
    for dtype in ("f32", "bf16"):
        for wrong in (-1, 10 ** 6, 2 ** 31 - 1):
            b = Batch(dtype, 8, 2, 64, 16, [4, 1, 3], [100, 50, 70])
            b.table[1, 2] = wrong
            with pytest.raises(B.BackendError) as e:
                b.run(ctx, buf)
            assert e.value.code == B.DEVICE_LOST and ctx.last_device_status() == 0x7C050009
            b.table[1, 2] = 0
            good = Batch(dtype, 8, 2, 64, 16, [4, 1, 3], [100, 50, 70])
            good.run(ctx, buf)                                 # the context goes on, and the other sequences were right
            good.check()
            assert torch.equal(b.out[:4], good.out[:4]) and torch.equal(b.out[5:8], good.out[5:8])


def test_attention_cuts_what_is_out_of_range(ctx, buf):
    """Starts outside the rows and a context beyond its table: cut, nothing else is read or written."""
    b = Batch("bf16", 8, 2, 64, 16, [5, 6], [64, 96], spare=0)
    b.run(ctx, buf)
    whole = b.out.clone()
    b.width = 6
    b.table = b.table[:, :6].contiguous()
    b.lens = [64, 10 ** 9]
    b.run(ctx, buf)
    assert torch.equal(b.out, whole)
    b.lens = [64, 96]
    for starts in ([0, 5, 10 ** 6], [-3, 5, 11], [0, 20, 30], [4, 2, 1]):
        b.starts = starts
        b.run(ctx, buf)
        torch.cuda.synchronize()


# ---- drafts ---------------------------------------------------------------------------------------------------------------------------


def run_verify(ctx, buf, target, draft, tokens, uniforms, starts, lens=True):
    R, V = target.shape
    n = len(starts) - 1
    out, accepted = torch.full((R,), -9, dtype=torch.int32, device="cuda"), torch.full((n,), -9, dtype=torch.int32, device="cuda")
    context = [100 + 10 * i for i in range(n)]
    kept = ints(context) if lens else None                     # in place
    ctx.verify_drafts(buf(target), buf(draft), buf(tokens), buf(uniforms), buf(ints(starts)), buf(out), buf(accepted), n, R, V, context_lens=buf(kept),
                      kept_lens=buf(kept))
    w_out, w_accepted = ref.verify(target, draft, tokens, uniforms, starts)
    assert out.tolist() == [-9 if x is None else x for x in w_out]
    assert accepted.tolist() == w_accepted
    if lens:
        assert kept.tolist() == [c - max(0, b - a - 1) + k for c, a, b, k in zip(context, starts, starts[1:], w_accepted)]


@pytest.mark.parametrize("V", [1, 7, 100, 1024, 4097, 32000, 50257])
@pytest.mark.parametrize("certain", [False, True])
def test_verify(ctx, buf, V, certain):
    g = torch.Generator(device="cuda").manual_seed(V)
    starts = [2, 3, 3, 8, 10, 45, 46]
    R = 48
    target = torch.softmax(2 * torch.randn(R, V, generator=g, device="cuda"), 1)
    draft = None if certain else torch.softmax(target.log() + 0.4 * torch.randn(R, V, generator=g, device="cuda"), 1)
    tokens = torch.multinomial(target if certain else draft, 1, generator=g)[:, 0].to(torch.int32).roll(1)
    u = torch.rand(R, generator=g, device="cuda")
    if certain:
        u *= 0.02
    run_verify(ctx, buf, target, draft, tokens, u, starts, lens=V != 7)


def test_verify_borders(ctx, buf):
    """Uniforms of 0 and almost 1, distributions with one token or zeros at the ends, equal distributions, no weight at all."""
    V = 515
    one = torch.zeros(6, V, device="cuda")
    one[:, 500] = 1.0
    flat = torch.full((6, V), 1.0 / V, device="cuda")
    ends = flat.clone()
    ends[:, :40] = 0
    ends[:, -40:] = 0
    zero = torch.zeros(6, V, device="cuda")
    odd = flat.clone()
    odd[:, 3] = math.nan
    odd[:, 4] = -1.0
    tokens = ints([0, 500, 500, 41, 600, -1])
    for p in (one, flat, ends, zero, odd):
        for q in (None, one, flat, ends, zero):
            for u in (0.0, 0.5, 1 - 2.0 ** -24):
                run_verify(ctx, buf, p, q, tokens, torch.full((6,), u, device="cuda"), [0, 6])
                run_verify(ctx, buf, p, q, tokens, torch.full((6,), u, device="cuda"), [0, 1, 4, 6])


@pytest.mark.parametrize("V", [600000, 600001])
def test_verify_large_vocabulary(ctx, buf, V):
    """Several vectors, or elements, of the drawn segment to a thread; weights at the segments' borders only too."""
    g = torch.Generator(device="cuda").manual_seed(V)
    target = torch.softmax(torch.randn(5, V, generator=g, device="cuda"), 1)
    draft = torch.softmax(target.log() + torch.randn(5, V, generator=g, device="cuda"), 1)
    few = torch.zeros(5, V, device="cuda")
    few[:, [0, 75000 - 1, 75000, 84375, V - 1]] = 0.2
    for u in (0.0, 0.3, 0.999):
        us = torch.full((5,), u, device="cuda")
        run_verify(ctx, buf, target, draft, ints([5, V - 1, 3, 7, 1]), us, [0, 3, 5])
        run_verify(ctx, buf, few, None, ints([5, 75000, 3, V - 1, 1]), us, [0, 2, 3, 5])


def test_verify_unaligned(ctx, buf):
    g = torch.Generator(device="cuda").manual_seed(1)
    both = torch.softmax(torch.randn(2, 3, 64, generator=g, device="cuda"), 2)
    flat = torch.empty(2, 3 * 64 + 1, device="cuda")
    flat[:, 1:] = both.reshape(2, -1)
    t, d = flat[0, 1:].reshape(3, 64), flat[1, 1:].reshape(3, 64)
    run_verify(ctx, buf, t, d, ints([1, 2, 3]), torch.rand(3, device="cuda"), [0, 3])


# ---- the operators as a host uses them --------------------------------------------------------------------------------------------------


class Server:
    """Two layers of a serving host over a paged cache: lengths and blocks live on the device, a step is enqueued without a wait."""

    def __init__(self, ctx, buf, dtype, seqs, most, H=8, KV=2, D=64, page=16, width=12, layers=2, V=211):
        self.ctx, self.buf, self.dtype, self.seqs, self.most = ctx, buf, dtype, seqs, most
        self.H, self.KV, self.D, self.page, self.width, self.layers, self.V = H, KV, D, page, width, layers, V
        self.dt, self.code = ref.DTYPES[dtype], CODE[dtype]
        g = torch.Generator(device="cuda").manual_seed(17)
        blocks = seqs * width
        self.table = torch.full((seqs, width), -1, dtype=torch.int32, device="cuda")
        self.free = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
        self.count = ints([blocks])
        self.lens, self.new, self.total = (torch.zeros(seqs, dtype=torch.int32, device="cuda") for _ in range(3))
        self.starts = torch.zeros(seqs + 1, dtype=torch.int32, device="cuda")
        self.pos, self.slots, self.out_tokens = (torch.zeros(most, dtype=torch.int32, device="cuda") for _ in range(3))
        self.accepted = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        self.tokens = torch.zeros(most, dtype=torch.int32, device="cuda")
        self.u = torch.zeros(most, device="cuda")
        self.p, self.qd = torch.zeros(most, V, device="cuda"), torch.zeros(most, V, device="cuda")
        self.cos, self.sin = ctx_tables(D, 400)
        self.wq, self.wk = 1 + 0.2 * torch.randn(D, generator=g, device="cuda"), 1 + 0.2 * torch.randn(D, generator=g, device="cuda")
        self.qkv = [torch.zeros(most, (H + 2 * KV) * D, dtype=self.dt, device="cuda") for _ in range(layers)]
        self.q = [torch.zeros(most, H, D, dtype=self.dt, device="cuda") for _ in range(layers)]
        self.out = [torch.zeros(most, H, D, dtype=self.dt, device="cuda") for _ in range(layers)]
        self.kc, self.vc = ([torch.full((blocks, KV, page, D), math.nan, dtype=self.dt, device="cuda") for _ in range(layers)] for _ in range(2))
        self.work = torch.empty(ctx.paged_chunk_workspace(seqs, most, H, KV, D, self.code), dtype=torch.uint8, device="cuda")
        self.b = {k: ([buf(x) for x in v] if isinstance(v, list) else buf(v)) for k, v in vars(self).items()
                  if torch.is_tensor(v) or (isinstance(v, list) and v and torch.is_tensor(v[0]))}

    def step(self, flags):
        c, b = self.ctx, self.b
        c.paged_reserve(b["lens"], b["new"], b["table"], b["free"], b["count"], b["starts"], b["total"], b["pos"], b["slots"], self.seqs, self.width,
                        self.page, self.most, flags=flags)
        for i in range(self.layers):
            c.paged_qkv(b["qkv"][i], b["wq"], b["wk"], b["cos"], b["sin"], b["pos"], b["slots"], b["q"][i], b["kc"][i], b["vc"][i], self.most, self.H,
                        self.KV, self.D, self.D, self.page, 1e-5, self.code, flags=flags | B.FLAG_ROPE_HALVES)
            c.paged_chunk_attention(b["q"][i], b["kc"][i], b["vc"][i], b["table"], b["starts"], b["total"], b["out"][i], self.seqs, self.most, self.H,
                                    self.KV, self.D, self.page, self.width, 1 / math.sqrt(self.D), self.code, b["work"], flags=flags | B.FLAG_ATTN_CAUSAL)
        c.verify_drafts(b["p"], b["qd"], b["tokens"], b["u"], b["starts"], b["out_tokens"], b["accepted"], self.seqs, self.most, self.V,
                        context_lens=b["total"], kept_lens=b["lens"], flags=flags)
        c.paged_release(b["lens"], b["table"], b["free"], b["count"], self.seqs, self.width, self.page, flags=flags)

    def load(self, g, new):
        """The next step's inputs, in place."""
        self.new.copy_(ints(new))
        logits = 2 * torch.randn(self.most, self.V, generator=g, device="cuda")
        self.p.copy_(torch.softmax(logits, 1))
        self.qd.copy_(torch.softmax(logits + 0.5 * torch.randn(self.most, self.V, generator=g, device="cuda"), 1))
        self.tokens.copy_(torch.multinomial(self.qd, 1, generator=g)[:, 0].to(torch.int32).roll(1))
        self.u.copy_(torch.rand(self.most, generator=g, device="cuda"))
        for x in self.qkv:
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))

    def expect(self, before, new):
        """What the step that has just run has to have left, from the state before it."""
        lens, table, free, count, kc, vc = before
        starts, total, pos, slots, table, count = ref.plan(lens.tolist(), new, table.tolist(), free.tolist(), int(count), self.page, self.most)
        assert self.starts.tolist() == starts and self.pos.tolist() == pos and self.slots.tolist() == slots and self.total.tolist() == total
        n = starts[-1]
        for i in range(self.layers):
            q, k, v, tq, tk = ref.qkv_step(self.qkv[i], self.wq, self.wk, self.cos, self.sin, self.pos, self.slots, self.H, self.KV, self.D, self.D,
                                           self.page, 1e-5, True, self.q[i], kc[i], vc[i])
            assert ((self.q[i].double() - q).abs() <= tq).all()
            assert ((self.kc[i].double() - k).abs() <= tk).logical_or(k.isnan()).all() and torch.equal(self.vc[i].double().nan_to_num(7), v.nan_to_num(7))
            out, _, tol, _ = ref.attention(self.q[i], self.kc[i], self.vc[i], ints(table), starts, total, 1 / math.sqrt(self.D), True)
            assert ((self.out[i][:n].double() - out[:n]).abs() <= tol[:n]).all()
        tokens, accepted = ref.verify(self.p, self.qd, self.tokens, self.u, starts)
        assert self.out_tokens.tolist()[:n] == tokens[:n] and self.accepted.tolist() == accepted
        kept = [t - max(0, d - 1) + a for t, d, a in zip(total, new, accepted)]
        assert self.lens.tolist() == kept
        table, free, count = ref.release(kept, table, free.tolist(), count, self.page)
        assert self.table.tolist() == table and self.free.tolist() == free and int(self.count) == count

    def state(self):
        return self.lens.clone(), self.table.clone(), self.free.clone(), self.count.clone(), [x.clone() for x in self.kc], [x.clone() for x in self.vc]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("captured", [False, True])
def test_serving_steps(backend, dtype, captured):
    """Steps of a serving host on a stream of its own: prompts in pieces, drafts, single tokens and waiting sequences, every operator enqueued without
    a wait; captured once and replayed with other lengths."""
    ctx = backend.create_context(0)
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    try:
        s = Server(ctx, Bufs(ctx), dtype, 5, 90)
        g = torch.Generator(device="cuda").manual_seed(23)
        graph = None
        if captured:
            s.load(g, [1, 1, 1, 1, 1])
            state = s.state()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                s.step(B.FLAG_NO_SYNC)
            assert torch.equal(s.table, state[1]) and int(s.count) == int(state[3])      # a capture runs nothing
        for new in [[40, 3, 0, 20, 25], [5, 5, 5, 5, 5], [1, 1, 30, 1, 1], [4, 0, 1, 50, 6], [1, 1, 1, 1, 1], [6, 5, 4, 3, 2]]:
            s.load(g, new)
            before = s.state()
            torch.cuda.synchronize()
            if graph is not None:
                graph.replay()
            else:
                s.step(B.FLAG_NO_SYNC)
            ctx.sync()
            torch.cuda.synchronize()
            s.expect(before, new)
        s.new.zero_()
        torch.cuda.synchronize()
        s.lens.zero_()
        torch.cuda.synchronize()
        ctx.paged_release(s.b["lens"], s.b["table"], s.b["free"], s.b["count"], 5, s.width, s.page)
        assert int(s.count) == 5 * s.width
        del graph
    finally:
        ctx.destroy()


def test_two_captured_calls_at_a_time(backend):
    """Two graphs of chunk attention, each with its workspace, replayed on two streams at once."""
    jobs = []
    for i, new in enumerate([[1, 200, 3], [130, 1, 1]]):
        ctx = backend.create_context(0)
        stream = torch.cuda.Stream()
        ctx.set_stream(stream.cuda_stream)
        b = Batch("bf16", 8, 2, 128, 16, new, [9000, 5000, 700], seed=40 + i)
        b.run(ctx, Bufs(ctx))
        torch.cuda.synchronize()
        want = b.out.clone(), b.lse.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            b.call(B.FLAG_NO_SYNC)
        jobs.append((ctx, stream, b, graph, want))
    for _ in range(5):
        for _, _, b, _, _ in jobs:
            b.out.zero_()
            b.lse.zero_()
        torch.cuda.synchronize()
        for _, stream, _, graph, _ in jobs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, _, b, _, want in jobs:
            assert torch.equal(b.out, want[0]) and torch.equal(b.lse, want[1])
    del graph
    for i, job in enumerate(jobs):
        ctx = job[0]
        jobs[i] = None
        del job
        ctx.destroy()


def test_many_chunk_calls_in_a_row(ctx, buf):
    """Hundreds of calls enqueued without a wait, each starting on the last one's end, over items of all kinds: the same bits every time."""
    b = Batch("f16", 8, 2, 128, 16, [1] * 12 + [70, 1, 5, 33], [3000 - 170 * i for i in range(12)] + [900, 64, 65, 400])
    b.run(ctx, buf)
    want = b.out.clone(), b.lse.clone()
    torch.cuda.synchronize()
    for _ in range(300):
        b.call(B.FLAG_NO_SYNC)
    ctx.sync()
    assert torch.equal(b.out, want[0]) and torch.equal(b.lse, want[1])
