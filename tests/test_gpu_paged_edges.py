"""Edges of the operators of a paged KV cache (lux/gpu/paged_ext.h): what lies beside a sequence's last key, faults that meet in one wait, rows of
many heads, block numbers out of range."""
import math
import random
import threading
import time

import pytest
import torch

import paged_reference as ref
from test_gpu_paged import Batch, Bufs, Pool, buf, ctx_tables, ints, run_verify  # noqa: F401  (buf is a fixture)
from webgpu_b200 import backend as B

pytestmark = pytest.mark.gpu


# ---- attention: values behind the last key ----------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D,page", [(128, 1), (128, 2), (128, 4), (128, 5), (128, 8), (128, 12), (128, 16), (128, 24), (128, 64), (64, 1), (64, 8), (64, 24)])
def test_attention_bits_do_not_depend_on_what_was_there_before(ctx, buf, dtype, D, page):
    """Sequences that end anywhere in a key tile, behind others whose values are no numbers: what an earlier tile (or call) left in shared memory
    behind the last key takes no part, so that the outputs are those of a call without it, bit for bit."""
    ends = [1, 8, 24, 40, 56, 1000, 9, 33, 64, 90, 108, 130, 186, 300]
    lens = [n for e in ends for n in (700, e)] * 4             # every other one is to be spoiled; several items to a CTA
    b = Batch(dtype, 8, 8, D, page, [1] * len(lens), lens)
    b.run(ctx, buf)
    b.check()
    want = b.out[1::2].clone(), b.lse[1::2].clone()
    for s in range(0, len(lens), 2):
        for at in b.table[s].tolist():
            if at >= 0:
                b.vc[at] = math.nan
    for _ in range(2):                                         # (the second time every CTA's ring has seen them)
        b.run(ctx, buf)
        torch.cuda.synchronize()
        assert b.out[::2].isnan().all()
        assert torch.equal(b.out[1::2], want[0]) and torch.equal(b.lse[1::2], want[1])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("H,KV,D,page,new,lens", [(8, 2, 128, 16, [1, 1], [70000, 40]), (8, 2, 64, 24, [70, 1], [3000, 20000]), (6, 2, 96, 8, [3, 65], [999, 700]),
                                                  (3, 1, 8, 16, [200], [1500]), (40, 1, 40, 5, [9], [3000])])
def test_attention_of_a_value_that_all_rows_see_and_is_no_number(ctx, buf, dtype, H, KV, D, page, new, lens):
    """One element of the first key's value is NaN: that column of every row is, and the others are as they were."""
    b = Batch(dtype, H, KV, D, page, new, lens)
    b.run(ctx, buf)
    plain, lse = b.out.clone(), b.lse.clone()
    for s in range(len(lens)):
        b.vc[int(b.table[s, 0]), :, 0, D - 3] = math.nan
    b.run(ctx, buf)
    torch.cuda.synchronize()
    assert b.out[:, :, D - 3].isnan().all() and torch.equal(b.lse, lse)
    rest = [c for c in range(D) if c != D - 3]
    clean = Batch(dtype, H, KV, D, page, new, lens)
    want, _, tol, _ = ref.attention(clean.q, clean.kc, clean.vc, clean.table, clean.starts, clean.lens, clean.scale, True)
    for out in (plain, b.out):
        assert ((out.double() - want).abs() <= tol)[:, :, rest].all()


def test_attention_of_such_values_takes_little_longer(ctx, buf):
    """A NaN that every row sees costs the rows once more, by whole warps (7 ms); a thread per row took 42 ms."""
    b = Batch("bf16", 32, 8, 128, 16, [256], [8192])
    b.vc[int(b.table[0, 0]), :, 0, 5] = math.nan
    b.run(ctx, buf)
    times = []
    for _ in range(5):
        torch.cuda.synchronize()
        t = time.perf_counter()
        b.call(0)
        times.append(time.perf_counter() - t)
    assert min(times) < 0.02, times


# ---- what only the device can see ---------------------------------------------------------------------------------------------------------


def test_several_faults_between_two_waits(ctx, buf):
    """A slot outside the cache and a position outside the tables in one call, and calls that each meet another fault without a wait in between:
    the status is that of a fault that was there, of the first call's where they run one after the other."""
    H, KV, D, page = 4, 2, 64, 16
    cos, sin = ctx_tables(D, 10)
    qkv = torch.randn(4, (H + 2 * KV) * D, device="cuda")
    q, kc, vc = torch.zeros(4, H, D, device="cuda"), torch.zeros(2, KV, page, D, device="cuda"), torch.zeros(2, KV, page, D, device="cuda")

    def step(slots, pos, flags=0):
        ctx.paged_qkv(buf(qkv), None, None, buf(cos), buf(sin), buf(ints(pos)), buf(ints(slots)), buf(q), buf(kc), buf(vc), 4, H, KV, D, D, page, 1e-5,
                      B.F32, flags=flags)

    def release(count):                                        # a list whose count is none of it
        ctx.paged_release(buf(ints([0])), buf(ints([-1])), buf(ints([0, 0])), buf(ints([count])), 1, 1, page, flags=B.FLAG_NO_SYNC)

    with pytest.raises(B.BackendError) as e:
        step([0, 32, 2, 3], [1, 1, 10, 1])
    assert e.value.code == B.DEVICE_LOST and ctx.last_device_status() in (0x7C050009, 0x7C05000A)
    good, slot, place = ([0, 1, 2, 3], [1, 1, 1, 1]), ([0, 32, 2, 3], [1, 1, 1, 1]), ([0, 1, 2, 3], [1, 1, 10, 1])
    for first, second, status in [(slot, place, 0x7C050009), (place, slot, 0x7C05000A), (good, slot, 0x7C050009)]:
        step(*first, flags=B.FLAG_NO_SYNC)
        step(*second, flags=B.FLAG_NO_SYNC)
        release(-1)
        with pytest.raises(B.BackendError):
            step(*good)
        assert ctx.last_device_status() == status
    release(3)
    step(*slot, flags=B.FLAG_NO_SYNC)
    with pytest.raises(B.BackendError):
        step(*good)
    assert ctx.last_device_status() == 0x7C05000B
    step(*good)                                                # and the context goes on
    assert ctx.last_device_status() == 0


@pytest.mark.parametrize("tokens", [9, 4000])
@pytest.mark.parametrize("page,block", [(16, 2 ** 28), (16, 2 ** 27), (16, 2 ** 28 + 3), (24, 2 ** 31 // 24 + 1), (2, 2 ** 30), (1, -7), (16, -1)])
def test_reserve_of_block_numbers_that_have_no_slots(ctx, buf, tokens, page, block):
    """A number from the free list, or one that the table holds, whose slots do not fit 31 bits: reported, and no slot of another block comes out."""
    def reserve(table, free, cached, new):
        t, f, count, starts, lens = ints(table), ints(free), ints([len(free)]), ints([0] * (len(new) + 1)), ints([0] * len(new))
        pos, slots = ints([-7] * tokens), ints([-7] * tokens)
        failed = False
        try:
            ctx.paged_reserve(buf(ints(cached)), buf(ints(new)), buf(t), buf(f), buf(count), buf(starts), buf(lens), buf(pos), buf(slots), len(new),
                              len(table[0]), page, tokens)
        except B.BackendError as e:
            assert e.code == B.DEVICE_LOST and ctx.last_device_status() == 0x7C050009
            failed = True
        return failed, pos.tolist(), slots.tolist(), int(count)

    # sequence 0 gets block 5, sequence 1 the bad one, sequence 2 block 3
    failed, pos, slots, count = reserve([[-1, -1]] * 3, [9, 3, block, 5], [0, 0, 0], [1, 1, 1])
    assert failed and pos[:3] == [0, 0, 0] and slots[:3] == [5 * page, -1, 3 * page] and slots[3:] == [-1] * (tokens - 3) and count == 1
    if block >= 0:                                             # (an entry below 0 is an empty one)
        failed, pos, slots, count = reserve([[block, -1], [4, -1]], [9], [0, 0], [1, 1])
        assert failed and slots[:2] == [-1, 4 * page] and count == 1
    failed, _, slots, _ = reserve([[-1, -1]], [(2 ** 31 - 1) // page - 1], [0], [1])     # the last number that has slots
    assert not failed and slots[0] == ((2 ** 31 - 1) // page - 1) * page


# ---- qkv: rings of different sizes ---------------------------------------------------------------------------------------------------------


def qkv_job(ctx, buf, H, KV, T=40, D=128, page=16):
    """A call of bf16 rows of H + 2 KV heads, and what it has to leave."""
    g = torch.Generator(device="cuda").manual_seed(H)
    qkv = torch.randn(T, (H + 2 * KV) * D, generator=g, device="cuda").bfloat16()
    q, kc, vc = torch.zeros(T, H, D, device="cuda").bfloat16(), *(torch.zeros(3, KV, page, D, device="cuda").bfloat16() for _ in range(2))
    held = [buf(x) for x in (qkv, ints(list(range(T))), q, kc, vc)]

    def call(flags=0):
        ctx.paged_qkv(held[0], None, None, None, None, None, *held[1:], T, H, KV, D, 0, page, 1e-5, B.BF16, flags=flags)

    call.held = buf                                            # (and the memory of what it wraps)

    def check():
        x = qkv.reshape(T, H + 2 * KV, D)
        assert torch.equal(q, x[:, :H])
        for cache, first in ((kc, H), (vc, H + KV)):
            assert torch.equal(cache.transpose(1, 2).reshape(3 * page, KV, D)[:T], x[:, first:first + KV])
        for t in (q, kc, vc):
            t.zero_()
        torch.cuda.synchronize()

    return call, check


def test_qkv_rows_of_many_heads_on_two_threads(backend):
    """Rows of 45 KB and of 21 KB, both of which need more shared memory than is open as it is, from two threads with a context each."""
    failed = []

    def work(H, KV):
        try:
            torch.cuda.set_device(0)
            mine = backend.create_context(0)
            call, check = qkv_job(mine, Bufs(mine), H, KV)
            for _ in range(2000):
                call(B.FLAG_NO_SYNC)
            mine.sync()
            check()
            mine.destroy()
        except Exception as e:                                 # noqa: BLE001  (told to the test's own thread)
            failed.append(repr(e))

    threads = [threading.Thread(target=work, args=a) for a in ((160, 8), (64, 8), (150, 10))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


def test_qkv_captured_before_a_call_of_smaller_rows(backend):
    """A graph of rows of 45 KB is instantiated and replayed after calls of rows of 21 KB."""
    mine = backend.create_context(0)
    stream = torch.cuda.Stream()
    mine.set_stream(stream.cuda_stream)
    large, check_large = qkv_job(mine, Bufs(mine), 160, 8)
    small, check_small = qkv_job(mine, Bufs(mine), 64, 8)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        large(B.FLAG_NO_SYNC)
        small(B.FLAG_NO_SYNC)
        large(B.FLAG_NO_SYNC)
    for _ in range(3):
        small()
        check_small()
        graph.replay()
        torch.cuda.synchronize()
        check_large()
        check_small()
    del graph
    mine.destroy()


# ---- offsets beyond 32 bits ------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_and_qkv_at_the_end_of_a_large_cache(ctx, buf, dtype):
    """Blocks behind the first 2^31 elements: attention reads them (a value that is no number among them, too), qkv writes them."""
    H, KV, D, page = 8, 2, 128, 16
    dt = ref.DTYPES[dtype]
    b = Batch(dtype, H, KV, D, page, [70, 1], [300, 1500])
    blocks, used = (1 << 31) // (KV * page * D) + 50, b.kc.shape[0]
    assert blocks * KV * page * D > 1 << 31 and used <= 150
    large = [torch.empty(blocks + used, KV, page, D, device="cuda", dtype=dt) for _ in range(2)]
    small = b.kc, b.vc, b.table
    for c, s in zip(large, small):
        c[:used] = math.nan                                    # where an offset that wraps would lead
        c[blocks:] = s
    b.kc, b.vc = large
    b.table = torch.where(b.table >= 0, b.table + blocks, b.table)
    b.run(ctx, buf)
    b.check()
    plain = b.out.clone()
    at = int(b.table[0, (300 - 20) // page])                   # a new token's value: the rows in front of it are done again, to rounding
    b.vc[at, :, (300 - 20) % page, 3] = math.nan
    b.run(ctx, buf)
    torch.cuda.synchronize()
    tol = ref.half_step(dt) * 4 if dtype != "f32" else 1e-5
    assert ((b.out[:50].float() - plain[:50].float()).abs() <= tol * (1 + plain[:50].float().abs())).all() and b.out[50:70, :, 3].isnan().all()
    T = 5
    qkv = torch.randn(T, (H + 2 * KV) * D, device="cuda").to(dt)
    slots = [(blocks + i) * page + 3 * i for i in range(T)]
    q = torch.zeros(T, H, D, device="cuda").to(dt)
    ctx.paged_qkv(buf(qkv), None, None, None, None, None, buf(ints(slots)), buf(q), buf(large[0]), buf(large[1]), T, H, KV, D, 0, page, 1e-5, b.code)
    x = qkv.reshape(T, H + 2 * KV, D)
    for i, s in enumerate(slots):
        assert torch.equal(large[0][s // page, :, s % page], x[i, H:H + KV]) and torch.equal(large[1][s // page, :, s % page], x[i, H + KV:])
    assert torch.equal(q, x[:, :H]) and large[0][:used].isnan().all()


def test_verify_of_many_rows(ctx, buf):
    """The last sequence's rows lie behind the first 2^31 elements."""
    V = 128256
    R = (1 << 31) // V + 40
    target = torch.zeros(R, V, device="cuda")
    starts = [0, R - 4, R - 1]
    g = torch.Generator(device="cuda").manual_seed(3)
    target[R - 4:] = torch.softmax(torch.randn(4, V, generator=g, device="cuda"), 1)
    target[0, 7] = 1.0
    tokens = torch.zeros(R, dtype=torch.int32, device="cuda")
    tokens[1], tokens[R - 3], tokens[R - 2] = 7, 11, 12
    u = torch.zeros(R, device="cuda")
    u[R - 2], u[R - 5] = 0.37, 0.5
    out, accepted = torch.full((R,), -9, dtype=torch.int32, device="cuda"), ints([0, 0])
    ctx.verify_drafts(buf(target), None, buf(tokens), buf(u), buf(ints(starts)), buf(out), buf(accepted), 2, R, V)
    # sequence 0: its draft 7 stands, then a token of row 1, which has no weight; sequence 1: both drafts stand (a uniform of 0), then a drawn one
    assert accepted.tolist() == [1, 2] and out[:3].tolist() == [7, -1, -1] and out[R - 4:R - 2].tolist() == [11, 12]
    w = target[R - 2].double().cpu()
    assert int(out[R - 2]) == int((w.cumsum(0) <= float(u[R - 2]) * w.sum()).sum())


# ---- many sequences --------------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("wide", [False, True])
def test_attention_of_more_sequences_than_a_cta_has_threads(ctx, buf, dtype, wide):
    """Shares of 1300 sequences, which a CTA sums in several rounds; `wide`: with tables so long that their costs do not fit 32 bits."""
    rng = random.Random(11)
    new = [rng.choice([0, 1, 1, 1, 1, 2, 5]) for _ in range(1300)]
    lens = [t + rng.choice([0, 3, 40, 64, 200]) for t in new]
    new[3], lens[3], new[900], lens[900], new[1299], lens[1299] = 70, 900, 40, 2500, 3, 700
    b = Batch(dtype, 4, 2, 64, 16, new, lens, pad=1)
    if wide:
        table = torch.full((1300, 1 << 15), -1, dtype=torch.int32, device="cuda")
        table[:, :b.width] = b.table
        b.table, b.width = table, 1 << 15
    b.run(ctx, buf)
    b.check()


def test_plan_of_as_many_sequences_as_there_may_be(ctx, buf):
    pool = Pool(8192, 3, 4, 8192 * 3)
    rng = random.Random(5)
    new = [rng.randint(0, 7) for _ in range(8192)]
    total = pool.reserve(ctx, buf, [0] * 8192, new, sum(new) + 3)
    assert total == new
    more = [rng.randint(0, 12 - n) for n in total]
    total = pool.reserve(ctx, buf, total, more, sum(more))
    pool.release(ctx, buf, [rng.choice([-1, 0, n, max(0, n - 3)]) for n in total])
    pool.release(ctx, buf, [0] * 8192)
    assert int(pool.count) == 8192 * 3


def test_verify_of_many_sequences(ctx, buf):
    g = torch.Generator(device="cuda").manual_seed(8)
    rng = random.Random(8)
    starts = [0]
    for _ in range(1500):
        starts.append(starts[-1] + rng.choice([0, 1, 2, 4]))
    R = starts[-1]
    target = torch.softmax(2 * torch.randn(R, 37, generator=g, device="cuda"), 1)
    draft = torch.softmax(target.log() + 0.5 * torch.randn(R, 37, generator=g, device="cuda"), 1)
    tokens = torch.multinomial(draft, 1, generator=g)[:, 0].to(torch.int32).roll(1)
    run_verify(ctx, buf, target, draft, tokens, torch.rand(R, generator=g, device="cuda"), starts)
