"""What the operators of a paged KV cache refuse, on the CPU: arguments are checked before anything touches a device, so a
context of zeros and buffers of made-up addresses are enough."""
import ctypes as C

import pytest

from webgpu_b200 import backend as B

BAD, NO = B.INVALID_ARGUMENT, B.NOT_SUPPORTED
BIG = 1 << 40


@pytest.fixture(scope="module")
def fake(backend):
    """A context (all zeros) and a maker of buffers: nothing behind their addresses is ever read."""
    memory = C.create_string_buffer(1 << 16)
    ctx = C.addressof(memory)
    made = []

    def buf(nbytes=BIG, at=1 << 20):
        h = backend.lib.lux_cuda_buffer_wrap(ctx, at, nbytes)
        made.append(h)
        return h

    yield backend.lib, ctx, buf, memory
    for h in made:
        backend.vt["buffer_free"](ctx, h)


def call(fn, names, good, **change):
    args = dict(good)
    assert set(change) <= set(names), change
    args.update(change)
    return fn(*[args[n] for n in names])


def test_reserve_and_release(fake):
    lib, ctx, buf, _ = fake
    names = ["ctx", "cached", "new", "table", "free", "count", "starts", "lens", "pos", "slots", "seqs", "width", "page", "tokens", "flags"]
    good = dict(ctx=ctx, cached=buf(40), new=buf(40), table=buf(10 * 7 * 4), free=buf(400), count=buf(4), starts=buf(44), lens=buf(40), pos=buf(80),
                slots=buf(80), seqs=10, width=7, page=16, tokens=20, flags=1)

    def refused(**k):
        assert call(lib.lux_cuda_paged_reserve, names, good, **k) == BAD, k

    refused(ctx=None)
    for n in ("cached", "new", "table", "free", "count", "starts", "lens", "pos", "slots"):
        refused(**{n: None})
        if n != "free":
            refused(**{n: buf(36 if n in ("cached", "new", "lens") else {"table": 276, "count": 3, "starts": 40}.get(n, 76))})
        refused(**{n: buf(at=(1 << 20) + 2)})
    refused(width=0)
    refused(page=0)
    refused(seqs=8193)
    refused(tokens=1 << 31)
    refused(table=buf(), width=1 << 20, page=1 << 11)          # a position would pass 31 bits

    names = ["ctx", "keep", "table", "free", "count", "seqs", "width", "page", "flags"]
    good = dict(ctx=ctx, keep=buf(40), table=buf(10 * 7 * 4), free=buf(400), count=buf(4), seqs=10, width=7, page=16, flags=1)
    for k in [dict(ctx=None), dict(keep=None), dict(keep=buf(36)), dict(table=buf(276)), dict(free=None), dict(count=buf(0)), dict(seqs=8193),
              dict(width=0), dict(page=0)]:
        assert call(lib.lux_cuda_paged_release, names, good, **k) == BAD, k


def test_qkv(fake):
    lib, ctx, buf, _ = fake
    names = ["ctx", "qkv", "wq", "wk", "cos", "sin", "pos", "slots", "q", "kc", "vc", "tokens", "stride", "heads", "kv", "dim", "rot", "page", "eps",
             "dtype", "flags"]
    good = dict(ctx=ctx, qkv=buf(5 * 8 * 64 * 2), wq=buf(256), wk=buf(256), cos=buf(), sin=buf(), pos=buf(20), slots=buf(20), q=buf(5 * 4 * 64 * 2),
                kc=buf(2 * 16 * 64 * 2), vc=buf(2 * 16 * 64 * 2), tokens=5, stride=0, heads=4, kv=2, dim=64, rot=64, page=16, eps=1e-6, dtype=B.F16,
                flags=1)

    def refused(**k):
        assert call(lib.lux_cuda_paged_qkv, names, good, **k) == BAD, k

    for n in ("ctx", "qkv", "wq", "wk", "cos", "sin", "pos", "slots", "q", "kc", "vc"):
        refused(**{n: None})
    refused(qkv=buf(5 * 8 * 64 * 2 - 2))
    refused(stride=511)
    refused(stride=600)                                        # the last row would pass the end
    refused(wk=buf(252))
    refused(cos=buf(124))
    refused(slots=buf(16))
    refused(pos=buf(16))
    refused(q=buf(5 * 4 * 64 * 2 - 2))
    refused(kc=buf(2 * 16 * 64 * 2 - 2))                       # not one block
    refused(kc=buf(at=(1 << 20) + 1))
    refused(dtype=3)
    refused(dim=0)
    refused(dim=63, rot=62)
    refused(rot=65)
    refused(rot=66)
    refused(rot=33)
    refused(dim=1026, rot=64, qkv=buf(), q=buf(), kc=buf(), vc=buf())
    refused(page=0)
    refused(heads=0, kv=0)
    refused(tokens=1 << 31, qkv=buf(1 << 60))
    refused(heads=0xffffffff, kv=0xffffffff, qkv=buf(1 << 60))


def test_chunk_attention(fake):
    lib, ctx, buf, _ = fake
    names = ["ctx", "q", "kc", "vc", "table", "starts", "lens", "out", "lse", "work", "seqs", "tokens", "heads", "kv", "dim", "page", "width", "scale",
             "dtype", "flags"]
    good = dict(ctx=ctx, q=buf(6 * 8 * 64 * 2), kc=buf(2 * 16 * 64 * 2), vc=buf(2 * 16 * 64 * 2), table=buf(3 * 5 * 4), starts=buf(16), lens=buf(12),
                out=buf(6 * 8 * 64 * 2), lse=buf(6 * 8 * 4), work=buf(), seqs=3, tokens=6, heads=8, kv=2, dim=64, page=16, width=5, scale=0.125,
                dtype=B.BF16, flags=1)

    def refused(code=BAD, **k):
        assert call(lib.lux_cuda_paged_chunk_attention, names, good, **k) == code, k

    for n in ("ctx", "q", "kc", "vc", "table", "starts", "lens", "out", "work"):
        refused(**{n: None})
    refused(q=buf(6 * 8 * 64 * 2 - 2))
    refused(out=buf(6 * 8 * 64 * 2 - 2))
    refused(vc=buf(2 * 16 * 64 * 2 - 2))
    refused(table=buf(56))
    refused(starts=buf(12))
    refused(lens=buf(8))
    refused(lse=buf(6 * 8 * 4 - 4))
    refused(work=buf(at=(1 << 20) + 8))
    refused(work=buf(8))
    refused(q=buf(at=(1 << 20) + 1))
    refused(heads=9)
    refused(heads=0)
    refused(kv=0)
    refused(dim=0)
    refused(page=0)
    refused(width=0)
    refused(dtype=7)
    refused(width=1 << 20, page=1 << 11, table=buf(), kc=buf(), vc=buf())
    refused(tokens=1 << 29, q=buf(1 << 60), out=buf(1 << 60), lse=None)
    refused(NO, dim=260, q=buf(), out=buf(), kc=buf(), vc=buf())
    size = lib.lux_cuda_paged_chunk_workspace
    assert size(ctx, 3, 6, 9, 2, 64, B.BF16) == 0 and size(ctx, 3, 6, 8, 2, 264, B.BF16) == 0 and size(ctx, 3, 6, 8, 2, 64, 3) == 0
    assert size(None, 3, 6, 8, 2, 64, B.BF16) == 0


def test_verify(fake):
    lib, ctx, buf, _ = fake
    names = ["ctx", "p", "q", "tokens", "u", "starts", "out", "accepted", "lens", "kept", "seqs", "rows", "vocab", "flags"]
    good = dict(ctx=ctx, p=buf(7 * 33 * 4), q=buf(7 * 33 * 4), tokens=buf(28), u=buf(28), starts=buf(16), out=buf(28), accepted=buf(12), lens=buf(12),
                kept=buf(12), seqs=3, rows=7, vocab=33, flags=1)

    def refused(**k):
        assert call(lib.lux_cuda_verify_drafts, names, good, **k) == BAD, k

    for n in ("ctx", "p", "tokens", "u", "starts", "out", "accepted", "lens", "kept"):
        refused(**{n: None})
    refused(p=buf(7 * 33 * 4 - 4))
    refused(q=buf(7 * 33 * 4 - 4))
    refused(tokens=buf(24))
    refused(u=buf(24))
    refused(starts=buf(12))
    refused(out=buf(24))
    refused(accepted=buf(8))
    refused(lens=buf(8))
    refused(kept=buf(8))
    refused(vocab=0)
    refused(rows=1 << 31, p=buf(1 << 60), q=None)
    refused(seqs=1 << 30)
