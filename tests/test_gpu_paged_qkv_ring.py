"""qkv of a paged cache (lux_cuda_paged_qkv) where a CTA takes token after token from its ring of rows: every place of the ring is filled several times,
beside padding and faults, for rings of two to four rows, of more shared memory than is open as it is, and for rows that are too long for a ring."""
import pytest
import torch

import paged_reference as ref
from test_gpu_paged import CODE, buf, ctx_tables  # noqa: F401  (buf is a fixture)
from webgpu_b200 import backend as B

pytestmark = pytest.mark.gpu

POSITIONS = 500


def expected(qkv, wq, wk, cos, sin, pos, slots, H, KV, D, rot, eps, halves):
    """Of the tokens that have a slot: q, k, v in 64 bits and the bounds of q and k, by the formula and the roundings that ref.qkv_step counts."""
    n = slots.numel()
    x = qkv.double().reshape(n, H + 2 * KV, D)
    y = x[:, :H + KV].clone()
    if wq is not None:
        y /= (y.square().mean(-1, keepdim=True) + eps).sqrt()
        y[:, :H] *= wq.double()
        y[:, H:] *= wk.double()
    z, size = y.clone(), y.abs()
    if rot:
        i = torch.arange(rot // 2, device=qkv.device)
        a, b = (i, i + rot // 2) if halves else (2 * i, 2 * i + 1)
        c, s = cos.double()[pos.long()][:, None], sin.double()[pos.long()][:, None]
        z[..., a], z[..., b] = y[..., a] * c - y[..., b] * s, y[..., a] * s + y[..., b] * c
        size[..., a], size[..., b] = (y[..., a] * c).abs() + (y[..., b] * s).abs(), (y[..., a] * s).abs() + (y[..., b] * c).abs()
    err = size * ref.U * ((16 + D / 16 + 5) / 2 + 9) + ref.rounded(z, qkv.dtype) * 1.001
    return z[:, :H], z[:, H:], x[:, H + KV:], err[:, :H], err[:, H:]


@pytest.mark.parametrize("dtype,H,KV,D,rot,page,halves,norm,ctas,ring", [
    ("bf16", 32, 8, 128, 128, 16, True, True, 5, 2),           # two rows of 12 KB
    ("f16", 16, 4, 128, 64, 8, False, True, 5, 4),             # four of 6 KB
    ("bf16", 20, 4, 96, 96, 24, True, False, 5, 4),            # four of 5.3 KB, heads that are no power of two
    ("f16", 24, 6, 128, 128, 16, False, False, 5, 2),          # two of 9 KB
    ("bf16", 20, 5, 128, 0, 16, False, True, 5, 3),            # three of 7.5 KB, no rotation
    ("bf16", 90, 10, 128, 128, 16, True, True, 3, 2),          # two of 28 KB: more than is open as it is, fewer CTAs per SM
    ("f16", 180, 10, 128, 128, 16, True, True, 2, 2),          # two of 50 KB, the longest that a ring takes
    ("bf16", 181, 10, 128, 128, 16, True, True, 5, 0),         # longer: straight from the input
    ("bf16", 4, 2, 1024, 512, 4, True, True, 5, 2)])           # heads that a warp goes over twice
@pytest.mark.parametrize("bad", [False, True])
def test_qkv_ring(ctx, buf, dtype, H, KV, D, rot, page, halves, norm, ctas, ring, bad):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    dt = ref.DTYPES[dtype]
    row = (H + 2 * KV) * D
    pitch = (2 * row + 127) // 128 * 128
    assert ring == (0 if pitch > 50 << 10 else min(4, max(2, (24 << 10) // pitch)))
    T = 5 * ctas * sms + 77                                    # every CTA has five tokens at least, so it fills every place again
    g = torch.Generator(device="cuda").manual_seed(H)
    qkv = torch.randn(T, row, generator=g, device="cuda").to(dt)
    wq, wk = (torch.randn(D, generator=g, device="cuda") for _ in range(2)) if norm else (None, None)
    cos, sin = ctx_tables(rot, POSITIONS)
    pos = torch.randint(0, POSITIONS, (T,), generator=g, device="cuda", dtype=torch.int32)
    blocks = (T + page - 1) // page + 1
    slots = torch.randperm(blocks * page, generator=g, device="cuda")[:T].to(torch.int32)
    slots[torch.rand(T, generator=g, device="cuda") < 0.1] = -1         # padding anywhere
    slots[3 * ctas * sms:3 * ctas * sms + 40] = -1
    good = slots >= 0
    if bad:                                                    # and faults, in the middle and at the end
        for t in (2 * ctas * sms + 5, 3 * ctas * sms - 1, T - 1):
            slots[t], good[t] = blocks * page + t % 3, False
        if rot:
            t = 4 * ctas * sms + 9
            slots[t], pos[t], good[t] = 0 if not (slots == 0).any() else -1, POSITIONS, False
    q = torch.full((T, H, D), 3.0, device="cuda").to(dt)
    kc, vc = (torch.full((blocks, KV, page, D), 3.0, device="cuda").to(dt) for _ in range(2))

    def call():
        ctx.paged_qkv(buf(qkv), buf(wq), buf(wk), buf(cos), buf(sin), buf(pos) if rot else None, buf(slots), buf(q), buf(kc), buf(vc), T, H, KV, D, rot, page,
                      1e-5, CODE[dtype], flags=B.FLAG_ROPE_HALVES if halves else 0)

    if bad:
        with pytest.raises(B.BackendError):
            call()
        assert ctx.last_device_status() in ((0x7C050009, 0x7C05000A) if rot else (0x7C050009,))
    else:
        call()
    at = slots[good].long()
    w_q, w_k, w_v, t_q, t_k = expected(qkv[good], wq, wk, cos, sin, pos[good], at, H, KV, D, rot, 1e-5, halves)
    assert ((q[good].double() - w_q).abs() <= t_q).all() and (q[~good] == 3).all()
    places = kc.transpose(1, 2).reshape(-1, KV, D), vc.transpose(1, 2).reshape(-1, KV, D)
    assert ((places[0][at].double() - w_k).abs() <= t_k).all() and torch.equal(places[1][at].double(), w_v)
    left = torch.ones(blocks * page, dtype=torch.bool, device="cuda")
    left[at] = False
    assert (places[0][left] == 3).all() and (places[1][left] == 3).all()
