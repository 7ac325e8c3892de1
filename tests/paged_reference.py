"""Plain 64-bit forms of the operators of a paged KV cache (torch, on whatever device the inputs are), with bounds on what the
kernels' arithmetic may differ by, derived from the number of roundings."""
import math

import torch

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24                      # half a step of f32
NO_KEYS = float(torch.tensor(-3.402823e38))     # as f32 holds it


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounded(want, dtype):
    """How far one rounding to `dtype` moves a value: half a step, and of subnormal numbers half the least one."""
    return want.abs() * half_step(dtype) + torch.finfo(dtype).smallest_normal * half_step(dtype)


def gather(cache, table, keys):
    """[kv_heads, keys, dim] of one sequence, 64 bits."""
    page = cache.shape[2]
    at = torch.arange(keys, device=cache.device)
    return cache[table[at // page].long(), :, at % page].double().transpose(0, 1)


def attention(q, kc, vc, table, starts, lens, scale, causal):
    """out [T, H, D], lse [T, H] and the bound of |out - computed|, |lse - computed|; rows of no sequence are NaN."""
    T, H, D = q.shape
    KV = kc.shape[1]
    G = H // KV
    dev = q.device
    out = torch.full((T, H, D), math.nan, dtype=torch.float64, device=dev)
    tol = torch.zeros((T, H, D), dtype=torch.float64, device=dev)
    lse = torch.full((T, H), math.nan, dtype=torch.float64, device=dev)
    ltol = torch.zeros((T, H), dtype=torch.float64, device=dev)
    for s in range(len(lens)):
        a, b, n = int(starts[s]), int(starts[s + 1]), max(0, int(lens[s]))
        t = b - a
        if t <= 0:
            continue
        k, v = gather(kc, table[s], n), gather(vc, table[s], n)
        at = torch.arange(n, device=dev)
        sees = torch.arange(t, device=dev) + (n - t) if causal else torch.full((t,), n - 1, device=dev)
        for h in range(H):
            x = (q[a:b, h].double() @ k[h // G].T) * scale
            hidden = at[None, :] > sees[:, None]
            x = x.masked_fill(hidden, -math.inf)
            some = ~hidden.all(1) if n else torch.zeros(t, dtype=torch.bool, device=dev)
            top = x.amax(1) if n else torch.zeros(t, dtype=torch.float64, device=dev)
            w = torch.exp(x - top[:, None]) if n else torch.zeros((t, 0), dtype=torch.float64, device=dev)
            w[~some] = 0
            # what a row must not see takes no part, whatever it holds
            vv = torch.where(torch.isfinite(v[h // G]), v[h // G], 0.0) if n else v[h // G]
            bad = (~torch.isfinite(v[h // G])).double() if n else v[h // G]
            l = w.sum(1)
            p = w / l.clamp(min=1e-300)[:, None]
            o = p @ vv
            o[(p @ bad) > 0] = math.nan
            out[a:b, h] = torch.where(some[:, None], o, 0.0)
            lse[a:b, h] = torch.where(some, top + torch.log(l.clamp(min=1e-300)), NO_KEYS)
            # a score: its products and their sum in f32 (on the tensor cores the sum is cut off, a whole step per 16 products), the scale
            # and the difference to the maximum; the power of two 2^-22; weights rounded to the data's type where that has 16 bits
            size = (q[a:b, h].double().abs() @ k[h // G].abs().T * abs(scale)).masked_fill(hidden, 0).nan_to_num(0, 0, 0)
            size = size.amax(1) if n else torch.zeros(t, dtype=torch.float64, device=dev)
            eps = 2.0 ** -22 + U * (D + 8 + D / 8) * size + U * 4 * (size + 1)
            parts = n / 16 + 64 + 160                       # sums over tiles, within one, and over the parts of a context
            rel = 2 * eps + 4 * parts * U + (half_step(q.dtype) * 1.01 if q.dtype != torch.float32 else 0)
            mass = p @ vv.abs()
            tol[a:b, h] = mass * rel[:, None] + rounded(o.nan_to_num(0), q.dtype) * (1 + rel[:, None])
            ltol[a:b, h] = 2 * eps + 2 * parts * U + U * (top.nan_to_num(0, 0, 0).abs() + 10) * 4
    return out, lse, tol, ltol


def qkv_step(qkv, wq, wk, cos, sin, pos, slots, H, KV, D, rot, page, eps, halves, q, kc, vc):
    """The 64-bit form of paged_qkv over copies of q, kc, vc (its own types' values where nothing is written), and the bounds."""
    q, kc, vc = q.double(), kc.double(), vc.double()
    dt = qkv.dtype
    tq, tk = torch.zeros_like(q), torch.zeros_like(kc)
    for t in range(qkv.shape[0]):
        slot = int(slots[t])
        if slot < 0:
            continue
        x = qkv[t, :(H + 2 * KV) * D].double().reshape(H + 2 * KV, D)
        y = x[:H + KV].clone()
        if wq is not None:
            y = y / torch.sqrt((y * y).mean(1, keepdim=True) + eps)
            y[:H] *= wq.double()
            y[H:] *= wk.double()
        i = torch.arange(rot // 2, device=qkv.device)
        a, b = (i, i + rot // 2) if halves else (2 * i, 2 * i + 1)
        z, size = y.clone(), y.abs()
        if rot:
            c, s = cos[int(pos[t])].double(), sin[int(pos[t])].double()
            z[:, a], z[:, b] = y[:, a] * c - y[:, b] * s, y[:, a] * s + y[:, b] * c
            size[:, a], size[:, b] = (y[:, a] * c).abs() + (y[:, b] * s).abs(), (y[:, a] * s).abs() + (y[:, b] * c).abs()
        # the sum of squares: chains of at most 16 + D / 16 terms, five steps over lanes, half of it through the root; then mean, root,
        # quotient, two products, and the rotation's two products and sum
        err = size * U * ((16 + D / 16 + 5) / 2 + 9) + rounded(z, dt) * 1.001
        q[t], tq[t] = z[:H], err[:H]
        kc[slot // page, :, slot % page], tk[slot // page, :, slot % page] = z[H:], err[H:]
        vc[slot // page, :, slot % page] = x[H + KV:]
    return q, kc, vc, tq, tk


def plan(cached, new, table, free, count, page, max_tokens):
    """Lists in, lists out: starts, lens, positions, slots, table, count; None if nothing is handed out."""
    table = [list(r) for r in table]
    starts, pos, slots = [0], [], []
    width = len(table[0]) if table else 0
    if count < 0 or count > len(free) or sum(new) > max_tokens or any(c < 0 or t < 0 or c + t > width * page for c, t in zip(cached, new)):
        return None
    for row, c, t in zip(table, cached, new):
        for p in range(c, c + t):
            if row[p // page] < 0:
                if count == 0:
                    return None
                count -= 1
                row[p // page] = free[count]
            pos.append(p)
            slots.append(row[p // page] * page + p % page)
        starts.append(starts[-1] + t)
    pos += [0] * (max_tokens - len(pos))
    slots += [-1] * (max_tokens - len(slots))
    return starts, [c + t for c, t in zip(cached, new)], pos, slots, table, count


def release(keep, table, free, count, page):
    table, free = [list(r) for r in table], list(free)
    back = []
    for row, k in zip(table, keep):
        if k < 0:
            continue
        for b in range((k + page - 1) // page, len(row)):
            if row[b] < 0:
                break
            back.append(row[b])
            row[b] = -1
    if count < 0 or count + len(back) > len(free):
        return None
    for b in reversed(back):
        free[count] = b
        count += 1
    return table, free, count


def verify(target, draft, tokens, uniforms, starts):
    """Lists of out tokens (-1 behind the drawn one; None: left as it is) and accepted counts, sums in 64 bits by math.fsum."""
    R, V = target.shape
    out, accepted = [None] * R, []
    p64 = target.double().cpu()
    q64 = draft.double().cpu() if draft is not None else None
    u = uniforms.double().cpu().tolist()
    tokens = tokens.tolist()
    for s in range(len(starts) - 1):
        a, b = starts[s], starts[s + 1]
        if a >= b:
            accepted.append(0)
            continue
        n = 0
        while n < b - a - 1:
            x = tokens[a + n + 1]
            if not 0 <= x < V or not u[a + n] * (1.0 if q64 is None else float(q64[a + n, x])) < float(p64[a + n, x]):
                break
            out[a + n] = x
            n += 1
        w = p64[a + n].clone()
        w = torch.where(w > 0, w, 0.0)
        if n < b - a - 1:
            r = p64[a + n].clone()
            if q64 is None:
                if 0 <= tokens[a + n + 1] < V:
                    r[tokens[a + n + 1]] -= 1.0
            else:
                r = r - q64[a + n]
            r = torch.where(r > 0, r, 0.0)
            if float(r.sum()) > 0:
                w = r
        w = w.tolist()
        goal, sum_, pick = u[b - 1] * math.fsum(w), 0.0, -1
        for i, x in enumerate(w):
            if x > 0:
                sum_ += x
                pick = i
                if sum_ > goal:
                    break
        out[a + n] = pick
        for i in range(a + n + 1, b):
            out[i] = -1
        accepted.append(n)
    return out, accepted
