"""Plain restatements, in Python and 64 bits on the CPU, of the operators of the paged 8-bit K/V cache
(``include/chia_paged.h``). Test infrastructure; nothing of the package imports it."""

import math

import torch

TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def pages_for(n, page):
    return -(-n // page)


def tables(seq_lens, new_lens, table, ring, state, page, max_tokens):
    """Lists in, lists out: slots, positions, cu_q, lengths, state, table; and whether all were served."""
    head, count = state
    table = [list(r) for r in table]
    slots, positions, cu, lens, wanted, taken, ok = [], [], [0], [], 0, 0, True
    for b, (n, m) in enumerate(zip(seq_lens, new_lens)):
        held, total = pages_for(n, page), pages_for(n + m, page)
        need = total - held if total <= len(table[b]) else 0
        wanted += need
        served = total <= len(table[b]) and (need == 0 or wanted <= count)
        ok &= served
        if served:
            for p in range(need):
                table[b][held + p] = ring[(head + wanted - need + p) % len(ring)]
            taken += need
        for t in range(n, n + m):
            slots.append(table[b][t // page] * page + t % page if served else -1)
            positions.append(t)
        cu.append(cu[-1] + m)
        lens.append(n + m if served else n)
    slots = (slots + [-1] * max_tokens)[:max_tokens]
    positions = (positions + [0] * max_tokens)[:max_tokens]
    return slots, positions, cu, lens, [(head + taken) % len(ring), count - taken], table, ok


def scale_for(x, top):
    """The smallest 2^e, e >= -64, that holds the finite values of x in units of top."""
    x = x[torch.isfinite(x)].abs()
    amax = float(x.max()) if x.numel() else 0.0
    e = -64
    while top * 2.0 ** e < amax:
        e += 1
    return 2.0 ** e


def round8(x, dtype):
    """64-bit values to the numbers of the cache's type (64-bit): nearest, ties to even, saturating."""
    top = TOP[dtype]
    if dtype == torch.int8:
        return torch.nan_to_num(x, nan=0.0, posinf=top, neginf=-top).round().clamp(-top, top)
    y = x.clamp(-top, top)
    _, e = torch.frexp(torch.nan_to_num(y).abs())
    unit = 2.0 ** ((e - 1).clamp(min=-6).double() - 3)
    return ((y / unit).round() * unit).clamp(-top, top)


def append(x, slots, cache, scale):
    """x [T, H, D]; cache (64-bit numbers) [pages, H, page, D] and scale [pages, H] are changed; dtype: the cache's."""
    cache, dtype = cache
    page = cache.shape[2]
    t = 0
    while t < len(slots):
        if slots[t] < 0:
            t += 1
            continue
        p, run = slots[t] // page, []
        while t < len(slots) and slots[t] >= 0 and slots[t] // page == p:
            run.append((t, slots[t] % page))
            t += 1
        if p >= cache.shape[0]:
            continue
        for h in range(cache.shape[1]):
            new = x[[r for r, _ in run], h].double()
            s, old = scale_for(new, TOP[dtype]), float(scale[p, h])
            if not any(o == 0 for _, o in run):
                s = max(s, old)
                if s != old:
                    cache[p, h] = round8(cache[p, h] * (old / s), dtype)
            cache[p, h, [o for _, o in run]] = round8(new / s, dtype)
            scale[p, h] = s


def attention(q, k, v, ks, vs, table, lens, cu, *, norm="softmax", mod="none", mask=None, scale=None, softcap=30.0,
              head_param=None, sig_bias=0.0, out_scale=1.0):
    """64-bit (out, lse, mass), mass = sum_j |p_j v_j|, the size of what was summed (for tolerances)."""
    T, H, D = q.shape
    hkv, page = k.shape[1], k.shape[2]
    out, mass = torch.zeros(T, H, D, dtype=torch.float64), torch.zeros(T, H, D, dtype=torch.float64)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64)
    scale = 1 / math.sqrt(D) if scale is None else scale
    for b, n in enumerate(lens):
        t0, t1 = cu[b], cu[b + 1]
        if n == 0 or t0 == t1:
            continue
        pg = torch.as_tensor(table[b][:pages_for(n, page)])
        kk = (k[pg].double() * ks[pg].double()[:, :, None, None]).transpose(0, 1).reshape(hkv, -1, D)[:, :n]
        vv = (v[pg].double() * vs[pg].double()[:, :, None, None]).transpose(0, 1).reshape(hkv, -1, D)[:, :n]
        i = torch.arange(n - (t1 - t0), n)[:, None]
        j = torch.arange(n)[None]
        see = torch.ones(t1 - t0, n, dtype=torch.bool)
        if mask.left >= 0:
            see &= i - j <= mask.left
        if mask.right >= 0:
            see &= j - i <= mask.right
        if mask.block:
            see &= i.div(mask.block, rounding_mode="floor") == j.div(mask.block, rounding_mode="floor")
        see &= (i - j) % mask.dilation == 0
        see |= j < mask.prefix
        for h in range(H):
            x = q[t0:t1, h].double() @ kk[h // (H // hkv)].T * scale
            if mod == "softcap":
                x = softcap * torch.tanh(x / softcap)
            elif mod == "alibi":
                x = x + float(head_param[h]) * (j - i)
            elif mod == "temp":
                x = x * float(head_param[h])
            val = vv[h // (H // hkv)]
            if norm == "sigmoid":
                p = torch.where(see, torch.sigmoid(x + sig_bias), 0.0)
            elif norm == "relu":
                p = torch.where(see, x.clamp(min=0), 0.0) * out_scale
            else:
                x = x.masked_fill(~see, -math.inf)
                z = torch.logsumexp(x, 1, keepdim=True)
                lse[t0:t1, h] = z[:, 0]
                p = torch.where(see, torch.exp(x - z), 0.0)
                p = torch.where(torch.isinf(z), 0.0, p)
            live = see.any(0)
            val = torch.where(live[:, None], val, 0.0)
            out[t0:t1, h] = p @ val
            mass[t0:t1, h] = p.abs() @ val.abs()
    return out, lse, mass
