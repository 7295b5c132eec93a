"""Plain restatements, in Python and 64 bits on the CPU, of the operators of drafted tokens (``include/chia_draft.h``) and
of the norm and rotation of queries and keys (``include/chia_rope.h``). Test infrastructure; nothing of the package imports
it."""

import math
import random

import torch

import paged_oracle as po


def tree(n, seed, chain=False, wide=False):
    """Parents of a tree of n nodes: in a row, all below node 0, or at random."""
    r = random.Random(seed)
    return [i - 1 if chain or i < 2 else 0 if wide else r.randrange(max(0, i - 7), i) for i in range(n)]


def paths(parents):
    """The nodes that each node sees, itself among them, from the root down."""
    out = []
    for i, p in enumerate(parents):
        out.append(([] if p < 0 else out[p]) + [i])
    return out


def tables(parents, cu, lens, rows):
    """Positions and words (as signed 64-bit numbers) of all rows."""
    pos, words = [0] * rows, [0] * rows
    for b, n in enumerate(lens):
        t0, t1 = cu[b], cu[b + 1]
        m = t1 - t0
        if m > 64:
            for i in range(m):
                pos[t0 + i] = n - m + i
            continue
        for i, path in enumerate(paths(parents[t0:t1])):
            pos[t0 + i] = n - m + len(path) - 1
            w = sum(1 << x for x in path)
            words[t0 + i] = w - 2 ** 64 if w >= 2 ** 63 else w
    return pos, words


def attention(q, k, v, ks, vs, table, lens, cu, parents, *, norm="softmax", mod="none", mask=None, scale=None,
              softcap=30.0, head_param=None, sig_bias=0.0, out_scale=1.0):
    """64-bit (out, lse, mass) as ``paged_oracle.attention``: each row attends to a cache of its own, the keys before the
    tree and its ancestors' in a row, where it is the last token. More than 64 queries are a chunk, which attends as
    without trees."""
    T, H, D = q.shape
    hkv, page = k.shape[1], k.shape[2]
    out, mass = torch.zeros(T, H, D, dtype=torch.float64), torch.zeros(T, H, D, dtype=torch.float64)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64)
    scale = 1 / math.sqrt(D) if scale is None else scale
    for b, n in enumerate(lens):
        t0, t1 = cu[b], cu[b + 1]
        m = t1 - t0
        if n == 0 or m == 0:
            continue
        pg = torch.as_tensor(table[b][:po.pages_for(n, page)])
        kk = (k[pg].double() * ks[pg].double()[:, :, None, None]).transpose(0, 1).reshape(hkv, -1, D)[:, :n]
        vv = (v[pg].double() * vs[pg].double()[:, :, None, None]).transpose(0, 1).reshape(hkv, -1, D)[:, :n]
        seen = paths(parents[t0:t1]) if m <= 64 else [None] * m
        for i, path in enumerate(seen):
            if path is None:  # a chunk: as without trees, the mask alone says what a query sees
                keys = pos = list(range(n))
                at = n - m + i
            else:
                keys = list(range(max(0, n - m))) + [n - m + x for x in path if n - m + x >= 0]
                pos = [j for j in range(max(0, n - m))] + [n - m + d for d, x in enumerate(path) if n - m + x >= 0]
                at = n - m + len(path) - 1
            keep = []
            for key, j in zip(keys, pos):
                ok = mask.left < 0 or at - j <= mask.left
                ok &= mask.right < 0 or j - at <= mask.right
                ok &= mask.block == 0 or at // mask.block == j // mask.block
                ok &= (at - j) % mask.dilation == 0
                if ok or j < mask.prefix:
                    keep.append((key, j))
            if not keep:
                continue
            idx = torch.tensor([x for x, _ in keep])
            away = torch.tensor([j - at for _, j in keep], dtype=torch.float64)
            qh = q[t0 + i].double().view(hkv, H // hkv, D)
            x = torch.einsum("gkd,ghd->ghk", kk[:, idx], qh).reshape(H, -1) * scale
            hp = None if head_param is None else torch.as_tensor(head_param).double()[:, None]
            if mod == "softcap":
                x = softcap * torch.tanh(x / softcap)
            elif mod == "alibi":
                x = x + hp * away
            elif mod == "temp":
                x = x * hp
            if norm == "sigmoid":
                p = torch.sigmoid(x + sig_bias)
            elif norm == "relu":
                p = x.clamp(min=0) * out_scale
            else:
                lse[t0 + i] = torch.logsumexp(x, 1)
                p = torch.softmax(x, 1)
            p = p.view(hkv, H // hkv, -1)
            out[t0 + i] = (p @ vv[:, idx]).reshape(H, D)
            mass[t0 + i] = (p.abs() @ vv[:, idx].abs()).reshape(H, D)
    return out, lse, mass


def verify(p, tokens, parents, cu, u, q, most):
    """Counts, tokens and path, as lists; plain Python numbers (64 bits), one request and one child after another."""
    counts, out, nodes = [], [], []
    clean = lambda row: [x if 0 < x < math.inf else 0.0 for x in row.double().tolist()]  # noqa: E731
    for b in range(len(cu) - 1):
        t0, n = cu[b], cu[b + 1] - cu[b]
        toks, path = [], [0]
        if n == 0 or n > 64:
            counts.append(0), out.append([-1] * most), nodes.append([-1] * most)
            continue
        node = 0
        while True:
            r, z, s = clean(p[t0 + node]), 1.0, 0.0
            qq = clean(q[t0 + node]) if q is not None else None
            taken = None
            for c in range(node + 1, n):
                if parents[t0 + c] != node or len(path) >= most:
                    continue
                x, uc = tokens[t0 + c], float(u[t0 + c])
                if not 0 <= x < len(r):
                    continue
                if qq is None:
                    if uc * z < r[x]:
                        taken = c
                        break
                    z, r[x] = z - r[x], 0.0
                else:
                    if uc * z * qq[x] < r[x] * (1.0 - s):
                        taken = c
                        break
                    if 1.0 - s > 0:
                        f = z / (1.0 - s)
                        r = [max(a - f * e, 0.0) for a, e in zip(r, qq)]
                        z = math.fsum(r)
                    s, qq[x] = s + qq[x], 0.0
            if taken is None:
                break
            toks.append(tokens[t0 + taken]), path.append(taken)
            node = taken
        if not math.fsum(r) > 0:
            r = clean(p[t0 + node])
        total, acc, x = math.fsum(r), 0.0, -1
        for i, a in enumerate(r):
            acc += a
            if a > 0:
                x = i
            if a > 0 and acc > float(u[t0]) * total:
                break
        toks.append(x)
        counts.append(len(toks))
        out.append(toks + [-1] * (most - len(toks)))
        nodes.append(path + [-1] * (most - len(path)))
    return counts, out, nodes


def compact(path, counts, cu, lens, table, cache, scale, dtype):
    """cache (64-bit numbers) [pages, H, page, D] and scale [pages, H] are changed; the lengths that are kept."""
    page, keep = cache.shape[2], []
    for b, n in enumerate(lens):
        base = n - (cu[b + 1] - cu[b])
        keep.append(base + counts[b])
        slot = lambda i: (table[b][(base + i) // page], (base + i) % page)  # noqa: E731
        moves = [(slot(x), slot(i)) for i, x in enumerate(path[b][:counts[b]]) if x != i]
        codes = [(cache[f[0], :, f[1]].clone(), scale[f[0]].clone()) for f, _ in moves]
        for pg in dict.fromkeys(t[0] for _, t in moves):
            old = scale[pg].clone()
            for (c, s), (_, t) in zip(codes, moves):
                if t[0] == pg:
                    scale[pg] = torch.maximum(scale[pg], s)
            for h in range(cache.shape[1]):
                if scale[pg, h] != old[h]:
                    cache[pg, h] = po.round8(cache[pg, h] * float(old[h] / scale[pg, h]), dtype)
        for (c, s), (_, t) in zip(codes, moves):
            for h in range(cache.shape[1]):
                cache[t[0], h, t[1]] = po.round8(c[h] * float(s[h] / scale[t[0], h]), dtype)
    return keep


def norm_rope(x, w, positions, inv_freq, eps, interleaved, offset):
    """x [B, H, S, D] in 64 bits (differentiable), positions [B, S]: the rows normed and turned."""
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if w is not None:
        y = y * (w + offset)
    half = len(inv_freq)
    if half == 0:
        return y
    angle = positions[:, None, :, None].double() * torch.tensor(inv_freq, dtype=torch.float64)
    cos, sin = angle.cos(), angle.sin()
    turned, rest = y[..., :2 * half], y[..., 2 * half:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1)
