"""The operators of speculative decoding over a paged 8-bit K/V cache: what is measured of them, and their plain forms.

A step checks a tree of drafted tokens for each request: queries and keys are normed head by head and turned to their
positions (``qk_norm_rope``, in training with its gradients), each drafted token attends to the cache and to its own
ancestors (``tree_tables``, ``paged_attention(tree=...)``), the drafts are verified against the target's probabilities
(``verify_drafts``), and the accepted path's keys and values move together in the cache (``cache_compact``).

Layouts. Activations ``[tokens, heads, head_dim]`` or ``[batch, heads, seq, head_dim]``; the cache as in
``operators.py``: ``[pages, heads_kv, page, head_dim]`` in float8_e4m3fn or int8, scales ``[pages, heads_kv]`` in fp32. A
request's tree is its last ``n`` tokens: node 0 is the token that is decided already, ``parents`` are nodes before their
children, -1 a root.
"""

import math
import random

import torch

own = False

E4M3, INT8 = torch.float8_e4m3fn, torch.int8
TOP = {E4M3: 448.0, INT8: 127.0}
MIN_EXP = -64  # the smallest scale is 2^-64
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------ the cases
def _norm(name, **kw):
    d = dict(name=name, op="norm", batch=0, tokens=64, heads=32, heads_kv=8, head_dim=128, rot=128, interleaved=False,
             dtype="bf16", weights="same", offset=0.0, base=10000.0, far=8192, train=False)
    d.update(kw)
    return d


def _tree(name, op, **kw):
    d = dict(name=name, op=op, batch=1, nodes=25, chain=False, ragged=False, page=64)
    if op == "attend":
        d.update(keys=512, heads=32, heads_kv=8, head_dim=128, cache="e4m3", dtype="bf16", kind="softmax", window=0)
    if op == "verify":
        d.update(vocab=32000, dtype="fp32", drafts=True, most=9)
    if op == "compact":
        d.update(heads_kv=8, head_dim=128, cache="e4m3", most=9)
    d.update(kw)
    return d


def listed():
    return [
        # one token of one request: nothing but latency
        _norm("norm one", tokens=1),
        # a prefill of long prompts, the queries and keys of one fused projection, half of the channels turned
        _norm("norm prompts", tokens=16421, rot=64, base=500000.0, far=100000),
        # a training step of this repository's benchmark (B4 H16 S4096 D128), forward and backward
        _norm("norm train", batch=4, tokens=4096, heads=16, heads_kv=16, train=True, weights="fp32"),
        # one user's chat: thirteen drafted tokens behind a short context
        _tree("attend one", "attend", nodes=13, keys=601),
        # continuous batching: trees of up to 25 nodes, unequal contexts, a padding row, a sliding window, int8, D = 64
        _tree("attend ragged", "attend", batch=48, keys=20000, ragged=True, heads=16, heads_kv=4, head_dim=64, cache="int8",
              dtype="fp16", page=16, window=1024),
        # the largest: full trees over long contexts, Gemma-2 style softcap
        _tree("attend wide", "attend", batch=32, nodes=64, keys=16384, ragged=True, heads=64, kind="softcap"),
        # the tables of one small tree, and of a full batch's
        _tree("tables one", "tables", nodes=13),
        _tree("tables batch", "tables", batch=64, nodes=64, ragged=True),
        # five drafted tokens in a row (each request's own model drafts greedily: no probabilities of the drafts)
        _tree("verify chain", "verify", batch=1, nodes=6, chain=True, drafts=False),
        # a full batch of trees, drafted by sampling without replacement, a large vocabulary
        _tree("verify trees", "verify", batch=64, ragged=True, vocab=131072),
        # an accepted path of one request; of a full batch over small pages, where most paths leave their page
        _tree("compact one", "compact", nodes=13),
        _tree("compact batch", "compact", batch=128, nodes=64, ragged=True, page=16, cache="int8"),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "attend", "attend", "tables", "verify", "compact"])
    page, head_dim, heads_kv = rng.choice([16, 32, 64, 128]), rng.choice([64, 128, 128]), rng.choice([1, 2, 4, 8])
    dtype, cache, ragged = rng.choice(["bf16", "bf16", "fp16"]), rng.choice(["e4m3", "e4m3", "int8"]), rng.random() < 0.7
    if op == "norm":
        train = rng.random() < 0.5
        batch = rng.choice([0, 1, 2, 4]) if train else 0
        heads = heads_kv * rng.choice([1, 2, 4, 7, 8])
        c = _norm("", batch=batch, heads=heads, heads_kv=heads_kv, head_dim=head_dim,
                  tokens=_spread(rng, 1, 400000 // (max(batch, 1) * (heads + heads_kv))),
                  rot=head_dim if rng.random() < 0.6 else 16 * rng.randint(1, head_dim // 16), train=train,
                  interleaved=rng.random() < 0.3, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                  weights=rng.choice(["same", "fp32", "none"]), offset=rng.choice([0.0, 0.0, 1.0]),
                  base=rng.choice([10000.0, 500000.0, 1000000.0]), far=rng.choice([4096, 131072, 2000000]))
        del c["name"]
        return c
    nodes, batch = _spread(rng, 2, 64), _spread(rng, 1, 64)
    c = _tree("", op, batch=batch, nodes=nodes, chain=rng.random() < 0.25, ragged=ragged, page=page)
    if op == "attend":
        c.update(keys=_spread(rng, 64, min(16384, 400000 // batch)), heads=heads_kv * rng.choice([1, 2, 4, 7, 8]),
                 heads_kv=heads_kv, head_dim=head_dim, cache=cache, dtype=dtype,
                 kind=rng.choice(["softmax", "softmax", "softcap", "alibi", "temp", "sigmoid", "relu"]),
                 window=_spread(rng, 4, 4096) if rng.random() < 0.3 else 0)
    if op == "verify":
        c.update(vocab=_spread(rng, 500, min(131072, 100000000 // (batch * nodes))), dtype=rng.choice(["fp32", "fp32", "bf16"]),
                 drafts=rng.random() < 0.7, most=rng.randint(1, 12))
    if op == "compact":
        c.update(heads_kv=heads_kv, head_dim=head_dim, cache=cache, most=rng.randint(2, 12))
    del c["name"]
    return c


def _pages(n, page):
    return -(-n // page)


def _lengths(c):
    """(keys of each request before its tree, nodes of its tree). Ragged: spread over the logarithm, the last of four
    requests or more is a padding row (no keys and no nodes)."""
    b, n = c["batch"], c["nodes"]
    keys = c.get("keys", 0)
    r = random.Random(1000003 * b + 1009 * keys + n)
    ks, ns = [], []
    for i in range(b):
        m = n if i == 0 or not c["ragged"] else _spread(r, 1, n)
        ns.append(m)
        if c["op"] == "attend":
            ks.append(max(0, (keys if i == 0 or not c["ragged"] else _spread(r, min(m, keys), keys)) - m))
        else:  # so much of a page that the cache is what the operator touches
            ks.append((11 * i + 5) % c["page"])
    if b >= 4 and c["ragged"]:
        ks[-1] = ns[-1] = 0
    return ks, ns


def _trees(c, seed):
    """The parents of each request's nodes: a chain, or a tree whose nodes have up to eight children."""
    r, out = random.Random(7919 * seed + c["nodes"]), []
    for n in _lengths(c)[1]:
        p, kids = [], [0] * n
        for i in range(n):
            if c["chain"] or i < 2:
                p.append(i - 1)
            else:
                p.append(r.choice([j for j in range(max(0, i - 9), i) if kids[j] < 8]))
            if p[-1] >= 0:
                kids[p[-1]] += 1
        out.append(p)
    return out


def _paths(c, seed):
    """Accepted paths of the compaction: node 0, then nodes that rise. Some requests keep their tokens where they are."""
    r, out = random.Random(104729 * seed + c["nodes"]), []
    for i, n in enumerate(_lengths(c)[1]):
        k = min(r.randint(1, c["most"]), (n + 1) // 2)
        out.append(list(range(k)) if i % 5 == 4 or k < 2 else [0] + sorted(r.sample(range(k, n), k - 1)))
    return out


def work(case):
    c = case
    if c["op"] == "norm":
        rows = max(c["batch"], 1) * c["tokens"] * (c["heads"] + c["heads_kv"])
        size = 4 if c["dtype"] == "fp32" else 2
        # queries and keys in and out; in training also the outputs' gradients in and the inputs' out
        return {"bytes": float(rows * c["head_dim"] * size * (4 if c["train"] else 2) + 4 * max(c["batch"], 1) * c["tokens"]),
                "flops": float(rows * c["head_dim"] * (30 if c["train"] else 8))}
    ks, ns = _lengths(c)
    rows = sum(ns)
    if c["op"] == "tables":  # parents, offsets and lengths in, a position and a word of ancestors out
        return {"bytes": float(rows * (4 + 4 + 8) + 8 * len(ns)), "flops": 0.0}
    if c["op"] == "attend":
        d, keys, pairs = c["head_dim"], 0, 0
        for k, n in zip(ks, ns):
            seen = min(k, c["window"] + n) if c["window"] else k
            keys += seen + n
            pairs += (seen + n / 4) * n
        # queries in and outputs out, the visible keys and values once, the scales of their pages
        return {"bytes": float(4 * rows * c["heads"] * d + 2 * keys * c["heads_kv"] * d + keys / c["page"] * c["heads_kv"] * 8 + 16 * rows),
                "flops": 4.0 * d * pairs * c["heads"]}
    if c["op"] == "verify":  # the row that the last token is drawn from, and its draft's
        served = sum(n > 0 for n in ns)
        row = c["vocab"] * (2 if c["dtype"] == "bf16" else 4)
        return {"bytes": float(served * row * (2 if c["drafts"] else 1) + 12 * rows), "flops": 3.0 * served * c["vocab"]}
    moved = sum(sum(k != x for k, x in enumerate(p)) for p in _paths(c, 1))
    return {"bytes": float(2 * 2 * moved * c["heads_kv"] * c["head_dim"] + 8 * rows), "flops": float(2 * moved * c["heads_kv"] * c["head_dim"])}


# ------------------------------------------------------------------ the inputs
def _exponent(amax, top):
    """The smallest e >= MIN_EXP with amax <= top * 2^e."""
    mant, exp = torch.frexp(amax.float())
    m, e = math.frexp(top)
    e = exp - e + (mant > m).to(exp.dtype)
    return torch.where(mant == 0, torch.full_like(e, MIN_EXP), e.clamp(min=MIN_EXP))


def _power(e):
    """2^e in fp32, exactly."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _to8(x, cache):
    """fp32 to the cache's 8 bits: to nearest, ties to even, the largest value for what is beyond it."""
    if cache == INT8:
        return torch.nan_to_num(x, nan=0.0, posinf=127.0, neginf=-127.0).round().clamp(-127, 127).to(INT8)
    return x.clamp(-448, 448).to(E4M3)


def _random_cache(shape, cache, channels, g):
    """A filled cache: keys or values with their channels' own sizes, quantised page by page and head by head."""
    q = torch.empty(shape, dtype=cache, device="cuda")
    scale = torch.empty(shape[:2], dtype=torch.float32, device="cuda")
    step = max(1, (1 << 28) // math.prod(shape[1:]))
    for a in range(0, shape[0], step):
        x = torch.randn((min(step, shape[0] - a),) + tuple(shape[1:]), device="cuda", generator=g) * channels
        e = _exponent(x.abs().amax((2, 3)), TOP[cache])
        scale[a:a + step] = _power(e)
        q[a:a + step] = _to8(x / scale[a:a + step, :, None, None], cache)
    return q, scale


def _channels(heads, d, g):
    """Sizes of a head's channels: a few of a key's channels are many times larger than the others."""
    s = torch.exp(0.4 * torch.randn(heads, 1, d, device="cuda", generator=g))
    return s * torch.where(torch.rand(heads, 1, d, device="cuda", generator=g) < 0.03, 6.0, 1.0)


def _prepare_norm(c, g):
    h, hkv, d, t = c["heads"], c["heads_kv"], c["head_dim"], c["tokens"]
    b = max(c["batch"], 1)
    dtype = TYPES[c["dtype"]]
    wtype = dtype if c["weights"] == "same" else torch.float32
    st = {"case": c}
    qkv = torch.randn(b, t, h + 2 * hkv, d, device="cuda", generator=g)
    qkv *= torch.exp(0.5 * torch.randn(b, t, h + 2 * hkv, 1, device="cuda", generator=g))
    q, k, _ = qkv.to(dtype).split([h, hkv, hkv], 2)  # one projection's output
    at = torch.randint(0, c["far"], (b, 1), device="cuda", generator=g)
    pos = at + torch.arange(t, device="cuda")
    if c["batch"]:
        q, k, st["positions"] = q.transpose(1, 2), k.transpose(1, 2), pos.to(torch.int32)
    else:
        q, k, st["positions"] = q[0], k[0], pos[0].to(torch.int32)
    st["q"], st["k"] = q.detach(), k.detach()
    for n in ("q_weight", "k_weight"):
        w = 1.0 - c["offset"] + 0.2 * torch.randn(d, device="cuda", generator=g)
        st[n] = None if c["weights"] == "none" else w.to(wtype)
    if c["train"]:
        st["dq"] = torch.randn(q.shape, device="cuda", generator=g).to(dtype)
        st["dk"] = torch.randn(k.shape, device="cuda", generator=g).to(dtype)
        st["leaves"] = [st[n].requires_grad_() for n in ("q", "k", "q_weight", "k_weight") if st[n] is not None]
    if own:
        import chia_proj_b200 as cp

        st["freqs"] = cp.rope_frequencies(c["rot"], base=c["base"])
    return st


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    if c["op"] == "norm":
        return _prepare_norm(c, g)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    ks, ns = _lengths(c)
    page, b, rows = c["page"], c["batch"], sum(ns)
    lens = [k + n for k, n in zip(ks, ns)]
    trees = _trees(c, seed)
    st = {"case": c, "page": page, "nodes": c["nodes"], "parents": ints([p for t in trees for p in t]),
          "cu_q": ints([sum(ns[:i]) for i in range(b + 1)]), "seq_lens": ints(lens)}
    if c["op"] == "tables":  # contexts of any length
        st["seq_lens"] += torch.randint(0, 100000, (b,), device="cuda", generator=g, dtype=torch.int32)
        return st
    if c["op"] == "verify":
        v, dtype = c["vocab"], TYPES[c["dtype"]]
        p = torch.empty(rows, v, device="cuda", dtype=dtype)
        q = torch.empty(rows, v, device="cuda", dtype=dtype) if c["drafts"] else None
        drawn, step = [], max(1, (1 << 26) // v)
        for a in range(0, rows, step):
            x = 3.0 * torch.randn(min(step, rows - a), v, device="cuda", generator=g)
            y = x + 0.8 * torch.randn(x.shape, device="cuda", generator=g)
            p[a:a + step] = torch.softmax(x, 1).to(dtype)
            y = torch.softmax(y, 1)
            if c["drafts"]:  # children by sampling without replacement: the largest of log q + Gumbel noise
                q[a:a + step] = y.to(dtype)
                y = q[a:a + step].float().log() - torch.log(-torch.log(torch.rand(x.shape, device="cuda", generator=g)))
            drawn.append(torch.topk(y, min(8, v), 1).indices)
        drawn, tokens, at = torch.cat(drawn).tolist() if rows else [], [], 0
        for t in trees:
            used = [0] * len(t)
            for i, par in enumerate(t):
                if par < 0:
                    tokens.append(17 % v)
                else:
                    tokens.append(drawn[at + par][used[par]])
                    used[par] += 1
            at += len(t)
        st.update(target_probs=p, draft_probs=q, tokens=ints(tokens), uniforms=torch.rand(rows, device="cuda", generator=g))
        return st
    cache, hkv, d = E4M3 if c["cache"] == "e4m3" else INT8, c["heads_kv"], c["head_dim"]
    kch, vch = _channels(hkv, d, g), _channels(hkv, d, g) * 0.5
    need = [_pages(n, page) for n in lens]
    total = sum(need) + 3
    perm = torch.randperm(total, device="cuda", generator=g).to(torch.int32)  # pages are handed out in any order
    at = torch.cumsum(torch.tensor([0] + need[:-1], device="cuda"), 0)
    col = torch.arange(max(max(need), 1), device="cuda")
    inside = col[None] < torch.tensor(need, device="cuda")[:, None]
    table = torch.where(inside, perm[(at[:, None] + col[None]).clamp(max=total - 1)], torch.zeros((), dtype=torch.int32, device="cuda"))
    st["block_table"] = table.contiguous()
    st["k_cache"], st["k_scale"] = _random_cache((total, hkv, page, d), cache, kch, g)
    st["v_cache"], st["v_scale"] = _random_cache((total, hkv, page, d), cache, vch, g)
    if c["op"] == "attend":
        st["q"] = torch.randn(rows, c["heads"], d, device="cuda", generator=g).to(TYPES[c["dtype"]])
        st["head_param"] = None
        if c["kind"] == "alibi":
            st["head_param"] = torch.pow(2.0, -8.0 * (torch.arange(c["heads"], device="cuda") + 1.0) / c["heads"])
        if c["kind"] == "temp":
            st["head_param"] = 0.5 + torch.arange(c["heads"], device="cuda") / c["heads"]
        return st
    # Compaction. A first page may have a smaller scale than those behind it, which share theirs: then a pass over what
    # the pass before left (its paths keep away from the places that it writes) gives the same again.
    for scale in (st["k_scale"], st["v_scale"]):
        for i in range(b):
            behind = table[i, 1:need[i]].long()
            if behind.numel():
                scale[behind] = scale[behind].amax(0)
                first = table[i, 0].long()
                scale[first] = torch.minimum(scale[first], scale[behind[0]]) * 2.0 ** -(i % 3)
    paths = _paths(c, seed)
    st["counts"] = ints([len(p) for p in paths])
    st["path"] = ints([p + [-1] * (c["most"] - len(p)) for p in paths])
    return st


# ------------------------------------------------------------------ one pass: the framework's calls
def _kind(c):
    kw = {"norm": c["kind"]} if c["kind"] in ("sigmoid", "relu") else {}
    if c["kind"] in ("softcap", "alibi", "temp"):
        kw["mod"] = c["kind"]
    return kw


def _own_run(s):
    import chia_proj_b200 as cp

    c = s["case"]
    if c["op"] == "norm":
        out = cp.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["freqs"], s["positions"],
                              interleaved=c["interleaved"], weight_offset=c["offset"])
        if not c["train"]:
            return list(out)
        return [o.detach() for o in out] + list(torch.autograd.grad(out, s["leaves"], [s["dq"], s["dk"]]))
    if c["op"] == "verify":
        return list(cp.verify_drafts(s["target_probs"], s["tokens"], s["parents"], s["cu_q"], s["uniforms"],
                                     draft_probs=s["draft_probs"], max_tokens=c["most"]))
    if c["op"] == "compact":
        caches = [s[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")]
        return caches + [cp.cache_compact(s["path"], s["counts"], s["cu_q"], s["seq_lens"], s["block_table"], *caches)]
    tree = cp.tree_tables(s["parents"], s["cu_q"], s["seq_lens"])
    if c["op"] == "tables":
        return list(tree)
    mask = cp.Mask(left=c["window"] - 1 if c["window"] else -1, right=0)
    return cp.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["block_table"],
                              s["seq_lens"], s["cu_q"], max_q=s["nodes"], mask=mask, softcap=50.0,
                              head_param=s["head_param"], sig_bias=-6.0, out_scale=0.001, tree=tree, **_kind(c))


# ------------------------------------------------------------------ one pass: the plain forms
def _turn(x, cos, sin, c, back=False):
    """The rotation of the first ``rot`` channels of the last dimension (``back``: its inverse)."""
    rot = c["rot"]
    if back:
        sin = -sin
    if c["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _plain_norm(s):
    c = s["case"]
    freq = c["base"] ** (torch.arange(0, c["rot"], 2, device="cuda", dtype=torch.float64) * (-1.0 / c["rot"]))
    angle = s["positions"][..., None].double() * freq  # far positions: 64 bits
    cos, sin = angle.cos().float(), angle.sin().float()
    cos, sin = (cos[:, None], sin[:, None])  # beside the heads: [T, 1, rot / 2] or [B, 1, S, rot / 2]
    outs, grads, weights = [], [], []
    for n, g in (("q", "dq"), ("k", "dk")):
        x, w = s[n].detach().float(), s[n + "_weight"]
        rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
        xhat = x * rstd
        wf = c["offset"] + w.detach().float() if w is not None else torch.ones((), device="cuda")
        outs.append(_turn(xhat * wf, cos, sin, c).to(s[n].dtype))
        if c["train"]:
            gn = _turn(s[g].float(), cos, sin, c, back=True)
            if w is not None:
                weights.append((gn * xhat).flatten(0, -2).sum(0, dtype=torch.float64).to(w.dtype))
            gx = gn * wf
            grads.append((rstd * (gx - xhat * (gx * xhat).mean(-1, keepdim=True))).to(s[n].dtype))
    return outs + grads + weights


def _plain_tables(s):
    """Positions, and of each node the bits of its ancestors and of itself."""
    cu, parents, lens = s["cu_q"].long(), s["parents"].long(), s["seq_lens"].long()
    rows = parents.numel()
    t = torch.arange(rows, device="cuda")
    r = torch.searchsorted(cu[1:], t, right=True)
    i = t - cu[r]
    word, up, depth = torch.ones_like(i) << i, parents, torch.zeros_like(i)
    at = torch.where(up >= 0, cu[r] + up, t)  # the node above, a root: itself
    own_bit = word
    for _ in range(s["nodes"]):
        depth = torch.where(up >= 0, depth[at] + 1, depth)
        word = own_bit | torch.where(up >= 0, word[at], torch.zeros_like(word))
    return [((lens - (cu[1:] - cu[:-1]))[r] + depth).to(torch.int32), word]


def _plain_attend(s):
    c, q = s["case"], s["q"]
    heads, d = q.shape[1:]
    hkv, page = s["k_cache"].shape[1:3]
    group, out = heads // hkv, []
    positions, words = _plain_tables(s)
    (ks, ns), t = _lengths(c), 0
    for b, (k0, n) in enumerate(zip(ks, ns)):
        if n == 0:
            continue
        keys = k0 + n
        pg = s["block_table"][b, :_pages(keys, page)].long()
        kf, vf = ((s[x + "_cache"][pg].float() * s[x + "_scale"][pg][..., None, None]).transpose(0, 1).reshape(hkv, 1, -1, d)[:, :, :keys]
                  for x in ("k", "v"))
        x = q[t:t + n].float().view(n, hkv, group, d).permute(1, 2, 0, 3) @ kf.transpose(2, 3) / math.sqrt(d)
        pos, word = positions[t:t + n].long()[:, None], words[t:t + n][:, None]
        j = torch.arange(keys, device="cuda")
        at = torch.cat([j[:k0], pos[:, 0]])[None]  # positions of the keys
        see = (j < k0)[None] | ((word >> (j - k0).clamp(min=0)[None]) & 1).bool()
        see = see & (at <= pos)
        if c["window"]:
            see = see & (pos - at < c["window"])
        hp = None if s["head_param"] is None else s["head_param"].view(hkv, group, 1, 1)
        if c["kind"] == "softcap":
            x = 50.0 * torch.tanh(x / 50.0)
        elif c["kind"] == "alibi":
            x = x + hp * (at - pos).float()
        elif c["kind"] == "temp":
            x = x * hp
        if c["kind"] == "sigmoid":
            p = torch.where(see, torch.sigmoid(x - 6.0), torch.zeros_like(x))
        elif c["kind"] == "relu":
            p = torch.where(see, x.clamp(min=0), torch.zeros_like(x)) * 0.001
        else:
            x = x.masked_fill(~see, float("-inf"))
            p = torch.exp(x - x.amax(-1, keepdim=True))
            p = p / p.sum(-1, keepdim=True)
        out.append((p @ vf).permute(2, 0, 1, 3).reshape(n, heads, d).to(q.dtype))
        t += n
    return torch.cat(out)


def _plain_verify(s):
    """A walk down each request's tree, all requests side by side. At a node the residual r begins as the target's row and
    its mass Z as one. Child x with the number u is accepted where u Z q(x) < r(x) (1 - s), s being what its earlier
    siblings had of q; otherwise r becomes max(r - Z / (1 - s) q, 0) and q(x) goes to s. (Without q: u Z < r(x), and Z loses
    r(x).) Behind the last accepted node a token is drawn from r."""
    c, p, q, tok = s["case"], s["target_probs"], s["draft_probs"], s["tokens"].long()
    cu, u, par = s["cu_q"].long(), s["uniforms"].double(), s["parents"].long()
    b, v, most = c["batch"], c["vocab"], c["most"]
    start, n = cu[:-1], cu[1:] - cu[:-1]
    rows = torch.arange(b, device="cuda")
    clean = lambda x: torch.where((x > 0) & (x < float("inf")), x.double(), torch.zeros((), dtype=torch.float64, device="cuda"))  # noqa: E731
    first = start.clamp(max=max(tok.numel() - 1, 0))
    r = clean(p[first])
    qr = clean(q[first]) if q is not None else None
    z, sib = torch.ones(b, dtype=torch.float64, device="cuda"), torch.zeros(b, dtype=torch.float64, device="cuda")
    node, count = torch.zeros_like(n), (n > 0).long()
    tokens = torch.full((b, most), -1, device="cuda", dtype=torch.long)
    path = tokens.clone()
    path[:, 0] = torch.where(n > 0, 0, -1)
    for i in range(1, max(_lengths(c)[1])):
        at = (start + i).clamp(max=tok.numel() - 1)
        here = (i < n) & (par[at] == node) & (count < most)
        x = tok[at]
        rx = r[rows, x]
        if q is not None:
            qx, d = qr[rows, x], 1.0 - sib
            yes = here & (u[at] * z * qx < rx * d)
        else:
            yes = here & (u[at] * z < rx)
        no = here & ~yes
        if q is not None:
            f = torch.where(no & (d > 0), z / d, torch.zeros_like(z))
            r = torch.where(no[:, None], (r - f[:, None] * qr).clamp(min=0), r)
            z = torch.where(no, r.sum(1), z)
            sib = torch.where(no, sib + qx, sib)
            qr[rows, x] = torch.where(no, torch.zeros_like(qx), qx)
        else:
            r[rows, x] = torch.where(no, torch.zeros_like(rx), rx)
            z = torch.where(no, z - rx, z)
        put = yes[:, None] & (torch.arange(most, device="cuda")[None] == count[:, None])
        path = torch.where(put, i, path)
        tokens = torch.where(yes[:, None] & (torch.arange(most, device="cuda")[None] == count[:, None] - 1), x[:, None], tokens)
        r = torch.where(yes[:, None], clean(p[at]), r)
        if q is not None:
            qr = torch.where(yes[:, None], clean(q[at]), qr)
        z, sib = torch.where(yes, torch.ones_like(z), z), torch.where(yes, torch.zeros_like(sib), sib)
        node, count = torch.where(yes, i, node), count + yes
    r = torch.where((r.sum(1) > 0)[:, None], r, clean(p[(start + node).clamp(max=tok.numel() - 1)]))
    sums = r.cumsum(1)
    x = (sums <= (u[first] * sums[:, -1])[:, None]).sum(1)
    last = v - 1 - (r.flip(1) > 0).int().argmax(1)
    x = torch.where(sums[:, -1] > 0, torch.minimum(x, last), -1)
    put = (n > 0)[:, None] & (torch.arange(most, device="cuda")[None] == count[:, None] - 1)
    tokens = torch.where(put, x[:, None], tokens)
    return [count.to(torch.int32), tokens.to(torch.int32), path.to(torch.int32)]


def _plain_compact(s):
    """Token ``path[k]`` goes to the place of token ``k``. A page takes the largest scale of the pages that its new tokens
    come from, where that is larger than its own, and what it holds is expressed in it."""
    path, counts, table, page = s["path"].long(), s["counts"].long(), s["block_table"].long(), s["page"]
    cu = s["cu_q"].long()
    base = s["seq_lens"].long() - (cu[1:] - cu[:-1])
    k = torch.arange(path.shape[1], device="cuda")[None]
    moves = (k < counts[:, None]) & (path != k)
    zero = torch.zeros_like(path)
    src, dst = (base[:, None] + torch.where(moves, x, zero) for x in (path, k))
    col = lambda x: (x // page).clamp(max=table.shape[1] - 1)  # noqa: E731
    sp, dp = table.gather(1, col(src)).flatten(), table.gather(1, col(dst)).flatten()
    so, do, moves = (src % page).flatten(), (dst % page).flatten(), moves.flatten()
    for n in ("k", "v"):
        cache, scale = s[n + "_cache"], s[n + "_scale"]
        codes = cache.view(torch.uint8)[sp, :, so].view(cache.dtype).float()  # [moves, heads, D]
        old = scale[sp]
        new = scale.clone().index_reduce_(0, dp, torch.where(moves[:, None], old, torch.zeros_like(old)), "amax")
        ratio = torch.where(new > scale, scale / new, torch.ones_like(scale))
        cache.copy_(_to8(cache.float() * ratio[:, :, None, None], cache.dtype))
        to, kept = new[dp], cache.view(torch.uint8)[dp, :, do]
        there = _to8(codes * (old / to)[:, :, None], cache.dtype).view(torch.uint8)
        # (places that nothing moves to stand for the request's first token, which stays; a padding row has none)
        cache.view(torch.uint8)[dp[moves], :, do[moves]] = torch.where(moves[:, None, None], there, kept)[moves]
        scale.copy_(new)
    return [s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], (base + counts).to(torch.int32)]


def run(state):
    if own:
        return _own_run(state)
    return {"norm": _plain_norm, "tables": _plain_tables, "attend": _plain_attend, "verify": _plain_verify,
            "compact": _plain_compact}[state["case"]["op"]](state)


# ------------------------------------------------------------------ the definition, in 64 bits
def _exact_norm(c, s):
    """As complex numbers: a pair of channels is multiplied by e^(i angle), its gradient by the conjugate."""
    half = c["rot"] // 2
    pos = s["positions"].double()
    phase = torch.stack([pos * math.exp(-math.log(c["base"]) * 2 * m / c["rot"]) for m in range(half)], -1)
    turn = torch.polar(torch.ones_like(phase), phase).unsqueeze(1)
    channel = torch.arange(c["rot"], device="cuda")
    one, two = (channel[0::2], channel[1::2]) if c["interleaved"] else (channel[:half], channel[half:])

    def rotate(x, by):
        z, y = torch.complex(x[..., one], x[..., two]) * by, x.clone()
        y[..., one], y[..., two] = z.real, z.imag
        return y

    outs, grads, weights = [], [], []
    for n in ("q", "k"):
        x, w = s[n].detach().double(), s[n + "_weight"]
        gain = w.detach().double() + c["offset"] if w is not None else torch.ones(c["head_dim"], dtype=torch.float64, device="cuda")
        size = torch.sqrt((x ** 2).sum(-1, keepdim=True) / c["head_dim"] + 1e-6)
        outs.append(rotate(x / size * gain, turn))
        if c["train"]:
            g = rotate(s["d" + n].double(), turn.conj())
            if w is not None:
                weights.append((g * x / size).flatten(0, -2).sum(0))
            g = g * gain
            grads.append(g / size - x * (g * x).sum(-1, keepdim=True) / (c["head_dim"] * size ** 3))
    return outs + grads + weights


def _exact_attend(c, s, seed):
    heads, d, page, out, t = c["heads"], c["head_dim"], c["page"], [], 0
    for b, (k0, n) in enumerate(zip(*_lengths(c))):
        if n == 0:
            continue
        parents, chains = _trees(c, seed)[b], []
        for i in range(n):  # the nodes that node i sees, in their order
            chains.append([i] if parents[i] < 0 else chains[parents[i]] + [i])
        pg = s["block_table"][b, :_pages(k0 + n, page)].long()
        k, v = ((s[x + "_cache"][pg].double() * s[x + "_scale"][pg].double()[:, :, None, None]).transpose(0, 1).flatten(1, 2)
                for x in ("k", "v"))
        for i in range(n):
            see = torch.tensor(list(range(k0)) + [k0 + a for a in chains[i]], device="cuda")
            away = torch.arange(see.numel(), device="cuda") - (see.numel() - 1)  # a path's positions follow one another
            if c["window"]:
                see, away = see[-c["window"]:], away[-c["window"]:]
            qs = s["q"][t + i].double().view(c["heads_kv"], -1, d)
            x = torch.einsum("hgd,hkd->hgk", qs, k[:, see]).reshape(heads, -1) * d ** -0.5
            hp = None if s["head_param"] is None else s["head_param"].double()[:, None]
            if c["kind"] == "softcap":
                x = 50 * torch.tanh(x / 50)
            if c["kind"] == "alibi":
                x = x + hp * away
            if c["kind"] == "temp":
                x = x * hp
            if c["kind"] == "sigmoid":
                w = torch.sigmoid(x - 6)
            elif c["kind"] == "relu":
                w = torch.relu(x) * 0.001
            else:
                w = torch.softmax(x, 1)
            out.append(torch.einsum("hgk,hkd->hgd", w.view(c["heads_kv"], -1, see.numel()), v[:, see]).reshape(heads, d))
        t += n
    return torch.stack(out)


def _exact_compact(c, s, seed):
    paths, (ks, ns), page = _paths(c, seed), _lengths(c), c["page"]
    table, whole = s["block_table"].cpu().tolist(), []
    for x in ("k", "v"):
        cache, scale = s[x + "_cache"].double(), s[x + "_scale"].double()
        before, old = cache.clone(), scale.clone()
        for b, p in enumerate(paths):
            moves = [(ks[b] + f, ks[b] + k) for k, f in enumerate(p) if f != k]
            places = [((table[b][f // page], f % page), (table[b][t // page], t % page)) for f, t in moves]
            for (sp, _), (dp, _) in places:
                scale[dp] = torch.maximum(scale[dp], old[sp])
            for dp in sorted({d[0] for _, d in places}):
                cache[dp] = _exact_round(before[dp] * (old[dp] / scale[dp])[:, None, None], c["cache"])
            for (sp, so), (dp, do) in places:
                cache[dp][:, do] = _exact_round(before[sp][:, so] * (old[sp] / scale[dp])[:, None], c["cache"])
        whole += [cache if c["cache"] == "e4m3" else None, scale]
    return [whole[0], whole[2], whole[1], whole[3], None]


def _exact_round(x, cache):
    if cache == "int8":
        return torch.round(x).clamp(-127, 127)
    _, e = torch.frexp(x.abs())
    unit = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)  # spacing of e4m3 numbers beside x
    return (torch.round(x / unit) * unit).clamp(-448, 448)


def exact(case, seed):
    c = case
    if c["op"] in ("tables", "verify"):  # whole numbers
        return None
    s = prepare(c, seed)
    if c["op"] == "norm":
        return _exact_norm(c, s)
    if c["op"] == "attend":
        ks, ns = _lengths(c)  # (the definition goes token by token)
        if sum(n * (5e-4 + 3e-9 * k * c["heads_kv"]) for k, n in zip(ks, ns)) > 15:
            return None
        return _exact_attend(c, s, seed)
    return _exact_compact(c, s, seed)
