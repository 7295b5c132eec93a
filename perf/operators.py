"""The operators of serving from a paged 8-bit K/V cache: what is measured of them, and their plain forms.

One step of a serving loop: the tables and slot maps of the step are built from the requests' lengths
(``page_tables``), the new tokens' keys and values go into the cache in 8 bits with a power-of-two scale for each
(page, head) (``cache_append``), and the step's queries attend to the cache (``paged_attention``).

Layouts. Caches ``[pages, heads_kv, page, head_dim]`` in float8_e4m3fn or int8, scales ``[pages, heads_kv]`` in
fp32; queries ``[tokens, heads, head_dim]``, requests one after another (``cu_q``); a request's queries are the last
tokens of its ``seq_lens`` keys; ``block_table[b, n]`` is the page of its tokens ``[n * page, (n + 1) * page)``.
"""

import math
import random

import torch

own = False

E4M3, INT8 = torch.float8_e4m3fn, torch.int8
TOP = {E4M3: 448.0, INT8: 127.0}
MIN_EXP = -64  # the smallest scale is 2^-64


# ------------------------------------------------------------------ the cases
def _attend(name, **kw):
    d = dict(name=name, op="attend", batch=1, q_len=1, keys=512, ragged=False, heads=32, heads_kv=8, head_dim=128,
             page=64, cache="e4m3", dtype="bf16", kind="softmax", window=0, prefix=0)
    d.update(kw)
    return d


def _append(name, **kw):
    d = dict(name=name, op="append", batch=1, q_len=1, ragged=False, heads_kv=8, head_dim=128, page=64, cache="e4m3",
             dtype="bf16")
    d.update(kw)
    return d


def _tables(name, **kw):
    d = dict(name=name, op="tables", batch=1, q_len=1, keys=512, ragged=False, page=64)
    d.update(kw)
    return d


def listed():
    return [
        # one user's chat on an otherwise idle GPU: nothing but latency
        _attend("attend one", keys=601),
        # the decode step of this repository's benchmark (B8 H32, 4 K/V heads, 8192 keys), Gemma-2 style softcap
        _attend("attend decode", batch=8, keys=8192, heads_kv=4, kind="softcap"),
        # continuous batching: very unequal lengths, a padding row with no keys, small pages
        _attend("attend ragged", batch=96, keys=16384, ragged=True, heads=64, page=16),
        # sliding window over long contexts: few pages of each request are read; int8, D = 64
        _attend("attend window", batch=48, keys=20000, ragged=True, head_dim=64, cache="int8", dtype="fp16", window=1024),
        # speculative decoding: up to five drafted tokens a request are checked in one pass, ALiBi
        _attend("attend drafts", batch=24, q_len=5, keys=4100, ragged=True, heads=16, heads_kv=4, page=32, kind="alibi"),
        # the largest: long contexts at a full batch
        _attend("attend long", batch=64, keys=32768, heads=64, page=128),
        # chunked prefill: chunks of up to 1024 new tokens over contexts already in the cache
        _attend("attend chunk", batch=4, q_len=1024, keys=8192, ragged=True),
        # a decode step's write: one token a request, most into a page that holds tokens already
        _append("append decode", batch=64),
        # a prefill's write: whole prompts, odd lengths
        _append("append prompts", batch=16, q_len=4099, ragged=True),
        # the tables of a decode step
        _tables("tables decode", batch=64, keys=8192, ragged=True),
        # the tables of a step that admits many prompts
        _tables("tables prompts", batch=512, q_len=300, keys=4096, ragged=True, page=16),
        # a whole decode step of one layer: tables, write, attention
        dict(_attend("step", batch=32, keys=4096, ragged=True, kind="temp"), op="step"),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "attend", "append", "append", "tables", "step"])
    page = rng.choice([16, 32, 64, 128])
    if op == "tables":
        c = _tables("", batch=_spread(rng, 1, 1024), q_len=rng.choice([1, 1, _spread(rng, 2, 300)]),
                    keys=_spread(rng, 64, 8192), ragged=rng.random() < 0.7, page=page)
        del c["name"]
        return c
    head_dim, heads_kv = rng.choice([64, 128, 128]), rng.choice([1, 2, 4, 8])
    cache, dtype = rng.choice(["e4m3", "e4m3", "int8"]), rng.choice(["bf16", "bf16", "fp16"])
    if op == "append":
        batch = _spread(rng, 1, 128)
        c = _append("", batch=batch, q_len=_spread(rng, 1, 60000 // batch) if rng.random() < 0.5 else 1,
                    ragged=rng.random() < 0.6, heads_kv=heads_kv, head_dim=head_dim, page=page, cache=cache, dtype=dtype)
        del c["name"]
        return c
    group = rng.choice([1, 2, 4, 4, 7, 8, 8])
    chunk = op == "attend" and rng.random() < 0.2
    if chunk:
        batch, q_len = _spread(rng, 1, 4), _spread(rng, 40, 1024)
        keys = _spread(rng, q_len, 8192)
        group = min(group, 4)
    else:
        batch, q_len = _spread(rng, 1, 96), 1 if op == "step" else rng.choice([1, 1, 1, 2, 3, 4])
        keys = _spread(rng, 64, min(32768, 800000 // batch))
    c = _attend("", batch=batch, q_len=q_len, keys=keys, ragged=rng.random() < 0.7, heads=group * heads_kv,
                heads_kv=heads_kv, head_dim=head_dim, page=page, cache=cache, dtype=dtype,
                kind=rng.choice(["softmax", "softmax", "softcap", "alibi", "temp", "sigmoid", "relu"]),
                window=_spread(rng, 64, 4096) if rng.random() < 0.25 else 0,
                prefix=_spread(rng, 1, 64) if rng.random() < 0.15 else 0)
    c["op"] = op
    del c["name"]
    return c


def _lengths(c):
    """(keys of each request, queries of each request); a property of the case. Ragged: spread over the logarithm,
    the last of four requests or more is a padding row (one query and no keys; no tokens in the other operators)."""
    b, q, attends = c["batch"], c["q_len"], c["op"] == "attend"
    keys = c.get("keys", c["page"])
    if not c["ragged"]:
        if attends or c["op"] == "append":
            return [max(keys, q)] * b, [q] * b
        return [max(keys, q) - (7 * i) % max(1, min(c["page"], keys - q)) for i in range(b)], [q] * b
    r = random.Random(1000003 * b + 1009 * keys + q)
    ks, qs = [], []
    for i in range(b):
        n = q if i == 0 else 1 + r.randrange(q)
        ks.append(max(keys, n) if i == 0 else _spread(r, n, max(keys, n)))
        qs.append(n)
    if b >= 4:
        ks[-1], qs[-1] = 0, 1 if attends else 0
    return ks, qs


def _context(c):
    """Tokens in the cache before an append; no more than a page, so that the cache is what the write touches."""
    _, qs = _lengths(c)
    if c["q_len"] > 8:  # prompts: from the start of a page, a third of them after a shared beginning
        return [(5 + i) % c["page"] if i % 3 == 2 else 0 for i in range(len(qs))]
    return [(11 * i) % c["page"] for i in range(len(qs))]


def _pages(n, page):
    return -(-n // page)


def _visible(c, n, q):
    """(keys that any of the request's queries sees, pairs of a query and a key that it sees)."""
    lo, pairs = n, 0
    w, pre = c["window"], min(c["prefix"], n)
    for i in range(q):
        p = n - q + i
        if p < 0:
            continue
        a = max(0, p - w + 1) if w else 0
        lo = min(lo, a)
        pairs += p + 1 - a + min(pre, a) + max(0, pre - p - 1)
    return n - lo + min(pre, lo), pairs


def work(case):
    c = case
    ks, qs = _lengths(c)
    tokens, one = sum(qs), 4
    out = {"bytes": 0.0, "flops": 0.0}
    if c["op"] in ("tables", "step"):
        new = sum(_pages(k, c["page"]) - _pages(k - q, c["page"]) for k, q in zip(ks, qs))
        # lengths in and out, new pages read and entered in the table, offsets, a slot and a position for each token
        out["bytes"] += one * (4 * len(ks) + 1 + 2 * new + 2 * tokens + 4)
    if c["op"] in ("append", "step"):
        d = c["heads_kv"] * c["head_dim"]
        ctx = _context(c) if c["op"] == "append" else [k - q for k, q in zip(ks, qs)]
        touched = sum(_pages(x + q, c["page"]) - x // c["page"] for x, q in zip(ctx, qs))
        # 16-bit keys and values in, 8-bit out, the slots, the scales of the touched pages in and out
        out["bytes"] += tokens * (2 * d * 3 + one) + touched * c["heads_kv"] * 2 * 2 * one
    if c["op"] in ("attend", "step"):
        seen = [_visible(c, k, q) for k, q in zip(ks, qs)]
        keys, pairs = sum(s[0] for s in seen), sum(s[1] for s in seen)
        d, p = c["head_dim"], sum(_pages(s[0], c["page"]) for s in seen)
        # queries in and outputs out, keys and values of the visible keys once, scales and table entries of their pages
        out["bytes"] += 4 * tokens * c["heads"] * d + 2 * keys * c["heads_kv"] * d + p * (c["heads_kv"] * 8 + 4)
        out["flops"] += 4.0 * d * pairs * c["heads"]
    return out


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


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    ks, qs = _lengths(c)
    page, b = c["page"], c["batch"]
    st = {"case": c, "page": page, "tokens": sum(qs), "q_len": c["q_len"]}
    if c["op"] != "tables":
        cache = E4M3 if c["cache"] == "e4m3" else INT8
        dtype = torch.bfloat16 if c["dtype"] == "bf16" else torch.float16
        hkv, d = c["heads_kv"], c["head_dim"]
        kch, vch = _channels(hkv, d, g), _channels(hkv, d, g) * 0.5
    if c["op"] == "append":
        ctx = _context(c)
        ks = [x + q for x, q in zip(ctx, qs)]
    else:
        ctx = [k - q for k, q in zip(ks, qs)]
    need = [_pages(max(k, 0), page) for k in ks]
    spare = 3 if c["op"] == "append" else 8
    held = [_pages(max(x, 0), page) for x in ctx] if c["op"] in ("tables", "step") else need
    total = sum(need) + spare
    perm = torch.randperm(total, device="cuda", generator=g).to(torch.int32)  # pages are handed out in any order
    width = max(need) + (4 if c["op"] in ("tables", "step") else 0)
    at = torch.cumsum(torch.tensor([0] + held[:-1], device="cuda"), 0)
    col = torch.arange(width, device="cuda")
    inside = col[None] < torch.tensor(held, device="cuda")[:, None]
    table = torch.where(inside, perm[(at[:, None] + col[None]).clamp(max=total - 1)], torch.zeros((), dtype=torch.int32, device="cuda"))
    st["block_table"] = table.contiguous()
    if c["op"] in ("tables", "step"):  # the pages that no request holds, in a ring that begins anywhere
        free, n = perm[sum(held):], total - sum(held)
        ring = torch.zeros(total, dtype=torch.int32, device="cuda")
        head = seed % total
        ring[(head + torch.arange(n, device="cuda")) % total] = free
        st.update(seq_lens=ints([max(x, 0) for x in ctx]), new_lens=ints(qs), free_pages=ring, free_state=ints([head, n]))
    if c["op"] in ("append", "step"):
        qkv = torch.randn(st["tokens"], (c.get("heads", 0) + 2 * hkv) * d, device="cuda", generator=g)
        h = c.get("heads", 0) * d
        qkv[:, h:h + hkv * d] *= kch.reshape(1, -1)
        qkv[:, h + hkv * d:] *= vch.reshape(1, -1)
        qkv = qkv.to(dtype).view(st["tokens"], -1, d)  # one projection's output: queries, keys and values beside one another
        st["q"], st["k"], st["v"] = qkv.split([c.get("heads", 0), hkv, hkv], 1)
    if c["op"] == "append":
        slots = []
        host = st["block_table"].cpu().tolist()
        for i in range(b):
            slots += [host[i][p // page] * page + p % page for p in range(ctx[i], ks[i])]
        st["slots"] = ints(slots)
    if c["op"] == "attend":
        st["q"] = torch.randn(st["tokens"], c["heads"], d, device="cuda", generator=g).to(dtype)
        st["seq_lens"] = ints(ks)
        st["cu_q"] = ints([sum(qs[:i]) for i in range(b + 1)])
    if c["op"] != "tables":
        st["k_cache"], st["k_scale"] = _random_cache((total, hkv, page, d), cache, kch, g)
        st["v_cache"], st["v_scale"] = _random_cache((total, hkv, page, d), cache, vch, g)
    if c["op"] in ("attend", "step"):
        heads = c["heads"]
        st["head_param"] = None
        if c["kind"] == "alibi":
            st["head_param"] = torch.pow(2.0, -8.0 * (torch.arange(heads, device="cuda") + 1.0) / heads)
        if c["kind"] == "temp":
            st["head_param"] = 0.5 + torch.arange(heads, device="cuda") / heads
    return st


# ------------------------------------------------------------------ one pass
def _own_attend(cp, s, q, seq_lens, cu_q):
    c = s["case"]
    kw = {"norm": c["kind"]} if c["kind"] in ("sigmoid", "relu") else {}
    if c["kind"] in ("softcap", "alibi", "temp"):
        kw["mod"] = c["kind"]
    mask = cp.Mask(left=c["window"] - 1 if c["window"] else -1, right=0, prefix=c["prefix"])
    return cp.paged_attention(q, s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["block_table"], seq_lens, cu_q,
                              max_q=s["q_len"], mask=mask, softcap=50.0, head_param=s["head_param"], sig_bias=-6.0,
                              out_scale=0.001, **kw)


def _own_run(s):
    import chia_proj_b200 as cp

    op = s["case"]["op"]
    if op == "attend":
        return _own_attend(cp, s, s["q"], s["seq_lens"], s["cu_q"])
    if op == "append":
        cp.cache_append(s["k"], s["v"], s["slots"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
        return [s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]]
    t = cp.page_tables(s["seq_lens"], s["new_lens"], s["block_table"], s["free_pages"], s["free_state"],
                       page_size=s["page"], max_tokens=s["tokens"])
    tables = [t.slots, t.positions, t.cu_q, t.seq_lens, t.free_state, s["block_table"]]
    if op == "tables":
        return tables
    cp.cache_append(s["k"], s["v"], t.slots, s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    out = _own_attend(cp, s, s["q"], t.seq_lens, t.cu_q)
    return [out] + tables + [s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]]


def _plain_tables(s):
    """Pages in request order from the ring's head: request b takes ceil((len + new) / page) - ceil(len / page)."""
    page, lens, new, table = s["page"], s["seq_lens"].long(), s["new_lens"].long(), s["block_table"]
    head, count = s["free_state"][0].long(), s["free_state"][1].long()
    ring = s["free_pages"]
    held = (lens + page - 1) // page
    need = (lens + new + page - 1) // page - held
    fits = held + need <= table.shape[1]
    need = torch.where(fits, need, torch.zeros_like(need))
    upto = need.cumsum(0)
    served = fits & ((need == 0) | (upto <= count))
    got = torch.where(served, need, torch.zeros_like(need))
    first = upto - need  # where the request's new pages begin, counted from the ring's head
    col = torch.arange(table.shape[1], device=table.device)[None]
    entry = ring[(head + first[:, None] + col - held[:, None]).remainder(ring.numel())]
    is_new = (col >= held[:, None]) & (col < (held + got)[:, None])
    table.copy_(torch.where(is_new, entry, table))
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device=table.device), new.cumsum(0)])
    t = torch.arange(s["tokens"], device=table.device)
    b = torch.searchsorted(cu[1:], t, right=True).clamp(max=lens.numel() - 1)
    pos = lens[b] + t - cu[b]
    at = table[b, (pos // page).clamp(max=table.shape[1] - 1)].long() * page + pos % page
    real = t < cu[-1]
    slots = torch.where(real & served[b], at, torch.full_like(at, -1))
    taken = got.sum()
    state = torch.stack([(head + taken).remainder(ring.numel()), count - taken])
    i32 = torch.int32
    return (slots.to(i32), torch.where(real, pos, torch.zeros_like(pos)).to(i32), cu.to(i32),
            torch.where(served, lens + new, lens).to(i32), state.to(i32))


def _plain_put(x, slots, cache, scale):
    """One of K and V into its cache. A page whose first slot is written begins anew; another keeps its scale or,
    where a new token needs a larger one, has its values expressed in that."""
    pages, heads, page, _ = cache.shape
    keep = slots >= 0
    x, at = x[keep].float(), slots[keep].long()
    where = at // page
    finite = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(2)
    amax = torch.zeros(pages, heads, device=x.device).index_reduce_(0, where, finite, "amax")
    marks = torch.zeros(2, pages, device=x.device)
    hit = marks[0].index_fill(0, where, 1.0) > 0
    fresh = marks[1].index_reduce(0, where, (at % page == 0).float(), "amax") > 0
    wanted = _power(_exponent(amax, TOP[cache.dtype]))
    new = torch.where(hit[:, None], torch.where(fresh[:, None], wanted, torch.maximum(wanted, scale)), scale)
    ratio = torch.where((hit & ~fresh)[:, None], scale / new, torch.ones_like(scale))
    cache.copy_(_to8(cache.float() * ratio[:, :, None, None], cache.dtype))
    cache.view(torch.uint8)[where, :, at % page] = _to8(x / new[where][:, :, None], cache.dtype).view(torch.uint8)
    scale.copy_(new)


def _plain_attend(s, q, seq_lens, cu_q):
    c = s["case"]
    heads, d = q.shape[1:]
    hkv, page = s["k_cache"].shape[1:3]
    group, n_q, b = heads // hkv, s["q_len"], seq_lens.numel()
    table = s["block_table"].long()
    table = table[:, :_pages(max(max(_lengths(c)[0]), 1), page)]
    keys = table.shape[1] * page

    def dense(cache, scale):  # [B, Hkv, keys, D]
        x = cache[table].float() * scale[table][..., None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(b, hkv, keys, d)

    i = torch.arange(n_q, device=q.device)
    lens, start = seq_lens.long(), cu_q.long()
    count = start[1:] - start[:-1]
    at = (start[:-1, None] + i).clamp(max=q.shape[0] - 1)
    qp = q[at].float().view(b, n_q, hkv, group, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, n_q * group, d)
    pos = (lens - count)[:, None] + i  # [B, n_q]
    j = torch.arange(keys, device=q.device)
    x = torch.matmul(qp, dense(s["k_cache"], s["k_scale"]).transpose(2, 3)).mul_(1.0 / math.sqrt(d))
    x = x.view(b, hkv, n_q, group, keys)
    hp = None if s["head_param"] is None else s["head_param"].view(hkv, 1, group, 1)
    if c["kind"] == "softcap":
        x = 50.0 * torch.tanh(x / 50.0)
    elif c["kind"] == "alibi":
        x = x + hp * (j[None, None] - pos[..., None]).float()[:, None, :, None]
    elif c["kind"] == "temp":
        x = x * hp
    see = j[None, None] <= pos[..., None]
    if c["window"]:
        see = see & (pos[..., None] - j < c["window"])
    see = (see | (j < c["prefix"])) & (j < lens[:, None, None])
    see = see[:, None, :, None]
    if c["kind"] == "sigmoid":
        p = torch.where(see, torch.sigmoid(x - 6.0), torch.zeros_like(x))
    elif c["kind"] == "relu":
        p = torch.where(see, x.clamp(min=0), torch.zeros_like(x))
    else:
        x = x.masked_fill(~see, float("-inf"))
        top = x.amax(-1, keepdim=True)
        p = torch.exp(x - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
        total = p.sum(-1, keepdim=True)
    # the masked places of a cache may hold anything
    live = (j < lens[:, None])[:, None, :, None]
    v = torch.where(live, dense(s["v_cache"], s["v_scale"]), torch.zeros((), device=q.device))
    o = torch.matmul(p.view(b, hkv, n_q * group, keys), v).view(b, hkv, n_q, group, d)
    if c["kind"] == "relu":
        o = o * 0.001
    elif c["kind"] != "sigmoid":
        o = torch.where(total > 0, o / total, torch.zeros_like(o))
    o = o.permute(0, 2, 1, 3, 4).reshape(b * n_q, heads, d)
    t = torch.arange(q.shape[0], device=q.device)
    r = torch.searchsorted(start[1:], t, right=True)
    return o[r * n_q + t - start[r]].to(q.dtype)


def run(state):
    if own:
        return _own_run(state)
    s, op = state, state["case"]["op"]
    caches = [s[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")] if op in ("append", "step") else []
    if op == "attend":
        return _plain_attend(s, s["q"], s["seq_lens"], s["cu_q"])
    if op == "append":
        _plain_put(s["k"], s["slots"], s["k_cache"], s["k_scale"])
        _plain_put(s["v"], s["slots"], s["v_cache"], s["v_scale"])
        return caches
    slots, positions, cu, lens, free = _plain_tables(s)
    tables = [slots, positions, cu, lens, free, s["block_table"]]
    if op == "tables":
        return tables
    _plain_put(s["k"], slots, s["k_cache"], s["k_scale"])
    _plain_put(s["v"], slots, s["v_cache"], s["v_scale"])
    return [_plain_attend(s, s["q"], lens, cu)] + tables + caches


# ------------------------------------------------------------------ the definition, in 64 bits
def _exact_power(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_round(x, cache):
    if cache == INT8:
        return torch.round(x).clamp(-127, 127)
    _, e = torch.frexp(x.abs())
    unit = _exact_power((e - 1).clamp(min=-6) - 3)  # spacing of e4m3 numbers beside x
    return (torch.round(x / unit) * unit).clamp(-448, 448)


def _exact_put(x, slots, cache, scale):
    """[pages, heads, page, D] values in units of the scale, and the scales, after the write; page by page."""
    q, sc, page = cache.double(), scale.double().clone(), cache.shape[2]
    by_page = {}
    for t, at in enumerate(slots):
        if at >= 0:
            by_page.setdefault(at // page, []).append((t, at % page))
    for p, rows in by_page.items():
        new = x[[t for t, _ in rows]].double().transpose(0, 1)  # [heads, n, D]
        m, e = torch.frexp((new.abs().amax((1, 2)) / TOP[cache.dtype]).clamp(min=2.0 ** MIN_EXP))
        want = _exact_power(e - (m == 0.5).int())
        if any(o == 0 for _, o in rows):
            s = want
        else:
            s = torch.maximum(want, sc[p])
            q[p] = _exact_round(q[p] * (sc[p] / s)[:, None, None], cache.dtype)
        sc[p] = s
        q[p][:, [o for _, o in rows]] = _exact_round(new / s[:, None, None], cache.dtype)
    return q, sc


def _exact_attend(c, q, kq, ks, vq, vs, table, lens, counts, hp):
    heads, d = q.shape[1:]
    hkv, page = kq.shape[1:3]
    group, out, t = heads // hkv, [], 0
    for b, (n, m) in enumerate(zip(lens, counts)):
        if n == 0:
            out.append(torch.zeros(m, heads, d, dtype=torch.float64, device=q.device))
            t += m
            continue
        pg = table[b, :_pages(n, page)].long()
        k = (kq[pg].double() * ks[pg].double()[:, :, None, None]).transpose(0, 1).reshape(hkv, -1, d)[:, :n]
        v = (vq[pg].double() * vs[pg].double()[:, :, None, None]).transpose(0, 1).reshape(hkv, -1, d)[:, :n]
        per = []
        for h in range(heads):
            x = q[t:t + m, h].double() @ k[h // group].T / math.sqrt(d)
            i = torch.arange(n - m, n, device=q.device)[:, None]
            j = torch.arange(n, device=q.device)[None]
            sees = (j <= i) & ((i - j < c["window"]) if c["window"] else (j >= 0)) | (j < c["prefix"])
            if c["kind"] == "softcap":
                x = 50 * torch.tanh(x / 50)
            if c["kind"] == "alibi":
                x = x + hp[h].double() * (j - i)
            if c["kind"] == "temp":
                x = x * hp[h].double()
            if c["kind"] == "sigmoid":
                p = torch.sigmoid(x - 6) * sees
            elif c["kind"] == "relu":
                p = x.clamp(min=0) * sees * 0.001
            else:
                p = torch.softmax(x.masked_fill(~sees, float("-inf")), 1)
            per.append(p @ v[h // group])
        out.append(torch.stack(per, 1))
        t += m
    return torch.cat(out)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    lens, counts = _lengths(c)
    none = [None] * 6  # the tables are whole numbers
    if c["op"] == "tables":
        return None
    if c["op"] == "attend":
        return _exact_attend(c, s["q"], s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"], s["block_table"], lens,
                             counts, s["head_param"])
    if c["op"] == "append":
        slots = s["slots"].tolist()
    else:  # give out the ring's pages one by one
        table, page = s["block_table"].cpu().tolist(), s["page"]
        ring, (head, _) = s["free_pages"].tolist(), s["free_state"].tolist()
        slots = []
        for b, (n, m) in enumerate(zip(lens, counts)):
            for p in range(_pages(n - m, page), _pages(n, page)):
                table[b][p] = ring[head % len(ring)]
                head += 1
            slots += [table[b][p // page] * page + p % page for p in range(n - m, n)]
        s["block_table"] = torch.tensor(table, device="cuda")
    k, ks = _exact_put(s["k"], slots, s["k_cache"], s["k_scale"])
    v, vs = _exact_put(s["v"], slots, s["v_cache"], s["v_scale"])
    caches = [k, v, ks, vs]
    if s["k_cache"].dtype == INT8:  # whole numbers have to be equal as they are
        caches = [None, None, ks, vs]
    if c["op"] == "append":
        return caches
    return [_exact_attend(c, s["q"], k, ks, v, vs, s["block_table"], lens, counts, s["head_param"])] + none + caches
