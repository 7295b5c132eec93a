"""Serving several requests at once from a paged 8-bit K/V cache.

A small decoder with random weights (attention layers only, of head size 128, with grouped K/V heads and capped scores,
every other layer with a sliding window) answers requests as they come: prompts go in by chunks, next to the single tokens
of the requests that answer already, and the pages of those that are done are handed out again. The host decides how many
tokens each request gets in a step; lengths, pages and tokens stay on the GPU, and no step waits for the host to read them.

    python examples/paged_serving.py [--requests 9] [--slots 4] [--new 12] [--dtype e4m3|int8]

At the end the logits are compared with those of the same layers over whole sequences in 16 bits.
"""

import argparse
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import chia_proj_b200 as cp  # noqa: E402

CAP = 50.0


class Decoder:
    """``layers`` of attention over a width of ``heads * 64``; layer 0, 2, .. see ``window`` tokens."""

    def __init__(self, layers=2, heads=8, heads_kv=2, head_dim=128, vocab=512, window=64, seed=0, device="cuda"):
        self.heads, self.heads_kv, self.head_dim = heads, heads_kv, head_dim
        width = heads * 64
        g = torch.Generator().manual_seed(seed)

        def weight(*shape):
            return (torch.randn(*shape, generator=g) * shape[0] ** -0.5).to(torch.bfloat16).to(device)

        self.embed = torch.randn(vocab, width, generator=g).to(torch.bfloat16).to(device)
        self.wqkv = [weight(width, (heads + 2 * heads_kv) * head_dim) for _ in range(layers)]
        # (averages over many keys are small; times four they weigh as much as the tokens themselves)
        self.wo = [weight(heads * head_dim, width) * 4 for _ in range(layers)]
        self.masks = [cp.CAUSAL if i % 2 else cp.Mask(left=window - 1, right=0) for i in range(layers)]
        freq = torch.exp(torch.arange(0, width, 2) * (-9.0 / width))
        self.freq = freq.to(device)

    def run(self, ids, positions, attend):
        """Logits ``[T, vocab]`` of tokens ``ids`` at ``positions``; ``attend(layer, q, k, v)`` on ``[T, heads, D]``."""
        angle = positions[:, None].float() * self.freq
        x = self.embed[ids].float() + torch.cat([angle.sin(), angle.cos()], -1)
        for i, (wqkv, wo) in enumerate(zip(self.wqkv, self.wo)):
            qkv = F.rms_norm(x, x.shape[-1:]).to(torch.bfloat16) @ wqkv
            q, k, v = qkv.view(len(ids), -1, self.head_dim).split([self.heads, self.heads_kv, self.heads_kv], 1)
            x = x + (attend(i, q, k, v).flatten(1) @ wo).float()
        return F.rms_norm(x, x.shape[-1:]).to(torch.bfloat16) @ self.embed.t()


class Server:
    """``slots`` requests at a time over ``pages`` pages of ``page_size`` tokens."""

    def __init__(self, model, slots=4, pages=64, page_size=16, most=512, dtype=torch.float8_e4m3fn, chunk=48):
        self.model, self.page_size, self.chunk = model, page_size, chunk
        dev = model.embed.device
        self.caches = [cp.new_cache(pages, model.heads_kv, model.head_dim, page_size=page_size, dtype=dtype, device=dev)
                       for _ in model.wqkv]
        self.table = torch.zeros(slots, -(-most // page_size), dtype=torch.int32, device=dev)
        self.free_pages = torch.arange(pages, dtype=torch.int32, device=dev)
        self.free_state = torch.tensor([0, pages], dtype=torch.int32, device=dev)
        self.lens = torch.zeros(slots, dtype=torch.int32, device=dev)
        self.last = torch.zeros(slots, dtype=torch.int64, device=dev)

    def step(self, prompt, answering):
        """One step. ``prompt[b]``: the prompt tokens that slot ``b`` takes now; ``answering[b]``: it takes the token it
        answered last. Logits ``[slots, vocab]`` of each slot's newest token, which decide the next answer."""
        new = [len(p) or int(a) for p, a in zip(prompt, answering)]
        total, dev = sum(new), self.lens.device
        known = torch.tensor([t for p, a in zip(prompt, answering) for t in (p or [-1] * int(a))]).to(dev)
        owner = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).to(dev)
        ids = torch.where(known < 0, self.last[owner], known)
        st = cp.page_tables(self.lens, torch.tensor(new, dtype=torch.int32).to(dev), self.table, self.free_pages,
                            self.free_state, page_size=self.page_size, max_tokens=total)

        def attend(i, q, k, v):
            cp.cache_append(k, v, st.slots, *self.caches[i])
            return cp.paged_attention(q, *self.caches[i], self.table, st.seq_lens, st.cu_q, max_q=max(new),
                                      mod="softcap", softcap=CAP, mask=self.model.masks[i])

        logits = self.model.run(ids, st.positions, attend)[(st.cu_q[1:].long() - 1).clamp_(min=0)]
        self.last = torch.where(torch.tensor(new).to(dev) > 0, logits.argmax(-1), self.last)
        self.lens, self.free_state = st.seq_lens, st.free_state
        return logits

    def release(self, done):
        """Give back the pages of the slots in ``done``."""
        if any(done):
            self.lens, self.free_state = cp.release_pages(
                torch.tensor(done, dtype=torch.int32).to(self.lens.device), self.lens, self.table, self.free_pages,
                self.free_state, page_size=self.page_size)


def serve(server, prompts, new):
    """Answer each of ``prompts`` with ``new`` tokens. Per request its answer and the logits that it was chosen by."""
    waiting, slots = list(range(len(prompts))), [None] * len(server.lens)
    answers, logits, steps = [[] for _ in prompts], [[] for _ in prompts], 0
    while waiting or any(s is not None for s in slots):
        for b in range(len(slots)):
            if slots[b] is None and waiting:
                slots[b] = [waiting.pop(0), 0]  # request, prompt tokens that are in
        chunk = [prompts[s[0]][s[1]:s[1] + server.chunk] if s else [] for s in slots]
        out = server.step(chunk, [s is not None and not c for s, c in zip(slots, chunk)])
        steps += 1
        done = [0] * len(slots)
        for b, s in enumerate(slots):
            if s is None:
                continue
            s[1] += len(chunk[b])
            if s[1] == len(prompts[s[0]]):  # the whole prompt is in: this step's logits answer
                answers[s[0]].append(server.last[b])
                logits[s[0]].append(out[b])
                if len(answers[s[0]]) == new:
                    slots[b], done[b] = None, 1
        server.release(done)
    cp.check_device_status(server.lens.device.index or 0)
    return [torch.stack(a).tolist() for a in answers], [torch.stack(x) for x in logits], steps


def whole(model, ids):
    """The same logits with every layer over the whole sequence in 16 bits."""
    ids = torch.tensor(ids, device=model.embed.device)

    def attend(i, q, k, v):
        q, k, v = (t.transpose(0, 1)[None] for t in (q, k, v))
        return cp.attention(q, k, v, mod="softcap", softcap=CAP, mask=model.masks[i])[0].transpose(0, 1)

    return model.run(ids, torch.arange(len(ids), device=ids.device), attend)


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--requests", type=int, default=9)
    ap.add_argument("--slots", type=int, default=4)
    ap.add_argument("--new", type=int, default=12)
    ap.add_argument("--dtype", choices=["e4m3", "int8"], default="e4m3")
    args = ap.parse_args(argv)
    model = Decoder()
    server = Server(model, slots=args.slots, dtype=torch.int8 if args.dtype == "int8" else torch.float8_e4m3fn)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 512, (int(torch.randint(1, 150, (1,), generator=g)),), generator=g).tolist()
               for _ in range(args.requests)]
    answers, logits, steps = serve(server, prompts, args.new)
    worst = 0.0
    for p, a, x in zip(prompts, answers, logits):
        want = whole(model, p + a)[len(p) - 1:-1].float()
        worst = max(worst, float((x.float() - want).norm() / want.norm()))
    print(f"{args.requests} requests, {sum(map(len, prompts))} prompt tokens, {args.requests * args.new} answered in "
          f"{steps} steps; free pages {int(server.free_state[1])} of {len(server.free_pages)}; "
          f"logits within {worst:.4f} (relative) of 16-bit attention over whole sequences")
    return worst, server


if __name__ == "__main__":
    main()
