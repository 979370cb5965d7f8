"""Serving a batch with one MX-quantised paged KV cache: shared prompt, drafted tokens, verification.

A small Llama with random MXFP4 weights answers several requests that continue one prompt.  The prompt is prefilled
once into shared pages; every step each request drafts the next tokens from its own history (the continuation of the
last bigram), the target runs over all of them in one pass (its K/V appended to the request's pages, attention over the
shared prompt and the own pages), and the verification keeps what the target would have said.

    python rust-fp4-blackwell_b200/examples/serve_mxkv.py --requests 6 --prompt 150 --tokens 40 --draft 3 --format mxfp8
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
from fp4x import ops  # noqa: E402


class Llama:
    """Random-weight Llama whose attention state lives in MxKvCache pages, one cache per layer."""

    def __init__(self, layers=2, dim=256, ffn=512, heads=8, kv_heads=2, head_dim=64, vocab=512, seed=1, max_pos=4096):
        self.heads, self.kv_heads, self.hd, self.vocab, self.max_pos = heads, kv_heads, head_dim, vocab, max_pos
        self.device = torch.device("cuda")
        g = torch.Generator(device="cuda").manual_seed(seed)

        def linear(n, k):  # held as MXFP4; this example multiplies with the values it stands for
            w = torch.randn((n, k), generator=g, device="cuda") / k ** 0.5
            return ops.dequantize_mxfp4(*ops.quantize_mxfp4(w))

        qkv = (heads + 2 * kv_heads) * head_dim
        self.layers = [dict(qkv=linear(qkv, dim), o=linear(dim, heads * head_dim), up=linear(2 * ffn, dim),
                            down=linear(dim, ffn)) for _ in range(layers)]
        self.embed = torch.randn((vocab, dim), generator=g, device="cuda")
        self.head = linear(vocab, dim) * 4.0
        self.cos, self.sin = ops.rope_tables(max_pos, head_dim, 10000.0)

    def _rope(self, x, pos):
        c, s = self.cos[pos][..., None, :], self.sin[pos][..., None, :]
        a, b = x.chunk(2, -1)
        return torch.cat((a * c - b * s, a * s + b * c), -1)

    def forward(self, tokens, pos, slots, attend):
        """tokens, pos, slots [batch][t]; attend(layer, q) runs the attention of q [batch][t][heads][hd]."""
        b, t = tokens.shape
        x = self.embed[tokens.long()]
        for i, w in enumerate(self.layers):
            h = torch.nn.functional.rms_norm(x, (x.shape[-1],), eps=1e-5)
            q, k, v = (h @ w["qkv"].T).view(b, t, -1, self.hd).split((self.heads, self.kv_heads, self.kv_heads), 2)
            q, k = self._rope(q, pos), self._rope(k, pos)
            ops.kv_append_mx(self.caches[i], slots.flatten(), k.flatten(0, 1), v.flatten(0, 1))
            x = x + attend(i, q.contiguous()).flatten(2) @ w["o"].T
            h = torch.nn.functional.rms_norm(x, (x.shape[-1],), eps=1e-5)
            gate, up = (h @ w["up"].T).chunk(2, -1)
            x = x + (torch.nn.functional.silu(gate) * up) @ w["down"].T
        return torch.nn.functional.rms_norm(x, (x.shape[-1],), eps=1e-5) @ self.head.T


def lookup_drafts(history, k):
    """Up to k tokens that followed the last bigram's previous occurrence."""
    for at in range(len(history) - 3, 0, -1):
        if history[at - 1:at + 1] == history[-2:]:
            return history[at + 1:at + 1 + k]
    return []


def serve(model, prompt, requests, n_tokens, draft, fmt="mxfp8", page=32, temperature=0.0, seed=0):
    """Continues `prompt` for every request (a list of its own first tokens).  Returns (tokens, target passes)."""
    B, P, dev = len(requests), len(prompt), model.device
    if not all(requests):
        raise ValueError("every request needs a token of its own")
    # A request may end with up to `draft` tokens more than it wanted, all but the last of them cached; while others go
    # on, passes still write their 1 + draft rows after them.
    most = max(map(len, requests)) + n_tokens + 2 * draft
    if P + most > model.max_pos:
        raise ValueError(f"{P + most} positions, and the model has {model.max_pos}")
    room = -(-most // page)  # own pages per request
    shared = -(-P // page)
    model.caches = [ops.MxKvCache.empty(shared + B * room, model.kv_heads, model.hd, page, fmt, dev) for _ in model.layers]
    prefix_pages = torch.arange(shared, dtype=torch.int32, device=dev)
    table = (shared + torch.arange(B * room, dtype=torch.int32, device=dev)).view(B, room)
    g = torch.Generator(device=dev).manual_seed(seed)

    # the prompt once, in passes of up to 64 tokens, as one sequence over the shared pages
    for at in range(0, P, 64):
        part = torch.tensor([prompt[at:at + 64]], dtype=torch.int32, device=dev)
        t = part.shape[1]
        pos = (at + torch.arange(t, device=dev))[None]
        lens = torch.tensor([at + t], dtype=torch.int32, device=dev)
        model.forward(part, pos, pos.int(),
                      lambda i, q: ops.attn_paged_mx(model.caches[i], q, prefix_pages[None], lens))

    def step(new, own):
        """Runs new [B][t] after own[b] cached positions; returns the logits."""
        t = new.shape[1]
        at = own[:, None] + torch.arange(t, device=dev)
        slots = (table.gather(1, (at // page).long()) * page + at % page).int()
        lens = (own + t).int()
        return model.forward(new, P + at, slots,
                             lambda i, q: ops.attn_shared_mx(model.caches[i], q, prefix_pages, P, table, lens))

    out = [list(r) for r in requests]
    own = torch.zeros(B, dtype=torch.long, device=dev)
    passes = 0
    while min(len(o) - len(r) for o, r in zip(out, requests)) < n_tokens:
        # tokens whose K/V are not cached yet, then the drafts; rows are padded to the longest
        done = own.tolist()
        known = [o[d:] for o, d in zip(out, done)]
        drafts = [lookup_drafts(prompt + o, draft) if len(o) - len(r) < n_tokens else [] for o, r in zip(out, requests)]
        width = max(map(len, known)) + draft
        rows = torch.tensor([(n + d + [0] * width)[:width] for n, d in zip(known, drafts)], dtype=torch.int32, device=dev)
        logits = step(rows, own)
        passes += 1
        first = torch.tensor([len(n) - 1 for n in known], device=dev)
        pick = logits.gather(1, (first[:, None] + torch.arange(draft + 1, device=dev))[..., None].expand(-1, -1, model.vocab))
        accepted, tokens, _ = ops.verify_drafts(
            pick, torch.tensor([(d + [0] * draft)[:draft] for d in drafts], dtype=torch.int32, device=dev).view(B, draft),
            torch.rand((B, draft), generator=g, device=dev),
            torch.empty((B, model.vocab), device=dev).exponential_(generator=g),
            draft_lens=torch.tensor(list(map(len, drafts)), dtype=torch.int32, device=dev),
            temperature=torch.full((B,), temperature, device=dev))
        # the known tokens and the accepted drafts are cached now; rejected rows are overwritten later
        for b, (n, row) in enumerate(zip(accepted.tolist(), tokens.tolist())):
            if len(out[b]) - len(requests[b]) < n_tokens:
                own[b] = done[b] + len(known[b]) + n
                out[b] += row[: n + 1]
    return [o[len(r):len(r) + n_tokens] for o, r in zip(out, requests)], passes


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--requests", type=int, default=6)
    ap.add_argument("--prompt", type=int, default=150)
    ap.add_argument("--tokens", type=int, default=40)
    ap.add_argument("--draft", type=int, default=3)
    ap.add_argument("--format", choices=("mxfp8", "mxfp4"), default="mxfp8")
    a = ap.parse_args(argv)
    model = Llama()
    g = torch.Generator().manual_seed(7)
    prompt = torch.randint(0, model.vocab, (a.prompt,), generator=g).tolist()
    requests = [torch.randint(0, model.vocab, (1 + i % 3,), generator=g).tolist() for i in range(a.requests)]
    plain, n0 = serve(model, prompt, requests, a.tokens, 0, a.format)
    drafted, n1 = serve(model, prompt, requests, a.tokens, a.draft, a.format)
    same = sum(x == y for p, d in zip(plain, drafted) for x, y in zip(p, d)) / (a.tokens * a.requests)
    print(f"{a.requests} requests, {a.tokens} tokens each: {n0} target passes without drafts, {n1} with up to {a.draft}; "
          f"{100 * same:.1f}% of the tokens alike")
    return plain, drafted, n0, n1


if __name__ == "__main__":
    main()
