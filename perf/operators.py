"""Workloads of the MX-quantised KV cache, the attention that reads it and the verification of drafted tokens.

Five operators, each with a plain form (elementary torch operations in 32 bits, rounded once at the end) and a call of
the framework:

  append  quantise new K/V rows into a paged cache (MXFP8 or MXFP4) and read the written rows back
  read    gather cached rows by slot and dequantise them
  attn    decode attention over the paged cache: 1..8 query tokens per sequence, ragged lengths, grouped heads
  shared  the same for a batch whose sequences continue one shared prefix
  verify  speculative verification of drafted tokens from given random numbers

Cache layout (K and V alike): codes [pages][kv heads][page size][row bytes], E8M0 scales [pages][kv heads][page size][hd/32].
A row holds dimension d = 32 b + 4 g + i (b < hd/32, g < 8, i < 4) at code position (g * hd/32 + b) * 4 + i; MXFP8 is one
E4M3 byte per code, MXFP4 one E2M1 nibble (low nibble first).  The value is code * 2^(scale - 127).
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

FMTS = ("mxfp8", "mxfp4")
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
DTYPE = {"bf16": torch.bfloat16, "f32": torch.float32}


def _ops():
    root = str(Path.cwd() / "rust-fp4-blackwell_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from fp4x import ops
    return ops


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one decode step of 64 requests: each adds one token (the smallest write, latency counts)
        dict(name="append_step_b64_hd128", op="append", fmt="mxfp8", tokens=64, n_kv=8, hd=128, page=64, dtype="f32"),
        # a long prompt written at once into a 4-bit cache
        dict(name="append_prompt_16k_mxfp4", op="append", fmt="mxfp4", tokens=16384, n_kv=8, hd=128, page=16, dtype="bf16"),
        # a short context handed to another consumer, odd length
        dict(name="read_817_hd64_mxfp4", op="read", fmt="mxfp4", tokens=817, n_kv=4, hd=64, page=32, dtype="f32"),
        # all contexts of a batch unpacked (hand-over to a path with a bf16 cache)
        dict(name="read_128k_hd128_mxfp8", op="read", fmt="mxfp8", tokens=131072, n_kv=8, hd=128, page=64, dtype="bf16"),
        # one interactive request with a 32k context
        dict(name="attn_b1_32k_hd128_mxfp8", op="attn", fmt="mxfp8", batch=1, n_kv=8, group=4, hd=128, q_len=1, max_len=32768,
             page=64, dtype="bf16", lens_seed=1),
        # a full batch of ragged contexts up to 16k, single tokens
        dict(name="attn_b64_16k_hd128_mxfp8", op="attn", fmt="mxfp8", batch=64, n_kv=8, group=4, hd=128, q_len=1, max_len=16384,
             page=64, dtype="bf16", lens_seed=2),
        # verification pass of 4 drafted tokens (5 query tokens), 64-wide heads, 4-bit cache, odd lengths
        dict(name="attn_b24_q5_6001_hd64_mxfp4", op="attn", fmt="mxfp4", batch=24, n_kv=4, group=8, hd=64, q_len=5, max_len=6001,
             page=16, dtype="f32", lens_seed=3),
        # few requests on a short system prompt
        dict(name="shared_b6_p1500_hd64_mxfp8", op="shared", fmt="mxfp8", batch=6, n_kv=4, group=8, hd=64, q_len=1, prefix=1500,
             max_len=300, page=32, dtype="f32", lens_seed=4),
        # many requests on one long document, short continuations of their own
        dict(name="shared_b96_p32k_hd128_mxfp8", op="shared", fmt="mxfp8", batch=96, n_kv=8, group=4, hd=128, q_len=1, prefix=32768,
             max_len=1000, page=64, dtype="bf16", lens_seed=5),
        # the same with drafted tokens to verify, 4-bit cache
        dict(name="shared_b32_q4_p8209_mxfp4", op="shared", fmt="mxfp4", batch=32, n_kv=8, group=4, hd=128, q_len=4, prefix=8209,
             max_len=2047, page=16, dtype="bf16", lens_seed=6),
        # one request, 3 drafted tokens, small vocabulary
        dict(name="verify_b1_k3_v32000", op="verify", batch=1, k=3, vocab=32000, dtype="f32", probs=True, lens_seed=7),
        # a batch, ragged drafts, large vocabulary
        dict(name="verify_b64_k5_v128256", op="verify", batch=64, k=5, vocab=128256, dtype="f32", probs=True, lens_seed=8),
    ]


def _log(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))
    n = max(lo, min(hi, n))
    return n - 1 if n == 3072 else n


def draw(rng):
    op = rng.choice(("append", "read", "attn", "attn", "shared", "shared", "verify"))
    if op == "verify":
        vocab = rng.choice((32000, 128256, _log(rng, 1000, 128256)))
        k = rng.randint(1, 8)
        batch = _log(rng, 1, max(1, min(128, 49_000_000 // ((k + 1) * vocab))))
        return dict(op=op, batch=batch, k=k, vocab=vocab, dtype=rng.choice(("f32", "f32", "bf16")), probs=rng.random() < 0.7,
                    lens_seed=rng.randrange(1 << 20))
    hd, n_kv = rng.choice((64, 128)), rng.choice((1, 2, 4, 8))
    case = dict(op=op, fmt=rng.choice(FMTS), n_kv=n_kv, hd=hd, page=rng.choice((16, 32, 64, 128)), dtype=rng.choice(("bf16", "f32")))
    if op in ("append", "read"):
        case["tokens"] = _log(rng, 1, (16384 if op == "append" else 131072) * 8 * 128 // (n_kv * hd * (2 if case["dtype"] == "f32" else 1)))
        return case
    case["group"] = rng.choice((1, 2, 4, 7, 8))
    case["q_len"] = rng.choice((1, 1, 1, rng.randint(2, 8)))
    per = n_kv * hd
    if op == "attn":
        batch = _log(rng, 1, 96)
        top = 64 * 16384 * 8 * 128 // (batch * per)
        if case["q_len"] * case["group"] > 16:
            top //= 4
        case.update(batch=batch, max_len=_log(rng, 1, max(1, min(32768, top))))
    else:
        batch = _log(rng, 2, 96)
        rows = batch * case["q_len"] * case["group"]
        top = 96 * 4 * 32768 * 8 * 128 // (rows * per)
        case.update(batch=batch, prefix=_log(rng, 16, max(16, min(32768, top))), max_len=_log(rng, 1, 2048))
    case["lens_seed"] = rng.randrange(1 << 20)
    return case


def _lens(case):
    """Own lengths of the sequences, the query tokens included: anywhere up to max_len, one of them max_len and, in a batch
    of 4 or more, one without any cached token."""
    rng = random.Random(case["lens_seed"])
    lens = [rng.randint(min(case["q_len"], case["max_len"]), case["max_len"]) for _ in range(case["batch"])]
    lens[rng.randrange(len(lens))] = case["max_len"]
    if len(lens) >= 4:
        i = rng.randrange(len(lens))
        if lens[i] != case["max_len"]:
            lens[i] = 0
    return lens


def _draft_lens(case):
    rng = random.Random(case["lens_seed"])
    return [rng.choice((case["k"], rng.randint(0, case["k"]))) for _ in range(case["batch"])]


def work(case):
    op = case["op"]
    if op == "verify":
        b, k, v = case["batch"], case["k"], case["vocab"]
        size = 4 if case["dtype"] == "f32" else 2
        rows = sum(n + 1 for n in _draft_lens(case))
        # every target row for its normaliser, then one row of draft probabilities and of noise per sequence
        return {"bytes": rows * v * size + b * v * 4 * (2 if case["probs"] else 1) + b * (k + 1) * 16, "flops": 4.0 * rows * v}
    hd, n_kv = case["hd"], case["n_kv"]
    row = (hd if case["fmt"] == "mxfp8" else hd // 2) + hd // 32
    size = 4 if case["dtype"] == "f32" else 2
    if op in ("append", "read"):
        vals = case["tokens"] * n_kv * hd * 2
        held = case["tokens"] * n_kv * row * 2
        return {"bytes": vals * size * (2 if op == "append" else 1) + held * (2 if op == "append" else 1) + 4 * case["tokens"],
                "flops": 2.0 * vals}
    t, heads = case["q_len"], n_kv * case["group"]
    lens = _lens(case)
    io = case["batch"] * t * heads * hd * size * 2
    pairs = sum(max(0, n - t + 1 + i) for n in lens for i in range(t))
    held = sum(lens)
    if op == "shared":
        pairs += case["batch"] * t * case["prefix"]
        held += case["prefix"]
    return {"bytes": held * n_kv * row * 2 + io + 4 * sum(-(-n // case["page"]) for n in lens), "flops": 4.0 * pairs * heads * hd}


# ------------------------------------------------------------------ inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _kv_values(g, rows, n_kv, hd):
    """K/V rows as a model makes them: unit normal with a few strong channels and a magnitude per token."""
    x = _normal(g, rows, n_kv, hd)
    gain = torch.exp2(2.0 * torch.rand((n_kv, hd), generator=g, device="cuda") ** 6)
    return x.mul_(gain).mul_(torch.exp2(_normal(g, rows, 1, 1) * 0.5))


def _quantise(x, fmt):
    """[rows][n_kv][hd] f32 -> (codes [rows][n_kv][row bytes], scales [rows][n_kv][hd/32]), uint8."""
    rows, n_kv, hd = x.shape
    nb = hd // 32
    x = x.float().reshape(rows, n_kv, nb, 8, 4)
    amax = x.abs().amax((-1, -2))
    top = 8 if fmt == "mxfp8" else 2
    e = torch.where(amax > 0, (torch.frexp(amax).exponent - 1 - top + 127).clamp(0, 254), 127)
    y = torch.ldexp(x, (127 - e)[..., None, None])
    y = y.transpose(2, 3).reshape(rows, n_kv, hd)  # row order: g, b, i
    if fmt == "mxfp8":
        codes = y.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        a = y.abs()
        c = torch.zeros(a.shape, dtype=torch.uint8, device=a.device)
        for edge in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0):  # nearest level, ties to the smaller magnitude
            c += a > edge
        c |= (y < 0).to(torch.uint8) << 3
        codes = c[..., 0::2] | (c[..., 1::2] << 4)
    return codes, e.to(torch.uint8)


def _dequantise(codes, scales, fmt):
    """codes [...][row bytes], scales [...][hd/32] -> f32 [...][hd]."""
    nb = scales.shape[-1]
    if fmt == "mxfp8":
        v = codes.view(torch.float8_e4m3fn).float()
    else:
        table = torch.tensor(E2M1, device=codes.device)
        v = table[torch.stack((codes & 15, codes >> 4), -1).flatten(-2).int()]
    v = v.unflatten(-1, (8, nb, 4)).transpose(-2, -3)  # [..][nb][8][4]
    v = v * torch.exp2(scales.float() - 127.0)[..., None, None]
    return v.flatten(-3)


def _pool(case, seed, g, n_pages, fill=True):
    """A page pool whose rows hold quantised K/V values; [pages][kv][page][...]."""
    n_kv, hd, page, fmt = case["n_kv"], case["hd"], case["page"], case["fmt"]
    rb = hd if fmt == "mxfp8" else hd // 2
    pool = []
    for _ in range(2):
        codes = torch.zeros((n_pages, n_kv, page, rb), dtype=torch.uint8, device="cuda")
        scales = torch.zeros((n_pages, n_kv, page, hd // 32), dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 26) // (n_kv * page * hd))
        for at in range(0, n_pages if fill else 0, step):
            n = min(step, n_pages - at)
            c, s = _quantise(_kv_values(g, n * page, n_kv, hd), fmt)
            codes[at:at + n] = c.view(n, page, n_kv, rb).transpose(1, 2)
            scales[at:at + n] = s.view(n, page, n_kv, -1).transpose(1, 2)
        pool += [codes, scales]
    return pool


def prepare(case, seed):
    g = _gen(seed)
    state = dict(case=case)
    op = case["op"]
    if op == "verify":
        b, k, v = case["batch"], case["k"], case["vocab"]
        logits = _normal(g, b, k + 1, v).mul_(2.5)
        # the draft model agrees with the target for the most part: its distribution is the target's, disturbed
        draft = logits[:, :k] + 0.7 * _normal(g, b, k, v)
        if case["probs"]:
            probs = torch.softmax(draft, -1)
            noise = torch.empty_like(probs).exponential_(generator=g)
            state["drafts"] = (probs / noise).argmax(-1).int()
            state["draft_probs"] = probs
        else:
            state["drafts"] = draft.argmax(-1).int()
            state["draft_probs"] = None
        state["logits"] = logits.to(DTYPE[case["dtype"]])
        state["draft_lens"] = torch.tensor(_draft_lens(case), dtype=torch.int32, device="cuda")
        state["uniforms"] = torch.rand((b, k), generator=g, device="cuda")
        state["noise"] = torch.empty((b, v), device="cuda").exponential_(generator=g)
        temp = 0.6 + 0.6 * torch.rand((b,), generator=g, device="cuda")
        temp[b // 2::5] = 0.0 if b > 1 else 1.0  # some requests of a batch decode greedily
        state["temperature"] = temp
        return state
    n_kv, hd, page = case["n_kv"], case["hd"], case["page"]
    if op in ("append", "read"):
        tokens = case["tokens"]
        n_pages = -(-tokens // page) + 3
        state["pool"] = _pool(case, seed, g, n_pages, fill=op == "read")
        order = torch.randperm(n_pages, generator=g, device="cuda")[: -(-tokens // page)]
        slots = (order[:, None] * page + torch.arange(page, device="cuda")).reshape(-1)[:tokens]
        state["slots"] = slots.int()
        if op == "append":
            # K and V come as slices of the fused QKV projection's output
            qkv = torch.cat((_normal(g, tokens, 4 * n_kv, hd), _kv_values(g, tokens, n_kv, hd), _kv_values(g, tokens, n_kv, hd)), 1)
            qkv = qkv.to(DTYPE[case["dtype"]])
            state["k"], state["v"] = qkv[:, 4 * n_kv:5 * n_kv], qkv[:, 5 * n_kv:]
    else:
        lens = _lens(case)
        pages = [-(-n // page) for n in lens]
        n_prefix = -(-case["prefix"] // page) if op == "shared" else 0
        n_pages = sum(pages) + n_prefix + 1
        state["pool"] = _pool(case, seed, g, n_pages)
        order = torch.randperm(n_pages, generator=g, device="cuda").int()
        table = torch.zeros((case["batch"], max(1, max(pages))), dtype=torch.int32, device="cuda")
        at = n_prefix
        for i, n in enumerate(pages):
            table[i, :n] = order[at:at + n]
            at += n
        state["page_table"] = table
        state["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        if op == "shared":
            state["prefix_pages"] = order[:n_prefix].contiguous()
        state["q"] = _normal(g, case["batch"], case["q_len"], n_kv * case["group"], hd).mul_(1.5).to(DTYPE[case["dtype"]])
    if own:
        state["cache"] = _ops().MxKvCache(*state["pool"])
    return state


# ------------------------------------------------------------------ plain forms

def _rows(pool, slots, page, fmt):
    page_of, at = slots.long() // page, slots.long() % page
    kc, ks, vc, vs = pool
    return _dequantise(kc[page_of, :, at], ks[page_of, :, at], fmt), _dequantise(vc[page_of, :, at], vs[page_of, :, at], fmt)


def _plain_append(s):
    case, pool = s["case"], s["pool"]
    page_of, at = s["slots"].long() // case["page"], s["slots"].long() % case["page"]
    for x, codes, scales in ((s["k"], pool[0], pool[1]), (s["v"], pool[2], pool[3])):
        c, e = _quantise(x, case["fmt"])
        codes[page_of, :, at] = c
        scales[page_of, :, at] = e
    return _plain_read(s)


def _plain_read(s):
    case = s["case"]
    k, v = _rows(s["pool"], s["slots"], case["page"], case["fmt"])
    return k.to(DTYPE[case["dtype"]]), v.to(DTYPE[case["dtype"]])


def _context(pool, table, case, n):
    """The first n positions behind a page table [..][pages] as f32 [..][n][kv][hd], K and V."""
    out = []
    for codes, scales in ((pool[0], pool[1]), (pool[2], pool[3])):
        x = _dequantise(codes[table.long()], scales[table.long()], case["fmt"])  # [..][pages][kv][page][hd]
        x = x.transpose(-2, -3).flatten(-4, -3)
        out.append(x[..., :n, :, :])
    return out


def _plain_attention(s):
    case = s["case"]
    b, t, hd, n_kv = case["batch"], case["q_len"], case["hd"], case["n_kv"]
    q = s["q"].float().view(b, t, n_kv, -1, hd).permute(0, 2, 1, 3, 4) / math.sqrt(hd)  # [b][kv][t][group][hd]
    k, v = _context(s["pool"], s["page_table"], case, case["max_len"])
    n = k.shape[1]
    score = torch.einsum("bhtgd,bnhd->bhtgn", q, k)
    seen = torch.arange(n, device="cuda") < (s["lens"][:, None, None] - t + 1 + torch.arange(t, device="cuda")[:, None])
    score = score.masked_fill(~seen[:, None, :, None, :], -math.inf)
    if case["op"] == "shared":
        pk, pv = _context(s["pool"], s["prefix_pages"], case, case["prefix"])
        score = torch.cat((torch.einsum("bhtgd,nhd->bhtgn", q, pk), score), -1)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)  # a row that sees nothing gives zeros
    out = torch.einsum("bhtgn,bnhd->bhtgd", p[..., -n:], v)
    if case["op"] == "shared":
        out = out + torch.einsum("bhtgn,nhd->bhtgd", p[..., :-n], pv)
    return out.permute(0, 2, 1, 3, 4).reshape(s["q"].shape).to(s["q"].dtype)


def _plain_verify(s):
    case = s["case"]
    b, k, v = case["batch"], case["k"], case["vocab"]
    logits, temp = s["logits"].float(), s["temperature"]
    greedy = temp <= 0
    best = logits.argmax(-1)
    x = logits / torch.where(greedy, 1.0, temp)[:, None, None]
    x = x - x.amax(-1, keepdim=True)
    p = torch.exp(x)
    total = p.sum(-1, keepdim=True)
    logp = x - torch.log(total)
    p = p / total
    p = torch.where(greedy[:, None, None], (torch.arange(v, device="cuda") == best[..., None]).float(), p)
    drafts = s["drafts"].long()
    if s["draft_probs"] is None:
        q = (torch.arange(v, device="cuda") == drafts[..., None]).float()
    else:
        q = s["draft_probs"]
    ratio_p = p[:, :k].gather(-1, drafts[..., None])[..., 0]
    ratio_q = q.gather(-1, drafts[..., None])[..., 0]
    ok = torch.where(greedy[:, None], drafts == best[:, :k], s["uniforms"] * ratio_q < ratio_p)
    ok = ok & (torch.arange(k, device="cuda") < s["draft_lens"][:, None])
    accepted = ok.int().cumprod(-1).sum(-1)
    rows = torch.arange(b, device="cuda")
    target = p[rows, accepted]
    rejected = accepted < s["draft_lens"]
    left = (target - q[rows, accepted.clamp(max=k - 1)]).clamp(min=0)
    left = torch.where((rejected & ~greedy)[:, None], left, target)
    left = torch.where((left.amax(-1, keepdim=True) > 0), left, target)
    last = torch.where(greedy, best[rows, accepted], (left / s["noise"]).argmax(-1))
    place = torch.arange(k + 1, device="cuda")
    padded = torch.cat((drafts, drafts[:, :1]), 1)
    tokens = torch.where(place < accepted[:, None], padded, torch.where(place == accepted[:, None], last[:, None], -1))
    logp = logp.gather(-1, tokens.clamp(min=0)[..., None])[..., 0]
    return accepted.int(), tokens.int(), torch.where(tokens >= 0, logp, 0.0)


def run(state):
    op = state["case"]["op"]
    if not own:
        if op == "append":
            return _plain_append(state)
        if op == "read":
            return _plain_read(state)
        return _plain_verify(state) if op == "verify" else _plain_attention(state)
    ops = _ops()
    if op == "append":
        ops.kv_append_mx(state["cache"], state["slots"], state["k"], state["v"])
        return ops.kv_read_mx(state["cache"], state["slots"], state["k"].dtype)
    if op == "read":
        return ops.kv_read_mx(state["cache"], state["slots"], DTYPE[state["case"]["dtype"]])
    if op == "verify":
        return ops.verify_drafts(state["logits"], state["drafts"], state["uniforms"], state["noise"],
                                 draft_probs=state["draft_probs"], draft_lens=state["draft_lens"],
                                 temperature=state["temperature"])
    if op == "shared":
        return ops.attn_shared_mx(state["cache"], state["q"], state["prefix_pages"], state["case"]["prefix"],
                                  state["page_table"], state["lens"], state["case"]["max_len"])
    return ops.attn_paged_mx(state["cache"], state["q"], state["page_table"], state["lens"], state["case"]["max_len"])


# ------------------------------------------------------------------ 64-bit definitions

def _value_table(fmt):
    """Value of every code, from the format's definition."""
    if fmt == "mxfp4":
        return list(E2M1)
    table = []
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = math.ldexp(m, -9) if e == 0 else math.ldexp(8 + m, e - 10)
        table.append(math.nan if c & 127 == 127 else -v if c & 128 else v)
    return table


def _exact_rows(codes, scales, fmt):
    """Cached rows [n][row bytes], [n][nb] -> f64 [n][hd], element by element through the position rule."""
    nb = scales.shape[-1]
    table = torch.tensor(_value_table(fmt), dtype=torch.float64, device=codes.device)
    d = torch.arange(32 * nb, device=codes.device)
    at = (d % 32 // 4 * nb + d // 32) * 4 + d % 4
    if fmt == "mxfp8":
        c = codes[..., at]
    else:
        c = codes[..., at // 2] >> (4 * (at % 2)).to(torch.uint8) & 15
    return table[c.long()] * torch.exp2(scales[..., d // 32].double() - 127)


def _exact_quantised(x, fmt):
    """What each value stands for once it is held in the format: nearest code of its block's scale, in 64 bits."""
    x = x.double()
    blocks = x.unflatten(-1, (-1, 32))
    amax = blocks.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(torch.where(amax > 0, amax, 1.0)))
    e = torch.where(torch.exp2(e) > amax, e - 1, torch.where(torch.exp2(e + 1) <= amax, e + 1, e))
    scale = torch.where(amax > 0, torch.exp2((e - (8 if fmt == "mxfp8" else 2)).clamp(-127, 127)), 1.0)
    y = (blocks / scale).abs()
    if fmt == "mxfp4":
        levels = torch.tensor(E2M1[:8], dtype=torch.float64, device=x.device)
        edges = (levels[1:] + levels[:-1]) / 2
        mag = levels[torch.bucketize(y, edges)]  # an edge itself goes down
    else:
        step = torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0 ** -6))) - 3)
        mag = (torch.round(y / step) * step).clamp(max=448.0)  # ties to even multiples of the step
    return (torch.where(blocks < 0, -mag, mag) * scale).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "append":
        return _exact_quantised(s["k"], case["fmt"]), _exact_quantised(s["v"], case["fmt"])
    if op == "read":
        out = []
        for codes, scales in ((s["pool"][0], s["pool"][1]), (s["pool"][2], s["pool"][3])):
            page_of, at = s["slots"].long() // case["page"], s["slots"].long() % case["page"]
            parts = [_exact_rows(codes[p, :, a], scales[p, :, a], case["fmt"])
                     for p, a in zip(page_of.split(8192), at.split(8192))]
            out.append(torch.cat(parts))
        return tuple(out)
    if op == "verify":
        return _exact_verify(case, s)
    b, t, n_kv, group, hd = case["batch"], case["q_len"], case["n_kv"], case["group"], case["hd"]
    kc, ks, vc, vs = s["pool"]

    def head(pages, n, h, codes, scales):
        p = pages[: -(-n // case["page"])].long()
        return _exact_rows(codes[p, h].flatten(0, 1)[:n], scales[p, h].flatten(0, 1)[:n], case["fmt"])

    out = torch.zeros((b, t, n_kv * group, hd), dtype=torch.float64, device="cuda")
    lens, prefix = _lens(case), case.get("prefix", 0)
    for h in range(n_kv):
        pk = head(s["prefix_pages"], prefix, h, kc, ks) if prefix else None
        pv = head(s["prefix_pages"], prefix, h, vc, vs) if prefix else None
        for i in range(b):
            k = head(s["page_table"][i], lens[i], h, kc, ks)
            v = head(s["page_table"][i], lens[i], h, vc, vs)
            if prefix:
                k, v = torch.cat((pk, k)), torch.cat((pv, v))
            q = s["q"][i, :, h * group:(h + 1) * group].double()  # [t][group][hd]
            score = (q.reshape(-1, hd) @ k.T / math.sqrt(hd)).view(t, group, -1)
            limit = prefix + lens[i] - t + 1 + torch.arange(t, device="cuda")
            if prefix:
                limit = limit.clamp(min=prefix)
            hidden = torch.arange(k.shape[0], device="cuda") >= limit[:, None]
            score = score.masked_fill(hidden[:, None], -math.inf)
            p = torch.softmax(score, -1) if k.shape[0] else score
            p = torch.nan_to_num(p)  # a row that sees nothing
            out[i, :, h * group:(h + 1) * group] = (p.view(t * group, -1) @ v).view(t, group, hd)
    return out


def _exact_verify(case, s):
    b, k = case["batch"], case["k"]
    accepted, tokens, logprobs = [], [], []
    lens, temps = _draft_lens(case), s["temperature"].tolist()
    drafts, u = s["drafts"].tolist(), s["uniforms"].tolist()
    for i in range(b):
        n, out, logp = 0, [], []
        while True:
            row = s["logits"][i, n].double()
            logps = torch.log_softmax(row / (temps[i] if temps[i] > 0 else 1.0), -1)
            if temps[i] <= 0:
                p = torch.zeros_like(row)
                p[int(row.argmax())] = 1.0
            else:
                p = torch.softmax(row / temps[i], -1)
            if n == lens[i]:
                left = p
                break
            d = drafts[i][n]
            if s["draft_probs"] is None:
                q = torch.zeros_like(p)
                q[d] = 1.0
            else:
                q = s["draft_probs"][i, n].double()
            if (float(p[d]) > 0.5) if temps[i] <= 0 else (u[i][n] * float(q[d]) < float(p[d])):
                out.append(d)
                logp.append(float(logps[d]))
                n += 1
                continue
            left = (p - q).clamp(min=0) if temps[i] > 0 else p
            left = left if float(left.amax()) > 0 else p
            break
        out.append(int((left / s["noise"][i].double()).argmax()) if temps[i] > 0 else int(p.argmax()))
        logp.append(float(logps[out[-1]]))
        accepted.append(n)
        tokens.append(out + [-1] * (k + 1 - len(out)))
        logprobs.append(logp + [0.0] * (k + 1 - len(logp)))
    return (torch.tensor(accepted, dtype=torch.int32), torch.tensor(tokens, dtype=torch.int32),
            torch.tensor(logprobs, dtype=torch.float64))
