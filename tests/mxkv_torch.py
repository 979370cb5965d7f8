"""Caches, batches and the 64-bit definition of the attention over the MX KV cache, in torch on the GPU."""
import torch

from fp4x import ops

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def filled(k, v, page, fmt):
    """A cache that holds rows k, v [n][n_kv][hd] in the order of its slots, and what it stands for in 64 bits."""
    n, n_kv, hd = k.shape
    cache = ops.MxKvCache.empty(-(-n // page), n_kv, hd, page, fmt)
    slots = torch.arange(n, dtype=torch.int32, device="cuda")
    ops.kv_append_mx(cache, slots, k, v)
    kk, vv = ops.kv_read_mx(cache, slots, torch.float32)
    return cache, kk.double(), vv.double()


def definition(q, k, v, seen):
    """q [t][H][hd], k, v [n][n_kv][hd] f64, seen [t][n]: the result, sum p |v| and max sum |q k| / sqrt(hd).  Positions
    that a query does not see do not exist for it, whatever they hold."""
    t, H, hd = q.shape
    n_kv = k.shape[1]
    qq = q.double().view(t, n_kv, H // n_kv, hd)
    out, mass, size = (torch.zeros((t, n_kv, H // n_kv, hd), dtype=torch.float64, device=q.device) for _ in range(3))
    for h in range(n_kv):
        s = torch.einsum("tgd,nd->tgn", qq[:, h], k[:, h]) / hd ** 0.5
        a = torch.einsum("tgd,nd->tgn", qq[:, h].abs(), k[:, h].abs()) / hd ** 0.5
        hidden = ~seen[:, None, :]
        p = torch.softmax(s.masked_fill(hidden, -torch.inf), -1)
        p = torch.where(seen.any(-1)[:, None, None], p, 0.0)
        missing = torch.einsum("tn,nd->td", seen.double(), v[:, h].isnan().double()) > 0
        vv = v[:, h].nan_to_num(0.0)
        out[:, h] = torch.einsum("tgn,nd->tgd", p, vv).masked_fill(missing[:, None], torch.nan)
        mass[:, h] = torch.einsum("tgn,nd->tgd", p, vv.abs())
        size[:, h] = a.masked_fill(hidden, 0.0).amax(-1, True)
    return out.view(q.shape), mass.view(q.shape), size.view(q.shape)


def check(got, want, mass, size, n):
    """The scores' error (f32 sums of 22-bit operands: 2^-20 of sum |q k|) moves every probability by that factor; the
    products, the statistics and the sums add 2^-18 of sum p |v|: between two additions in f32 the tensor core's
    accumulator takes at most 48 that cut off up to an ulp (2^-23) of a sum that grows evenly, 24 x 2^-23 together.
    bf16 queries: P has 16 bits (2^-16 of sum p |v|), the chain of accumulations may be a segment's (n / 128 tiles of a
    warp, two additions each: n 2^-30); the result is the rounding of a value that near, so it lies between the
    roundings of the ends.  NaN where the definition has it, and nowhere else."""
    assert torch.equal(got.isnan(), want.isnan())
    fine = ~want.isnan()
    got, want, off = got[fine], want[fine], ((2.0 ** -18 + 2.0 ** -19 * size) * mass)[fine]
    if got.dtype == torch.float32:
        off = off + 2.0 ** -149
        worst = float(((got.double() - want).abs() / off).max()) if got.numel() else 0.0
        assert worst <= 1.0, worst
        return
    off = off + (2.0 ** -16 + n * 2.0 ** -30) * mass[fine]
    assert bool((got >= (want - off).to(got.dtype)).all() and (got <= (want + off).to(got.dtype)).all())


class Batch:
    """Sequences of `lens` own positions, the last q_len of them the queries', after a shared prefix, on scattered pages
    of one pool."""

    def __init__(self, g, lens, page, prefix=0, q_len=1, max_len=None):
        self.lens, self.page, self.prefix, self.q_len = lens, page, prefix, q_len
        self.max_len = max(1, max(lens)) if max_len is None else max_len
        need = [-(-n // page) for n in lens]
        shared = -(-prefix // page)
        self.n_pages = shared + sum(need) + 1
        order = torch.randperm(self.n_pages, generator=g, device="cuda").int()
        self.prefix_pages = order[:shared].contiguous()
        self.table = torch.zeros((len(lens), max(1, -(-self.max_len // page))), dtype=torch.int32, device="cuda")
        at = shared
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.tl = torch.tensor(lens, dtype=torch.int32, device="cuda")

    def slots(self, b):
        """Slots of the positions that sequence b's queries can see, the prefix first."""
        pages = torch.cat((self.prefix_pages, self.table[b]))
        slots = (pages[:, None].long() * self.page + torch.arange(self.page, device="cuda")).flatten()
        n = self.prefix_pages.numel() * self.page
        return torch.cat((slots[:self.prefix], slots[n:n + self.lens[b]]))

    def attend(self, cache, q, **kw):
        if self.prefix:
            return ops.attn_shared_mx(cache, q, self.prefix_pages, self.prefix, self.table, self.tl, self.max_len, **kw)
        return ops.attn_paged_mx(cache, q, self.table, self.tl, self.max_len, **kw)

    def check(self, got, q, k, v, gone=None, only=None):
        """got against the definition for every sequence (or those in `only`); k, v [slots][n_kv][hd]; `gone(b)`: those of
        slots(b) that lie in no page."""
        for b in range(len(self.lens)) if only is None else only:
            slots = self.slots(b)
            if slots.numel() == 0:
                assert not got[b].any()
                continue
            limit = self.prefix + (self.lens[b] - self.q_len + 1 + torch.arange(self.q_len, device="cuda")).clamp(min=0)
            seen = torch.arange(slots.numel(), device="cuda") < limit[:, None]
            if gone is not None:
                seen = seen & ~gone(b)
            check(got[b], *definition(q[b], k[slots], v[slots], seen), slots.numel())
