"""Attention over the MX cache at lengths where a CTA takes many tiles and segments: accuracy of the sums, rescaling."""
import pytest

torch = pytest.importorskip("torch")
from fp4x import ops  # noqa: E402

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _cache(k, v, page, fmt):
    """A cache that holds rows k, v [n][n_kv][hd] in the order of its slots, and what it stands for in 64 bits."""
    n, n_kv, hd = k.shape
    cache = ops.MxKvCache.empty(-(-n // page), n_kv, hd, page, fmt)
    slots = torch.arange(n, dtype=torch.int32, device="cuda")
    ops.kv_append_mx(cache, slots, k, v)
    kk, vv = ops.kv_read_mx(cache, slots, torch.float32)
    return cache, kk.double(), vv.double()


def _definition(q, k, v, seen):
    """q [t][H][hd], k, v [n][n_kv][hd] f64, seen [t][n]: the result, sum p |v| and max sum |q k| / sqrt(hd)."""
    t, H, hd = q.shape
    n_kv = k.shape[1]
    qq = q.double().view(t, n_kv, H // n_kv, hd)
    out, mass, size = (torch.zeros((t, n_kv, H // n_kv, hd), dtype=torch.float64, device=q.device) for _ in range(3))
    for h in range(n_kv):
        s = torch.einsum("tgd,nd->tgn", qq[:, h], k[:, h]) / hd ** 0.5
        a = torch.einsum("tgd,nd->tgn", qq[:, h].abs(), k[:, h].abs()) / hd ** 0.5
        hidden = ~seen[:, None, :]
        p = torch.softmax(s.masked_fill(hidden, -torch.inf), -1).nan_to_num(0.0)
        out[:, h], mass[:, h] = torch.einsum("tgn,nd->tgd", p, v[:, h]), torch.einsum("tgn,nd->tgd", p, v[:, h].abs())
        size[:, h] = a.masked_fill(hidden, 0.0).amax(-1, True)
    return out.view(q.shape), mass.view(q.shape), size.view(q.shape)


def _close(got, want, mass, size, n):
    """The scores' error (f32 sums of 22-bit operands: 2^-20 of sum |q k|) moves every probability by that factor; the
    products, the statistics and the sums add 2^-18 of sum p |v|: between two additions in f32 the tensor core's
    accumulator takes at most 48 that cut off up to an ulp (2^-23) of a sum that grows evenly, 24 x 2^-23 together.
    bf16 queries: P has 16 bits (2^-16 of sum p |v|), the chain of accumulations may be a segment's (n / 128 tiles of a
    warp, two additions each: n 2^-30); the result is the rounding of a value that near, so it lies between the
    roundings of the ends."""
    off = (2.0 ** -18 + 2.0 ** -19 * size) * mass
    if got.dtype == torch.float32:
        worst = float(((got.double() - want).abs() / off).max())
        assert worst <= 1.0, worst
        return
    off = off + (2.0 ** -16 + n * 2.0 ** -30) * mass
    assert bool((got >= (want - off).to(got.dtype)).all() and (got <= (want + off).to(got.dtype)).all())


@pytest.mark.parametrize("group,hd,fmt", [(4, 128, "mxfp8"), (8, 64, "mxfp4"), (16, 64, "mxfp8"), (16, 128, "mxfp8"),
                                          (9, 128, "mxfp4"), (32, 64, "mxfp4"), (17, 128, "mxfp8"),
                                          (64, 128, "mxfp8"), (40, 64, "mxfp4")])
def test_sums_do_not_drift_with_the_length(group, hd, fmt):
    """Near-equal scores and values of one sign over 32768 positions, a segment per CTA: the f32 sums stay f32 sums."""
    n, n_kv, batch, page = 32768, 8, 37, 64
    g = _gen(group)
    cache, k, v = _cache(torch.randn((n, n_kv, hd), generator=g, device="cuda"),
                         torch.randn((n, n_kv, hd), generator=g, device="cuda").abs(), page, fmt)
    q = torch.randn((batch, 1, n_kv * group, hd), generator=g, device="cuda") * 0.01
    table = torch.arange(n // page, dtype=torch.int32, device="cuda").expand(batch, -1).contiguous()
    lens = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    got = ops.attn_paged_mx(cache, q, table, lens)
    seen = torch.ones((batch, n), dtype=torch.bool, device="cuda")
    _close(got[:, 0], *_definition(q[:, 0], k, v, seen), n)
    # the same bits again, and from a workspace with other contents
    ws = ops.attn_mx_workspace(cache, batch, n_kv * group, 1, 0, n)
    ws.fill_(0xFF)
    assert torch.equal(got, ops.attn_paged_mx(cache, q, table, lens, workspace=ws))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("group,hd,fmt", [(1, 128, "mxfp8"), (7, 64, "mxfp4"), (12, 128, "mxfp8"), (16, 64, "mxfp4"),
                                          (32, 64, "mxfp8"), (20, 128, "mxfp4"), (33, 128, "mxfp8"), (64, 64, "mxfp4")])
def test_maximum_that_grows_late(group, hd, fmt, dtype):
    """Single positions whose scores pass all before by more than the kernels leave standing (16 powers of two), with as
    much of the probability as the thousands before them: what was summed before is rescaled, in registers and out."""
    n, n_kv, batch, page = 20000, 8, 37, 32
    g = _gen(group + hd)
    k = torch.randn((n, n_kv, hd), generator=g, device="cuda") * 0.05
    k[:, :, 0] = 0.0
    for at, up in ((3000, 11.5), (9001, 23.0), (9002, 23.0), (16007, 34.5), (19990, 46.0)):
        k[at:, :, 0] = up - 4.5    # the run of positions after it is below it by what 90 of them make up
        k[at, :, 0] = up
    cache, k, v = _cache(k, torch.randn((n, n_kv, hd), generator=g, device="cuda"), page, fmt)
    q = torch.randn((batch, 1, n_kv * group, hd), generator=g, device="cuda")
    q[..., 0] = hd ** 0.5
    q = q.to(DT[dtype])
    table = torch.arange(n // page, dtype=torch.int32, device="cuda").expand(batch, -1).contiguous()
    for length in (n, 16100, 9100):
        lens = torch.full((batch,), length, dtype=torch.int32, device="cuda")
        got = ops.attn_paged_mx(cache, q, table, lens)
        seen = (torch.arange(n, device="cuda") < length).expand(batch, n)
        _close(got[:, 0], *_definition(q[:, 0], k, v, seen), n)


@pytest.mark.parametrize("group,hd,fmt", [(4, 128, "mxfp8"), (64, 128, "mxfp8"), (48, 64, "mxfp4")])
def test_bf16_results_have_no_bias(group, hd, fmt):
    """bf16 results over 32768 positions, spread over a power of two: their rounding errors average out, a sum that
    loses a little with every addition does not."""
    n, n_kv, batch, page = 32768, 8, 37, 64
    g = _gen(group)
    spread = torch.exp2(torch.arange(hd, device="cuda") / hd)
    cache, k, v = _cache(torch.randn((n, n_kv, hd), generator=g, device="cuda"),
                         torch.randn((n, n_kv, hd), generator=g, device="cuda").abs() * spread, page, fmt)
    q = (torch.randn((batch, 1, n_kv * group, hd), generator=g, device="cuda") * 0.5).bfloat16()
    table = torch.arange(n // page, dtype=torch.int32, device="cuda").expand(batch, -1).contiguous()
    lens = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    got = ops.attn_paged_mx(cache, q, table, lens)[:, 0]
    want, mass, size = _definition(q[:, 0], k, v, torch.ones((batch, n), dtype=torch.bool, device="cuda"))
    _close(got, want, mass, size, n)
    # at most 128 additions that cut off up to an ulp of an evenly growing sum (64 x 2^-23); rounding errors of at most
    # 2^-8 of the result, evenly spread (deviation 2^-8 / sqrt(3)): five deviations of their mean
    bias = float(((got.double() - want) / want).mean())
    assert abs(bias) <= 2.0 ** -17 + 5 * 2.0 ** -8 / (3 * want.numel()) ** 0.5, bias
