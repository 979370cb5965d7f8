"""Attention over the MX cache at lengths where a CTA takes many tiles and segments: accuracy of the sums, rescaling."""
import pytest

torch = pytest.importorskip("torch")
from fp4x import ops  # noqa: E402
from mxkv_torch import DT, Batch, check, definition, filled, gen, normal  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group,hd,fmt", [(4, 128, "mxfp8"), (8, 64, "mxfp4"), (16, 64, "mxfp8"), (16, 128, "mxfp8"),
                                          (9, 128, "mxfp4"), (32, 64, "mxfp4"), (17, 128, "mxfp8"),
                                          (64, 128, "mxfp8"), (40, 64, "mxfp4")])
def test_sums_do_not_drift_with_the_length(group, hd, fmt):
    """Near-equal scores and values of one sign over 32768 positions, a segment per CTA: the f32 sums stay f32 sums."""
    n, n_kv, batch, page = 32768, 8, 37, 64
    g = gen(group)
    cache, k, v = filled(torch.randn((n, n_kv, hd), generator=g, device="cuda"),
                         torch.randn((n, n_kv, hd), generator=g, device="cuda").abs(), page, fmt)
    q = torch.randn((batch, 1, n_kv * group, hd), generator=g, device="cuda") * 0.01
    table = torch.arange(n // page, dtype=torch.int32, device="cuda").expand(batch, -1).contiguous()
    lens = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    got = ops.attn_paged_mx(cache, q, table, lens)
    seen = torch.ones((batch, n), dtype=torch.bool, device="cuda")
    check(got[:, 0], *definition(q[:, 0], k, v, seen), n)
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
    g = gen(group + hd)
    k = torch.randn((n, n_kv, hd), generator=g, device="cuda") * 0.05
    k[:, :, 0] = 0.0
    for at, up in ((3000, 11.5), (9001, 23.0), (9002, 23.0), (16007, 34.5), (19990, 46.0)):
        k[at:, :, 0] = up - 4.5    # the run of positions after it is below it by what 90 of them make up
        k[at, :, 0] = up
    cache, k, v = filled(k, torch.randn((n, n_kv, hd), generator=g, device="cuda"), page, fmt)
    q = torch.randn((batch, 1, n_kv * group, hd), generator=g, device="cuda")
    q[..., 0] = hd ** 0.5
    q = q.to(DT[dtype])
    table = torch.arange(n // page, dtype=torch.int32, device="cuda").expand(batch, -1).contiguous()
    for length in (n, 16100, 9100):
        lens = torch.full((batch,), length, dtype=torch.int32, device="cuda")
        got = ops.attn_paged_mx(cache, q, table, lens)
        seen = (torch.arange(n, device="cuda") < length).expand(batch, n)
        check(got[:, 0], *definition(q[:, 0], k, v, seen), n)


@pytest.mark.parametrize("group,hd,fmt", [(4, 128, "mxfp8"), (64, 128, "mxfp8"), (48, 64, "mxfp4")])
def test_bf16_results_have_no_bias(group, hd, fmt):
    """bf16 results over 32768 positions, spread over a power of two: their rounding errors average out, a sum that
    loses a little with every addition does not."""
    n, n_kv, batch, page = 32768, 8, 37, 64
    g = gen(group)
    spread = torch.exp2(torch.arange(hd, device="cuda") / hd)
    cache, k, v = filled(torch.randn((n, n_kv, hd), generator=g, device="cuda"),
                         torch.randn((n, n_kv, hd), generator=g, device="cuda").abs() * spread, page, fmt)
    q = (torch.randn((batch, 1, n_kv * group, hd), generator=g, device="cuda") * 0.5).bfloat16()
    table = torch.arange(n // page, dtype=torch.int32, device="cuda").expand(batch, -1).contiguous()
    lens = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    got = ops.attn_paged_mx(cache, q, table, lens)[:, 0]
    want, mass, size = definition(q[:, 0], k, v, torch.ones((batch, n), dtype=torch.bool, device="cuda"))
    check(got, want, mass, size, n)
    # at most 128 additions that cut off up to an ulp of an evenly growing sum (64 x 2^-23); rounding errors of at most
    # 2^-8 of the result, evenly spread (deviation 2^-8 / sqrt(3)): five deviations of their mean
    bias = float(((got.double() - want) / want).mean())
    assert abs(bias) <= 2.0 ** -17 + 5 * 2.0 ** -8 / (3 * want.numel()) ** 0.5, bias


def _tiles(batch, n_kv, rows, tn, tile_rows=128, sms=None):
    """How the 128-row kernel's work falls to its CTAs, from the rule in its source: (segment, tiles) per CTA.  A segment
    is a sequence x 128 rows x KV head; it costs its chunks of 128 positions and 2 more; CTA c starts at cost
    floor(c * total / CTAs)."""
    sms = sms or torch.cuda.get_device_properties(0).multi_processor_count
    row_tiles = -(-rows // tile_rows)
    lens = [n for n in batch for _ in range(row_tiles * n_kv)]
    segments, at = [], 0
    for n in lens:
        c = -(-n // 128)
        if c:
            segments.append((at, c, n))
            at += c + 2
    ctas = min(sms, -(-max(batch) // 128) * len(batch) * n_kv * row_tiles)
    out = []
    for c in range(ctas):
        lo, hi = c * at // ctas, (c + 1) * at // ctas
        mine = []
        for start, chunks, n in segments:
            a, b = max(lo - start - 2, 0), min(hi - start - 2, chunks)
            if lo < start + 2 + chunks and hi > start and a < b:
                mine.append(-(-(min(b * 128, n) - a * 128) // tn))
        out.append(mine)
    return out


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd,fmt,page", [(128, "mxfp8", 64), (64, "mxfp4", 16)])
@pytest.mark.parametrize("rising", [False, True])
def test_many_tiles_of_a_shared_prefix(hd, fmt, page, rising, dtype):
    """300 rows on a prefix of 20011 positions x 8 KV heads: more than twice as many tiles in a row as between two
    additions to the sum, buffers and their barriers several times around."""
    g = gen(hd)
    n_kv, group, prefix, lens = 8, 4, 20011, [0, 130, 1] * 25
    tiles = _tiles([prefix], n_kv, group * len(lens), 64 if dtype == "f32" else 128)
    assert max(map(max, tiles)) > 2 * 8  # the sums take O every 2 (f32) or 4 tiles
    batch = Batch(g, lens, page, prefix)
    k = normal(g, batch.n_pages * page, n_kv, hd)
    if rising:  # scores grow along the prefix: O is rescaled in late tiles, in and out of step with the sums
        order = batch.slots(0)
        k[order] *= 0.1
        k[order, :, 0] = torch.linspace(0.0, 90.0, prefix, device="cuda")[:, None]
    cache, k, v = filled(k, normal(g, batch.n_pages * page, n_kv, hd), page, fmt)
    q = normal(g, len(lens), 1, n_kv * group, hd)
    if rising:
        q[..., 0] = hd ** 0.5 * torch.linspace(0.2, 2.0, n_kv * group, device="cuda")
    q = q.to(DT[dtype])
    got = batch.attend(cache, q)
    batch.check(got, q, k, v, only=[0, 1, 2, 40, 73, 74])
    assert torch.equal(got, batch.attend(cache, q))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd,fmt,page,group,q_len", [(128, "mxfp8", 64, 4, 40), (64, "mxfp4", 32, 12, 11), (128, "mxfp4", 16, 64, 1)])
def test_many_segments_of_own_positions(hd, fmt, page, group, q_len, dtype):
    """More segments than CTAs, of ragged lengths (0 among them): a CTA takes several of them, whole and in parts."""
    g = gen(group)
    n_kv = 8
    lens = [700, 0, 1, 129, 2300, 40, 64, 0, 513, 128, 300, 17, 1000, 90] * 3
    tiles = _tiles(lens, n_kv, group * q_len, 64 if dtype == "f32" else 128)
    assert max(map(len, tiles)) >= 3 and max(map(sum, tiles)) >= 8
    batch = Batch(g, lens, page, 0, q_len)
    k, v = (normal(g, batch.n_pages * page, n_kv, hd) for _ in range(2))
    cache, k, v = filled(k, v, page, fmt)
    q = normal(g, len(lens), q_len, n_kv * group, hd).to(DT[dtype])
    got = batch.attend(cache, q)
    batch.check(got, q, k, v)
    assert torch.equal(got, batch.attend(cache, q))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("group,q_len,n", [(4, 1, 32768), (1, 1, 40001), (16, 1, 32000), (64, 1, 32768), (8, 64, 9000)])
def test_one_long_sequence(group, q_len, n, dtype):
    """One sequence and one KV head over all CTAs: up to some 300 partial results of one row are joined."""
    g = gen(n)
    batch = Batch(g, [n], 16, 0, q_len)
    k, v = (normal(g, batch.n_pages * 16, 1, 128) for _ in range(2))
    cache, k, v = filled(k, v, 16, "mxfp8")
    q = normal(g, 1, q_len, group, 128).to(DT[dtype])
    got = batch.attend(cache, q)
    batch.check(got, q, k, v)
    assert torch.equal(got, batch.attend(cache, q))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("q_len", [17, 32, 63, 64])
@pytest.mark.parametrize("group,hd,fmt,prefix", [(1, 64, "mxfp4", 0), (4, 128, "mxfp8", 0), (7, 64, "mxfp8", 100), (4, 128, "mxfp4", 700)])
def test_prompt_passes(group, hd, fmt, prefix, q_len, dtype):
    """Query tokens up to the most that a call takes, as the first positions of a sequence and after many others."""
    g = gen(q_len)
    batch = Batch(g, [q_len, 500 + q_len, q_len - 3, 0, 130], 32, prefix, q_len)
    k, v = (normal(g, batch.n_pages * 32, 2, hd) for _ in range(2))
    cache, k, v = filled(k, v, 32, fmt)
    q = normal(g, 5, q_len, 2 * group, hd).to(DT[dtype])
    batch.check(batch.attend(cache, q), q, k, v)
