"""Attention over the MX cache at lengths where a CTA takes many tiles and segments: accuracy of the sums, rescaling."""
import pytest

torch = pytest.importorskip("torch")
from fp4x import ops  # noqa: E402
from mxkv_torch import DT, check, definition, filled, gen  # noqa: E402

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
