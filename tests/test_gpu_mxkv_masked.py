"""What positions hold that a query does not see must not matter: hidden tokens, rows past the length, missing pages."""
import pytest

torch = pytest.importorskip("torch")
from mxkv_torch import DT, Batch, filled, gen, normal  # noqa: E402

pytestmark = pytest.mark.gpu

# query heads per KV head and query tokens: 5 to 128 rows, on both kernels
ROWS = [(1, 5), (4, 4), (4, 8), (8, 5), (2, 64), (24, 5)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("prefix", [0, 70])
@pytest.mark.parametrize("fmt,hd,page", [("mxfp8", 128, 16), ("mxfp4", 64, 32), ("mxfp8", 64, 64), ("mxfp4", 128, 16)])
@pytest.mark.parametrize("group,q_len", ROWS, ids=str)
def test_nan_in_a_later_query_token(group, q_len, fmt, hd, page, prefix, dtype):
    """A NaN that one of the query tokens brings into the cache, in V or in K, reaches the queries that see it alone."""
    g = gen(group + q_len)
    n_kv = 2
    batch = Batch(g, [q_len + 3, 1, 0, 65 + q_len, 700, q_len], page, prefix, q_len, max_len=800)
    k, v = (normal(g, batch.n_pages * page, n_kv, hd) for _ in range(2))
    for b, n in enumerate(batch.lens):
        slots = batch.slots(b)[prefix:]
        for back, dims in ((1, (0, 37)), (q_len // 2, (5, 63)), (q_len - 1, (hd - 1,))):
            if n > back >= 1:
                v[slots[n - back], b % 2, list(dims)] = torch.nan
    k[batch.slots(4)[-1], 1, 7] = torch.nan       # the last key of one sequence: its last query alone
    cache, k, v = filled(k, v, page, fmt)
    q = normal(g, len(batch.lens), q_len, n_kv * group, hd).to(DT[dtype])
    got = batch.attend(cache, q)
    assert got.isnan().any() and not got[2].isnan().any()
    batch.check(got, q, k, v)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("prefix", [0, 33])
@pytest.mark.parametrize("group,q_len", [(4, 3), (20, 4)], ids=str)
def test_values_past_the_range_in_a_later_query_token(group, q_len, prefix, dtype):
    """Codes and a scale that make more than 2^128, in V of the last query token: the ones before do not see it."""
    g = gen(3)
    batch = Batch(g, [q_len, 200], 32, prefix, q_len)
    k, v = (normal(g, batch.n_pages * 32, 1, 64) for _ in range(2))
    cache, k, v = filled(k, v, 32, "mxfp8")
    for b in range(2):
        slot = int(batch.slots(b)[-1])
        cache.v[slot // 32, 0, slot % 32] = 0x7E
        cache.v_scales[slot // 32, 0, slot % 32] = 254
    q = normal(g, 2, q_len, group, 64).to(DT[dtype])
    got = batch.attend(cache, q)
    assert not got[:, -1].isfinite().any()
    got[:, -1] = torch.nan
    for b in range(2):
        v[batch.slots(b)[-1]] = torch.nan
    batch.check(got, q, k, v)
