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


def _dirty(cache, fmt, live):
    """NaN codes and scales in every row of the pool that `live` [slots] leaves out."""
    n_pages, n_kv, page, _ = cache.k.shape
    gone = ~live.view(n_pages, 1, page).expand(n_pages, n_kv, page)
    for t in (cache.k, cache.v):
        t[gone] = 0x7F if fmt == "mxfp8" else 0xFF
    for t in (cache.k_scales, cache.v_scales):
        t[gone] = 255


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("prefix", [0, 37, 200])
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("group,q_len", [(8, 5), (40, 1), (4, 33)], ids=str)
def test_rows_past_the_length_are_not_used(group, q_len, fmt, prefix, dtype):
    """More than 32 rows per KV head: NaN in the rows past the lengths and in free pages changes no bit."""
    g = gen(8)
    batch = Batch(g, [45, 3, 0, 70, 129, 500], 32, prefix, q_len, max_len=600)
    k, v = (normal(g, batch.n_pages * 32, 2, 128) for _ in range(2))
    cache, k, v = filled(k, v, 32, fmt)
    q = normal(g, 6, q_len, 2 * group, 128).to(DT[dtype])
    clean = batch.attend(cache, q)
    live = torch.zeros(k.shape[0], dtype=torch.bool, device="cuda")
    for b in range(6):
        live[batch.slots(b)] = True
    _dirty(cache, fmt, live)
    got = batch.attend(cache, q)
    assert torch.equal(got, clean) and got.isfinite().all()
    batch.check(got, q, k, v)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fmt,hd", [("mxfp8", 128), ("mxfp4", 64), ("mxfp8", 64), ("mxfp4", 128)])
@pytest.mark.parametrize("group,q_len,prefix", [(4, 1, 0), (6, 5, 0), (8, 5, 0), (64, 1, 0), (8, 5, 520), (4, 2, 2050)], ids=str)
def test_pages_outside_the_cache_are_masked(group, q_len, prefix, fmt, hd, dtype):
    """Page ids outside the cache at several places of a tile, in both of its halves, over a whole tile, and as all pages
    of a sequence: the result is that of the other positions, and the device error word is set."""
    import test_gpu_mxkv as T
    g = gen(9)
    batch = Batch(g, [600, 77, 16, 1000], 16, prefix, q_len)
    k, v = (normal(g, batch.n_pages * 16, 2, hd) for _ in range(2))
    cache, k, v = filled(k, v, 16, fmt)
    q = normal(g, 4, q_len, 2 * group, hd).to(DT[dtype])
    good = batch.table.clone(), batch.prefix_pages.clone()
    bad = [[0, 3, 4, 7, *range(16, 24), 33], [2], [0], [8, 9, 15, 60, 61]]
    lost = torch.zeros(batch.n_pages, dtype=torch.bool, device="cuda")
    for b, at in enumerate(bad):
        lost[good[0][b, at].long()] = True
        batch.table[b, at] = torch.tensor([batch.n_pages, -1, 2**31 - 1], dtype=torch.int32, device="cuda").repeat(5)[:len(at)]
    if prefix:
        at = [1, 6, *range(24, 32)]
        lost[good[1][at].long()] = True
        batch.prefix_pages[at] = -7
    assert T._errors() == (0, 0)
    got = batch.attend(cache, q)
    st, bits = T._errors()
    assert st == 3 and bits & 4
    batch.table, batch.prefix_pages = good
    batch.check(got, q, k, v, gone=lambda b: lost[batch.slots(b) // 16])
    batch.check(batch.attend(cache, q), q, k, v)
    assert T._errors() == (0, 0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("prefix", [0, 130])
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_value_scales_of_every_size(fmt, prefix, dtype):
    """More than 32 rows: V of very different sizes (2^-30 to 2^30), and the probability on the small ones."""
    g = gen(12)
    group, hd = 40, 64
    batch = Batch(g, [300, 5, 140], 16, prefix)
    n = batch.n_pages * 16
    k = normal(g, n, 1, hd) * 0.5
    v = normal(g, n, 1, hd) * torch.exp2(torch.randint(-30, 30, (n, 1, 1), generator=g, device="cuda").float())
    # where V is large the keys point away from the queries
    k[..., 0] = torch.where(v.abs().amax(-1) > 2.0 ** -10, -30.0, 0.0)
    cache, k, v = filled(k, v, 16, fmt)
    q = normal(g, 3, 1, group, hd)
    q[..., 0] = torch.linspace(0, 12, group, device="cuda")
    q = q.to(DT[dtype])
    batch.check(batch.attend(cache, q), q, k, v)


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_pages_past_4_gib(fmt):
    """More than 32 rows on pages far apart: offsets pass 32 bits; the bits are those of a dense pool."""
    from fp4x import ops
    n_kv, hd, page, n_pages, far = 2, 128, 64, 20, 300 << 20
    row = hd if fmt == "mxfp8" else hd // 2
    base = torch.zeros(n_pages * far, dtype=torch.uint8, device="cuda")
    code, scale = n_kv * page * row, n_kv * page * 4

    def part(off, last):
        return torch.as_strided(base, (n_pages, n_kv, page, last), [far, page * last, last, 1], off)

    far_cache = ops.MxKvCache(part(0, row), part(2 * code, 4), part(code, row), part(2 * code + scale, 4))
    dense = ops.MxKvCache.empty(n_pages, n_kv, hd, page, fmt)
    g = gen(1)
    k, v = (normal(g, n_pages * page, n_kv, hd) for _ in range(2))
    slots = torch.randperm(n_pages * page, generator=g, device="cuda").int()
    for c in (far_cache, dense):
        ops.kv_append_mx(c, slots, k, v)
    table = torch.randperm(n_pages, generator=g, device="cuda").int()[None].repeat(2, 1)
    lens = torch.tensor([n_pages * page, n_pages * page - 100], dtype=torch.int32, device="cuda")
    for dtype in DT.values():
        q = normal(g, 2, 5, 16, hd).to(dtype)
        assert torch.equal(ops.attn_paged_mx(far_cache, q, table, lens), ops.attn_paged_mx(dense, q, table, lens))
        one = table[0].contiguous()
        assert torch.equal(ops.attn_shared_mx(far_cache, q, one, 1270, table, lens),
                           ops.attn_shared_mx(dense, q, one, 1270, table, lens))


def test_another_stream_and_a_graph():
    """More than 32 rows: own stream, and a captured call that sees new lengths."""
    from fp4x import ops
    g = gen(6)
    batch = Batch(g, [160, 3, 77, 0], 16, 150, 5, max_len=200)
    k, v = (normal(g, batch.n_pages * 16, 2, 128) for _ in range(2))
    cache, k, v = filled(k, v, 16, "mxfp8")
    q = normal(g, 4, 5, 16, 128).bfloat16()
    ws = ops.attn_mx_workspace(cache, 4, 16, 5, 150, 200)
    want = batch.attend(cache, q)
    batch.check(want, q, k, v)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = batch.attend(cache, q, workspace=ws)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = batch.attend(cache, q, workspace=ws)
    batch.lens = [100, 0, 77, 2]
    batch.table[3, 0] = batch.table[0, 0]
    batch.tl.copy_(torch.tensor(batch.lens))
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, batch.attend(cache, q))
    batch.check(out, q, k, v)
