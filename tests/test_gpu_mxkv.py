"""MX-quantised paged KV cache: writing, reading and the attention over it, against 64-bit definitions."""
import numpy as np
import pytest

import mxkv_ref as R

torch = pytest.importorskip("torch")
import fp4x  # noqa: E402
from fp4x import ops  # noqa: E402

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _values(rng, rows, n_kv, hd):
    x = rng.standard_normal((rows, n_kv, hd)) * np.exp2(rng.normal(0, 1, (rows, 1, 1)))
    x[:, :, rng.integers(0, hd, 3)] *= 6.0
    return x.astype(np.float32)


def _filled(rng, n_pages, n_kv, hd, page, fmt, values=None):
    """A cache of quantised values written from the host, and its K/V in 64 bits [pages][kv][page][hd]."""
    cache = ops.MxKvCache.empty(n_pages, n_kv, hd, page, fmt)
    vals = []
    for codes, scales in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)):
        x = values if values is not None else _values(rng, n_pages * page, n_kv, hd)
        c, s = R.encode(x, fmt)
        c = c.reshape(n_pages, page, n_kv, -1).transpose(0, 2, 1, 3)
        s = s.reshape(n_pages, page, n_kv, -1).transpose(0, 2, 1, 3)
        codes.copy_(torch.from_numpy(np.ascontiguousarray(c)))
        scales.copy_(torch.from_numpy(np.ascontiguousarray(s)))
        vals.append(R.decode(c, s, fmt))
    return cache, vals[0], vals[1]


def _errors():
    import ctypes
    bits = ctypes.c_uint32(0)
    st = fp4x.lib().fp4x_device_error(torch.cuda.current_stream().cuda_stream, ctypes.byref(bits))
    return st, bits.value


# ------------------------------------------------------------------ append, read

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("n,n_kv,hd,page", [(1, 1, 64, 16), (37, 4, 64, 32), (130, 8, 128, 64), (257, 3, 128, 256),
                                            (19, 2, 128, 128)])
def test_append_and_read_are_exact(fmt, dtype, n, n_kv, hd, page):
    rng = np.random.default_rng(n + hd)
    n_pages = -(-n // page) + 2
    cache = ops.MxKvCache.empty(n_pages, n_kv, hd, page, fmt)
    for t in (cache.k, cache.v, cache.k_scales, cache.v_scales):
        t.fill_(0x5A)
    slots = rng.permutation(n_pages * page)[:n].astype(np.int32)
    keep = slots.copy()
    if n > 8:
        slots[3] = slots[7] = -1  # padding rows
    # K and V are slices of a wider projection
    qkv = torch.from_numpy(_values(rng, n, 4 * n_kv, hd)).to(DT[dtype]).cuda()
    k, v = qkv[:, 2 * n_kv:3 * n_kv], qkv[:, 3 * n_kv:]
    ops.kv_append_mx(cache, torch.from_numpy(slots).cuda(), k, v)
    gk, gv = ops.kv_read_mx(cache, torch.from_numpy(slots).cuda(), torch.float32)
    hk, hv = ops.kv_read_mx(cache, torch.from_numpy(slots).cuda(), torch.bfloat16)
    for x, codes, scales, got, half in ((k, cache.k, cache.k_scales, gk, hk), (v, cache.v, cache.v_scales, gv, hv)):
        c, s = R.encode(x.float().cpu().numpy(), fmt)
        codes, scales = codes.cpu().numpy(), scales.cpu().numpy()
        untouched = np.ones((n_pages, page), bool)
        want = R.decode(c, s, fmt)
        for i, slot in enumerate(slots):
            if slot < 0:
                want[i] = 0
                continue
            untouched[slot // page, slot % page] = False
            assert np.array_equal(codes[slot // page, :, slot % page], c[i])
            assert np.array_equal(scales[slot // page, :, slot % page], s[i])
        assert np.all(codes.transpose(0, 2, 1, 3)[untouched] == 0x5A)
        assert np.all(scales.transpose(0, 2, 1, 3)[untouched] == 0x5A)
        # a code has at most four significant bits: exact in both types
        assert np.array_equal(got.cpu().numpy().astype(np.float64), want)
        assert np.array_equal(half.float().cpu().numpy().astype(np.float64), want)
    assert keep.shape == slots.shape


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_append_special_values(fmt):
    hd, page = 64, 16
    rows = np.zeros((12, 1, hd), np.float32)
    rows[1] = 1e-45                                # smallest subnormal
    rows[2, 0, :32] = np.linspace(-3.4e38, 3.4e38, 32)
    rows[3, 0, 5] = np.inf
    rows[3, 0, 6] = -np.inf
    rows[4, 0, 40] = np.nan
    rows[4, 0, 41] = 7.0
    rows[5] = -0.0
    rows[6, 0] = np.tile(np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], np.float32), 8)  # ties of E2M1
    rows[7, 0] = np.tile(np.array([464.0, 479.0, 511.0, 448.0, 432.0, 17.0, 19.0, 0.001], np.float32), 8)
    rows[8, 0] = -np.exp2(np.arange(64) - 32.0)
    rows[9, 0, 0] = 2.0 ** -126
    rows[10, 0, :3] = [3e38, 1e-30, -1e-30]
    rows[11] = 1.1754944e-38 * np.arange(64)
    cache = ops.MxKvCache.empty(2, 1, hd, page, fmt)
    x = torch.from_numpy(rows).cuda()
    slots = torch.arange(12, dtype=torch.int32, device="cuda")
    ops.kv_append_mx(cache, slots, x, x)
    c, s = R.encode(rows, fmt)
    got_c, got_s = cache.k[0, 0, :12].cpu().numpy(), cache.k_scales[0, 0, :12].cpu().numpy()
    assert np.array_equal(got_s, s[:, 0])
    nan_block = np.repeat(s[:, 0] == 255, 32, -1)
    if fmt == "mxfp8":
        assert np.array_equal(got_c, c[:, 0])
    else:  # codes of a NaN block mean nothing
        assert np.array_equal(np.where(nan_block, 0, R.decode(got_c, np.where(s[:, 0] == 255, 127, s[:, 0]), fmt)),
                              np.where(nan_block, 0, R.decode(c[:, 0], np.where(s[:, 0] == 255, 127, s[:, 0]), fmt)))
    k, v = ops.kv_read_mx(cache, slots, torch.float32)
    want = R.decode(c, s, fmt)
    with np.errstate(over="ignore"):
        assert np.array_equal(k.cpu().numpy(), want.astype(np.float32), equal_nan=True)
    assert torch.equal(k.isnan(), v.isnan())


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_append_bf16_ties_and_zeros(fmt):
    """Every bf16 value between 2^-4 and 8 beside a fixed block maximum, both signs, zeros of both signs."""
    bits = np.concatenate([np.arange(0x3D80, 0x4100), [0]]).astype(np.uint32)
    vals = (bits << 16).view(np.float32)
    vals = np.concatenate([vals, -vals])
    n = -(-len(vals) // 62)
    rows = np.zeros((n, 1, 64), np.float32)
    body = np.zeros(n * 62, np.float32)
    body[: len(vals)] = vals
    rows[:, 0, :31], rows[:, 0, 32:63] = body.reshape(n, 62)[:, :31], body.reshape(n, 62)[:, 31:]
    rows[:, 0, 31], rows[:, 0, 63] = 7.0, -7.5
    cache = ops.MxKvCache.empty(-(-n // 16), 1, 64, 16, fmt)
    x = torch.from_numpy(rows).to(torch.bfloat16).cuda()
    assert torch.equal(x.float().cpu(), torch.from_numpy(rows))
    ops.kv_append_mx(cache, torch.arange(n, dtype=torch.int32, device="cuda"), x, x)
    c, s = R.encode(rows, fmt)
    assert np.array_equal(cache.k[:, 0].flatten(0, 1)[:n].cpu().numpy(), c[:, 0])
    assert np.array_equal(cache.v_scales[:, 0].flatten(0, 1)[:n].cpu().numpy(), s[:, 0])


def test_slots_past_the_cache_are_skipped_and_reported():
    cache = ops.MxKvCache.empty(2, 2, 64, 16, "mxfp8")
    cache.k.fill_(1), cache.v.fill_(1), cache.k_scales.fill_(127), cache.v_scales.fill_(127)
    x = torch.ones((3, 2, 64), device="cuda")
    ops.kv_append_mx(cache, torch.tensor([0, 32, 2**31 - 1], dtype=torch.int32, device="cuda"), x, x)
    st, bits = _errors()
    assert st == 3 and bits & 4
    assert int((cache.k != 1).any(-1).sum()) == 2  # one slot, two heads
    k, _ = ops.kv_read_mx(cache, torch.tensor([0, 40], dtype=torch.int32, device="cuda"), torch.float32)
    assert _errors()[0] == 3
    assert torch.all(k[0] == 1) and torch.all(k[1] == 0)
    assert _errors() == (0, 0)


# ------------------------------------------------------------------ attention

def _attention_case(rng, cache, kv, vv, lens, page, group, q_len, dtype, prefix=0, max_len=None, q=None):
    """Runs the operator and the definition; returns (got, want, mass, size)."""
    n_pages, n_kv, _, hd = kv.shape
    B = len(lens)
    max_len = max(max(lens), 1) if max_len is None else max_len
    order = rng.permutation(n_pages)
    n_prefix = -(-prefix // page)
    width = -(-max_len // page)
    table = np.full((B, width), -1, np.int32)  # unused entries are no pages
    at = n_prefix
    for b, n in enumerate(lens):
        need = -(-n // page)
        table[b, :need] = order[at:at + need]
        at += need
    assert at <= n_pages
    H = n_kv * group
    if q is None:
        q = rng.standard_normal((B, q_len, H, hd)).astype(np.float32) * 2
    # q as a slice of the fused projection
    wide = torch.zeros((B, q_len, H + 2 * n_kv, hd), dtype=DT[dtype], device="cuda")
    wide[:, :, :H] = torch.from_numpy(q).cuda()
    tq = wide[:, :, :H]
    args = (torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), max_len)
    if prefix:
        pp = torch.from_numpy(order[:n_prefix].astype(np.int32)).cuda()
        got = ops.attn_shared_mx(cache, tq, pp, prefix, *args)
    else:
        got = ops.attn_paged_mx(cache, tq, *args)
    qq = tq.float().cpu().numpy().astype(np.float64)
    want, mass, size = np.zeros_like(qq), np.zeros_like(qq), np.zeros(qq.shape[:3] + (1,))

    def rows(x, pages, n):
        return x[pages].transpose(0, 2, 1, 3).reshape(-1, n_kv, hd)[:n]

    for b, n in enumerate(lens):
        pages = table[b, : -(-n // page)]
        k, v = rows(kv, pages, n), rows(vv, pages, n)
        if prefix:
            k = np.concatenate((rows(kv, order[:n_prefix], prefix), k))
            v = np.concatenate((rows(vv, order[:n_prefix], prefix), v))
        limits = [prefix + max(0, n - q_len + 1 + i) for i in range(q_len)]
        want[b], mass[b], size[b] = R.attention(qq[b], k, v, limits)
    return got, want, mass, size


def _close(got, want, mass, size, dtype):
    """bf16: half a bf16 step of the result, and probabilities rounded to at least bf16 (2^-9 of sum p|v|).
    f32: the scores' error (f32 accumulation and 22-bit operands: 2^-20 of sum |q k|) shifts every p by that factor,
    the products and sums add 2^-20 of sum p|v|."""
    assert got.dtype == DT[dtype]
    g = got.float().cpu().numpy().astype(np.float64)
    assert np.isfinite(g).all()
    bound = 2.0 ** -9 * (np.abs(want) + mass) if dtype == "bf16" else 0.0
    bound = bound + 2.0 ** -20 * mass * (2 + 2 * size) + 1e-37
    bad = np.abs(g - want) > bound
    assert not bad.any(), (np.abs(g - want) / bound).max()


SHAPES = [
    # n_kv, group, hd, page, q_len, lens
    (1, 1, 64, 16, 1, [1]),
    (1, 1, 128, 64, 1, [1, 0, 2]),
    (2, 4, 128, 16, 1, [15, 16, 17, 31, 32, 33]),
    (8, 4, 128, 64, 1, [700]),
    (4, 8, 64, 32, 1, [513, 0, 1, 1000]),
    (2, 7, 128, 128, 1, [255, 129, 5]),
    (3, 2, 64, 256, 1, [300, 256]),
    (1, 16, 128, 16, 1, [97, 64]),
    (2, 4, 128, 16, 5, [200, 5, 4, 1, 0, 65]),  # queries that see nothing where the length is below q_len
    (1, 8, 64, 64, 3, [1, 2, 3, 130]),
    (2, 1, 64, 32, 8, [8, 77]),
    (1, 4, 128, 64, 16, [400, 16]),
]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_paged_attention(shape, fmt, dtype):
    n_kv, group, hd, page, q_len, lens = shape
    rng = np.random.default_rng(hd + group + len(lens))
    n_pages = sum(-(-n // page) for n in lens) + 1
    cache, kv, vv = _filled(rng, n_pages, n_kv, hd, page, fmt)
    got, want, mass, size = _attention_case(rng, cache, kv, vv, lens, page, group, q_len, dtype,
                                            max_len=max(lens) + 40)
    _close(got, want, mass, size, dtype)
    assert _errors() == (0, 0)


SHARED = [
    # n_kv, group, hd, page, q_len, prefix, lens
    (1, 1, 64, 16, 1, 1, [0, 1]),
    (2, 4, 128, 64, 1, 127, [0, 3, 64]),
    (2, 4, 128, 16, 1, 128, [1, 200, 17]),
    (4, 8, 64, 32, 1, 1000, [33, 0]),
    (1, 4, 128, 64, 4, 600, [10] * 11),
    (1, 7, 64, 128, 3, 259, [2, 0, 150, 3] * 5),
    (1, 8, 128, 16, 2, 513, list(range(1, 20))),
    (2, 2, 128, 64, 1, 384, [5] * 140),
]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("shape", SHARED, ids=lambda s: str(s[:6]) + f"x{len(s[6])}")
def test_shared_attention(shape, fmt, dtype):
    n_kv, group, hd, page, q_len, prefix, lens = shape
    rng = np.random.default_rng(hd + group + prefix)
    n_pages = sum(-(-n // page) for n in lens) + -(-prefix // page) + 1
    cache, kv, vv = _filled(rng, n_pages, n_kv, hd, page, fmt)
    got, want, mass, size = _attention_case(rng, cache, kv, vv, lens, page, group, q_len, dtype, prefix=prefix)
    _close(got, want, mass, size, dtype)
    assert _errors() == (0, 0)


def test_shared_without_prefix_and_without_own_positions():
    rng = np.random.default_rng(9)
    cache, kv, vv = _filled(rng, 12, 2, 64, 16, "mxfp8")
    q = torch.randn((3, 1, 8, 64), device="cuda")
    table = torch.arange(9, dtype=torch.int32, device="cuda").view(3, 3)
    lens = torch.tensor([40, 0, 17], dtype=torch.int32, device="cuda")
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    a, b = ops.attn_shared_mx(cache, q, none, 0, table, lens), ops.attn_paged_mx(cache, q, table, lens)
    assert torch.equal(a, b) and torch.all(b[1] == 0)
    # nothing of their own: every sequence sees the prefix alone
    empty_table = torch.empty((3, 0), dtype=torch.int32, device="cuda")
    zero = torch.zeros(3, dtype=torch.int32, device="cuda")
    c = ops.attn_shared_mx(cache, q, table[0].contiguous(), 40, empty_table, zero, 0)
    d = ops.attn_paged_mx(cache, q, table[:1].expand(3, 3).contiguous(), torch.full_like(lens, 40))
    torch.testing.assert_close(c, d, rtol=1e-5, atol=1e-5)
    assert torch.all(ops.attn_paged_mx(cache, q, empty_table, zero, 0) == 0)


@pytest.mark.parametrize("prefix", [0, 37])
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_rows_past_the_length_are_not_used(fmt, prefix):
    """NaN codes and NaN scales in rows past the length (and in pages of no sequence) change nothing."""
    page, n_kv, hd, lens = 32, 2, 128, [45, 3, 0, 70]
    outs = []
    for dirty in (False, True):
        rng = np.random.default_rng(4)
        cache, kv, vv = _filled(rng, 16, n_kv, hd, page, fmt)
        order = np.random.default_rng(8).permutation(16)
        table = np.zeros((4, 3), np.int32)
        at = 2
        live = torch.zeros((16, page), dtype=torch.bool)
        for b, n in enumerate(lens):
            for j in range(-(-n // page)):
                table[b, j] = order[at]
                live[order[at], : min(page, n - j * page)] = True
                at += 1
        for j in range(-(-prefix // page)):
            live[order[j], : min(page, prefix - j * page)] = True
        if dirty:
            gone = ~live.cuda()[:, None, :].expand(16, n_kv, page)
            for t in (cache.k, cache.v):
                t[gone] = 0x7F if fmt == "mxfp8" else 0xFF
            for t in (cache.k_scales, cache.v_scales):
                t[gone] = 255
        g = torch.Generator(device="cuda").manual_seed(3)
        q = torch.randn((4, 2, 8, hd), generator=g, device="cuda")
        args = (torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"))
        for dtype in (torch.float32, torch.bfloat16):
            if prefix:
                pp = torch.from_numpy(order[:2].astype(np.int32)).cuda()
                outs.append(ops.attn_shared_mx(cache, q.to(dtype), pp, prefix, *args))
            else:
                outs.append(ops.attn_paged_mx(cache, q.to(dtype), *args))
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])
    assert torch.isfinite(outs[2]).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("prefix", [0, 48])
def test_value_scales_of_every_size(dtype, prefix):
    """Positions whose V is 2^60 times another's, with the probability on the small ones: nothing underflows."""
    rng = np.random.default_rng(12)
    page, n_kv, hd = 16, 1, 64
    n = 48
    v = rng.standard_normal((10 * page, n_kv, hd)).astype(np.float32)
    v *= np.exp2(rng.integers(-30, 30, (10 * page, 1, 1))).astype(np.float32)
    cache, kv, vv = _filled(rng, 10, n_kv, hd, page, "mxfp8", values=v)
    _, kv2, _ = None, None, None
    # keys equal to the values' rows would make scores huge: small keys, so that probabilities stay comparable
    k = (rng.standard_normal((10 * page, n_kv, hd)) * 0.5).astype(np.float32)
    c, s = R.encode(k, "mxfp8")
    cc, ss = c.reshape(10, page, n_kv, -1).transpose(0, 2, 1, 3), s.reshape(10, page, n_kv, -1).transpose(0, 2, 1, 3)
    cache.k.copy_(torch.from_numpy(np.ascontiguousarray(cc)))
    cache.k_scales.copy_(torch.from_numpy(np.ascontiguousarray(ss)))
    kv = R.decode(cc, ss, "mxfp8")
    lens = [n, 5]
    got, want, mass, size = _attention_case(rng, cache, kv, vv, lens, page, 4, 1, dtype, prefix=prefix)
    _close(got, want, mass, size, dtype)


def test_probability_on_small_values():
    """One position takes almost all of the probability and has V 2^25 times smaller than the rest, whose probability is
    far below 2^-25: the result is the small value, to the accuracy of the sum."""
    page, hd = 16, 64
    for fmt in ("mxfp8", "mxfp4"):
        rng = np.random.default_rng(1)
        n = 40
        k = np.zeros((3 * page, 1, hd), np.float32)
        k[:, 0, 0] = -4.0
        k[21, 0, 0] = 4.0
        v = rng.choice([1.0, 1.5, 2.0, 3.0], (3 * page, 1, hd)).astype(np.float32)
        v[21] *= 2.0 ** -25
        cache = ops.MxKvCache.empty(3, 1, hd, page, fmt)
        slots = torch.arange(3 * page, dtype=torch.int32, device="cuda")
        ops.kv_append_mx(cache, slots, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda())
        kk, vv = (x.double().cpu().numpy() for x in ops.kv_read_mx(cache, slots, torch.float32))
        q = np.zeros((1, 1, 4, hd), np.float32)
        q[..., 0] = [30.0, 40.0, 60.0, 100.0]
        for dtype in ("f32", "bf16"):
            got = ops.attn_paged_mx(cache, torch.from_numpy(q).to(DT[dtype]).cuda(),
                                    torch.arange(3, dtype=torch.int32, device="cuda")[None],
                                    torch.tensor([n], dtype=torch.int32, device="cuda"))
            want, mass, size = R.attention(q[0].astype(np.float64), kk, vv, [n])
            _close(got, want[None], mass[None], size[None], dtype)


def test_invalid_pages_are_masked_and_reported():
    rng = np.random.default_rng(2)
    cache, kv, vv = _filled(rng, 6, 1, 64, 16, "mxfp8")
    q = torch.randn((2, 1, 4, 64), device="cuda")
    table = torch.tensor([[0, 6, 2], [3, 4, 5]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([48, 48], dtype=torch.int32, device="cuda")
    out = ops.attn_paged_mx(cache, q, table, lens)
    st, bits = _errors()
    assert st == 3 and bits & 4 and torch.isfinite(out).all()
    clean = torch.tensor([[0, 2, 2], [3, 4, 5]], dtype=torch.int32, device="cuda")
    want = ops.attn_paged_mx(cache, q, clean, torch.tensor([32, 48], dtype=torch.int32, device="cuda"))
    torch.testing.assert_close(out, want, rtol=1e-5, atol=1e-5)
    assert _errors() == (0, 0)


def test_lengths_outside_the_table_are_clamped():
    rng = np.random.default_rng(2)
    cache, kv, vv = _filled(rng, 6, 1, 64, 16, "mxfp4")
    q = torch.randn((2, 1, 4, 64), device="cuda")
    table = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32, device="cuda")
    a = ops.attn_paged_mx(cache, q, table, torch.tensor([2**31 - 1, -5], dtype=torch.int32, device="cuda"))
    b = ops.attn_paged_mx(cache, q, table, torch.tensor([48, 0], dtype=torch.int32, device="cuda"))
    assert torch.equal(a, b)


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_pages_of_one_allocation_past_4_gib(fmt):
    """K and V pages in turn in one allocation, pages far apart: offsets pass 32 bits."""
    n_kv, hd, page, n_pages = 2, 128, 64, 20
    row = hd if fmt == "mxfp8" else hd // 2
    far = 300 << 20
    base = torch.zeros(n_pages * far, dtype=torch.uint8, device="cuda")
    code, scale = n_kv * page * row, n_kv * page * 4

    def part(off, shape):
        inner = [shape[1] * shape[2], shape[2], 1]
        return torch.as_strided(base, (n_pages,) + shape, [far] + inner, off)

    views = [part(0, (n_kv, page, row)), part(2 * code, (n_kv, page, 4)), part(code, (n_kv, page, row)),
             part(2 * code + scale, (n_kv, page, 4))]
    cache = ops.MxKvCache(*views)
    dense = ops.MxKvCache.empty(n_pages, n_kv, hd, page, fmt)
    n = n_pages * page
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn((n, n_kv, hd), generator=g, device="cuda") for _ in range(2))
    slots = torch.randperm(n, generator=g, device="cuda").int()
    for c in (cache, dense):
        ops.kv_append_mx(c, slots, k, v)
    for a, b in zip(ops.kv_read_mx(cache, slots), ops.kv_read_mx(dense, slots)):
        assert torch.equal(a, b)
    q = torch.randn((2, 1, 8, hd), generator=g, device="cuda")
    table = torch.randperm(n_pages, generator=g, device="cuda").int()[None].repeat(2, 1)
    lens = torch.tensor([n, n - 100], dtype=torch.int32, device="cuda")
    assert torch.equal(ops.attn_paged_mx(cache, q, table, lens), ops.attn_paged_mx(dense, q, table, lens))
    assert torch.equal(ops.attn_shared_mx(cache, q, table[0].contiguous(), n, table, lens),
                       ops.attn_shared_mx(dense, q, table[0].contiguous(), n, table, lens))


@pytest.mark.parametrize("prefix", [0, 700])
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_long_batches_against_torch(fmt, prefix):
    """Sizes at which the work is split over many CTAs, against 64-bit torch on the same rows; twice: the same bits."""
    rng = np.random.default_rng(6)
    page, n_kv, group, hd, q_len = 64, 4, 4, 128, 2
    lens = [5000, 1, 0, 12345, 64, 3000, 2, 777]
    n_pages = sum(-(-n // page) for n in lens) + -(-prefix // page)
    cache = ops.MxKvCache.empty(n_pages, n_kv, hd, page, fmt)
    g = torch.Generator(device="cuda").manual_seed(5)
    k, v = (torch.randn((n_pages * page, n_kv, hd), generator=g, device="cuda") for _ in range(2))
    ops.kv_append_mx(cache, torch.arange(n_pages * page, dtype=torch.int32, device="cuda"), k, v)
    table = torch.full((len(lens), -(-max(lens) // page)), -1, dtype=torch.int32, device="cuda")
    order = torch.from_numpy(rng.permutation(n_pages).astype(np.int32)).cuda()
    at = -(-prefix // page)
    pages = order[:at].contiguous()
    for b, n in enumerate(lens):
        table[b, : -(-n // page)] = order[at:at - (-n // page)]
        at -= -n // page
    tl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for dtype in ("bf16", "f32"):
        q = torch.randn((len(lens), q_len, n_kv * group, hd), generator=g, device="cuda").to(DT[dtype])

        def call():
            return (ops.attn_shared_mx(cache, q, pages, prefix, table, tl) if prefix
                    else ops.attn_paged_mx(cache, q, table, tl))

        got = call()
        want, mass, size = (torch.zeros(q.shape, dtype=torch.float64, device="cuda") for _ in range(3))
        ar = torch.arange(page, device="cuda")
        for b, n in enumerate(lens):
            ids = torch.cat((pages, table[b, : -(-n // page)])).long()
            keep = torch.cat((torch.arange(len(pages) * page, device="cuda") < prefix,
                              torch.arange((-(-n // page)) * page, device="cuda") < n))
            slots = (ids[:, None] * page + ar).reshape(-1)[keep].int()
            kk, vv = (x.double().repeat_interleave(group, 1) for x in ops.kv_read_mx(cache, slots, torch.float32))
            if kk.shape[0] == 0:
                continue
            s = torch.einsum("thd,nhd->thn", q[b].double(), kk) / hd ** 0.5
            size[b] = (torch.einsum("thd,nhd->thn", q[b].double().abs(), kk.abs()) / hd ** 0.5).amax(-1, True)
            lim = prefix + (n - q_len + 1 + torch.arange(q_len, device="cuda")).clamp(min=0)
            s = s.masked_fill(torch.arange(kk.shape[0], device="cuda") >= lim[:, None, None], -torch.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0)
            want[b], mass[b] = torch.einsum("thn,nhd->thd", p, vv), torch.einsum("thn,nhd->thd", p, vv.abs())
        _close(got, want.cpu().numpy(), mass.cpu().numpy(), size.cpu().numpy(), dtype)
        assert torch.equal(got, call())


def test_attention_on_another_stream_and_in_a_graph():
    rng = np.random.default_rng(6)
    cache, kv, vv = _filled(rng, 40, 2, 128, 16, "mxfp8")
    q = torch.randn((4, 1, 8, 128), device="cuda", dtype=torch.bfloat16)
    table = torch.arange(40, dtype=torch.int32, device="cuda").view(4, 10)
    lens = torch.tensor([160, 3, 77, 0], dtype=torch.int32, device="cuda")
    pages = table[0].contiguous()
    slots = torch.tensor([159], dtype=torch.int32, device="cuda")
    want = ops.attn_paged_mx(cache, q, table, lens)
    want2 = ops.attn_shared_mx(cache, q, pages, 150, table, lens)
    ws = ops.attn_mx_workspace(cache, 4, 8, 1, 150, 160)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        a = ops.attn_paged_mx(cache, q, table, lens)
        b = ops.attn_shared_mx(cache, q, pages, 150, table, lens, workspace=ws)
    side.synchronize()
    assert torch.equal(a, want) and torch.equal(b, want2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        k = torch.ones((1, 2, 128), device="cuda")
        ops.kv_append_mx(cache, slots, k, k)
        out = ops.attn_shared_mx(cache, q, pages, 150, table, lens, workspace=ws)
        one = ops.attn_paged_mx(cache, q, table, lens)
    lens.copy_(torch.tensor([160, 160, 0, 9]))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ops.attn_shared_mx(cache, q, pages, 150, table, lens))
    assert torch.equal(one, ops.attn_paged_mx(cache, q, table, lens))


def test_wrappers_refuse():
    cache = ops.MxKvCache.empty(4, 2, 64, 16, "mxfp8")
    q = torch.zeros((2, 1, 8, 64), device="cuda")
    table = torch.zeros((2, 2), dtype=torch.int32, device="cuda")
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        ops.attn_paged_mx(cache, q.half(), table, lens)
    with pytest.raises(ValueError):
        ops.attn_paged_mx(cache, q[..., :32], table, lens)
    with pytest.raises(ValueError):
        ops.attn_paged_mx(cache, q, table.long(), lens)
    with pytest.raises(ValueError):
        ops.attn_paged_mx(cache, q, table[:1], lens)
    with pytest.raises(fp4x.Fp4xError):
        ops.attn_paged_mx(cache, q, table, lens, max_len=33)
    with pytest.raises(ValueError):
        ops.attn_shared_mx(cache, q, lens, 33, table, lens)
    with pytest.raises(ValueError):
        ops.attn_paged_mx(cache, torch.zeros((2, 8, 3, 64), device="cuda").transpose(1, 2), table, lens)
    with pytest.raises(ValueError):
        ops.attn_paged_mx(cache, q.cpu(), table, lens)
    x = torch.zeros((3, 2, 64), device="cuda")
    with pytest.raises(ValueError):
        ops.kv_append_mx(cache, lens, x, x)
    with pytest.raises(ValueError):
        ops.kv_append_mx(cache, torch.zeros(3, dtype=torch.int64, device="cuda"), x, x)
    with pytest.raises(ValueError):
        ops.MxKvCache(cache.k, cache.k_scales, cache.v[:2], cache.v_scales)
