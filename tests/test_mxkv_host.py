"""MX KV cache and draft verification: refusals (host checks, nothing launched) and the reference definitions."""
import ctypes

import numpy as np
import pytest

import fp4x
import mxkv_ref as R


def _cache(**kw):
    d = dict(k=4096, k_scales=8192, v=1 << 20, v_scales=1 << 21, page_stride=64 * 8 * 128, scale_page_stride=64 * 8 * 4,
             n_pages=4, page_size=64, n_kv_heads=8, head_dim=128, format=0)
    d.update(kw)
    return fp4x.MxKv(**d)


BAD_CACHES = [dict(page_size=48), dict(page_size=8), dict(head_dim=96), dict(format=2), dict(n_pages=0),
              dict(n_kv_heads=0), dict(k=None), dict(v_scales=None), dict(k=4104), dict(page_stride=64 * 8 * 128 - 16),
              dict(page_stride=64 * 8 * 128 + 8), dict(scale_page_stride=64 * 8 * 4 - 8), dict(k_scales=8196),
              dict(scale_page_stride=64 * 8 * 4 + 4), dict(n_pages=1 << 25), dict(page_stride=1 << 32), dict(scale_page_stride=1 << 32)]


def _p(c):
    return None if c is None else ctypes.addressof(c)


def _append(c, n=4, slots=64, dtype=0, k=4096, ks=1024, v=4096, vs=1024):
    return fp4x.lib().llama_kv_append_mx(None, _p(c), n, slots, dtype, k, ks, v, vs)


def _attn(c, batch=2, heads=32, q_len=1, prefix=None, prefix_len=0, table=64, stride=16, lens=64, max_len=1024, dtype=1,
          q=4096, q_stride=4096, out=4096, ws=4096, nbytes=1 << 40):
    L = fp4x.lib()
    if prefix is None and prefix_len == 0:
        return L.llama_attn_paged_mx(None, _p(c), batch, heads, q_len, table, stride, lens, max_len, dtype, q, q_stride,
                                     out, ws, nbytes)
    return L.llama_attn_shared_mx(None, _p(c), batch, heads, q_len, prefix, prefix_len, table, stride, lens, max_len,
                                  dtype, q, q_stride, out, ws, nbytes)


def _verify(batch=2, k=3, vocab=100, dtype=0, logits=4096, stride=100, probs=4096, drafts=4096, lens=None, u=4096,
            noise=4096, temp=None, acc=4096, tok=4096, lp=None, ws=4096, nbytes=1 << 40):
    return fp4x.lib().llama_verify_drafts(None, batch, k, vocab, dtype, logits, stride, probs, drafts, lens, u, noise,
                                          temp, acc, tok, lp, ws, nbytes)


@pytest.mark.parametrize("bad", BAD_CACHES, ids=lambda b: "-".join(b))
def test_bad_caches_are_refused(bad):
    c = _cache(**bad)
    for call in (lambda: _append(c), lambda: _attn(c),
                 lambda: fp4x.lib().llama_kv_read_mx(None, _p(c), 4, 64, 0, 4096, 4096)):
        assert call() == 1 and fp4x.last_error()
    assert _append(None) == 1 and b"null cache" in fp4x.lib().fp4x_last_error()


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(slots=None), dict(k=None), dict(k=4104), dict(ks=1022),
                                 dict(vs=1020), dict(dtype=1, ks=1028)], ids=str)
def test_append_refuses(bad):
    assert _append(_cache(), **bad) == 1


def test_read_refuses():
    f = fp4x.lib().llama_kv_read_mx
    c = _cache()
    assert f(None, _p(c), 4, 64, 7, 4096, 4096) == 1
    assert f(None, _p(c), 4, None, 0, 4096, 4096) == 1
    assert f(None, _p(c), 4, 64, 0, 4096, 4100) == 1


@pytest.mark.parametrize("bad", [dict(heads=30), dict(heads=0), dict(q_len=0), dict(q_len=65), dict(table=None),
                                 dict(lens=None), dict(stride=15), dict(dtype=3), dict(q=4104), dict(out=None),
                                 dict(q_stride=4092), dict(q_stride=4088), dict(prefix=None, prefix_len=5),
                                 dict(max_len=0x7FFFFFFF, stride=1 << 26), dict(prefix=64, prefix_len=0xFFFFFFFF)],
                         ids=str)
def test_attention_refuses(bad):
    assert _attn(_cache(), **bad) == 1


def test_attention_refuses_a_small_workspace():
    c = _cache()
    need = fp4x.lib().llama_attn_mx_workspace_size(_p(c), 2, 32, 1, 0, 1024)
    if need:
        assert _attn(c, nbytes=need - 1) == 1
        assert _attn(c, ws=4104) == 1
    assert fp4x.lib().llama_attn_mx_workspace_size(None, 2, 32, 1, 0, 1024) == 0


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(vocab=0), dict(stride=99), dict(k=256), dict(batch=70000),
                                 dict(logits=None), dict(logits=4098), dict(noise=None), dict(drafts=None), dict(u=None),
                                 dict(acc=None), dict(tok=None)], ids=str)
def test_verify_refuses(bad):
    assert _verify(**bad) == 1


def test_verify_refuses_a_small_workspace():
    need = fp4x.lib().llama_verify_workspace_size(2, 3, 100)
    if need:
        assert _verify(nbytes=need - 1) == 1


def test_empty_calls_do_nothing():
    assert _append(_cache(), n=0) == 0
    assert fp4x.lib().llama_kv_read_mx(None, _p(_cache()), 0, None, 0, None, None) == 0
    assert _attn(_cache(), batch=0) == 0
    assert _verify(batch=0) == 0


@pytest.mark.parametrize("fmt,top,rel", [("mxfp8", 448.0, 2.0 ** -4), ("mxfp4", 6.0, 2.0 ** -2)])
def test_reference_encode_decode(fmt, top, rel):
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((50, 128)) * np.exp2(rng.integers(-20, 20, (50, 1)))).astype(np.float32)
    rows, scales = R.encode(x, fmt)
    y = R.decode(rows, scales, fmt)
    block = np.repeat(np.abs(x).reshape(50, 4, 32).max(-1), 32, -1)
    # half a step of the code (rel of the value, at least the smallest step); values past the largest code saturate
    limit = np.maximum(np.abs(x) * rel, block * 2.0 ** -2 * (1 if fmt == "mxfp4" else 2.0 ** -6))
    unit = np.repeat(np.exp2(scales.astype(np.float64) - 127), 32, -1)
    limit = np.where(np.abs(x) > top * unit, np.abs(x) - top * unit, limit)
    assert np.all(np.abs(x - y) <= limit)
    assert np.array_equal(R.decode(*R.encode(y, fmt), fmt), y)


def test_reference_verify_keeps_the_target_distribution():
    # over many draws the emitted first token follows the target's softmax, whatever the draft proposes
    rng = np.random.default_rng(5)
    V, n = 5, 20000
    logits = np.broadcast_to(rng.standard_normal(V), (n, 2, V))
    p = np.exp(logits[0, 0]) / np.exp(logits[0, 0]).sum()
    q = rng.dirichlet(np.ones(V))
    drafts = rng.choice(V, (n, 1), p=q)
    acc, tok, _ = R.verify(logits, drafts, rng.random((n, 1)), rng.exponential(size=(n, V)),
                           probs=np.broadcast_to(q, (n, 1, V)))
    got = np.bincount(tok[:, 0], minlength=V) / n
    # binomial deviation: five standard deviations
    assert np.all(np.abs(got - p) <= 5 * np.sqrt(p * (1 - p) / n))
    assert abs(acc.mean() - np.minimum(p, q).sum()) <= 5 * 0.5 / np.sqrt(n)


@pytest.mark.parametrize("own,prefix", [(0x7FFFFF80, 0), (0x7FFFFF00, 0), (0x7FFFFFFE, 0), (0, 0x7FFFFF80), (0x3FFFFFFF, 0x3FFFFFFF)],
                         ids=str)
def test_lengths_whose_last_tile_passes_31_bits_are_refused(own, prefix):
    """A tile of up to 128 positions that starts below such a length ends past 2^31."""
    assert _attn(_cache(), max_len=own, stride=1 << 26, prefix=64 if prefix else None, prefix_len=prefix) == 1
    assert b"2^31" in fp4x.lib().fp4x_last_error()
