"""Verification of drafted tokens against the 64-bit definition."""
import numpy as np
import pytest

import mxkv_ref as R

torch = pytest.importorskip("torch")
from fp4x import ops  # noqa: E402

pytestmark = pytest.mark.gpu


def _case(seed, B, k, V, dtype=torch.float32, probs=True, agree=0.7):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*s):
        return torch.randn(s, generator=g, device="cuda")

    logits = (normal(B, k + 1, V) * 2.5).to(dtype)
    draft = logits[:, :k].float() + agree * normal(B, k, V)
    q = torch.softmax(draft, -1)
    drafts = (q / torch.empty_like(q).exponential_(generator=g)).argmax(-1).int()
    u = torch.rand((B, k), generator=g, device="cuda")
    noise = torch.empty((B, V), device="cuda").exponential_(generator=g)
    return logits, drafts, u, noise, q if probs else None


def _check(args, **kw):
    logits, drafts, u, noise, q = args
    acc, tok, lp = ops.verify_drafts(logits, drafts, u, noise, draft_probs=q, **kw)

    def host(t):
        return None if t is None else t.double().cpu().numpy()

    want = R.verify(host(logits), drafts.cpu().numpy(), host(u), host(noise), host(q),
                    host(kw.get("draft_lens")), host(kw.get("temperature")))
    assert np.array_equal(acc.cpu().numpy(), want[0])
    assert np.array_equal(tok.cpu().numpy(), want[1])
    # f32 sums of up to V terms and one exp/log: 2^-20 relative of the sum, 2^-22 of the shifted logit
    got = lp.double().cpu().numpy()
    fine = np.isfinite(want[2])
    assert np.array_equal(fine, np.isfinite(got))
    assert np.all(np.abs(got - want[2])[fine] <= 2.0 ** -20 + 2.0 ** -21 * np.abs(want[2][fine]))
    return want


@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,k,V", [(1, 1, 7), (3, 4, 1000), (2, 3, 32000), (5, 8, 4097), (9, 2, 1025), (1, 5, 128256),
                                   (40, 4, 2001), (2, 0, 300), (1, 15, 1)])
def test_verify(B, k, V, dtype, probs):
    args = _case(B + k + V, B, k, V, dtype, probs)
    lens = torch.tensor([(3 * b + 1) % (k + 1) for b in range(B)], dtype=torch.int32, device="cuda")
    temp = torch.tensor([(0.7, 1.0, 0.0, 1.6)[b % 4] for b in range(B)], device="cuda")
    want = _check(args)
    _check(args, draft_lens=lens)
    _check(args, draft_lens=lens, temperature=temp)
    if B >= 40:
        assert len(set(want[0].tolist())) > 2  # the draws reach different lengths


def test_verify_everything_agrees_or_nothing():
    logits, drafts, u, noise, _ = _case(3, 4, 3, 500)
    q = torch.softmax(logits[:, :3].float(), -1)
    _check((logits, drafts, u * 0.999, noise, q))      # u q < p: p == q up to rounding, u below 1
    _check((logits, drafts, u * 0 + 1.0, noise, q * 2))  # never accepted; q above p everywhere: falls back to p
    best = logits[:, :3].float().argmax(-1).int()
    zero = torch.zeros(4, device="cuda")
    want = _check((logits, best, u, noise, None), temperature=zero)
    assert want[0].tolist() == [3, 3, 3, 3]


def test_verify_masked_logits():
    """-inf, NaN and +inf logits, rows without any mass, drafts outside the vocabulary."""
    logits, drafts, u, noise, q = _case(11, 8, 3, 300)
    logits[0, :, 5:] = -torch.inf
    drafts[0, 0] = 7
    logits[1, 0] = -torch.inf                     # no token is possible
    logits[2, :, 17] = torch.nan
    drafts[2, 0] = 17
    logits[3, 1, 4] = torch.inf
    drafts[4, 0], drafts[4, 1], drafts[5, 0] = -1, 300, 2**31 - 1
    logits[6, 1] = torch.nan
    logits[7, 0, :] = 3.4e38
    u[7] = 0
    for qq in (q, None):
        for t in (None, torch.full((8,), 0.5, device="cuda"), torch.zeros(8, device="cuda"),
                  torch.full((8,), torch.nan, device="cuda")):
            with np.errstate(all="ignore"):
                acc, tok, lp = ops.verify_drafts(logits, drafts, u, noise, draft_probs=qq, temperature=t)
                want = R.verify(logits.double().cpu().numpy(), drafts.cpu().numpy(), u.double().cpu().numpy(),
                                noise.double().cpu().numpy(), None if qq is None else qq.double().cpu().numpy(), None,
                                None if t is None else t.double().cpu().numpy())
            assert np.array_equal(acc.cpu().numpy(), want[0]) and np.array_equal(tok.cpu().numpy(), want[1])
            assert not np.isnan(lp.cpu().numpy()).any()


def test_verify_ties_go_to_the_lowest_index():
    logits = torch.zeros((2, 3, 5000), device="cuda")
    logits[:, :, [40, 700, 4999]] = 4.0
    drafts = torch.tensor([[40, 700], [40, 40]], dtype=torch.int32, device="cuda")
    u, noise = torch.full((2, 2), 0.5, device="cuda"), torch.ones((2, 5000), device="cuda")
    acc, tok, _ = ops.verify_drafts(logits, drafts, u, noise, temperature=torch.zeros(2, device="cuda"))
    assert acc.tolist() == [1, 2] and tok.tolist() == [[40, 40, -1], [40, 40, 40]]
    _, tok, _ = ops.verify_drafts(logits, drafts, u, noise, draft_lens=torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert tok[:, 0].tolist() == [40, 40]


def test_verify_strided_logits_and_stream():
    """Rows of a padded vocabulary, unaligned, on another stream."""
    wide = torch.randn((3, 5, 1100), device="cuda") * 2
    for off, V in ((0, 1001), (1, 1000), (3, 1097)):
        logits = wide[..., off:off + V]
        _, drafts, u, noise, q = _case(off, 3, 4, V)
        a = ops.verify_drafts(logits, drafts, u, noise, draft_probs=q)
        b = ops.verify_drafts(logits.contiguous(), drafts, u, noise, draft_probs=q)
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            c = ops.verify_drafts(logits, drafts, u, noise, draft_probs=q)
        side.synchronize()
        for x, y, z in zip(a, b, c):
            torch.testing.assert_close(x, y, rtol=1e-5, atol=1e-5)
            assert torch.equal(x, z)
        _check((logits, drafts, u, noise, q))


def test_verify_samples_the_target():
    """Over many sequences the first emitted token follows the target's softmax (five standard deviations)."""
    B, V = 20000, 6
    g = torch.Generator(device="cuda").manual_seed(2)
    row = torch.randn(V, generator=g, device="cuda")
    logits = row.expand(B, 2, V).contiguous()
    q = torch.softmax(torch.randn(V, generator=g, device="cuda"), -1)
    drafts = torch.multinomial(q, B, replacement=True, generator=g).int()[:, None].contiguous()
    u = torch.rand((B, 1), generator=g, device="cuda")
    noise = torch.empty((B, V), device="cuda").exponential_(generator=g)
    acc, tok, _ = ops.verify_drafts(logits, drafts, u, noise, draft_probs=q.expand(B, 1, V).contiguous())
    p = torch.softmax(row.double(), -1).cpu().numpy()
    got = np.bincount(tok[:, 0].cpu().numpy(), minlength=V) / B
    assert np.all(np.abs(got - p) <= 5 * np.sqrt(p * (1 - p) / B))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("temp", [float("inf"), 3e38, 1e20])
def test_verify_at_temperatures_without_end(temp, probs, dtype):
    """+inf and very large temperatures: every token that is not masked is as likely as any other."""
    for B, k, V in ((1, 1, 4), (6, 3, 1001), (3, 4, 9000)):
        args = _case(B + V, B, k, V, dtype, probs)
        args[0][0, :, V // 2:] = -torch.inf
        args[0][-1, 0, 1] = torch.nan
        t = torch.full((B,), temp, device="cuda")
        t[1:B - 1:2] = 0.8  # beside ordinary ones
        want = _check(args, temperature=t)
        _check(args, temperature=t, draft_lens=torch.zeros(B, dtype=torch.int32, device="cuda"))
        assert np.isfinite(want[2]).all()
