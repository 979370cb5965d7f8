"""The serving example's scheduling (pages, positions, rows of a pass) on the CPU: the model and the operators are stand-ins
whose indexing is checked by torch."""
import sys
import types
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")
sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "rust-fp4-blackwell_b200" / "examples"))
import serve_mxkv  # noqa: E402


class Cache:
    def __init__(self, n_pages, page):
        self.rows = torch.zeros(n_pages * page, dtype=torch.bool)

    @classmethod
    def empty(cls, n_pages, n_kv, hd, page, fmt, device):
        return cls(n_pages, page)


class Model:
    kv_heads, hd, vocab, layers, device = 1, 64, 16, [None], torch.device("cpu")

    def __init__(self, max_pos=4096):
        self.max_pos, self.cos = max_pos, torch.zeros(max_pos)

    def forward(self, tokens, pos, slots, attend):
        assert tokens.shape == pos.shape == slots.shape and int(tokens.min()) >= 0 and int(tokens.max()) < self.vocab
        self.cos[pos]  # raises past the table
        for s in slots:
            assert len(set(s.tolist())) == len(s)
            self.caches[0].rows[s.long()] = True
        attend(0, None)
        return torch.nn.functional.one_hot((tokens.long() + 1) % 8, self.vocab)  # the texts count to 8, over and over


def _run(monkeypatch, accepts, requests, n_tokens, draft, page, prompt=20, max_pos=4096):
    """accepts(b): whether request b's drafts are all accepted (else none of them)."""
    seen = []

    def shared(cache, q, prefix_pages, prefix, table, lens):
        assert int(lens.max()) <= table.shape[1] * page
        seen.append(lens.tolist())
        for b, n in enumerate(lens.tolist()):
            slots = (table[b][:, None] * page + torch.arange(page)).flatten()[:n].long()
            assert bool(cache.rows[slots].all())  # every position that is attended to has been written

    def verify(logits, drafts, uniforms, noise, draft_lens=None, temperature=None):
        n = torch.tensor([int(draft_lens[b]) if accepts(b) else 0 for b in range(len(draft_lens))])
        tokens = torch.full((len(n), drafts.shape[1] + 1), -1)
        for b, k in enumerate(n.tolist()):
            tokens[b, :k], tokens[b, k] = drafts[b, :k], logits[b, k].argmax()
        return n.int(), tokens, None

    monkeypatch.setattr(serve_mxkv, "ops", types.SimpleNamespace(
        MxKvCache=Cache, attn_paged_mx=lambda *a: None, attn_shared_mx=shared, verify_drafts=verify))
    out, passes = serve_mxkv.serve(Model(max_pos), [i % 8 for i in range(prompt)], requests, n_tokens, draft, page=page)
    assert passes == len(seen)
    for o, r in zip(out, requests):
        assert o == [(r[-1] + 1 + i) % 8 for i in range(n_tokens)]
    return out


@pytest.mark.parametrize("draft", [0, 1, 3, 6])
@pytest.mark.parametrize("n_tokens", range(1, 18))
def test_pages_hold_what_a_pass_writes(monkeypatch, n_tokens, draft):
    """One request takes all of its drafts and is done early, the others go on; every alignment with the pages' ends."""
    for page in (1, 2, 16):
        _run(monkeypatch, lambda b: b == 0, [[4, 5, 6], [4], [4, 5]], n_tokens, draft, page)
        _run(monkeypatch, lambda b: True, [[4], [4, 5]], n_tokens, draft, page)


def test_what_does_not_fit_is_refused(monkeypatch):
    _run(monkeypatch, lambda b: b == 0, [[4, 5], [4]], 10, 3, 16, prompt=20, max_pos=38)
    with pytest.raises(ValueError):
        _run(monkeypatch, lambda b: True, [[4, 5], [4]], 10, 3, 16, prompt=20, max_pos=37)
    with pytest.raises(ValueError):
        _run(monkeypatch, lambda b: True, [[4], []], 4, 1, 16)
