"""Arguments of the MX cache's wrappers that would make a kernel read somewhere else are refused before any launch."""
import pytest

torch = pytest.importorskip("torch")
import fp4x  # noqa: E402
from fp4x import ops  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture
def a():
    """Valid arguments of every call."""
    def i32(*shape):
        return torch.zeros(shape, dtype=torch.int32, device="cuda")

    class A:
        cache = ops.MxKvCache.empty(4, 2, 64, 16, "mxfp8")
        slots, table, lens, pages = i32(3), i32(2, 2), i32(2), i32(2)
        k = torch.zeros((3, 2, 64), device="cuda")
        q = torch.zeros((2, 1, 8, 64), device="cuda")
        logits, drafts = torch.zeros((2, 3, 50), device="cuda"), i32(2, 2)
        u, noise = torch.zeros((2, 2), device="cuda"), torch.ones((2, 50), device="cuda")

    for t in (A.cache.k, A.cache.v, A.cache.k_scales, A.cache.v_scales):
        t.zero_()
    return A


def _calls(a, **kw):
    def x(name):
        return kw.get(name, getattr(a, name, None))

    return {
        "append": lambda: ops.kv_append_mx(a.cache, x("slots"), x("k"), x("v") if "v" in kw else x("k")),
        "read": lambda: ops.kv_read_mx(a.cache, x("slots")),
        "paged": lambda: ops.attn_paged_mx(a.cache, x("q"), x("table"), x("lens"), workspace=x("ws")),
        "shared": lambda: ops.attn_shared_mx(a.cache, x("q"), x("pages"), 20, x("table"), x("lens"), workspace=x("ws")),
        "verify": lambda: ops.verify_drafts(x("logits"), x("drafts"), x("u"), x("noise"), draft_probs=x("probs"),
                                            draft_lens=x("dl"), temperature=x("temp"), workspace=x("ws")),
    }


@pytest.mark.parametrize("call,names", [("append", ["slots", "k", "v"]), ("read", ["slots"]),
                                        ("paged", ["q", "table", "lens", "ws"]),
                                        ("shared", ["q", "pages", "table", "lens", "ws"]),
                                        ("verify", ["logits", "drafts", "u", "noise", "probs", "dl", "temp", "ws"])])
def test_tensors_of_the_host_are_refused(a, call, names):
    _calls(a)[call]()
    host = dict(slots=a.slots.cpu(), k=a.k.cpu(), v=a.k.cpu(), q=a.q.cpu(), table=a.table.cpu(), lens=a.lens.cpu(),
                pages=a.pages.cpu(), ws=torch.zeros(1 << 22, dtype=torch.uint8), logits=a.logits.cpu(), drafts=a.drafts.cpu(),
                u=a.u.cpu(), noise=a.noise.cpu(), probs=torch.zeros(2, 2, 50), dl=torch.zeros(2, dtype=torch.int32),
                temp=torch.ones(2))
    for name in names:
        with pytest.raises(ValueError):
            _calls(a, **{name: host[name]})[call]()
    with pytest.raises(ValueError):
        _calls(a, **{name: host[name] for name in names})[call]()
    torch.cuda.synchronize()


def test_slots_have_one_dimension(a):
    two = torch.zeros((3, 5), dtype=torch.int32, device="cuda")
    for call in ("append", "read"):
        with pytest.raises(ValueError):
            _calls(a, slots=two)[call]()


@pytest.mark.parametrize("call", ["paged", "shared", "verify"])
def test_workspaces(a, call):
    """Of any type: its bytes count; too small, strided or misaligned ones are refused."""
    need = {"paged": ops.attn_mx_workspace(a.cache, 2, 8, 1, 0, 32).numel(),
            "shared": ops.attn_mx_workspace(a.cache, 2, 8, 1, 20, 32).numel(),
            "verify": fp4x.lib().llama_verify_workspace_size(2, 2, 50)}[call]
    _calls(a, ws=torch.zeros(-(-need // 4), dtype=torch.float32, device="cuda"))[call]()
    flat = torch.zeros(2 * need + 32, dtype=torch.uint8, device="cuda")
    for ws in (flat[: need // 2], flat[8:need + 24]):
        with pytest.raises(fp4x.Fp4xError):
            _calls(a, ws=ws)[call]()
    with pytest.raises(ValueError):
        _calls(a, ws=flat[::2])[call]()


def test_caches_without_pages_are_refused():
    with pytest.raises(ValueError):
        ops.MxKvCache.empty(0, 2, 64, 16, "mxfp8")
    with pytest.raises(ValueError):
        ops.MxKvCache(*[torch.zeros((4, 16, 64), dtype=torch.uint8, device="cuda")] * 4)


def test_stream_of_a_call(monkeypatch):
    """The handle that the wrappers pass is the current stream's, with torch's private call and without it."""
    side = torch.cuda.Stream()
    for raw in (ops._raw_stream, None):
        monkeypatch.setattr(ops, "_raw_stream", raw)
        assert ops._stream() == torch.cuda.current_stream().cuda_stream
        with torch.cuda.stream(side):
            assert ops._stream() == side.cuda_stream
