"""torch-facing wrappers over the C ABI: each call hands device pointers of CUDA
tensors and the current torch stream to libfp4x.so.  Tensors must be CUDA and
contiguous; nothing here computes on the host."""
from __future__ import annotations

import ctypes

import torch

from . import MxKv, check, lib


# The current device, and its stream's handle without building a torch.cuda.Stream (3 us per call): by torch's own cheap
# calls where it has them.
_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream():
    return torch.cuda.current_stream().cuda_stream if _raw_stream is None else _raw_stream(_device())


def _ptr(t: torch.Tensor):
    if not t.is_cuda:
        raise ValueError("fp4x operators take CUDA tensors (no CPU fallback)")
    if not t.is_contiguous():
        raise ValueError("fp4x operators take contiguous tensors")
    return t.data_ptr()


def quantize_mxfp4(w: torch.Tensor):
    n, k = w.shape
    packed = torch.empty((n, k // 2), dtype=torch.uint8, device=w.device)
    scales = torch.empty((n, k // 32), dtype=torch.uint8, device=w.device)
    check(lib().fp4_quantize_mxfp4(_stream(), n, k, _ptr(w), _ptr(packed), _ptr(scales)))
    return packed, scales


def quantize_nvfp4(w: torch.Tensor, global_scale: float = 1.0):
    """f32 [n][k] -> NVFP4 (packed [n][k/2], UE4M3 scales [n][k/16])."""
    n, k = w.shape
    packed = torch.empty((n, k // 2), dtype=torch.uint8, device=w.device)
    scales = torch.empty((n, k // 16), dtype=torch.uint8, device=w.device)
    check(lib().fp4_quantize_nvfp4(_stream(), n, k, _ptr(w), _ptr(packed), _ptr(scales), global_scale))
    return packed, scales


def quantize_ref(w: torch.Tensor):
    n, k = w.shape
    packed = torch.empty((n, k // 8), dtype=torch.int32, device=w.device)
    scales = torch.empty((n, k // 32), dtype=torch.float32, device=w.device)
    check(lib().fp4_quantize_ref(_stream(), n, k, _ptr(w), _ptr(packed), _ptr(scales)))
    return packed, scales


def dequantize_mxfp4(packed: torch.Tensor, scales: torch.Tensor):
    n = packed.shape[0]
    k = packed.shape[1] * 2
    out = torch.empty((n, k), dtype=torch.float32, device=packed.device)
    check(lib().fp4_dequantize_mxfp4(_stream(), n, k, _ptr(packed), _ptr(scales), _ptr(out)))
    return out


def fill_normal(n: int, seed: int, sigma: float = 1.0, offset: int = 0, dtype=torch.float32, device="cuda"):
    out = torch.empty(n, dtype=dtype, device=device)
    if dtype == torch.float32:
        check(lib().fp4x_fill_normal_f32(_stream(), seed, offset, sigma, _ptr(out), n))
    elif dtype == torch.bfloat16:
        check(lib().fp4x_fill_normal_bf16(_stream(), seed, offset, sigma, _ptr(out), n))
    else:
        raise ValueError(dtype)
    return out


def init_mxfp4(n: int, k: int, seed: int, sigma: float = 0.02, device="cuda"):
    packed = torch.empty((n, k // 2), dtype=torch.uint8, device=device)
    scales = torch.empty((n, k // 32), dtype=torch.uint8, device=device)
    check(lib().fp4x_init_mxfp4(_stream(), seed, sigma, n, k, _ptr(packed), _ptr(scales)))
    return packed, scales


def gemv(packed: torch.Tensor, scales: torch.Tensor, x: torch.Tensor, out: torch.Tensor | None = None):
    """y = W x on native MXFP4 storage; x bf16 (fp4_gemv) or f32 (fp4_gemv_f32x)."""
    n = packed.shape[0]
    k = packed.shape[1] * 2
    y = out if out is not None else torch.empty(n, dtype=torch.float32, device=packed.device)
    if x.dtype == torch.bfloat16:
        check(lib().fp4_gemv(_stream(), n, k, _ptr(packed), _ptr(scales), _ptr(x), _ptr(y)))
    elif x.dtype == torch.float32:
        check(lib().fp4_gemv_f32x(_stream(), n, k, _ptr(packed), _ptr(scales), _ptr(x), _ptr(y)))
    else:
        raise ValueError(x.dtype)
    return y


def gemv_ref(words: torch.Tensor, scales: torch.Tensor, x: torch.Tensor):
    """The reference's storage: u32 words (as int32), f32 scales, f32 x."""
    n = words.shape[0]
    k = x.shape[0]
    y = torch.empty(n, dtype=torch.float32, device=words.device)
    check(lib().fp4_gemv_ref(_stream(), n, k, _ptr(words), _ptr(scales), _ptr(x), _ptr(y)))
    return y


def mma(a: torch.Tensor, sa: torch.Tensor, w: torch.Tensor, sw: torch.Tensor, out_dtype=torch.bfloat16):
    """d[m][n] = A W^T for MXFP4 A [m][k/2] (+ E8M0 scales [m][k/32]) and W [n][k/2]
    (+ [n][k/32]) on tcgen05.mma.kind::mxf4; bf16 (fp4_mma) or fp32 (fp4_mma_f32) out."""
    m, n, k = a.shape[0], w.shape[0], a.shape[1] * 2
    if w.shape[1] * 2 != k or sa.shape != (m, k // 32) or sw.shape != (n, k // 32):
        raise ValueError("fp4 mma: operand shapes disagree")
    d = torch.empty((m, n), dtype=out_dtype, device=a.device)
    if out_dtype == torch.float32:
        check(lib().fp4_mma_f32(_stream(), m, n, k, _ptr(a), _ptr(sa), _ptr(w), _ptr(sw), _ptr(d)))
        return d
    if out_dtype != torch.bfloat16:
        raise ValueError(out_dtype)
    ws_bytes = lib().fp4_mma_workspace_size(m, n, k)
    ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=a.device)
    check(lib().fp4_mma(_stream(), m, n, k, _ptr(a), _ptr(sa), _ptr(w), _ptr(sw), _ptr(d), _ptr(ws), ws_bytes))
    return d


def mma_nvf4(a, sa, w, sw, alpha: float = 1.0, out_dtype=torch.bfloat16):
    """NVFP4 GEMM: d[m][n] = alpha * A W^T, UE4M3 scales per 16 values."""
    m, n, k = a.shape[0], w.shape[0], a.shape[1] * 2
    if w.shape[1] * 2 != k or sa.shape != (m, k // 16) or sw.shape != (n, k // 16):
        raise ValueError("nvf4 mma: operand shapes disagree")
    d = torch.empty((m, n), dtype=out_dtype, device=a.device)
    if out_dtype == torch.float32:
        check(lib().fp4_mma_nvf4_f32(_stream(), m, n, k, _ptr(a), _ptr(sa), _ptr(w), _ptr(sw), alpha, _ptr(d)))
        return d
    ws_bytes = lib().fp4_mma_nvf4_workspace_size(m, n, k)
    ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=a.device)
    check(lib().fp4_mma_nvf4(_stream(), m, n, k, _ptr(a), _ptr(sa), _ptr(w), _ptr(sw), alpha, _ptr(d), _ptr(ws),
                             ws_bytes))
    return d


def mma_allones(device="cuda"):
    """The reference's all-ones known-answer test on tcgen05: [16][8], every value 64.0."""
    out = torch.full((16, 8), -1.0, dtype=torch.float32, device=device)
    check(lib().fp4_mma_allones(_stream(), _ptr(out)))
    return out


def rmsnorm(x, w, eps=1e-5):
    y = torch.empty_like(x)
    check(lib().llama_rmsnorm(_stream(), x.numel(), eps, _ptr(x), _ptr(w), _ptr(y)))
    return y


def rope_tables(n_pos: int, head_dim: int, theta: float, device="cuda"):
    c = torch.empty((n_pos, head_dim // 2), dtype=torch.float32, device=device)
    s = torch.empty_like(c)
    check(lib().llama_rope_tables(_stream(), n_pos, head_dim, float(theta), _ptr(c), _ptr(s)))
    return c, s


def rope_(q, num_heads, head_dim, cos_base, cos_t, sin_t):
    check(lib().llama_rope(_stream(), num_heads, head_dim, cos_base, _ptr(cos_t), _ptr(sin_t), _ptr(q)))
    return q


def copy_into_(dst, src, off):
    check(lib().llama_copy_into(_stream(), src.numel(), off, _ptr(src), _ptr(dst)))
    return dst


def kv_append_bf16_(dst, src, off):
    check(lib().llama_kv_append_bf16(_stream(), src.numel(), off, _ptr(src), _ptr(dst)))
    return dst


def swiglu(g, u):
    out = torch.empty_like(g)
    check(lib().llama_swiglu(_stream(), g.numel(), _ptr(g), _ptr(u), _ptr(out)))
    return out


def residual_(x, y):
    check(lib().llama_residual(_stream(), x.numel(), _ptr(y), _ptr(x)))
    return x


def argmax(logits):
    out = torch.empty(1, dtype=torch.int32, device=logits.device)
    check(lib().llama_argmax(_stream(), logits.numel(), _ptr(logits), _ptr(out)))
    return out


def attn_decode(q, kc, vc, n_heads, n_kv, seq):
    """Reference signature: f32, head_dim 64, cache [seq][n_kv][64]."""
    out = torch.empty(n_heads * 64, dtype=torch.float32, device=q.device)
    check(lib().llama_attn_decode(_stream(), n_heads, n_kv, seq, _ptr(q), _ptr(kc), _ptr(vc), _ptr(out)))
    return out


def attn_workspace(batch, n_heads, n_kv, head_dim, seq, device="cuda"):
    nbytes = lib().llama_attn_workspace_size(batch, n_heads, n_kv, head_dim, seq)
    return torch.empty(max(nbytes, 16), dtype=torch.uint8, device=device), nbytes


def attn_decode_hd(q, kc, vc, n_heads, n_kv, head_dim, seq, split=True):
    out = torch.empty(n_heads * head_dim, dtype=torch.float32, device=q.device)
    ws, nbytes = attn_workspace(1, n_heads, n_kv, head_dim, seq, q.device) if split else (None, 0)
    check(lib().llama_attn_decode_hd(_stream(), n_heads, n_kv, head_dim, seq, _ptr(q), _ptr(kc), _ptr(vc),
                                     _ptr(out), _ptr(ws) if ws is not None else None, nbytes))
    return out


def attn_decode_bf16(q, kc, vc, seq, split=True):
    """q [B][H][hd] bf16; kc/vc [B][max_seq][n_kv][hd] bf16 -> out [B][H][hd] bf16."""
    B, H, hd = q.shape
    max_seq, n_kv = kc.shape[1], kc.shape[2]
    out = torch.empty_like(q)
    ws, nbytes = attn_workspace(B, H, n_kv, hd, seq, q.device) if split else (None, 0)
    check(lib().llama_attn_decode_bf16(_stream(), B, H, n_kv, hd, seq, max_seq, _ptr(q), _ptr(kc), _ptr(vc),
                                       _ptr(out), _ptr(ws) if ws is not None else None, nbytes))
    return out


# ------------------------------------------------------------ MX KV cache
_DTYPES = {torch.float32: 0, torch.bfloat16: 1}


def _dtype(t: torch.Tensor) -> int:
    d = _DTYPES.get(t.dtype)
    if d is None:
        raise ValueError(f"fp4x: {t.dtype} is not float32 or bfloat16")
    return d


def _flat(t: torch.Tensor):
    if not t.is_contiguous():
        raise ValueError("fp4x operators take contiguous tensors")
    return t.data_ptr()


# of tensors that _together has seen
def _i32(t: torch.Tensor, name: str):
    if t.dtype != torch.int32:
        raise ValueError(f"{name} must be int32, not {t.dtype}")
    return _flat(t)


def _f32(t: torch.Tensor, name: str):
    if t.dtype != torch.float32:
        raise ValueError(f"{name} must be float32, not {t.dtype}")
    return _flat(t)


def _together(*tensors):
    """All tensors of a call (None: not given) lie on the current CUDA device."""
    dev = _device()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"fp4x operators take CUDA tensors of the current device (cuda:{dev}), not {t.device}")


def _work(ws: torch.Tensor):
    """Pointer and bytes of a workspace of any type."""
    return _flat(ws), ws.numel() * ws.element_size()


def _rows(t: torch.Tensor, n: int):
    """Pointer and row stride of [rows][n] data whose leading dimension may be strided."""
    return t.data_ptr(), (t.stride(0) if t.shape[0] > 1 else n)


class MxKvCache:
    """Paged KV cache in MXFP8 (E4M3) or MXFP4 (E2M1) with one E8M0 scale per 32 values.

    k, v: uint8 [n_pages][n_kv][page_size][head_dim or head_dim/2], k_scales, v_scales: uint8
    [n_pages][n_kv][page_size][head_dim/32]; the page dimension may be strided (alike for K and V), as in one
    allocation that holds K and V pages in turn.  Row layout: see fp4x_mxkv in fp4x.h.
    """

    def __init__(self, k, k_scales, v, v_scales):
        if k.dim() != 4 or k.shape[0] == 0:
            raise ValueError("an MX cache is [n_pages][n_kv][page_size][row], with a page at least")
        n_pages, n_kv, page, row = k.shape
        head_dim = 32 * k_scales.shape[-1]
        if row not in (head_dim, head_dim // 2):
            raise ValueError(f"row of {row} bytes does not hold head_dim {head_dim}")
        if v.shape != k.shape or k_scales.shape != (n_pages, n_kv, page, head_dim // 32) \
                or v_scales.shape != k_scales.shape:
            raise ValueError("K, V and their scales disagree in shape")
        for t in (k, k_scales, v, v_scales):
            if t.dtype != torch.uint8 or not t.is_cuda or t.device != k.device:
                raise ValueError("an MX cache is uint8 CUDA tensors of one device")
            if not t[0].is_contiguous():
                raise ValueError("every page must be contiguous")
        if n_pages > 1 and (k.stride(0) != v.stride(0) or k_scales.stride(0) != v_scales.stride(0)):
            raise ValueError("K and V must have the same page stride")
        self.k, self.k_scales, self.v, self.v_scales = k, k_scales, v, v_scales
        self.n_pages, self.n_kv, self.page_size, self.head_dim = n_pages, n_kv, page, head_dim
        self.format = "mxfp8" if row == head_dim else "mxfp4"
        strides = (k.stride(0), k_scales.stride(0)) if n_pages > 1 else (k[0].numel(), k_scales[0].numel())
        self._struct = MxKv(k.data_ptr(), k_scales.data_ptr(), v.data_ptr(), v_scales.data_ptr(), *strides, n_pages,
                            page, n_kv, head_dim, 0 if row == head_dim else 1)
        self.ptr = ctypes.addressof(self._struct)

    @classmethod
    def empty(cls, n_pages, n_kv, head_dim, page_size=64, fmt="mxfp8", device="cuda"):
        """A cache of `n_pages` pages; nothing is read from a row before it is written."""
        if fmt not in ("mxfp8", "mxfp4"):
            raise ValueError(fmt)
        row = head_dim if fmt == "mxfp8" else head_dim // 2
        shape = (n_pages, n_kv, page_size)
        new = [torch.empty(shape + (n,), dtype=torch.uint8, device=device) for n in (row, head_dim // 32) * 2]
        return cls(*new)


def kv_append_mx(cache: MxKvCache, slots, k, v):
    """Quantise rows k, v [n][n_kv][head_dim] (f32 or bf16, rows may be strided) into the cache's slots [n] int32."""
    _together(cache.k, slots, k, v)
    if slots.dim() != 1:
        raise ValueError("slots must be [n]")
    n = slots.shape[0]
    shape = (n, cache.n_kv, cache.head_dim)
    if k.shape != shape or v.shape != shape or k.dtype != v.dtype:
        raise ValueError(f"k and v must be {shape} of one type")
    hd = cache.head_dim
    for t in (k, v):
        if t.stride(2) != 1 or (t.stride(1) != hd and cache.n_kv > 1):
            raise ValueError("k and v rows must be contiguous")
    row = cache.n_kv * hd
    (kp, ks), (vp, vs) = _rows(k, row), _rows(v, row)
    check(lib().llama_kv_append_mx(_stream(), cache.ptr, n, _i32(slots, "slots"), _dtype(k), kp, ks, vp, vs))


def kv_read_mx(cache: MxKvCache, slots, dtype=torch.bfloat16):
    """The cached rows in slots [n] int32 as K, V [n][n_kv][head_dim] of `dtype`; zeros for negative slots."""
    _together(cache.k, slots)
    if slots.dim() != 1:
        raise ValueError("slots must be [n]")
    n = slots.shape[0]
    k, v = cache.k.new_empty((2, n, cache.n_kv, cache.head_dim), dtype=dtype).unbind(0)
    check(lib().llama_kv_read_mx(_stream(), cache.ptr, n, _i32(slots, "slots"), _dtype(k), k.data_ptr(), v.data_ptr()))
    return k, v


def attn_mx_workspace(cache: MxKvCache, batch, n_heads, q_len, prefix_len, max_len):
    """Workspace of attn_paged_mx (prefix_len 0) and attn_shared_mx for this shape."""
    nbytes = lib().llama_attn_mx_workspace_size(cache.ptr, batch, n_heads, q_len, prefix_len, max_len)
    return cache.k.new_empty(max(nbytes, 16))


def _attn_args(cache, q, page_table, lens, max_len, *others):
    _together(cache.k, q, page_table, lens, *others)
    if q.dim() != 4 or q.shape[3] != cache.head_dim:
        raise ValueError(f"q must be [batch][q_len][n_heads][{cache.head_dim}]")
    B, T, H, hd = q.shape
    sb, st, sh, sd = q.stride()
    row = st if T > 1 else sb if B > 1 else H * hd
    if sd != 1 or (sh != hd and H > 1) or (B > 1 and sb != T * row):
        raise ValueError("q token rows must be contiguous and evenly spaced")
    if page_table.dim() != 2 or page_table.shape[0] != B or lens.shape != (B,):
        raise ValueError("page_table must be [batch][pages] and lens [batch]")
    if max_len is None:
        max_len = page_table.shape[1] * cache.page_size
    return B, T, H, row, max_len


def attn_paged_mx(cache: MxKvCache, q, page_table, lens, max_len=None, workspace=None):
    """Attention of q [batch][q_len][n_heads][hd] over each sequence's own pages; lens [batch] int32 counts the cached
    positions with the q_len new ones as the last.  Returns a tensor shaped like q."""
    B, T, H, row, max_len = _attn_args(cache, q, page_table, lens, max_len, workspace)
    ws = workspace if workspace is not None else attn_mx_workspace(cache, B, H, T, 0, max_len)
    out = q.new_empty(q.shape)
    check(lib().llama_attn_paged_mx(_stream(), cache.ptr, B, H, T, _i32(page_table, "page_table"), page_table.shape[1],
                                    _i32(lens, "lens"), max_len, _dtype(q), q.data_ptr(), row, out.data_ptr(),
                                    *_work(ws)))
    return out


def attn_shared_mx(cache: MxKvCache, q, prefix_pages, prefix_len, page_table, lens, max_len=None, workspace=None):
    """attn_paged_mx for sequences that continue one prefix of prefix_len positions behind prefix_pages int32."""
    B, T, H, row, max_len = _attn_args(cache, q, page_table, lens, max_len, prefix_pages, workspace)
    if prefix_pages.numel() * cache.page_size < prefix_len:
        raise ValueError("prefix_pages hold fewer than prefix_len positions")
    ws = workspace if workspace is not None else attn_mx_workspace(cache, B, H, T, prefix_len, max_len)
    out = q.new_empty(q.shape)
    check(lib().llama_attn_shared_mx(_stream(), cache.ptr, B, H, T, _i32(prefix_pages, "prefix_pages"), prefix_len,
                                     _i32(page_table, "page_table"), page_table.shape[1], _i32(lens, "lens"), max_len,
                                     _dtype(q), q.data_ptr(), row, out.data_ptr(), *_work(ws)))
    return out


def verify_drafts(logits, drafts, uniforms, noise, draft_probs=None, draft_lens=None, temperature=None,
                  workspace=None):
    """Speculative verification: logits [batch][k+1][vocab] (f32 or bf16) of the target, drafts [batch][k] int32,
    uniforms [batch][k], noise [batch][vocab] exponential draws, draft_probs [batch][k][vocab] (None: certain drafts),
    draft_lens [batch] int32, temperature [batch].  Returns (accepted [batch] int32, tokens [batch][k+1] int32,
    logprobs [batch][k+1])."""
    _together(logits, drafts, uniforms, noise, draft_probs, draft_lens, temperature, workspace)
    B, K1, V = logits.shape
    k = K1 - 1
    if drafts.shape != (B, k) or uniforms.shape != (B, k) or noise.shape != (B, V):
        raise ValueError("verify_drafts: drafts, uniforms and noise disagree with the logits' shape")
    if draft_probs is not None and draft_probs.shape != (B, k, V):
        raise ValueError("verify_drafts: draft_probs must be [batch][k][vocab]")
    if (draft_lens is not None and draft_lens.shape != (B,)) or (temperature is not None and temperature.shape != (B,)):
        raise ValueError("verify_drafts: draft_lens and temperature must be [batch]")
    stride = logits.stride(1) if K1 > 1 else logits.stride(0) if B > 1 else V
    if logits.stride(2) != 1 or (B > 1 and logits.stride(0) != K1 * stride):
        raise ValueError("verify_drafts: logits must be CUDA rows, evenly spaced")
    accepted, tokens = drafts.new_empty(B), drafts.new_empty((B, K1))
    logprobs = uniforms.new_empty((B, K1))
    if workspace is None:
        workspace = drafts.new_empty(max(lib().llama_verify_workspace_size(B, k, V), 16), dtype=torch.uint8)
    check(lib().llama_verify_drafts(
        _stream(), B, k, V, _dtype(logits), logits.data_ptr(), stride,
        None if draft_probs is None else _f32(draft_probs, "draft_probs"), _i32(drafts, "drafts"),
        None if draft_lens is None else _i32(draft_lens, "draft_lens"), _f32(uniforms, "uniforms"),
        _f32(noise, "noise"), None if temperature is None else _f32(temperature, "temperature"), accepted.data_ptr(),
        tokens.data_ptr(), logprobs.data_ptr(), *_work(workspace)))
    return accepted, tokens, logprobs
