"""Operators of batched serving: a paged KV cache and its attention, attention
of packed prompts, and the draw of the next token.

The reference decodes one sequence at a time (``CompressedKVCache``,
polarflash_rt/kv_cache/compressed_kv.py:22-282; ``PFlashAttentionBlock``,
polarflash_core/model_integration.py:63-147) and leaves the choice of the
token to its caller; these are the same steps for several sequences of
different lengths.  Every call launches on torch's current stream of its
tensors' device, allocates nothing but its outputs (and the attention's
workspace, unless it is given), and can be captured in a CUDA graph.  They
compute no gradients.  There is no CPU path.
"""
import ctypes
import functools
from typing import Optional, Union

import torch

from . import _lib
from .kv_cache import KV_MODES

PAGE_MODES = dict(KV_MODES, fp16=8, bf16=9)
PAGE_SIZES = (16, 32, 64, 128, 256)
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_ROW_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "int8": torch.int8, "2bit": torch.uint8,
               "2bit_asym": torch.uint8}


try:  # the stream's handle without building a Stream object: a call's host time is a few microseconds
    from torch._C import _cuda_getCurrentRawStream as _raw_stream
except ImportError:  # pragma: no cover
    def _raw_stream(index: int) -> int:
        return torch.cuda.current_stream(index).cuda_stream


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _call(fn, what: str, index: int, *args) -> None:
    """fn(*args, stream) with device `index` current, on torch's current stream there."""
    if torch.cuda.current_device() == index:
        st = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            st = fn(*args, _raw_stream(index))
    if st:
        _lib.check(st, what)


def _need(t: torch.Tensor, name: str, index: int, dtype, shape=None) -> None:
    """A contiguous tensor of `dtype` (and shape) on CUDA device `index`."""
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == index and t.is_contiguous() and \
            (shape is None or t.shape == shape):
        return
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.get_device() != index:
        raise ValueError(f"{name}: a tensor on cuda:{index} is needed (no CPU path)")
    if t.dtype is not dtype:
        raise ValueError(f"{name}: {dtype} is needed, not {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} has to be contiguous")
    raise ValueError(f"{name}: shape {tuple(shape)} is needed, not {tuple(t.shape)}")


def _rows(t: torch.Tensor, name: str, index: int, dtypes):
    """(rows, heads, dim, elements between rows) of t [rows, heads, dim] whose rows are contiguous."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.get_device() != index:
        raise ValueError(f"{name}: a tensor on cuda:{index} is needed (no CPU path)")
    if t.dtype not in dtypes:
        raise ValueError(f"{name}: one of {', '.join(str(d) for d in dtypes)} is needed, not {t.dtype}")
    shape = t.shape
    if len(shape) != 3:
        raise ValueError(f"{name}: [rows, heads, head_dim] is needed, not {tuple(shape)}")
    n, h, d = shape
    if t.is_contiguous():
        return n, h, d, h * d
    s = t.stride()
    if (h > 1 and s[1] != d) or (d > 1 and s[2] != 1):
        raise ValueError(f"{name}: a row's heads have to be contiguous")
    return n, h, d, s[0] if n > 1 else h * d


class KVPages:
    """One layer's pages: rows k, v [num_pages, kv_heads, page_size, row] (fp16
    / bf16 values, int8 codes, or uint8 bytes of four 2-bit codes) and, for the
    quantized modes, fp32 scales (and zeros, "2bit_asym") [num_pages, kv_heads,
    page_size]: the formulas of CompressedKVCache
    (polarflash_rt/kv_cache/compressed_kv.py:68-150) as torch evaluates them on
    a CUDA device, where dividing by a number is multiplying by its reciprocal.
    kv_cache.kv_quantize divides, as on a CPU: its scales differ by at most
    3 * 2^-24 of themselves, its codes by one where a value lies on the border
    of two."""

    __slots__ = ("mode", "k", "v", "k_scales", "v_scales", "k_zeros", "v_zeros", "num_pages", "kv_heads", "page_size",
                 "head_dim", "index", "desc")

    def __init__(self, mode: str, k: torch.Tensor, v: torch.Tensor, k_scales: Optional[torch.Tensor] = None,
                 v_scales: Optional[torch.Tensor] = None, k_zeros: Optional[torch.Tensor] = None,
                 v_zeros: Optional[torch.Tensor] = None):
        row_dtype = _ROW_DTYPES.get(mode)
        if row_dtype is None:
            raise ValueError(f"KVPages mode {mode!r}: one of {', '.join(PAGE_MODES)}")
        if not isinstance(k, torch.Tensor) or not k.is_cuda:
            raise ValueError("KVPages: k is a CUDA tensor (no CPU path)")
        if k.dim() != 4:
            raise ValueError(f"KVPages: k [num_pages, kv_heads, page_size, row] is needed, not {tuple(k.shape)}")
        shape = k.shape
        P, H, S, R = shape
        hd = R * 4 if row_dtype is torch.uint8 else R
        if P < 1 or H < 1 or S not in PAGE_SIZES or hd not in (64, 128):
            raise ValueError(f"KVPages: {P} pages of {S} slots, {H} heads of {hd}: at least one page and head, "
                             f"page_size one of {PAGE_SIZES} and head_dim 64 or 128 are needed")
        index = k.get_device()
        _need(k, "k", index, row_dtype)
        _need(v, "v", index, row_dtype, shape)
        pks = pvs = pkz = pvz = None
        if mode in KV_MODES:
            shape = shape[:3]
            _need(k_scales, "k_scales", index, torch.float32, shape)
            _need(v_scales, "v_scales", index, torch.float32, shape)
            pks, pvs = k_scales.data_ptr(), v_scales.data_ptr()
        else:
            k_scales = v_scales = None
        if mode == "2bit_asym":
            _need(k_zeros, "k_zeros", index, torch.float32, shape)
            _need(v_zeros, "v_zeros", index, torch.float32, shape)
            pkz, pvz = k_zeros.data_ptr(), v_zeros.data_ptr()
        else:
            k_zeros = v_zeros = None
        self.mode, self.k, self.v = mode, k, v
        self.k_scales, self.v_scales, self.k_zeros, self.v_zeros = k_scales, v_scales, k_zeros, v_zeros
        self.num_pages, self.kv_heads, self.page_size, self.head_dim, self.index = P, H, S, hd, index
        self.desc = _lib.PFKVPages(PAGE_MODES[mode], P, S, H, hd, 0, k.data_ptr(), v.data_ptr(), pks, pvs, pkz, pvz)

    @property
    def device(self) -> torch.device:
        return self.k.device

    @classmethod
    def empty(cls, mode: str, num_pages: int, page_size: int, kv_heads: int, head_dim: int, device) -> "KVPages":
        """Zero-filled pages."""
        if mode not in PAGE_MODES:
            raise ValueError(f"KVPages mode {mode!r}: one of {', '.join(PAGE_MODES)}")
        row = head_dim // 4 if mode.startswith("2bit") else head_dim
        shape = (num_pages, kv_heads, page_size)
        z = lambda s, dt: torch.zeros(s, dtype=dt, device=device)  # noqa: E731
        sc = [z(shape, torch.float32) for _ in range(2)] if mode in KV_MODES else [None, None]
        ze = [z(shape, torch.float32) for _ in range(2)] if mode == "2bit_asym" else [None, None]
        return cls(mode, z(shape + (row,), _ROW_DTYPES[mode]), z(shape + (row,), _ROW_DTYPES[mode]), *sc, *ze)

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scales, self.v_scales, self.k_zeros,
                                                          self.v_zeros) if t is not None)


def _table(block_table: torch.Tensor, seq_lens: torch.Tensor, index: int):
    if not isinstance(block_table, torch.Tensor) or block_table.dim() != 2:
        raise ValueError("block_table: [sequences, pages] is needed")
    B, W = block_table.shape
    if W < 1:
        raise ValueError("block_table: at least one page per sequence is needed")
    _need(block_table, "block_table", index, torch.int32)
    _need(seq_lens, "seq_lens", index, torch.int32, (B,))
    return B, W


def paged_rope_kv(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, cos: Optional[torch.Tensor],
                  sin: Optional[torch.Tensor], pages: KVPages, block_table: torch.Tensor, seq_lens: torch.Tensor,
                  cu_seqlens: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                  q_out: Optional[torch.Tensor] = None, return_kv: bool = False):
    """Rotates new tokens' q and k and writes k and v into their pages.

    q [tokens, heads, head_dim] (None: only the cache is written), k and v
    [tokens, kv_heads, head_dim] of one dtype (fp32, fp16, bf16; rows may be
    strided), cos and sin [tokens, head_dim / 2] fp32 of each token's position
    (None: no rotation; halves rotate as apply_rotary_pos_emb does,
    polarflash_core/model_integration.py:40-60).  block_table [sequences, width]
    and seq_lens [sequences] int32, the lengths counting the new tokens in;
    cu_seqlens [sequences + 1] int32 gives each sequence's rows (None: one new
    token per sequence).  Returns (q, k, v) rotated, in `out_dtype` (k and v
    None unless `return_kv`); `q_out` takes q's place, and may be q itself.  Rows
    behind cu_seqlens[-1] are left out of the cache and of the outputs (whose rows
    there are undefined); so are, of the cache, positions outside the table and
    pages outside the cache.  No page may be written by two sequences of a call."""
    dev = pages.index
    T, nkv, hd, ks = _rows(k, "k", dev, _DTYPES)
    dtype = k.dtype
    vT, vh, vd, vs = _rows(v, "v", dev, (dtype,))
    if vT != T or vh != nkv or vd != hd or nkv != pages.kv_heads or hd != pages.head_dim:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)}: equal rows of {pages.kv_heads} heads of "
                         f"{pages.head_dim} are needed")
    if out_dtype is None:
        out_dtype = dtype
    elif out_dtype not in _DTYPES:
        raise ValueError(f"out_dtype {out_dtype}: one of {', '.join(str(d) for d in _DTYPES)}")
    nh = qs = 0
    if q is not None:
        qT, nh, qd, qs = _rows(q, "q", dev, (dtype,))
        if qT != T or qd != hd or nh < 1:
            raise ValueError(f"q {tuple(q.shape)}: [{T}, heads, {hd}] is needed")
        if q_out is None:
            q_out = torch.empty((T, nh, hd), dtype=out_dtype, device=k.device)
        else:
            _need(q_out, "q_out", dev, out_dtype, (T, nh, hd))
    elif q_out is not None:
        raise ValueError("q_out without q")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin go together")
    if cos is not None:
        _need(cos, "cos", dev, torch.float32, (T, hd // 2))
        _need(sin, "sin", dev, torch.float32, (T, hd // 2))
    B, W = _table(block_table, seq_lens, dev)
    if cu_seqlens is not None:
        _need(cu_seqlens, "cu_seqlens", dev, torch.int32, (B + 1,))
    elif T != B:
        raise ValueError(f"{T} tokens of {B} sequences: cu_seqlens is needed")
    ko = vo = None
    if return_kv:
        ko, vo = (torch.empty((T, nkv, hd), dtype=out_dtype, device=k.device) for _ in range(2))
    if T and B:
        _call(_lib.load().pf_paged_rope_kv, "pf_paged_rope_kv", dev, ctypes.byref(pages.desc), _ptr(q), qs,
              k.data_ptr(), ks, v.data_ptr(), vs, _DTYPES[dtype], _ptr(cos), _ptr(sin), T, _ptr(cu_seqlens),
              seq_lens.data_ptr(), block_table.data_ptr(), W, B, nh, _ptr(q_out), _ptr(ko), _ptr(vo),
              _DTYPES[out_dtype])
    return q_out, ko, vo


def paged_attention_workspace_bytes(n_heads: int, n_kv_heads: int, head_dim: int, seqs: int, device) -> int:
    """Bytes of paged_attention's workspace on a device."""
    device = torch.device(device)
    return _workspace_bytes(torch.cuda.current_device() if device.index is None else device.index, n_heads, n_kv_heads,
                            head_dim, seqs)


@functools.lru_cache(maxsize=None)
def _workspace_bytes(index: int, n_heads: int, n_kv_heads: int, head_dim: int, seqs: int) -> int:
    with torch.cuda.device(index):
        return int(_lib.load().pf_paged_attention_workspace_size(n_heads, n_kv_heads, head_dim, seqs))


def paged_attention(q: torch.Tensor, pages: KVPages, block_table: torch.Tensor, seq_lens: torch.Tensor,
                    scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                    workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale q k^T) v of one new token per sequence over its cached
    positions 0..seq_lens - 1 (PFlashAttentionBlock's attention,
    polarflash_core/model_integration.py:126-145, over pages).

    q [sequences, heads, head_dim] (fp32, fp16 or bf16; contiguous), heads a
    multiple of the cache's KV heads; out the same.  block_table [sequences,
    width] and seq_lens [sequences] int32.  `scale` defaults to
    1 / sqrt(head_dim).  A sequence of length 0 gives zeros; positions whose page
    is not one of the cache's are left out.  `workspace`: a uint8 tensor of
    paged_attention_workspace_bytes, used by one call at a time; by default one
    is allocated."""
    dev = pages.index
    code = _DTYPES.get(q.dtype) if isinstance(q, torch.Tensor) else None
    if code is None or q.dim() != 3:
        raise ValueError("q: [sequences, heads, head_dim] in fp32, fp16 or bf16 is needed")
    _need(q, "q", dev, q.dtype)
    B, W = _table(block_table, seq_lens, dev)
    n, nh, hd = q.shape
    if n != B or hd != pages.head_dim or nh < 1 or nh % pages.kv_heads:
        raise ValueError(f"q {tuple(q.shape)}: [{B}, a multiple of {pages.kv_heads}, {pages.head_dim}] is needed")
    if out is None:
        out = torch.empty_like(q)
    else:
        _need(out, "out", dev, q.dtype, (n, nh, hd))
    if B == 0:
        return out
    need = _workspace_bytes(dev, nh, pages.kv_heads, hd, B)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    else:
        _need(workspace, "workspace", dev, torch.uint8)
        if workspace.numel() < need:
            raise ValueError(f"workspace of {workspace.numel()} bytes < {need} needed")
    _call(_lib.load().pf_paged_attention, "pf_paged_attention", dev, ctypes.byref(pages.desc), q.data_ptr(), code,
          out.data_ptr(), block_table.data_ptr(), W, seq_lens.data_ptr(), B, nh,
          hd ** -0.5 if scale is None else float(scale), workspace.data_ptr(), need)
    return out


def check_serving_status(device) -> None:
    """Raises RuntimeError when a bounded wait of a prompt_attention kernel on
    `device` gave up since the last check (its rows are NaN then), in a replayed
    graph too.  Waits for the device's current stream."""
    device = torch.device(device)
    index = torch.cuda.current_device() if device.index is None else device.index
    st = ctypes.c_int(_lib.OK)
    _call(_lib.load().pf_prompt_status, "pf_prompt_status", index, 1, ctypes.byref(st))
    _lib.check(st.value, "pf_prompt_attention")


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor,
                     cu_seqlens_k: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of packed prompts of different lengths
    (PFlashAttentionBlock.forward for several tokens,
    polarflash_core/model_integration.py:126-145).

    q [total_q, heads, head_dim], k and v [total_k, kv_heads, head_dim] in fp16
    or bf16 (one dtype; rows may be strided, as slices of a fused projection
    are), head_dim a multiple of 8 up to 128.  Sequence b has the query rows
    cu_seqlens_q[b]..cu_seqlens_q[b + 1] - 1 and the key rows cu_seqlens_k[b]..
    cu_seqlens_k[b + 1] - 1 (int32, ascending from 0; cu_seqlens_k defaults to
    cu_seqlens_q); its last query sees its last key, so that keys before the
    queries' own (a cached prefix) are seen by all.  Rows that see no key give
    zeros; rows of `out` (none of q, k and v) behind cu_seqlens_q[-1] are left as
    they were.  `scale` (above 0) defaults to 1 / sqrt(head_dim).  Softmax weights
    are rounded to the inputs' type before they meet v.  A wait of the kernel
    that gave up shows as NaN rows and in check_serving_status."""
    if not isinstance(q, torch.Tensor) or not q.is_cuda:
        raise ValueError("prompt_attention needs CUDA tensors (no CPU path)")
    dev, dts = q.get_device(), (torch.float16, torch.bfloat16)
    T, nh, hd, qs = _rows(q, "q", dev, dts)
    dtype = q.dtype
    TK, nkv, kd, ks = _rows(k, "k", dev, (dtype,))
    vT, vh, vd, vs = _rows(v, "v", dev, (dtype,))
    if vT != TK or vh != nkv or vd != kd or kd != hd or nkv < 1 or nh < 1 or nh % nkv:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}: equal k and v, one head_dim "
                         "and a multiple of the KV heads are needed")
    if cu_seqlens_k is None:
        cu_seqlens_k = cu_seqlens_q
        if TK != T:
            raise ValueError(f"{T} queries and {TK} keys: cu_seqlens_k is needed")
    if not isinstance(cu_seqlens_q, torch.Tensor) or cu_seqlens_q.dim() != 1 or cu_seqlens_q.numel() < 1:
        raise ValueError("cu_seqlens_q: [sequences + 1] is needed")
    _need(cu_seqlens_q, "cu_seqlens_q", dev, torch.int32)
    B = cu_seqlens_q.numel() - 1
    _need(cu_seqlens_k, "cu_seqlens_k", dev, torch.int32, (B + 1,))
    if out is None:
        out = torch.empty((T, nh, hd), dtype=dtype, device=q.device)
        os = nh * hd
    else:
        oT, oh, od, os = _rows(out, "out", dev, (dtype,))
        if oT != T or oh != nh or od != hd:
            raise ValueError(f"out {tuple(out.shape)}: {tuple(q.shape)} is needed")
    if T and B:
        _call(_lib.load().pf_prompt_attention, "pf_prompt_attention", dev, q.data_ptr(), qs, k.data_ptr(), ks,
              v.data_ptr(), vs, out.data_ptr(), os, _DTYPES[dtype], cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(),
              B, T, TK, nh, nkv, hd, hd ** -0.5 if scale is None else float(scale), None)
    return out


_Param = Union[float, int, torch.Tensor]


def sample_logits(logits: torch.Tensor, u: torch.Tensor, temperature: _Param = 1.0, top_k: _Param = 0,
                  top_p: _Param = 1.0, min_p: _Param = 0.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token per row of logits [rows, vocab] (fp32, fp16 or bf16; rows may
    be strided), int64 [rows], from uniform numbers u [rows] (fp32, in [0, 1)).

    With w = exp((logits - max) / temperature): top_k keeps the top_k largest (the
    lowest indices of equal ones; <= 0 keeps all), of these top_p keeps those
    with less than top_p of their total weight before them in falling order (>= 1
    keeps all, the largest always stays), min_p those with w >= min_p; the token
    is the first whose running sum, in index order, exceeds u times the total.
    temperature <= 0 takes the lowest index of the largest logit.  Each may be a
    number or a tensor [rows] (fp32; top_k int32).  NaN logits count as -inf; a
    row without a finite or +inf value gives -1."""
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
        raise ValueError("sample_logits needs CUDA tensors (no CPU path)")
    code, dev = _DTYPES.get(logits.dtype), logits.get_device()
    if code is None or logits.dim() != 2:
        raise ValueError("logits: [rows, vocab] in fp32, fp16 or bf16 is needed")
    R, V = logits.shape
    step, inner = logits.stride()
    if V < 1 or V > 360000:
        raise ValueError(f"vocab {V}: 1 to 360000")
    if V > 1 and inner != 1:
        raise ValueError("logits: a row has to be contiguous")
    _need(u, "u", dev, torch.float32, (R,))
    t, k, p, m = temperature, top_k, top_p, min_p
    tp = kp = pp = mp = None
    if isinstance(t, torch.Tensor):
        _need(t, "temperature", dev, torch.float32, (R,))
        tp, t = t.data_ptr(), 0.0
    if isinstance(k, torch.Tensor):
        _need(k, "top_k", dev, torch.int32, (R,))
        kp, k = k.data_ptr(), 0
    else:
        k = max(0, min(int(k), V))
    if isinstance(p, torch.Tensor):
        _need(p, "top_p", dev, torch.float32, (R,))
        pp, p = p.data_ptr(), 0.0
    if isinstance(m, torch.Tensor):
        _need(m, "min_p", dev, torch.float32, (R,))
        mp, m = m.data_ptr(), 0.0
    if out is None:
        out = torch.empty(R, dtype=torch.int64, device=logits.device)
    else:
        _need(out, "out", dev, torch.int64, (R,))
    if R:
        _call(_lib.load().pf_sample_logits, "pf_sample_logits", dev, logits.data_ptr(), step if R > 1 else V, code, R,
              V, u.data_ptr(), tp, float(t), kp, k, pp, float(p), mp, float(m), out.data_ptr())
    return out
