"""Grouped-query attention: whole prompts, and an 8-bit paged cache.

For the layers and draft models that a serving engine runs beside the
latent-attention ones (the reference has none of it), and for dense prompts
of latent attention with its heads expanded (d_qk 192, d_v 128).  The
functions make one serving path:

* ``gqa_prefill_fwd``        attention over packed whole prompts;
* ``gqa_cache_append``       their (or a decode step's) K and V into the cache;
* ``gqa_decode_fwd``         attention of each sequence's last tokens over it;
* ``gqa_attention_weights``  the weight that each cached position drew;
* ``gqa_cache_evict``        keeps the heaviest and the newest positions.

The cache: ``k_cache`` and ``v_cache`` float8_e4m3fn (or uint8) [num_blocks,
P, h_kv, d] with any 16-byte aligned strides (a [num_blocks, h_kv, P, d]
pool is passed as ``pool.transpose(1, 2)``), P a power of two from 16 to
1024, d 64 or 128; ``k_scale`` and ``v_scale`` fp32 [num_blocks, h_kv]: a
stored value stands for e4m3 * scale of its block and head.  Position t of
sequence i lies in block ``block_table[i, t // P]``, row t % P;
``context_lens`` int32 [b] counts each sequence's positions, a table holds at
most 2^30.  Block ids out of range hold nothing: reads leave them out, writes
skip them.

All run on the current stream without a host synchronisation and can be
captured in CUDA graphs.  Errors raise RuntimeError.  See include/dsv4b.h
for the exact contracts.
"""
from __future__ import annotations

import ctypes
import struct
from typing import Optional, Tuple

import torch

from ._lib import check, lib
from .ops import _on_device

_i32, _i64, _f32, _vp = ctypes.c_int32, ctypes.c_int64, ctypes.c_float, ctypes.c_void_p
_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
_FP8 = (torch.float8_e4m3fn, torch.uint8)
_MAX_FP32 = torch.finfo(torch.float32).max
_MAX_POSITIONS = 1 << 30  # of a sequence, its weights and its budget


class GqaCache(ctypes.Structure):
    """dsv4b_gqa_cache."""
    _fields_ = [
        ("k", _vp), ("v", _vp), ("k_scale", _vp), ("v_scale", _vp),
        ("stride_k_block", _i64), ("stride_k_row", _i64), ("stride_k_head", _i64),
        ("stride_v_block", _i64), ("stride_v_row", _i64), ("stride_v_head", _i64),
        ("num_blocks", _i32), ("page_block_size", _i32), ("h_kv", _i32), ("d", _i32),
        ("block_table", _vp), ("stride_block_table", _i64), ("table_width", _i32), ("b", _i32),
        ("context_lens", _vp),
    ]


class GqaQuery(ctypes.Structure):
    """dsv4b_gqa_query."""
    _fields_ = [
        ("dtype", _i32), ("s_q", _i32), ("h_q", _i32), ("sm_scale", _f32),
        ("q", _vp), ("stride_q_b", _i64), ("stride_q_s", _i64), ("stride_q_h", _i64),
    ]


class GqaEvictParams(ctypes.Structure):
    """dsv4b_gqa_evict_params."""
    _fields_ = [
        ("budget", _i32), ("recent", _i32), ("weights", _vp), ("stride_w_b", _i64), ("stride_w_h", _i64),
        ("width", _i32), ("new_width", _i32), ("new_weights", _vp), ("stride_nw_b", _i64), ("stride_nw_h", _i64),
        ("kept", _vp), ("new_lens", _vp), ("new_table", _vp), ("stride_new_table", _i64), ("new_table_width", _i32),
    ]


class GqaPrefillParams(ctypes.Structure):
    """dsv4b_gqa_prefill_params."""
    _fields_ = [
        ("dtype", _i32), ("b", _i32), ("h_q", _i32), ("h_kv", _i32), ("d_qk", _i32), ("d_v", _i32), ("causal", _i32),
        ("sm_scale", _f32), ("total_q", _i64), ("total_k", _i64),
        ("q", _vp), ("stride_q_t", _i64), ("stride_q_h", _i64),
        ("k", _vp), ("stride_k_t", _i64), ("stride_k_h", _i64),
        ("v", _vp), ("stride_v_t", _i64), ("stride_v_h", _i64),
        ("cu_seqlens_q", _vp), ("cu_seqlens_k", _vp),
        ("out", _vp), ("stride_o_t", _i64), ("stride_o_h", _i64), ("lse", _vp),
    ]


# The structures are packed in one call each (a ctypes structure filled field
# by field took a fifth of a decode call's host time).
_CODES = {_i32: "i", _i64: "q", _f32: "f", _vp: "P"}


def _packer(cls) -> struct.Struct:
    return struct.Struct("@" + "".join(_CODES[t] for _, t in cls._fields_))


_PACK_CACHE, _PACK_QUERY = _packer(GqaCache).pack, _packer(GqaQuery).pack
_PACK_EVICT, _PACK_PREFILL = _packer(GqaEvictParams).pack, _packer(GqaPrefillParams).pack

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(dev: torch.device) -> int:
    """The current stream's handle (the public accessor takes 2 us of a call)."""
    return torch.cuda.current_stream(dev).cuda_stream if _raw_stream is None else _raw_stream(dev.index)


def _require(ok: bool, message: str) -> None:
    if not ok:
        raise RuntimeError(message)


def _int32(t: torch.Tensor, n: int, name: str, dev: torch.device) -> int:
    """Pointer of a contiguous int32 tensor of n elements."""
    if t.dtype != torch.int32 or t.dim() != 1 or t.numel() != n or not t.is_contiguous() or t.device != dev:
        raise RuntimeError(f"{name} must be a contiguous int32 tensor of shape {(n,)} on {dev}, got "
                           f"{t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _table(t: torch.Tensor, b: int, name: str, dev: torch.device):
    """Pointer, row stride and width of a block table."""
    if t.dtype != torch.int32 or t.dim() != 2 or t.device != dev:
        raise RuntimeError(f"{name} must be int32 [b, blocks] on {dev}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    n, width = t.shape
    stride, unit = t.stride()
    if n != b or width < 1 or (unit != 1 and width > 1):
        raise RuntimeError(f"{name} must be int32 [{b}, blocks] with a contiguous last dim, got {tuple(t.shape)}")
    return t.data_ptr(), stride, width


def _rows16(t: torch.Tensor, name: str, distinct: bool = False):
    """Pointer and strides of a tensor whose rows are read or written 16 bytes
    at a time; ``distinct``: no two rows may be the same memory."""
    ptr, st = t.data_ptr(), t.stride()
    bits = 0
    for x in st[:-1]:
        bits |= x & 7
    if bits or st[-1] != 1 or ptr & 15 or (distinct and 0 in st):
        # strides of dims of one element are never used
        st = [x if n > 1 else 8 for x, n in zip(st[:-1], t.shape)] + [st[-1]]
        if st[-1] != 1 or any(x % 8 for x in st[:-1]) or ptr % 16 or (distinct and 0 in st):
            raise RuntimeError(f"{name} needs a contiguous last dim, other strides in multiples of 8 elements (not 0, if "
                               f"it is written to or loaded by tiles) and a 16-byte aligned base, got strides {t.stride()}")
    return ptr, st


def _row_starts(t: torch.Tensor, base: int) -> torch.Tensor:
    """Where the rows of a tensor begin, in elements from ``base`` on, ascending (on the host)."""
    at = torch.tensor([(t.data_ptr() - base) // t.element_size()], device="cpu")
    for n, x in zip(t.shape[:-1], t.stride()):
        at = (at[:, None] + torch.arange(n, device="cpu") * x).view(-1)
    return at.sort()[0]


def _own_rows(t: torch.Tensor, name: str) -> None:
    """Refuses a tensor, to be written, of which two rows share an element."""
    if t.is_contiguous():
        return
    width = need = t.size(-1)
    for x, n in sorted((x, n) for x, n in zip(t.stride()[:-1], t.shape) if n > 1):
        if x < need:  # rows inside one another's gaps?
            at = _row_starts(t, t.data_ptr())
            _require(bool((at[1:] - at[:-1] >= width).all()), f"{name}'s rows overlap: strides {t.stride()}")
            return
        need += x * (n - 1)


def _fp8_cache(t: torch.Tensor, scale: torch.Tensor, name: str, dev: torch.device):
    """The pointers and the three byte strides of a cache tensor and its scales."""
    if t.dtype not in _FP8 or t.dim() != 4 or t.device != dev:
        raise RuntimeError(f"{name}_cache must be float8_e4m3fn / uint8 [num_blocks, P, h_kv, d] on {dev}")
    nb, page, h, d = t.shape
    ptr, (sb, sr, sh, sd) = t.data_ptr(), t.stride()
    if nb <= 1 or h <= 1:  # dims of one element: any stride will do
        _require(nb > 0 and h > 0, f"{name}_cache has no blocks or heads")
        sb = sb if nb > 1 else max(page * sr, d)
        sh = sh if h > 1 else max(sr, d)
    if sd != 1 or (sb | sr | sh | ptr) & 15 or min(sb, sr, sh) < d:
        raise RuntimeError(f"{name}_cache needs a contiguous last dim, other strides in multiples of 16 bytes and a "
                           f"16-byte aligned base, got strides {t.stride()}")
    if scale.dtype != torch.float32 or scale.shape != (nb, h) or not scale.is_contiguous() or scale.device != dev:
        raise RuntimeError(f"{name}_scale must be contiguous float32 {[nb, h]} on {dev}")
    return ptr, scale.data_ptr(), sb, sr, sh


class _Cache:
    """A checked cache: its packed structure, and the sizes that the calls need."""

    __slots__ = ("packed", "dev", "b", "page", "h_kv", "d", "width", "table_ptr")

    def __init__(self, k_cache, v_cache, k_scale, v_scale, block_table, context_lens):
        dev = self.dev = k_cache.device
        _require(k_cache.is_cuda, "the cache must be a CUDA tensor")
        b = self.b = context_lens.numel()
        _require(b > 0, "context_lens is empty")
        ctx = _int32(context_lens, b, "context_lens", dev)
        self.table_ptr, stride, self.width = _table(block_table, b, "block_table", dev)
        k, ks, kb, kr, kh = _fp8_cache(k_cache, k_scale, "k", dev)
        shape = k_cache.shape
        if v_cache is None:
            v = vs = vb = vr = vh = 0
        else:
            if v_cache.shape != shape:
                raise RuntimeError("k_cache and v_cache must have one shape")
            v, vs, vb, vr, vh = _fp8_cache(v_cache, v_scale, "v", dev)
        nb, self.page, self.h_kv, self.d = shape
        if self.page not in _PAGES or self.d not in (64, 128):
            raise RuntimeError(f"blocks of {self.page} positions, d {self.d}: a power of two from 16 to 1024, and 64 or "
                               "128, are supported")
        self.packed = _PACK_CACHE(k, v, ks, vs, kb, kr, kh, vb, vr, vh, nb, self.page, self.h_kv, self.d,
                                  self.table_ptr, stride, self.width, b, ctx)


_PAGES = (16, 32, 64, 128, 256, 512, 1024)


def _scale(sm_scale: Optional[float], d: int) -> float:
    scale = d ** -0.5 if sm_scale is None else float(sm_scale)
    if not 0.0 < scale <= _MAX_FP32:
        raise RuntimeError(f"sm_scale must be positive, in fp32 too, got {scale}")
    return scale


def _query(q, c: _Cache, sm_scale: Optional[float]):
    """The packed query, s_q and h_q."""
    if q.dim() != 4 or q.dtype not in _DTYPES or q.device != c.dev:
        raise RuntimeError(f"q must be bf16 / fp16 [b, s_q, h_q, d] on {c.dev}")
    b, s_q, h_q, d = q.shape
    if b != c.b or d != c.d or s_q < 1 or h_q < 1 or h_q % c.h_kv:
        raise RuntimeError(f"q {tuple(q.shape)} does not match {c.b} sequences, {c.h_kv} KV heads, d {c.d}")
    ptr, st = _rows16(q, "q")
    scale = _scale(sm_scale, d)
    return _PACK_QUERY(_DTYPES[q.dtype], s_q, h_q, scale, ptr, st[0], st[1], st[2]), s_q, h_q


def gqa_prefill_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor,
                    cu_seqlens_k: Optional[torch.Tensor] = None, sm_scale: Optional[float] = None,
                    causal: bool = True, out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention over whole prompts of packed sequences.

    q [total_q, h_q, d_qk], k [total_k, h_kv, d_qk], v [total_k, h_kv, d_v],
    bf16 or fp16, (d_qk, d_v) = (64, 64), (128, 128) or (192, 128), h_q a
    multiple of h_kv; cu_seqlens int32 [b + 1] (``cu_seqlens_k`` defaults to
    ``cu_seqlens_q``).  With ``causal`` the last query of a sequence sees
    all its keys, the one before it one less, and so on.  Returns (out
    [total_q, h_q, d_v], lse fp32 [total_q, h_q], natural log); a query that
    sees no key gets 0 and -inf.  Rows behind the last sequence are not
    written.  ``out`` may be q itself, but share no memory with k or v."""
    dev = q.device
    _require(q.is_cuda, "q must be a CUDA tensor")
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        if t.dim() != 3 or t.dtype != q.dtype or t.dtype not in _DTYPES or t.device != dev:
            raise RuntimeError(f"{name} must be bf16 / fp16 [tokens, heads, d], as q is, on {dev}")
    total_q, h_q, d_qk = q.shape
    total_k, h_kv, d_v = v.shape
    _require(k.shape == (total_k, h_kv, d_qk), "k does not match q and v")
    if (d_qk, d_v) not in ((64, 64), (128, 128), (192, 128)):
        raise RuntimeError(f"(d_qk, d_v) = {(d_qk, d_v)}: (64, 64), (128, 128) or (192, 128) is supported")
    if h_kv < 1 or h_q < 1 or h_q % h_kv:
        raise RuntimeError(f"{h_q} query heads are not a multiple of {h_kv} KV heads")
    scale = _scale(sm_scale, d_qk)
    b = cu_seqlens_q.numel() - 1
    _require(b >= 1, "cu_seqlens_q must have b + 1 >= 2 entries")
    cq = _int32(cu_seqlens_q, b + 1, "cu_seqlens_q", dev)
    if cu_seqlens_k is None:
        _require(total_k == total_q, "k and q have different lengths: pass cu_seqlens_k")
        ck = cq
    else:
        ck = _int32(cu_seqlens_k, b + 1, "cu_seqlens_k", dev)
    if out is None:
        out = q.new_empty((total_q, h_q, d_v))
    elif out.dtype != q.dtype or out.shape != (total_q, h_q, d_v) or out.device != dev:
        raise RuntimeError(f"out must be {q.dtype} {[total_q, h_q, d_v]} on {dev}")
    else:
        _own_rows(out, "out")
    lse = torch.empty((total_q, h_q), dtype=torch.float32, device=dev)
    if total_q == 0:
        return out, lse
    qp, qs = _rows16(q, "q", True)
    kp, ks = _rows16(k, "k", True)
    vp, vs = _rows16(v, "v", True)
    op, os_ = _rows16(out, "out", True)
    p = _PACK_PREFILL(_DTYPES[q.dtype], b, h_q, h_kv, d_qk, d_v, 1 if causal else 0, scale, total_q, total_k, qp, qs[0],
                      qs[1], kp, ks[0], ks[1], vp, vs[0], vs[1], cq, ck, op, os_[0], os_[1], lse.data_ptr())
    with _on_device(dev):
        check("dsv4b_gqa_prefill", lib.dsv4b_gqa_prefill(p, _stream(dev)))
    return out, lse


def gqa_cache_append(k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, context_lens: torch.Tensor,
                     block_table: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                     v_scale: torch.Tensor) -> None:
    """Appends tokens to the cache: rows cu_seqlens[i] .. cu_seqlens[i + 1] - 1
    of k and v (bf16 / fp16 [n, h_kv, d]) become the last positions of
    sequence i, whose ``context_lens`` counts them already.

    A block and head's scale is the smallest power of two (at least 2^-100)
    that holds its largest value; a block with earlier positions keeps a
    larger scale, or has them rounded again to the new one.  Infinities are
    stored as +-448 of the finite values' scale, NaN as NaN.  No block may
    be written by two sequences of one call."""
    c = _Cache(k_cache, v_cache, k_scale, v_scale, block_table, context_lens)
    dev = c.dev
    n = k.size(0) if k.dim() else 0
    if k.dim() != 3 or k.dtype not in _DTYPES or v.dtype != k.dtype or k.shape != (n, c.h_kv, c.d) or \
            v.shape != k.shape or k.device != dev or v.device != dev:
        raise RuntimeError(f"k and v must be bf16 / fp16 [n, {c.h_kv}, {c.d}] on {dev}")
    kp, ks = _rows16(k, "k")
    vp, vs = _rows16(v, "v")
    cu = _int32(cu_seqlens, c.b + 1, "cu_seqlens", dev)
    with _on_device(dev):
        check("dsv4b_gqa_cache_append",
              lib.dsv4b_gqa_cache_append(c.packed, _DTYPES[k.dtype], kp, ks[0], ks[1], vp, vs[0], vs[1], cu, n,
                                         _stream(dev)))


_ws_bytes: dict = {}  # (device index, d) -> bytes


def _decode_workspace(dev: torch.device, d: int) -> torch.Tensor:
    n = _ws_bytes.get((dev.index, d))
    if n is None:
        size = ctypes.c_size_t()
        check("dsv4b_gqa_decode_workspace_bytes",
              lib.dsv4b_gqa_decode_workspace_bytes(dev.index, d, ctypes.byref(size)))
        n = _ws_bytes[(dev.index, d)] = int(size.value)
    # each call's own: calls on several streams, or captured in several graphs, share none
    return torch.empty(n, dtype=torch.uint8, device=dev)


def gqa_decode_fwd(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                   v_scale: torch.Tensor, block_table: torch.Tensor, context_lens: torch.Tensor,
                   sm_scale: Optional[float] = None,
                   out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention of each sequence's last s_q positions over the cache.

    q bf16 / fp16 [b, s_q, h_q, d]; ``context_lens`` counts the queries' own
    positions, and query x sees those up to its own.  Returns (out [b, s_q,
    h_q, d] in q's type, lse fp32 [b, h_q, s_q], natural log); a query that
    sees no position gets 0 and -inf.  ``out`` may be q itself."""
    c = _Cache(k_cache, v_cache, k_scale, v_scale, block_table, context_lens)
    dev = c.dev
    qq, s_q, h_q = _query(q, c, sm_scale)
    if out is None:
        out = q.new_empty(q.shape)
    elif out.dtype != q.dtype or out.shape != q.shape or out.device != dev:
        raise RuntimeError(f"out must be {q.dtype} {list(q.shape)} on {dev}")
    else:
        _own_rows(out, "out")
    op, so = _rows16(out, "out", True)
    lse = torch.empty((c.b, h_q, s_q), dtype=torch.float32, device=dev)
    with _on_device(dev):
        ws = _decode_workspace(dev, c.d)
        check("dsv4b_gqa_decode",
              lib.dsv4b_gqa_decode(c.packed, qq, op, so[0], so[1], so[2], lse.data_ptr(), ws.data_ptr(), ws.numel(),
                                   _stream(dev)))
    return out, lse


def gqa_attention_weights(q: torch.Tensor, lse: torch.Tensor, k_cache: torch.Tensor, k_scale: torch.Tensor,
                          block_table: torch.Tensor, context_lens: torch.Tensor, sm_scale: Optional[float] = None,
                          weights: Optional[torch.Tensor] = None, accumulate: bool = False,
                          max_context: Optional[int] = None) -> torch.Tensor:
    """The attention weight that each cached position drew from ``q``, summed
    over the queries and over the query heads of a KV head.

    q and lse as for / from ``gqa_decode_fwd`` (a prompt's last queries, or
    a decode step's).  Returns fp32 [b, h_kv, width]: ``weights`` if given,
    which ``accumulate`` adds to (behind the context it is left as it was;
    without ``accumulate`` zeros go there), else a new tensor of width
    ``max_context`` (default: the block table's)."""
    c = _Cache(k_cache, None, k_scale, None, block_table, context_lens)
    dev = c.dev
    qq, s_q, h_q = _query(q, c, sm_scale)
    if lse.dtype != torch.float32 or lse.shape != (c.b, h_q, s_q) or not lse.is_contiguous() or lse.device != dev:
        raise RuntimeError(f"lse must be contiguous float32 {[c.b, h_q, s_q]} on {dev}")
    if weights is None:
        _require(not accumulate, "accumulate needs weights to add to")
        width = c.width * c.page if max_context is None else int(max_context)
        if not 0 < width <= _MAX_POSITIONS:
            raise RuntimeError(f"max_context must be positive and at most 2^30, got {width}")
        weights = torch.empty((c.b, c.h_kv, width), dtype=torch.float32, device=dev)
    else:
        _require(max_context is None, "max_context is for a new tensor: weights has a width already")
        width = _weights(weights, c, "weights", True)
    sb, sh, _ = weights.stride()
    with _on_device(dev):
        check("dsv4b_gqa_attention_weights",
              lib.dsv4b_gqa_attention_weights(c.packed, qq, lse.data_ptr(), weights.data_ptr(), sb, sh, width,
                                              1 if accumulate else 0, _stream(dev)))
    return weights


def _weights(t: torch.Tensor, c: _Cache, name: str, written: bool) -> int:
    """The width of a weights tensor."""
    if t.dtype != torch.float32 or t.dim() != 3 or t.shape[:2] != (c.b, c.h_kv) or t.size(2) < 1 or \
            t.size(2) > _MAX_POSITIONS or t.stride(2) != 1 or t.device != c.dev:
        raise RuntimeError(f"{name} must be float32 [{c.b}, {c.h_kv}, width <= 2^30] on {c.dev} with a contiguous last dim")
    if written:
        _own_rows(t, name)
    return t.size(2)


def _apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two [b, h_kv, width] tensors of one type share no element."""
    pa, pb, sa, sb = a.data_ptr(), b.data_ptr(), a.stride(), b.stride()

    def end(t, p, st):
        return p + t.element_size() * (sum((n - 1) * x for n, x in zip(t.shape, st)) + 1)

    if end(a, pa, sa) <= pb or end(b, pb, sb) <= pa:
        return True
    x, y = _row_starts(a, pa), _row_starts(b, pa)
    behind = torch.searchsorted(x, y)  # the first row of a at or behind each of b's
    after = torch.where(behind < len(x), x[behind.clamp(max=len(x) - 1)], y + b.size(2))
    before = torch.where(behind > 0, x[(behind - 1).clamp(min=0)], y - a.size(2))
    return bool((after >= y + b.size(2)).all() and (before + a.size(2) <= y).all())


def gqa_cache_evict(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                    block_table: torch.Tensor, context_lens: torch.Tensor, weights: torch.Tensor, budget: int,
                    recent: int, new_block_table: torch.Tensor, new_weights: Optional[torch.Tensor] = None
                    ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Keeps ``budget`` positions of every sequence and KV head, each head
    its own: the newest ``recent``, and of the others those of the largest
    ``weights`` (fp32 [b, h_kv, width]; equal ones: the lowest position
    first), all of them where there are no more.  They become, in order, the
    first positions of the blocks of ``new_block_table`` [b, >= ceil(budget /
    P)], which must be blocks that the call does not read, none twice.

    ``new_weights``, if given, must share no memory with ``weights``.  A
    sequence counts as at most width positions long.

    Returns (kept int32 [b, h_kv, budget], -1 behind the new length;
    new_weights fp32 [b, h_kv, >= budget], the kept positions' weights, 0
    behind; new context_lens int32 [b]).  The old blocks keep what they
    hold."""
    c = _Cache(k_cache, v_cache, k_scale, v_scale, block_table, context_lens)
    dev = c.dev
    budget, recent = int(budget), int(recent)
    if not 1 <= budget <= _MAX_POSITIONS or not 0 <= recent <= budget:
        raise RuntimeError(f"budget {budget}, recent {recent}: 0 <= recent <= budget, 1 <= budget <= 2^30")
    width = _weights(weights, c, "weights", False)
    new_table, new_stride, new_blocks = _table(new_block_table, c.b, "new_block_table", dev)
    _require(new_table != c.table_ptr, "new_block_table must not be block_table")
    _require(new_blocks * c.page >= min(budget, width, c.width * c.page),
             "new_block_table has fewer blocks than the budget needs")
    if new_weights is None:
        new_width = budget
        new_weights = torch.empty((c.b, c.h_kv, budget), dtype=torch.float32, device=dev)
    else:
        new_width = _weights(new_weights, c, "new_weights", True)
        _require(new_width >= budget, "new_weights is narrower than the budget")
        _require(_apart(weights, new_weights), "new_weights must not share memory with weights")
    kept = torch.empty((c.b, c.h_kv, budget), dtype=torch.int32, device=dev)
    new_lens = torch.empty((c.b,), dtype=torch.int32, device=dev)
    ws, ns = weights.stride(), new_weights.stride()
    p = _PACK_EVICT(budget, recent, weights.data_ptr(), ws[0], ws[1], width, new_width, new_weights.data_ptr(), ns[0],
                    ns[1], kept.data_ptr(), new_lens.data_ptr(), new_table, new_stride, new_blocks)
    with _on_device(dev):
        check("dsv4b_gqa_cache_evict", lib.dsv4b_gqa_cache_evict(c.packed, p, _stream(dev)))
    return kept, new_weights, new_lens


def gqa_status(device: Optional[torch.device] = None) -> int:
    """Status word of the grouped-query kernels (0 = no error; 1 = a wait
    timed out and a call's outputs are invalid); clears it.  Synchronises."""
    device = torch.device("cuda" if device is None else device)
    _require(device.type == "cuda", f"{device} is not a CUDA device")
    if device.index is None:
        device = torch.device(device.type, torch.cuda.current_device())
    flags = ctypes.c_int()
    with torch.cuda.device(device):
        check("dsv4b_gqa_status", lib.dsv4b_gqa_status(ctypes.byref(flags), _stream(device)))
    return int(flags.value)
