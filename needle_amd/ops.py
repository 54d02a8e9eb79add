"""torch-facing wrappers of the HIP paged-KV operations.

Each function mirrors one seam of needle/layers/attention.py (rms_norm and
silu_mul: the decoder layer's elementwise ops around it, needle/model/qwen2.py:52-65)
and forwards device pointers to the C ABI (include/needle_amd.h) on torch's current
stream.  Nothing here computes on the host: the HIP library is required.

Argument meaning follows the reference:
  kv_cache      [2, num_blocks, num_kv_heads, block_size, head_dim]   (attention.py:9-10)
  block_table   int32 [num_seqs, max_blocks_per_seq]                  (runner.py:220-235)
  context_lens  int32 [num_seqs], tokens already cached               (runner.py:204-218)
  cu_seqlens    int32 [num_seqs + 1], packed token offsets           (runner.py:217)
"""
from __future__ import annotations

import contextlib
import os
from typing import NamedTuple, Optional

import torch
import torch.nn.functional as F
from torch.autograd import forward_ad

from . import _lib

_DTYPES = {torch.bfloat16: _lib.NDL_DTYPE_BF16, torch.float16: _lib.NDL_DTYPE_F16,
           torch.float32: _lib.NDL_DTYPE_F32}


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(dev: torch.device) -> int:
    """The raw handle of torch's current stream on dev (what current_stream(dev).cuda_stream
    gives, without building a Stream object on every call where torch exposes the handle)."""
    if _raw_stream is None:
        return torch.cuda.current_stream(dev).cuda_stream
    idx = dev.index
    return _raw_stream(torch.cuda.current_device() if idx is None else idx)


def _on(dev: torch.device):
    """dev as the current device while a launch is sized and made (no guard where it is)."""
    if dev.index is None or dev.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(dev)


def _require(cond: bool, msg: str, exc=ValueError) -> None:
    if not cond:
        raise exc(msg)


def _check_cache(kv_cache: torch.Tensor) -> None:
    if kv_cache.dim() != 5 or kv_cache.shape[0] != 2:
        raise ValueError("kv_cache must be [2, num_blocks, num_kv_heads, block_size, "
                         f"head_dim], got {tuple(kv_cache.shape)}")
    _require(kv_cache.is_cuda, "kv_cache must be a GPU tensor")
    _require(kv_cache.is_contiguous(), "kv_cache must be contiguous")
    if kv_cache.dtype not in _DTYPES:
        raise TypeError(f"unsupported kv_cache dtype {kv_cache.dtype}")


def _check_int32(name: str, t: torch.Tensor, dim: int, device) -> None:
    # Messages are formatted only on failure: these checks run on every launch.
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    if t.dim() != dim:
        raise ValueError(f"{name} must have {dim} dims, got {t.dim()}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    if t.stride(-1) != 1:
        raise ValueError(f"{name} must be contiguous along its last dim")


def _rows(name: str, x: torch.Tensor, n_heads: int, head_dim: int, device) -> int:
    """Token stride of a [T, n_heads, head_dim] tensor with contiguous inner rows."""
    if x.dim() != 3 or x.shape[1] != n_heads or x.shape[2] != head_dim:
        raise ValueError(f"{name} must be [T, {n_heads}, {head_dim}], got {tuple(x.shape)}")
    if x.device != device:
        raise ValueError(f"{name} must be on {device}")
    if x.stride(2) != 1 or x.stride(1) != head_dim:
        raise ValueError(f"{name} rows must be contiguous (strides {x.stride()})")
    return x.stride(0) if x.shape[0] > 1 else n_heads * head_dim


def _validate_enabled() -> bool:
    return os.environ.get("NEEDLE_AMD_VALIDATE", "") not in ("", "0")


def _validate_slots(block_table, num_blocks, name="block_table") -> None:
    """Opt-in host check (syncs) that mirrors the reference's index errors."""
    if block_table.numel() == 0:
        return
    lo, hi = int(block_table.min()), int(block_table.max())
    if lo < 0 or hi >= num_blocks:
        raise IndexError(f"{name} holds block id outside [0, {num_blocks}): [{lo}, {hi}]")


def kv_append(k: torch.Tensor, v: torch.Tensor, kv_cache: torch.Tensor,
              block_table: torch.Tensor, context_lens: torch.Tensor,
              cu_seqlens: Optional[torch.Tensor] = None) -> None:
    """Scatter k/v [T, Hkv, D] into kv_cache in place.

    cu_seqlens=None is the decode form (attention.py:141-154: token i belongs
    to sequence i); otherwise the varlen form of _write_kv (attention.py:204-246).
    """
    _check_cache(kv_cache)
    dev = kv_cache.device
    _, num_blocks, hkv, bs, d = kv_cache.shape
    _require(k.dtype == kv_cache.dtype and v.dtype == kv_cache.dtype,
             "k/v dtype must match kv_cache", TypeError)
    ks = _rows("k", k, hkv, d, dev)
    vs = _rows("v", v, hkv, d, dev)
    _require(k.shape[0] == v.shape[0], "k and v token counts differ")
    _check_int32("block_table", block_table, 2, dev)
    _check_int32("context_lens", context_lens, 1, dev)
    n_seqs = block_table.shape[0]
    _require(context_lens.shape[0] == n_seqs, "context_lens/block_table batch mismatch")
    n_tok = k.shape[0]
    if cu_seqlens is None:
        _require(n_tok == n_seqs, f"decode append needs one token per sequence "
                 f"({n_tok} tokens, {n_seqs} sequences)")
    else:
        _check_int32("cu_seqlens", cu_seqlens, 1, dev)
        _require(cu_seqlens.shape[0] == n_seqs + 1, "cu_seqlens must be [num_seqs + 1]")
    if n_tok == 0:
        return
    _require(block_table.shape[1] > 0, "block_table has no columns")
    if _validate_enabled():
        _validate_slots(block_table, num_blocks)
    lib = _lib.load()
    rc = lib.ndl_kv_append(
        kv_cache.data_ptr(), num_blocks, hkv, bs, d, _DTYPES[kv_cache.dtype],
        k.data_ptr(), ks, v.data_ptr(), vs,
        block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
        _ptr(cu_seqlens), context_lens.data_ptr(), n_seqs, n_tok, _stream(dev))
    _lib.check(rc, "ndl_kv_append")


def rope_kv_append(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor,
                   cos: torch.Tensor, sin: torch.Tensor, kv_cache: torch.Tensor,
                   block_table: torch.Tensor, context_lens: torch.Tensor,
                   cu_seqlens: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Rotate q/k by (cos, sin) and append rotated k and v to kv_cache; returns rotated q.

    Same result as _apply_rope (attention.py:88, :277-288) followed by the append
    of attention.py:141-154 (cu_seqlens=None) or _write_kv (:204-246), bit for bit.
    q [T, H, D], k/v [T, Hkv, D], cos/sin [T, D] in the cache dtype (bf16, fp16 or fp32).
    q=None rotates and appends k (and appends v) only, and returns None: the form that
    precedes rope_varlen_prefill, which rotates q itself.
    """
    if q is None and out is None and cu_seqlens is not None and _lib.NATIVE is not None:
        if _lib.NATIVE.rope_kv_append(k, v, cos, sin, kv_cache, block_table, context_lens,
                                      cu_seqlens):
            return None
    _check_cache(kv_cache)
    dev = kv_cache.device
    _, num_blocks, hkv, bs, d = kv_cache.shape
    for name, x in (("q", q), ("k", k), ("v", v), ("cos", cos), ("sin", sin)):
        if x is not None and x.dtype != kv_cache.dtype:
            raise TypeError(f"{name} dtype must match kv_cache")
    ks = _rows("k", k, hkv, d, dev)
    vs = _rows("v", v, hkv, d, dev)
    n_tok = k.shape[0]
    if q is not None:
        if q.dim() != 3:
            raise ValueError(f"q must be [T, H, {d}], got {tuple(q.shape)}")
        h = q.shape[1]
        qs = _rows("q", q, h, d, dev)
        _require(q.shape[0] == n_tok, "q/k/v token counts differ")
        if h % hkv:
            raise ValueError(f"num_heads {h} not a multiple of num_kv_heads {hkv}")
    else:
        _require(out is None, "out is the rotated q: pass q with it")
        h, qs = hkv, 0
    _require(v.shape[0] == n_tok, "q/k/v token counts differ")
    if d % 16:
        raise ValueError(f"head_dim {d} must be a multiple of 16")
    for name, x in (("cos", cos), ("sin", sin)):
        if x.dim() != 2 or x.shape[0] != n_tok or x.shape[1] != d:
            raise ValueError(f"{name} must be [{n_tok}, {d}], got {tuple(x.shape)}")
        if x.device != dev or x.stride(1) != 1:
            raise ValueError(f"{name} rows must be contiguous on {dev}")
    _require(cos.stride(0) == sin.stride(0) or n_tok <= 1, "cos and sin token strides differ")
    cs = cos.stride(0) if n_tok > 1 else d
    _check_int32("block_table", block_table, 2, dev)
    _check_int32("context_lens", context_lens, 1, dev)
    n_seqs = block_table.shape[0]
    _require(context_lens.shape[0] == n_seqs, "context_lens/block_table batch mismatch")
    if cu_seqlens is None:
        _require(n_tok == n_seqs, f"decode append needs one token per sequence "
                 f"({n_tok} tokens, {n_seqs} sequences)")
    else:
        _check_int32("cu_seqlens", cu_seqlens, 1, dev)
        _require(cu_seqlens.shape[0] == n_seqs + 1, "cu_seqlens must be [num_seqs + 1]")
    if q is None:
        pass
    elif out is None:
        out = torch.empty((n_tok, h, d), dtype=q.dtype, device=dev)
    else:
        _require(out.shape == (n_tok, h, d) and out.is_contiguous() and out.dtype == q.dtype
                 and out.device == dev, "out must be a contiguous [T, H, D] tensor like q")
    if n_tok == 0:
        return out
    _require(block_table.shape[1] > 0, "block_table has no columns")
    if _validate_enabled():
        _validate_slots(block_table, num_blocks)
    lib = _lib.load()
    rc = lib.ndl_rope_kv_append(
        _ptr(out), _ptr(q), qs, k.data_ptr(), ks, v.data_ptr(), vs,
        cos.data_ptr(), sin.data_ptr(), cs,
        kv_cache.data_ptr(), num_blocks, h, hkv, bs, d, _DTYPES[kv_cache.dtype],
        block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
        _ptr(cu_seqlens), context_lens.data_ptr(), n_seqs, n_tok, _stream(dev))
    _lib.check(rc, "ndl_rope_kv_append")
    return out


def write_kv(k, v, kv_cache, block_table, cu_seqlens, context_lens) -> None:
    """Same signature and effect as the reference _write_kv (attention.py:204-246)."""
    kv_append(k, v, kv_cache, block_table, context_lens, cu_seqlens=cu_seqlens)


def decode_workspace_bytes(num_seqs: int, num_heads: int, num_kv_heads: int, head_dim: int,
                           max_blocks_per_seq: int, block_size: int = 16,
                           partition_tokens: int = 0, dtype: Optional[torch.dtype] = None) -> int:
    """Bytes of the workspace paged_decode uses for this shape: for a pool of dtype (float32's
    split has a size of its own), or, without one, enough for any."""
    lib = _lib.load()
    f32 = 0
    if dtype in (None, torch.float32) and partition_tokens == 0:
        f32 = int(lib.ndl_paged_decode_f32_workspace_bytes(
            num_seqs, num_heads, num_kv_heads, head_dim, max_blocks_per_seq, block_size))
        if f32 and dtype is not None:
            return f32   # 0: a shape the launch refuses, sized (and refused) as the other formats'
    need = int(lib.ndl_paged_decode_workspace_bytes(
        num_seqs, num_heads, num_kv_heads, head_dim, max_blocks_per_seq, block_size,
        partition_tokens))
    return max(need, f32) if need else 0


def paged_decode(q: torch.Tensor, kv_cache: torch.Tensor, block_table: torch.Tensor,
                 context_lens: torch.Tensor, scale: float, num_heads: int, num_kv_heads: int,
                 head_dim: int, *, partition_tokens: int = 0,
                 out: Optional[torch.Tensor] = None,
                 workspace: Optional[torch.Tensor] = None,
                 new_k: Optional[torch.Tensor] = None,
                 new_v: Optional[torch.Tensor] = None,
                 cos: Optional[torch.Tensor] = None,
                 sin: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Paged decode attention; same signature as _decode_pytorch (attention.py:291).

    Sequence i attends min(context_lens[i] + 1, W * block_size) cached tokens.
    Returns [num_seqs, num_heads, head_dim] in q's dtype.  partition_tokens: 0 lets the
    library choose the split; -1 asks for one 8-wave workgroup per (kv head, sequence);
    a positive multiple of 16 asks for the stream split with that many tokens per wave.

    new_k / new_v ([num_seqs, num_kv_heads, head_dim]): the decode append of this step
    (attention.py:141-154) done in the same launch, with the same cache bytes and output as
    kv_append followed by paged_decode.  Requires that no two sequences attend the same
    block (as BlockAllocator's tables guarantee).

    cos / sin ([num_seqs, head_dim], with new_k / new_v): q and new_k are the projections'
    outputs, not yet rotated; the launch applies the rotary embedding of attention.py:88 to
    both first (bit-identical to rope_kv_append followed by paged_decode).
    """
    _check_cache(kv_cache)
    dev = kv_cache.device
    _, num_blocks, hkv, bs, d = kv_cache.shape
    _require(hkv == num_kv_heads and d == head_dim, "kv_cache shape disagrees with head counts")
    _require(q.dtype == kv_cache.dtype, "q dtype must match kv_cache", TypeError)
    qs = _rows("q", q, num_heads, head_dim, dev)
    _check_int32("block_table", block_table, 2, dev)
    _check_int32("context_lens", context_lens, 1, dev)
    n_seqs = q.shape[0]
    _require(block_table.shape[0] == n_seqs and context_lens.shape[0] == n_seqs,
             "q / block_table / context_lens batch mismatch")
    if out is None:
        out = torch.empty((n_seqs, num_heads, head_dim), dtype=q.dtype, device=dev)
    else:
        _require(out.shape == (n_seqs, num_heads, head_dim) and out.is_contiguous()
                 and out.dtype == q.dtype and out.device == dev, "bad out tensor")
    if n_seqs == 0:
        return out
    _require(block_table.shape[1] > 0, "block_table has no columns")
    if _validate_enabled():
        _validate_slots(block_table, num_blocks)
    lib = _lib.load()
    w = block_table.shape[1]
    need = decode_workspace_bytes(n_seqs, num_heads, num_kv_heads, head_dim, w, bs,
                                  partition_tokens, q.dtype)
    _require(need > 0, "unsupported decode shape")
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = decode_workspace(need, dev)
    f32_split = q.dtype == torch.float32 and partition_tokens == 0

    def decode_f32(ks=0, vs=0, cs=0):
        rc = lib.ndl_paged_decode_f32(
            out.data_ptr(), q.data_ptr(), qs, _ptr(new_k), ks, _ptr(new_v), vs, _ptr(cos),
            _ptr(sin), cs, kv_cache.data_ptr(), num_blocks, block_table.data_ptr(),
            block_table.stride(0), w, context_lens.data_ptr(), n_seqs, num_heads, num_kv_heads,
            head_dim, bs, float(scale), workspace.data_ptr(), need, _stream(dev))
        _lib.check(rc, "ndl_paged_decode_f32")
        return out

    if new_k is None and new_v is None:
        _require(cos is None and sin is None, "cos / sin need new_k / new_v")
        if f32_split:
            return decode_f32()
        rc = lib.ndl_paged_decode(
            out.data_ptr(), q.data_ptr(), qs, kv_cache.data_ptr(), num_blocks,
            block_table.data_ptr(), block_table.stride(0), w,
            context_lens.data_ptr(), n_seqs, num_heads, num_kv_heads, head_dim, bs,
            _DTYPES[q.dtype], float(scale), partition_tokens, workspace.data_ptr(), need,
            _stream(dev))
        _lib.check(rc, "ndl_paged_decode")
        return out
    _require(new_k is not None and new_v is not None, "new_k and new_v go together")
    for name, x in (("new_k", new_k), ("new_v", new_v)):
        _require(x.dtype == kv_cache.dtype, f"{name} dtype must match kv_cache", TypeError)
        _require(x.shape[0] == n_seqs, f"{name} must have one row per sequence")
    ks = _rows("new_k", new_k, num_kv_heads, head_dim, dev)
    vs = _rows("new_v", new_v, num_kv_heads, head_dim, dev)
    if cos is not None or sin is not None:
        _require(cos is not None and sin is not None, "cos and sin go together")
        for name, x in (("cos", cos), ("sin", sin)):
            _require(x.dtype == kv_cache.dtype, f"{name} dtype must match kv_cache", TypeError)
            _require(x.dim() == 2 and x.shape[0] == n_seqs and x.shape[1] == head_dim,
                     f"{name} must be [{n_seqs}, {head_dim}], got {tuple(x.shape)}")
            _require(x.device == dev and x.stride(1) == 1, f"{name} rows must be contiguous")
        _require(cos.stride(0) == sin.stride(0) or n_seqs <= 1, "cos and sin strides differ")
        cs = cos.stride(0) if n_seqs > 1 else head_dim
        if f32_split:
            return decode_f32(ks, vs, cs)
        rc = lib.ndl_rope_paged_decode_append(
            out.data_ptr(), q.data_ptr(), qs, new_k.data_ptr(), ks, new_v.data_ptr(), vs,
            cos.data_ptr(), sin.data_ptr(), cs,
            kv_cache.data_ptr(), num_blocks, block_table.data_ptr(), block_table.stride(0), w,
            context_lens.data_ptr(), n_seqs, num_heads, num_kv_heads, head_dim, bs,
            _DTYPES[q.dtype], float(scale), partition_tokens, workspace.data_ptr(), need,
            _stream(dev))
        _lib.check(rc, "ndl_rope_paged_decode_append")
        return out
    if f32_split:
        return decode_f32(ks, vs)
    rc = lib.ndl_paged_decode_append(
        out.data_ptr(), q.data_ptr(), qs, new_k.data_ptr(), ks, new_v.data_ptr(), vs,
        kv_cache.data_ptr(), num_blocks, block_table.data_ptr(), block_table.stride(0), w,
        context_lens.data_ptr(), n_seqs, num_heads, num_kv_heads, head_dim, bs,
        _DTYPES[q.dtype], float(scale), partition_tokens, workspace.data_ptr(), need,
        _stream(dev))
    _lib.check(rc, "ndl_paged_decode_append")
    return out


def decode_workspace(nbytes: int, device) -> torch.Tensor:
    """Scratch for ndl_paged_decode (no contents are assumed; calls that share one must
    run in stream order)."""
    return torch.empty(max(nbytes, 1), dtype=torch.uint8, device=device)


def varlen_prefill(q: torch.Tensor, kv_cache: torch.Tensor, block_table: torch.Tensor,
                   cu_seqlens: torch.Tensor, context_lens: torch.Tensor, max_seqlen: int,
                   scale: float, num_heads: int, num_kv_heads: int, head_dim: int, *,
                   max_context_len: int = 0, out: Optional[torch.Tensor] = None,
                   cos: Optional[torch.Tensor] = None,
                   sin: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of packed prompts over the paged cache (after kv_append).

    Equals the reference _prefill_pytorch (attention.py:120-134) when every
    context_lens entry is 0; with a cached prefix the prefix is attended too.
    Returns [num_tokens, num_heads, head_dim].
    max_context_len bounds context_lens (0: nothing cached).  Results do not depend on it; few
    tokens after a long prefix are split over the GPU only where it says so.
    With cos/sin ([T, D] rows of the packed tokens), q is the raw projection and each row
    is rotated inside the kernel (ndl_rope_varlen_prefill): the output is bit-identical to
    rope_kv_append's rotated q fed to this function, with k already rotated in the cache
    (rope_kv_append with q=None).
    """
    if out is None and _lib.NATIVE is not None:
        out = _lib.NATIVE.varlen_prefill(q, kv_cache, block_table, cu_seqlens, context_lens,
                                         max_seqlen, scale, num_heads, num_kv_heads, head_dim,
                                         max_context_len, cos, sin)
        if out is not None:
            return out
    _check_cache(kv_cache)
    dev = kv_cache.device
    _, num_blocks, hkv, bs, d = kv_cache.shape
    _require(hkv == num_kv_heads and d == head_dim, "kv_cache shape disagrees with head counts")
    _require(q.dtype == kv_cache.dtype, "q dtype must match kv_cache", TypeError)
    qs = _rows("q", q, num_heads, head_dim, dev)
    _check_int32("block_table", block_table, 2, dev)
    _check_int32("cu_seqlens", cu_seqlens, 1, dev)
    _check_int32("context_lens", context_lens, 1, dev)
    n_seqs = block_table.shape[0]
    _require(cu_seqlens.shape[0] == n_seqs + 1 and context_lens.shape[0] == n_seqs,
             "cu_seqlens / context_lens / block_table batch mismatch")
    n_tok = q.shape[0]
    _require((cos is None) == (sin is None), "pass both cos and sin, or neither")
    cs = 0
    if cos is not None:
        for name, x in (("cos", cos), ("sin", sin)):
            if x.dtype != q.dtype:
                raise TypeError(f"{name} dtype must match q")
            if x.dim() != 2 or x.shape[0] != n_tok or x.shape[1] != head_dim:
                raise ValueError(f"{name} must be [{n_tok}, {head_dim}], got {tuple(x.shape)}")
            if x.device != dev or x.stride(1) != 1:
                raise ValueError(f"{name} rows must be contiguous on {dev}")
        _require(cos.stride(0) == sin.stride(0) or n_tok <= 1, "cos and sin token strides differ")
        cs = cos.stride(0) if n_tok > 1 else head_dim
    if out is None:
        out = torch.empty((n_tok, num_heads, head_dim), dtype=q.dtype, device=dev)
    else:
        _require(out.shape == (n_tok, num_heads, head_dim) and out.is_contiguous()
                 and out.dtype == q.dtype and out.device == dev,
                 f"out must be a contiguous {q.dtype} [{n_tok}, {num_heads}, {head_dim}] "
                 f"tensor on {dev}")
    if n_tok == 0 or n_seqs == 0:
        return out
    _require(block_table.shape[1] > 0, "block_table has no columns")
    if _validate_enabled():
        _validate_slots(block_table, num_blocks)
    lib = _lib.load()
    args = (kv_cache.data_ptr(), num_blocks,
            block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
            cu_seqlens.data_ptr(), context_lens.data_ptr(), n_seqs, n_tok, int(max_seqlen),
            int(max_context_len), num_heads, num_kv_heads, head_dim, bs, _DTYPES[q.dtype],
            float(scale))
    # few query tiles over many keys: split over workgroups, the pieces in a workspace
    need = 0
    blocks = min(block_table.shape[1], -(-(int(max_context_len) + int(max_seqlen)) // max(bs, 1)))
    if blocks * bs >= _lib.NDL_PREFILL_SPLIT_MIN_KEYS:
        need = lib.ndl_varlen_prefill_workspace_bytes(
            n_seqs, n_tok, int(max_seqlen), blocks, num_heads, num_kv_heads, head_dim, bs,
            _DTYPES[q.dtype])
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        rc = lib.ndl_varlen_prefill_split(out.data_ptr(), q.data_ptr(), qs, _ptr(cos), _ptr(sin),
                                          cs, *args, ws.data_ptr(), need, _stream(dev))
        _lib.check(rc, "ndl_varlen_prefill_split")
        return out
    tail = (*args, _stream(dev))
    if cos is None:
        rc = lib.ndl_varlen_prefill(out.data_ptr(), q.data_ptr(), qs, *tail)
        _lib.check(rc, "ndl_varlen_prefill")
    else:
        rc = lib.ndl_rope_varlen_prefill(out.data_ptr(), q.data_ptr(), qs, cos.data_ptr(),
                                         sin.data_ptr(), cs, *tail)
        _lib.check(rc, "ndl_rope_varlen_prefill")
    return out


def kv_block_copy(dst_pools, src_pools, src_ids: torch.Tensor, dst_ids: torch.Tensor) -> None:
    """Copy block src_ids[j] to block dst_ids[j] in every layer's pool, both planes, in one
    launch (the KV swap copies; the reference copies per layer and block,
    runner.py:175-192).

    dst_pools / src_pools: equal-length lists of [2, NB, Hkv, bs, D] tensors (or of Fp8KVCache:
    two launches, codes and scales), each on the GPU or in pinned CPU memory (pin_memory=True).
    src_ids / dst_ids: int32 [pairs] on the GPU or pinned.  Enqueued on the current stream of
    the GPU the pools (or ids) live on.
    """
    import ctypes
    _require(len(dst_pools) == len(src_pools), "dst_pools and src_pools differ in length")
    if not dst_pools:
        return
    if any(isinstance(p, Fp8KVCache) for p in (*dst_pools, *src_pools)):
        _require(all(isinstance(p, Fp8KVCache) for p in (*dst_pools, *src_pools)),
                 "an 8-bit pool copies to an 8-bit pool", TypeError)
        for part in (0, 1):
            kv_block_copy([_as_16bit_pool(p)[part] for p in dst_pools],
                          [_as_16bit_pool(p)[part] for p in src_pools], src_ids, dst_ids)
        return
    ref = dst_pools[0]
    _require(ref.dim() == 5 and ref.shape[0] == 2, "pools must be [2, NB, Hkv, bs, D]")
    dev = next((t.device for t in list(dst_pools) + list(src_pools) + [src_ids, dst_ids]
                if t.is_cuda), None)
    _require(dev is not None, "at least one of the pools or ids must be on the GPU")

    def check_pool(t, nb):
        _require(t.dim() == 5 and tuple(t.shape[2:]) == tuple(ref.shape[2:]) and t.shape[0] == 2
                 and t.shape[1] == nb, f"pool shape {tuple(t.shape)} differs from its set")
        _require(t.dtype == ref.dtype and t.dtype in _DTYPES, "pools must share one supported dtype",
                 TypeError)
        _require(t.is_contiguous(), "pools must be contiguous")
        _require(t.device == dev or (t.device.type == "cpu" and t.is_pinned()),
                 "a CPU pool must be pinned (pin_memory=True)")

    dst_nb, src_nb = dst_pools[0].shape[1], src_pools[0].shape[1]
    for t in dst_pools:
        check_pool(t, dst_nb)
    for t in src_pools:
        check_pool(t, src_nb)
    for name, t in (("src_ids", src_ids), ("dst_ids", dst_ids)):
        _require(t.dtype == torch.int32 and t.dim() == 1 and t.is_contiguous(),
                 f"{name} must be a contiguous int32 vector", TypeError)
        _require(t.device == dev or (t.device.type == "cpu" and t.is_pinned()),
                 f"{name} must be on {dev} or pinned")
    _require(src_ids.numel() == dst_ids.numel(), "src_ids and dst_ids differ in length")
    n = src_ids.numel()
    if n == 0:
        return
    arr = ctypes.c_void_p * len(dst_pools)
    dsts = arr(*[t.data_ptr() for t in dst_pools])
    srcs = arr(*[t.data_ptr() for t in src_pools])
    _, _, hkv, bs, d = ref.shape
    lib = _lib.load()
    rc = lib.ndl_kv_block_copy(dsts, dst_nb, srcs, src_nb, len(dst_pools), hkv, bs, d,
                               _DTYPES[ref.dtype], src_ids.data_ptr(), dst_ids.data_ptr(), n,
                               _stream(dev))
    _lib.check(rc, "ndl_kv_block_copy")


def _row_stride(name: str, x: torch.Tensor, width: int, dtype, device) -> int:
    """Row stride of a [rows, width] tensor whose rows are contiguous and 16-byte aligned."""
    if x.dim() != 2 or x.shape[1] != width:
        raise ValueError(f"{name} must be [rows, {width}], got {tuple(x.shape)}")
    if x.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {x.dtype}")
    if x.device != device:
        raise ValueError(f"{name} must be on {device}, got {x.device}")
    if x.stride(1) != 1 and x.shape[1] != 1:
        raise ValueError(f"{name} rows must be contiguous")
    stride = x.stride(0) if x.shape[0] > 1 else width
    if stride % 8 or x.data_ptr() % 16:
        raise ValueError(f"{name} rows must start 16-byte aligned (row stride {stride})")
    return stride


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float,
             residual: Optional[torch.Tensor] = None):
    """RMSNorm of the rows of x (needle/layers/norm.py:14-17), in one kernel.

    Without residual: returns weight * round(x * rsqrt(mean(x^2) + eps)).
    With residual: h = round(x + residual) (the decoder layer's residual add,
    needle/model/qwen2.py:58, :63) and returns (norm of h, h) as new tensors.
    x: [rows, hidden] with contiguous rows; residual: [rows, hidden]; weight: [hidden];
    one dtype (bfloat16, float16 or float32), on one GPU.
    """
    if _lib.NATIVE is not None:
        done = _lib.NATIVE.rms_norm(x, weight, eps, residual)
        if done is not None:
            return done
    _require(x.is_cuda, "x must be a GPU tensor")
    if x.dtype not in _DTYPES:
        raise TypeError(f"unsupported dtype {x.dtype}")
    if x.dim() != 2:
        raise ValueError(f"x must be [rows, hidden], got {tuple(x.shape)}")
    rows, hidden = x.shape
    stride = _row_stride("x", x, hidden, x.dtype, x.device)
    if (weight.shape != (hidden,) or weight.dtype != x.dtype or weight.device != x.device
            or not weight.is_contiguous()):
        raise ValueError(f"weight must be a contiguous [{hidden}] {x.dtype} tensor on {x.device}")
    out = torch.empty((rows, hidden), dtype=x.dtype, device=x.device)
    res_out = None
    if residual is not None:
        if residual.shape != x.shape or not residual.is_contiguous():
            raise ValueError(f"residual must be a contiguous {tuple(x.shape)} tensor")
        _row_stride("residual", residual, hidden, x.dtype, x.device)
        res_out = torch.empty_like(out)
    lib = _lib.load()
    rc = lib.ndl_rms_norm(out.data_ptr(), _ptr(res_out), x.data_ptr(), stride, _ptr(residual),
                          weight.data_ptr(), rows, hidden, float(eps), _DTYPES[x.dtype],
                          _stream(x.device))
    _lib.check(rc, "ndl_rms_norm")
    return out if residual is None else (out, res_out)


def silu_mul(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """silu(gate) * up of the SwiGLU MLP (needle/model/llama.py:37), in one kernel, with
    torch's roundings (the SiLU rounded to the dtype, then the product).  gate, up:
    [rows, intermediate] with contiguous rows (e.g. the two halves of one fused gate/up
    projection output); returns a new [rows, intermediate] tensor."""
    if _lib.NATIVE is not None:
        done = _lib.NATIVE.silu_mul(gate, up)
        if done is not None:
            return done
    _require(gate.is_cuda, "gate must be a GPU tensor")
    if gate.dtype not in _DTYPES:
        raise TypeError(f"unsupported dtype {gate.dtype}")
    if gate.dim() != 2:
        raise ValueError(f"gate must be [rows, intermediate], got {tuple(gate.shape)}")
    rows, inter = gate.shape
    gs = _row_stride("gate", gate, inter, gate.dtype, gate.device)
    us = _row_stride("up", up, inter, gate.dtype, gate.device)
    if up.shape[0] != rows:
        raise ValueError(f"up has {up.shape[0]} rows, gate {rows}")
    out = torch.empty((rows, inter), dtype=gate.dtype, device=gate.device)
    lib = _lib.load()
    rc = lib.ndl_silu_mul(out.data_ptr(), gate.data_ptr(), gs, up.data_ptr(), us, rows, inter,
                          _DTYPES[gate.dtype], _stream(gate.device))
    _lib.check(rc, "ndl_silu_mul")
    return out


# Rows up to which ndl_skinny_linear runs a projection: past them (more than four 16-row
# tiles) its activations outweigh the weights it streams and the library's GEMM takes over.
SKINNY_ROWS = 64


def _skinny_rows(n: int, k: int) -> int:
    """The rows up to which the kernel is the faster one for a single output of n columns.  Past
    16,384 columns the library streams large weights as fast, and the kernel's re-read of the
    activations shows from the third 16-row tile on (us, here / library, at 32, 48 and 64 rows:
    152,064 x 3,584 222 / 264, 221 / 203, 242 / 210; 18,944 x 3,584 31.2 / 33.1, 37.6 / 34.3,
    41.2 / 35.1; 128,256 x 4,096 210 / 205, 210 / 215, 228 / 218), at short k from the fourth
    (151,936 x 896 58 / 66, 67 / 73, 72.9 / 70.4).  Narrower ones keep all 64 (4,608 x 3,584
    12.1 / 13.3, 12.7 / 19.6, 14.2 / 19.0; 3,584 x 18,944 41 / 111, 46 / 114, 53 / 92), and so does
    the gate/up form, which saves the library's second launch (37,888 x 3,584 52.0 / 58.6, 58.6 /
    61.4, 63.4 / 65.3)."""
    if n <= 16384 or k <= 512:
        return SKINNY_ROWS
    return 48 if k <= 1024 else 32


_TENSORS = (torch.Tensor, torch.nn.Parameter)


def skinny_linear_takes(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor],
                        halves: int = 1) -> bool:
    """True where linear (halves = 1) or linear_silu (halves = 2: weight holds the gate and
    the up rows) runs the HIP kernel: up to 64 contiguous, aligned rows of a 16-bit format
    on the current GPU, k a multiple of 64 and the output columns of 16.  Everything that looks
    at the operation rather than its values (autograd, autocast, tracing, function
    transforms, dispatch modes, tensor subclasses) gets torch's own."""
    if (type(x) not in _TENSORS or torch.compiler.is_compiling() or x.dim() != 2
            or not x.is_cuda or not 0 < x.shape[0] <= SKINNY_ROWS):
        return False
    dtype = x.dtype
    if dtype != torch.bfloat16 and dtype != torch.float16:
        return False
    rows, k = x.shape
    n = weight.shape[0]
    if (weight.layout != torch.strided or weight.dim() != 2 or weight.shape[1] != k or k == 0
            or k % 64 or n == 0 or n % (16 * halves) or k > 1 << 24 or n > 1 << 28 or weight.dtype != dtype
            or weight.device != x.device or not weight.is_contiguous()):
        return False
    if halves == 1 and rows > 32 and rows > _skinny_rows(n, k):
        return False
    if not _plain_call():   # before any address: a transform's tensors have none
        return False
    st = x.stride(0) if rows > 1 else k
    if x.stride(1) != 1 or st < k or st % 8 or st > 1 << 24:
        return False
    if bias is not None and (bias.dtype != dtype or bias.device != x.device
                             or bias.shape != (n,) or not bias.is_contiguous()
                             or not _plain(bias) or bias.data_ptr() % 16):
        return False
    return (_plain(x) and _plain(weight) and (x.data_ptr() | weight.data_ptr()) % 16 == 0
            and not torch.is_autocast_enabled("cuda")
            and torch.cuda.current_device() == x.device.index)


def _plain(t: torch.Tensor) -> bool:
    """An ordinary tensor that nothing records."""
    return (type(t) in _TENSORS and not (t.requires_grad and torch.is_grad_enabled())
            and not t.is_conj() and not t.is_neg())


def _plain_call() -> bool:
    """An ordinary call: nothing differentiates, traces, transforms or intercepts it.  torch
    has no public names for most of these; where one is missing the answer is no."""
    try:
        return (forward_ad._current_level < 0
                and torch._C._functorch.peek_interpreter_stack() is None
                and torch._C._len_torch_dispatch_stack() == 0
                and torch._C._len_torch_function_stack() == 0
                and not torch.jit.is_tracing())
    except AttributeError:
        return False


def linear(x: torch.Tensor, weight: torch.Tensor,
           bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """torch's F.linear; on up to SKINNY_ROWS rows (a decode step) one weight-streaming HIP
    kernel, with fp32 sums and one rounding as the library's GEMM (skinny_linear_takes says
    where).  Graph-capturable either way."""
    if not skinny_linear_takes(x, weight, bias):
        return F.linear(x, weight, bias)
    rows, k = x.shape
    n = weight.shape[0]
    out = torch.empty((rows, n), dtype=x.dtype, device=x.device)
    rc = _lib.load().ndl_skinny_linear(
        out.data_ptr(), x.data_ptr(), x.stride(0) if rows > 1 else k, weight.data_ptr(),
        _ptr(bias), rows, n, k, _DTYPES[x.dtype], _stream(x.device))
    _lib.check(rc, "ndl_skinny_linear")
    return out


def linear_silu(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    """silu(gate) * up of x's gate/up projection (needle/model/llama.py:36-37), weight holding
    the gate rows and then the up rows: linear followed by silu_mul, with the same roundings,
    in one kernel on the rows skinny_linear_takes(x, weight, None, halves=2) accepts."""
    inter = weight.shape[0] // 2
    if skinny_linear_takes(x, weight, None, halves=2):
        return skinny_linear_silu(x, weight)
    gate_up = F.linear(x, weight)
    return silu_mul(gate_up[:, :inter], gate_up[:, inter:])


def skinny_linear_silu(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    """linear_silu's kernel, for a caller that has asked skinny_linear_takes(.., halves=2)."""
    inter = weight.shape[0] // 2
    rows, k = x.shape
    out = torch.empty((rows, inter), dtype=x.dtype, device=x.device)
    rc = _lib.load().ndl_skinny_linear_silu(
        out.data_ptr(), x.data_ptr(), x.stride(0) if rows > 1 else k, weight.data_ptr(),
        rows, inter, k, _DTYPES[x.dtype], _stream(x.device))
    _lib.check(rc, "ndl_skinny_linear_silu")
    return out


def greedy_argmax(logits: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The index of each row's maximum, in torch's argmax order (needle/model/sampler.py:
    27-28, for the whole batch: one or two launches, the slices' partials in a workspace
    allocated here, from the graph's pool under capture).  logits: [rows, vocab]; the kernel
    reads contiguous rows that start 16-byte aligned, and other rows (a vocabulary that is not
    a multiple of 8 elements wide, a column slice, a transposed view) are first copied into
    such a buffer on the GPU.  out: int32 or int64 [rows] on the same GPU (a new int64 tensor
    by default).  Graph-capturable."""
    _require(logits.is_cuda, "logits must be a GPU tensor")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"unsupported dtype {logits.dtype}")
    if logits.dim() != 2:
        raise ValueError(f"logits must be [rows, vocab], got {tuple(logits.shape)}")
    rows, vocab = logits.shape
    if rows > 0 and vocab > 0:
        st = logits.stride(0) if rows > 1 else vocab
        if (logits.stride(1) != 1 and vocab > 1) or st % 8 or logits.data_ptr() % 16:
            padded = torch.empty((rows, (vocab + 7) // 8 * 8), dtype=logits.dtype,
                                 device=logits.device)
            padded[:, :vocab].copy_(logits)
            logits = padded[:, :vocab]
    stride = _row_stride("logits", logits, vocab, logits.dtype, logits.device)
    if out is None:
        out = torch.empty(rows, dtype=torch.int64, device=logits.device)
    if (out.dtype not in (torch.int32, torch.int64) or out.shape != (rows,) or
            not out.is_contiguous() or out.device != logits.device):
        raise ValueError(f"out must be a contiguous int32 or int64 [{rows}] tensor on "
                         f"{logits.device}")
    lib = _lib.load()
    nbytes = lib.ndl_greedy_argmax_workspace_bytes(rows, vocab) if rows > 0 else 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=logits.device) if nbytes else None
    rc = lib.ndl_greedy_argmax(out.data_ptr(), int(out.dtype == torch.int64),
                               logits.data_ptr(), stride, rows, vocab, _DTYPES[logits.dtype],
                               _ptr(ws), nbytes, _stream(logits.device))
    _lib.check(rc, "ndl_greedy_argmax")
    return out


# ---------------------------------------------------------------- the 8-bit pool

class Fp8KVCache(NamedTuple):
    """A layer's 8-bit pool, where kv_cache stands for a 16-bit one (Attention.forward): e4m3
    codes [2, num_blocks, num_kv_heads, block_size, head_dim] and a byte per row (token, head),
    [2, num_blocks, num_kv_heads, block_size].  A row's values are code * 2^(byte - 127)."""
    codes: torch.Tensor
    scales: torch.Tensor

    @property
    def shape(self):
        return self.codes.shape


def fp8_kv_pool(num_blocks: int, num_kv_heads: int, block_size: int, head_dim: int, device=None,
                pin_memory: bool = False) -> Fp8KVCache:
    """A zero-filled pool (every value 0)."""
    shape = (2, num_blocks, num_kv_heads, block_size)
    codes = torch.zeros((*shape, head_dim), dtype=torch.uint8, device=device,
                        pin_memory=pin_memory)
    scales = torch.zeros(shape, dtype=torch.uint8, device=device, pin_memory=pin_memory)
    return Fp8KVCache(codes.view(torch.float8_e4m3fn), scales)


def _as_16bit_pool(pool: Fp8KVCache):
    """The bytes of an 8-bit pool as two 16-bit pools, codes and scales, for kv_block_copy (which
    moves raw bits): a block's codes, and its row of scale bytes, of whole 16-byte pieces."""
    _, nb, hkv, bs, d = pool.codes.shape
    return (pool.codes.view(torch.uint8).view(torch.bfloat16),
            pool.scales.view(torch.bfloat16).view(2, nb, 1, hkv * bs // 16, 8))


_FP8_CODES = (torch.float8_e4m3fn, torch.uint8)


def _check_fp8_cache(kv_codes: torch.Tensor, kv_scales: torch.Tensor):
    """(num_blocks, num_kv_heads, block_size, head_dim) of an 8-bit pool."""
    if kv_codes.dim() != 5 or kv_codes.shape[0] != 2:
        raise ValueError("kv_codes must be [2, num_blocks, num_kv_heads, block_size, head_dim], "
                         f"got {tuple(kv_codes.shape)}")
    if kv_codes.dtype not in _FP8_CODES or kv_scales.dtype != torch.uint8:
        raise TypeError("kv_codes must be float8_e4m3fn (or its bytes, uint8) and kv_scales "
                        f"uint8, got {kv_codes.dtype} and {kv_scales.dtype}")
    if kv_scales.shape != kv_codes.shape[:4]:
        raise ValueError(f"kv_scales must be {tuple(kv_codes.shape[:4])}, got "
                         f"{tuple(kv_scales.shape)}")
    _require(kv_codes.is_cuda and kv_scales.device == kv_codes.device,
             "kv_codes and kv_scales must be on one GPU")
    _require(kv_codes.is_contiguous() and kv_scales.is_contiguous(),
             "kv_codes and kv_scales must be contiguous")
    _, nb, hkv, bs, d = kv_codes.shape
    if d not in (64, 128):
        raise ValueError(f"the 8-bit pool is built for head_dim 64 and 128, got {d}")
    if bs < 16 or bs > 1024 or bs & (bs - 1):
        raise ValueError("the 8-bit pool is built for blocks of a power of two from 16 to 1024 "
                         f"tokens, got {bs}")
    return nb, hkv, bs, d


def _check_16bit(name: str, dtype: torch.dtype) -> None:
    if dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"{name} must be bfloat16 or float16 with an 8-bit pool, got {dtype}")


def _check_table(block_table: torch.Tensor, num_blocks: int, device) -> int:
    _check_int32("block_table", block_table, 2, device)
    if _validate_enabled():
        _validate_slots(block_table, num_blocks)
    return block_table.shape[0]


def _check_rope(cos, sin, dtype, n_tok, d, dev) -> int:
    """Token stride of cos and sin [n_tok, d]."""
    for name, x in (("cos", cos), ("sin", sin)):
        if x.dtype != dtype:
            raise TypeError(f"{name} dtype must match k")
        if x.dim() != 2 or x.shape[0] != n_tok or x.shape[1] != d:
            raise ValueError(f"{name} must be [{n_tok}, {d}], got {tuple(x.shape)}")
        if x.device != dev or x.stride(1) != 1:
            raise ValueError(f"{name} rows must be contiguous on {dev}")
    _require(cos.stride(0) == sin.stride(0) or n_tok <= 1, "cos and sin token strides differ")
    return cos.stride(0) if n_tok > 1 else d


def kv_append_fp8(k: torch.Tensor, v: torch.Tensor, kv_codes: torch.Tensor,
                  kv_scales: torch.Tensor, block_table: torch.Tensor,
                  context_lens: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None, *,
                  q: Optional[torch.Tensor] = None, cos: Optional[torch.Tensor] = None,
                  sin: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """kv_append into an 8-bit pool (Fp8KVCache): k/v [T, Hkv, D] in bfloat16 or float16, each
    row quantised as it is written: e4m3 codes of its values divided by the smallest power of
    two (at least 2^-126) that leaves none above 448, rounded to nearest even; NaN where a value
    is not finite.

    cos / sin [T, D] rotate k first, with rope_kv_append's roundings, and q [T, H, D] too if it
    is given: then the rotated q is returned (written to out, contiguous, if that is given; it
    may be q).
    cu_seqlens None: one token per sequence.
    """
    if out is None and _lib.NATIVE is not None:
        done = _lib.NATIVE.kv_append_fp8(k, v, kv_codes, kv_scales, block_table, context_lens,
                                         cu_seqlens, q, cos, sin)
        if done is not None:
            return None if q is None else done
    nb, hkv, bs, d = _check_fp8_cache(kv_codes, kv_scales)
    dev, dtype = kv_codes.device, k.dtype
    _check_16bit("k", dtype)
    for name, x in (("v", v), ("q", q), ("cos", cos), ("sin", sin)):
        if x is not None and x.dtype != dtype:
            raise TypeError(f"{name} dtype must match k")
    ks, vs, n_tok = _rows("k", k, hkv, d, dev), _rows("v", v, hkv, d, dev), k.shape[0]
    _require(v.shape[0] == n_tok, "k and v token counts differ")
    _require((cos is None) == (sin is None), "pass both cos and sin, or neither")
    h, qs, cs = 0, 0, 0
    if cos is not None:
        cs = _check_rope(cos, sin, dtype, n_tok, d, dev)
    if q is not None:
        _require(cos is not None, "q is passed to be rotated: pass cos and sin")
        if q.dim() != 3:
            raise ValueError(f"q must be [T, H, {d}], got {tuple(q.shape)}")
        h = q.shape[1]
        qs = _rows("q", q, h, d, dev)
        _require(q.shape[0] == n_tok, "q/k/v token counts differ")
        _require(h > 0, "q has no heads")
        if out is None:
            out = torch.empty((n_tok, h, d), dtype=dtype, device=dev)
        else:
            _require(out.shape == (n_tok, h, d) and out.is_contiguous() and out.dtype == dtype
                     and out.device == dev, "out must be a contiguous [T, H, D] tensor like q")
    else:
        _require(out is None, "out is the rotated q: pass q with it")
    n_seqs = _check_table(block_table, nb, dev)
    _check_int32("context_lens", context_lens, 1, dev)
    _require(context_lens.shape[0] == n_seqs, "context_lens/block_table batch mismatch")
    if cu_seqlens is None:
        _require(n_tok == n_seqs, f"decode append needs one token per sequence "
                 f"({n_tok} tokens, {n_seqs} sequences)")
    else:
        _check_int32("cu_seqlens", cu_seqlens, 1, dev)
        _require(cu_seqlens.shape[0] == n_seqs + 1, "cu_seqlens must be [num_seqs + 1]")
    if n_tok == 0:
        return out
    _require(block_table.shape[1] > 0, "block_table has no columns")
    with _on(dev):
        rc = _lib.load().ndl_kv_append_fp8(
            kv_codes.data_ptr(), kv_scales.data_ptr(), nb, hkv, bs, d, _DTYPES[dtype],
            k.data_ptr(), ks, v.data_ptr(), vs, _ptr(out), _ptr(q), qs, h, _ptr(cos), _ptr(sin), cs,
            block_table.data_ptr(), block_table.stride(0), block_table.shape[1], _ptr(cu_seqlens),
            context_lens.data_ptr(), n_seqs, n_tok, _stream(dev))
    _lib.check(rc, "ndl_kv_append_fp8")
    return out


def kv_read_fp8(kv_codes: torch.Tensor, kv_scales: torch.Tensor, block_table: torch.Tensor,
                first: torch.Tensor, cu_seqlens: torch.Tensor, num_tokens: int, *,
                dtype: torch.dtype = torch.bfloat16):
    """Ranges of cached tokens in 16 bits: (k, v) [num_tokens, Hkv, D], packed by cu_seqlens, of
    the tokens first[i], first[i] + 1, .. of each sequence.  bfloat16 has every value of the pool
    exactly; float16 every one that came from a float16 row, but for its smallest subnormals and
    the codes of entries of 63,488 and more, which are 65,536 and read as infinity.
    first: int32 [num_seqs].  Rows outside cu_seqlens hold nothing in particular."""
    if _lib.NATIVE is not None:
        done = _lib.NATIVE.kv_read_fp8(kv_codes, kv_scales, block_table, first, cu_seqlens,
                                       num_tokens, _DTYPES.get(dtype))
        if done is not None:
            return done
    nb, hkv, bs, d = _check_fp8_cache(kv_codes, kv_scales)
    dev = kv_codes.device
    _check_16bit("dtype", dtype)
    n_seqs = _check_table(block_table, nb, dev)
    _check_int32("first", first, 1, dev)
    _check_int32("cu_seqlens", cu_seqlens, 1, dev)
    _require(first.shape[0] == n_seqs, "first/block_table batch mismatch")
    _require(cu_seqlens.shape[0] == n_seqs + 1, "cu_seqlens must be [num_seqs + 1]")
    _require(num_tokens >= 0, "num_tokens is negative")
    k = torch.empty((num_tokens, hkv, d), dtype=dtype, device=dev)
    v = torch.empty_like(k)
    if num_tokens == 0 or n_seqs == 0:
        return k, v
    _require(block_table.shape[1] > 0, "block_table has no columns")
    with _on(dev):
        rc = _lib.load().ndl_kv_read_fp8(
            k.data_ptr(), v.data_ptr(), kv_codes.data_ptr(), kv_scales.data_ptr(), nb, hkv, bs, d,
            _DTYPES[dtype], block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
            first.data_ptr(), cu_seqlens.data_ptr(), n_seqs, num_tokens, _stream(dev))
    _lib.check(rc, "ndl_kv_read_fp8")
    return k, v


def _fp8_attention(q, kv_codes, kv_scales, block_table, cu_seqlens, context_lens, max_seqlen,
                   max_keys, scale, num_heads, num_kv_heads, head_dim, out, workspace, *new):
    """new: what a decode step appends and its rotation, (new_k, new_v, cos, sin), or nothing."""
    if out is None and workspace is None and _lib.NATIVE is not None:
        out = _lib.NATIVE.fp8_attention(q, kv_codes, kv_scales, block_table, cu_seqlens,
                                        context_lens, max_seqlen, max_keys, scale, num_heads,
                                        num_kv_heads, head_dim, *new)
        if out is not None:
            return out
    nb, hkv, bs, d = _check_fp8_cache(kv_codes, kv_scales)
    dev = kv_codes.device
    _require(hkv == num_kv_heads and d == head_dim, "kv_codes shape disagrees with head counts")
    _check_16bit("q", q.dtype)
    qs = _rows("q", q, num_heads, head_dim, dev)
    if num_heads % num_kv_heads or num_heads // num_kv_heads > 16:
        raise ValueError(f"num_heads {num_heads} must be 1 to 16 times num_kv_heads "
                         f"{num_kv_heads}")
    n_seqs, n_tok = _check_table(block_table, nb, dev), q.shape[0]
    _check_int32("context_lens", context_lens, 1, dev)
    _require(context_lens.shape[0] == n_seqs, "context_lens/block_table batch mismatch")
    if cu_seqlens is None:
        _require(n_tok == n_seqs, "q / block_table batch mismatch")
    else:
        _check_int32("cu_seqlens", cu_seqlens, 1, dev)
        _require(cu_seqlens.shape[0] == n_seqs + 1, "cu_seqlens must be [num_seqs + 1]")
    if out is None:
        out = torch.empty((n_tok, num_heads, head_dim), dtype=q.dtype, device=dev)
    else:
        _require(out.shape == (n_tok, num_heads, head_dim) and out.is_contiguous()
                 and out.dtype == q.dtype and out.device == dev,
                 f"out must be a contiguous {q.dtype} [{n_tok}, {num_heads}, {head_dim}] "
                 f"tensor on {dev}")
    ks = vs = cs = 0
    new_k, new_v, cos, sin = new or (None,) * 4
    if new:
        _require(new_k is not None and new_v is not None, "new_k and new_v go together")
        for name, x in (("new_k", new_k), ("new_v", new_v)):
            _require(x.dtype == q.dtype, f"{name} dtype must match q", TypeError)
            _require(x.shape[0] == n_seqs, f"{name} must have one row per sequence")
        ks = _rows("new_k", new_k, num_kv_heads, head_dim, dev)
        vs = _rows("new_v", new_v, num_kv_heads, head_dim, dev)
        _require((cos is None) == (sin is None), "cos and sin go together")
        if cos is not None:
            cs = _check_rope(cos, sin, q.dtype, n_seqs, head_dim, dev)
    if n_tok == 0 or n_seqs == 0:
        return out
    w = block_table.shape[1]
    _require(w > 0, "block_table has no columns")
    _require(max_seqlen > 0, "max_seqlen must be positive")
    max_keys = min(w * bs, max_keys) if max_keys else w * bs
    lib = _lib.load()
    with _on(dev):
        need = lib.ndl_fp8_attention_workspace_bytes(n_seqs, n_tok, max_seqlen, max_keys, num_heads,
                                                     num_kv_heads, head_dim, bs)
        if need and (workspace is None or workspace.numel() * workspace.element_size() < need
                     or workspace.device != dev):
            workspace = decode_workspace(need, dev)
        if new:
            rc = lib.ndl_fp8_decode_append(
                out.data_ptr(), q.data_ptr(), qs, new_k.data_ptr(), ks, new_v.data_ptr(), vs,
                _ptr(cos), _ptr(sin), cs, kv_codes.data_ptr(), kv_scales.data_ptr(), nb,
                block_table.data_ptr(), block_table.stride(0), w, context_lens.data_ptr(),
                n_seqs, num_heads, num_kv_heads, head_dim, bs, _DTYPES[q.dtype], float(scale),
                _ptr(workspace) if need else None, need, _stream(dev))
            _lib.check(rc, "ndl_fp8_decode_append")
            return out
        rc = lib.ndl_fp8_attention(
            out.data_ptr(), q.data_ptr(), qs, kv_codes.data_ptr(), kv_scales.data_ptr(), nb,
            block_table.data_ptr(), block_table.stride(0), w, _ptr(cu_seqlens),
            context_lens.data_ptr(), n_seqs, n_tok, max_seqlen, max_keys, num_heads, num_kv_heads,
            head_dim, bs, _DTYPES[q.dtype], float(scale), _ptr(workspace) if need else None, need,
            _stream(dev))
    _lib.check(rc, "ndl_fp8_attention")
    return out


def fp8_attention_workspace_bytes(num_seqs: int, num_tokens: int, max_seqlen: int, max_keys: int,
                                  num_heads: int, num_kv_heads: int, head_dim: int,
                                  block_size: int = 16) -> int:
    """Bytes of the workspace paged_decode_fp8 (num_tokens num_seqs, max_seqlen 1, max_keys the
    table's) or varlen_prefill_fp8 uses on the current GPU; 0 where none is used."""
    return int(_lib.load().ndl_fp8_attention_workspace_bytes(
        num_seqs, num_tokens, max_seqlen, max_keys, num_heads, num_kv_heads, head_dim,
        block_size))


def paged_decode_fp8(q: torch.Tensor, kv_codes: torch.Tensor, kv_scales: torch.Tensor,
                     block_table: torch.Tensor, context_lens: torch.Tensor, scale: float,
                     num_heads: int, num_kv_heads: int, head_dim: int, *,
                     out: Optional[torch.Tensor] = None,
                     workspace: Optional[torch.Tensor] = None,
                     new_k: Optional[torch.Tensor] = None, new_v: Optional[torch.Tensor] = None,
                     cos: Optional[torch.Tensor] = None,
                     sin: Optional[torch.Tensor] = None) -> torch.Tensor:
    """paged_decode over an 8-bit pool (Fp8KVCache): q [num_seqs, H, D] in bfloat16 or float16,
    sequence i attends min(context_lens[i] + 1, W * block_size) tokens.  Append (and rotate q)
    with kv_append_fp8 first, or hand the step's rows to this call.  workspace: as
    decode_workspace gives, of fp8_attention_workspace_bytes, for one call at a time.

    new_k / new_v ([num_seqs, Hkv, D]): the step's append, done in the same launch, with the same
    pool bytes and output as kv_append_fp8 followed by this call.  Requires that no two sequences
    attend the same block that one of them writes (as BlockAllocator's tables guarantee).
    cos / sin ([num_seqs, D], with new_k / new_v): q and new_k are not yet rotated; the launch
    rotates both first."""
    new = ()
    if new_k is not None or new_v is not None:
        new = (new_k, new_v, cos, sin)
    else:
        _require(cos is None and sin is None, "cos / sin need new_k / new_v")
    return _fp8_attention(q, kv_codes, kv_scales, block_table, None, context_lens, 1, 0, scale,
                          num_heads, num_kv_heads, head_dim, out, workspace, *new)


def varlen_prefill_fp8(q: torch.Tensor, kv_codes: torch.Tensor, kv_scales: torch.Tensor,
                       block_table: torch.Tensor, cu_seqlens: torch.Tensor,
                       context_lens: torch.Tensor, max_seqlen: int, scale: float,
                       num_heads: int, num_kv_heads: int, head_dim: int, *,
                       max_context_len: int = 0, out: Optional[torch.Tensor] = None,
                       workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """varlen_prefill over an 8-bit pool (Fp8KVCache): causal attention of packed chunks of new
    tokens, from one per sequence to whole prompts, over what is cached and the chunk itself
    (after kv_append_fp8).  Token j of sequence i attends min(context_lens[i] + j + 1,
    W * block_size) tokens.  max_seqlen bounds a sequence's tokens, max_context_len its cached
    ones (0: not known, the table's width then): sequences past these bounds are not attended
    whole.  Long chunks (224 rows of max_seqlen times H / Hkv and 2^24 scores by these bounds)
    unpack the keys into a 16-bit workspace first, of as many sequences of the bounds' keys as 4 GiB
    hold (one at least) at a time, and are attended by varlen_prefill's kernels."""
    return _fp8_attention(q, kv_codes, kv_scales, block_table, cu_seqlens, context_lens,
                          int(max_seqlen),
                          int(max_context_len) + int(max_seqlen) if max_context_len else 0,
                          scale, num_heads, num_kv_heads, head_dim, out, workspace)


def _check_f32(name, t, shape, dev):
    if t.dtype != torch.float32:
        raise TypeError(f"{name} must be float32, got {t.dtype}")
    if t.shape != shape or t.device != dev or (t.numel() and t.stride(-1) != 1
                                               and shape[-1] != 1):
        raise ValueError(f"{name} must be {list(shape)} with contiguous rows on {dev}, got "
                         f"{tuple(t.shape)}")


def _check_verify(logits, ids, cu_seqlens, uniforms, temperature):
    """(device, rows, vocab, sequences) of a verification's rows."""
    _require(logits.is_cuda, "logits must be a GPU tensor")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"unsupported dtype {logits.dtype}")
    if logits.dim() != 2:
        raise ValueError(f"logits must be [rows, vocab], got {tuple(logits.shape)}")
    rows, vocab = logits.shape
    dev = logits.device
    _require(vocab > 0, "logits have no columns")
    _require(logits.stride(1) == 1 or vocab == 1, "logits rows must be contiguous")
    _require(rows <= 1 or logits.stride(0) >= vocab, "logits rows overlap")
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"ids must be int32 or int64, got {ids.dtype}")
    if ids.shape != (rows,) or not ids.is_contiguous() or ids.device != dev:
        raise ValueError(f"ids must be a contiguous [{rows}] tensor on {dev}")
    _check_int32("cu_seqlens", cu_seqlens, 1, dev)
    n_seqs = cu_seqlens.shape[0] - 1
    _require(n_seqs >= 0, "cu_seqlens must be [num_seqs + 1]")
    _require(rows >= n_seqs, f"every sequence has a row: {rows} rows, {n_seqs} sequences")
    _check_f32("uniforms", uniforms, (rows,), dev)
    if temperature is not None:
        _check_f32("temperature", temperature, (n_seqs,), dev)
    return dev, rows, vocab, n_seqs


def verify_drafts(logits: torch.Tensor, ids: torch.Tensor, cu_seqlens: torch.Tensor,
                  uniforms: torch.Tensor, *, temperature: Optional[torch.Tensor] = None,
                  draft_probs: Optional[torch.Tensor] = None):
    """Speculative decoding's verification: (tokens [T], accepted int32 [num_seqs]).

    logits [T, vocab] (bfloat16, float16 or float32, rows contiguous, any row stride) are the
    target's rows for the packed chunks ids [T] (int32 or int64): a sequence's newest token and
    its drafts, at least one row each.  Row r decides on the draft ids[r + 1]; a sequence's last row
    on none.  With p = softmax(logits[r] / temperature[i]) and q row r - i of draft_probs
    (float32 [T - num_seqs, vocab]; None: the drafts have probability 1) a draft x is accepted
    while uniforms[r] * q(x) < p(x), for it and all before it.  The next token follows
    max(p - q, 0) of the first rejected row, or p of the last row, by the inverse of its
    cumulative distribution at the sequence's last uniform: together distributed as the target.

    temperature float32 [num_seqs] (None: 1); 0 takes the argmax, as does a row whose maximum is
    not finite.  uniforms float32 [T] in [0, 1).  A draft whose row draft_probs has not (after a
    sequence without rows) is rejected.  tokens, in ids' type: the accepted drafts, the next token,
    then -1; rows outside cu_seqlens hold nothing in particular.  Graph-capturable; no host
    synchronisation."""
    if _lib.NATIVE is not None:
        done = _lib.NATIVE.verify_drafts(logits, ids, cu_seqlens, uniforms, temperature,
                                         draft_probs)
        if done is not None:
            return done
    dev, rows, vocab, n_seqs = _check_verify(logits, ids, cu_seqlens, uniforms, temperature)
    ds = vocab
    if draft_probs is not None:
        _check_f32("draft_probs", draft_probs, (rows - n_seqs, vocab), dev)
        if rows - n_seqs > 1:
            ds = draft_probs.stride(0)
            _require(ds >= vocab, "draft_probs rows overlap")
    tokens = torch.empty_like(ids)
    accepted = torch.empty(n_seqs, dtype=torch.int32, device=dev)
    if n_seqs == 0:
        return tokens, accepted
    lib = _lib.load()
    need = lib.ndl_verify_drafts_workspace_bytes(rows, n_seqs, vocab)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    # no draft rows may have no address either: one of which nothing is read says that they are given
    probs = draft_probs if draft_probs is None or rows > n_seqs else uniforms
    with _on(dev):
        rc = lib.ndl_verify_drafts(
            tokens.data_ptr(), accepted.data_ptr(), logits.data_ptr(),
            logits.stride(0) if rows > 1 else vocab, _DTYPES[logits.dtype], ids.data_ptr(),
            int(ids.dtype == torch.int64), cu_seqlens.data_ptr(), uniforms.data_ptr(),
            _ptr(temperature), _ptr(probs), ds, rows - n_seqs, rows, n_seqs, vocab, ws.data_ptr(),
            need, _stream(dev))
    _lib.check(rc, "ndl_verify_drafts")
    return tokens, accepted


# ---------------------------------------------------------------- drafted trees

def tree_mask(parents: torch.Tensor, cu_seqlens: torch.Tensor, max_seqlen: int):
    """Which nodes a drafted tree's tokens attend: (mask int64 [T, ceil(max_seqlen / 64)],
    depth int32 [T]), once a step for tree_attention of every layer.

    parents int32 [T]: for each packed token the node of its own sequence (0 .. its rows) that it
    follows.  Node 0 is the sequence's newest token, and parents come before their children: any other
    number (-1, say) stands for a node that follows the cached tokens alone.  Bit b % 64 of word
    b // 64 is set for the token itself and its ancestors; depth counts the ancestors, so that
    context_lens[i] + depth is the token's position for the rotary embedding.  max_seqlen bounds a
    sequence's tokens.  Rows outside cu_seqlens hold nothing in particular."""
    if _lib.NATIVE is not None:
        done = _lib.NATIVE.tree_mask(parents, cu_seqlens, max_seqlen)
        if done is not None:
            return done
    _require(parents.is_cuda, "parents must be a GPU tensor")
    dev = parents.device
    _check_int32("parents", parents, 1, dev)
    _check_int32("cu_seqlens", cu_seqlens, 1, dev)
    n_seqs, n_tok = cu_seqlens.shape[0] - 1, parents.shape[0]
    _require(n_seqs >= 0, "cu_seqlens must be [num_seqs + 1]")
    max_seqlen = int(max_seqlen)
    _require(max_seqlen > 0, "max_seqlen must be positive")
    words = (max_seqlen + 63) // 64
    mask = torch.empty((n_tok, words), dtype=torch.int64, device=dev)
    depth = torch.empty(n_tok, dtype=torch.int32, device=dev)
    if n_tok == 0 or n_seqs == 0:
        return mask, depth
    with _on(dev):
        rc = _lib.load().ndl_tree_mask(
            mask.data_ptr(), words, words, depth.data_ptr(), parents.data_ptr(),
            cu_seqlens.data_ptr(), n_seqs, n_tok, max_seqlen, _stream(dev))
    _lib.check(rc, "ndl_tree_mask")
    return mask, depth


def tree_attention_workspace_bytes(num_seqs: int, max_seqlen: int, max_keys: int, num_heads: int,
                                   num_kv_heads: int, head_dim: int, block_size: int = 16,
                                   fp8: bool = False) -> int:
    """Bytes of the workspace tree_attention uses over a 16-bit (fp8: an 8-bit) pool on the current
    GPU, max_keys at most the table's; 0 where none is used."""
    lib = _lib.load()
    query = (lib.ndl_fp8_tree_attention_workspace_bytes if fp8
             else lib.ndl_tree_attention_workspace_bytes)
    return int(query(num_seqs, max_seqlen, max_keys, num_heads, num_kv_heads, head_dim,
                     block_size))


def _check_out(out, n_tok, num_heads, head_dim, like):
    shape = (n_tok, num_heads, head_dim)
    if out is None:
        return torch.empty(shape, dtype=like.dtype, device=like.device)
    _require(out.shape == shape and out.is_contiguous() and out.dtype == like.dtype
             and out.device == like.device,
             f"out must be a contiguous {like.dtype} {list(shape)} tensor on {like.device}")
    return out


def _check_group(num_heads, num_kv_heads):
    if num_kv_heads <= 0 or num_heads % num_kv_heads or not 0 < num_heads // num_kv_heads <= 16:
        raise ValueError(f"num_heads {num_heads} must be 1 to 16 times num_kv_heads "
                         f"{num_kv_heads}")


def tree_attention(q: torch.Tensor, kv_cache, block_table: torch.Tensor,
                   cu_seqlens: torch.Tensor, context_lens: torch.Tensor, mask: torch.Tensor,
                   max_seqlen: int, scale: float, num_heads: int, num_kv_heads: int,
                   head_dim: int, *, max_context_len: int = 0,
                   out: Optional[torch.Tensor] = None,
                   workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """varlen_prefill for drafted trees: each token of a sequence's chunk attends what is cached and
    those of the chunk's tokens whose bits its row of mask (tree_mask) has, itself among them.
    The chunk's K and V are in the cache already (kv_append, kv_append_fp8), token j of sequence i at
    position context_lens[i] + j, whatever position its rotary embedding stands for.

    q [T, H, D] in bfloat16 or float16; kv_cache a 16-bit pool of the same type, or an Fp8KVCache.
    mask int64 [T, words]: bit b % 64 of word b // 64 for token b of the sequence.  A token that
    attends nothing gets zeros.  max_seqlen bounds a sequence's tokens, max_context_len its cached
    ones (0: not known, the table's width then): sequences past these bounds are not attended
    whole."""
    if out is None and workspace is None and _lib.NATIVE is not None:
        pool, scales = kv_cache if isinstance(kv_cache, Fp8KVCache) else (kv_cache, None)
        out = _lib.NATIVE.tree_attention(q, pool, scales, block_table, cu_seqlens, context_lens,
                                         mask, max_seqlen, max_context_len, scale, num_heads,
                                         num_kv_heads, head_dim)
        if out is not None:
            return out
    pool = kv_cache.codes if isinstance(kv_cache, Fp8KVCache) else kv_cache
    _check_cache(pool) if pool is kv_cache else _check_fp8_cache(*kv_cache)
    dev = pool.device
    _, nb, hkv, bs, d = pool.shape
    _require(hkv == num_kv_heads and d == head_dim, "kv_cache shape disagrees with head counts")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"q must be bfloat16 or float16, got {q.dtype}")
    if pool is kv_cache:
        _require(q.dtype == pool.dtype, "q dtype must match kv_cache", TypeError)
    qs = _rows("q", q, num_heads, head_dim, dev)
    _check_group(num_heads, num_kv_heads)
    n_seqs, n_tok = _check_table(block_table, nb, dev), q.shape[0]
    _check_int32("cu_seqlens", cu_seqlens, 1, dev)
    _check_int32("context_lens", context_lens, 1, dev)
    _require(cu_seqlens.shape[0] == n_seqs + 1 and context_lens.shape[0] == n_seqs,
             "cu_seqlens / context_lens / block_table batch mismatch")
    if mask.dtype != torch.int64:
        raise TypeError(f"mask must be int64, got {mask.dtype}")
    if mask.dim() != 2 or mask.shape[0] != n_tok or mask.shape[1] < 1:
        raise ValueError(f"mask must be [{n_tok}, words], got {tuple(mask.shape)}")
    words = mask.shape[1]
    if mask.device != dev or (n_tok and words > 1 and mask.stride(1) != 1):
        raise ValueError(f"mask rows must be contiguous on {dev}")
    ms = mask.stride(0) if n_tok > 1 else words
    _require(ms >= words, "mask rows overlap")
    out = _check_out(out, n_tok, num_heads, head_dim, q)
    if n_tok == 0 or n_seqs == 0:
        return out
    w = block_table.shape[1]
    _require(w > 0, "block_table has no columns")
    max_seqlen, max_context_len = int(max_seqlen), int(max_context_len)
    _require(max_seqlen > 0, "max_seqlen must be positive")
    _require(max_context_len >= 0, "max_context_len is negative")
    max_keys = min(w * bs, max_context_len + max_seqlen) if max_context_len else w * bs
    lib = _lib.load()
    fp8 = pool is not kv_cache
    with _on(dev):
        need = tree_attention_workspace_bytes(n_seqs, max_seqlen, max_keys, num_heads,
                                              num_kv_heads, head_dim, bs, fp8)
        if need and (workspace is None or workspace.numel() * workspace.element_size() < need
                     or workspace.device != dev):
            workspace = decode_workspace(need, dev)
        tail = (nb, block_table.data_ptr(), block_table.stride(0), w, cu_seqlens.data_ptr(),
                context_lens.data_ptr(), mask.data_ptr(), ms, words, n_seqs, n_tok, max_seqlen,
                max_keys, num_heads, num_kv_heads, head_dim, bs, _DTYPES[q.dtype], float(scale),
                _ptr(workspace) if need else None, need, _stream(dev))
        if fp8:
            rc = lib.ndl_fp8_tree_attention(out.data_ptr(), q.data_ptr(), qs, pool.data_ptr(),
                                            kv_cache.scales.data_ptr(), *tail)
        else:
            rc = lib.ndl_tree_attention(out.data_ptr(), q.data_ptr(), qs, pool.data_ptr(), *tail)
    _lib.check(rc, "ndl_fp8_tree_attention" if fp8 else "ndl_tree_attention")
    return out


def verify_tree(logits: torch.Tensor, ids: torch.Tensor, parents: torch.Tensor,
                cu_seqlens: torch.Tensor, uniforms: torch.Tensor, *,
                temperature: Optional[torch.Tensor] = None):
    """verify_drafts for drafted trees: (tokens [T], accepted int32 [num_seqs], path int32 [T]).

    logits [T, vocab] (bfloat16, float16 or float32, rows contiguous, any row stride) are the
    target's rows for the nodes ids [T] (int32 or int64) of each sequence's tree, parents int32 [T]
    as for tree_mask; node 0 is the sequence's newest token.  From there, with
    p = softmax(logits[r] / temperature[i]) of the node r, the path goes on to the first of its
    children (in the order of their rows) whose token's p, added to those of the children before it,
    is more than uniforms[r]; a token that several children have counts once.  Where there is none,
    the next token is drawn from the node's p without its children's tokens, by the inverse of the
    cumulative distribution at the sequence's last uniform (its last node is a leaf): together
    distributed as the target.  A chain gives what verify_drafts gives without draft_probs.

    temperature float32 [num_seqs] (None: 1); 0 takes the argmax, as does a row whose maximum is
    not finite.  uniforms float32 [T] in [0, 1).  A sequence's rows past its 1,024th are no part of
    its tree.  tokens, in ids' type: the path's tokens after node 0, the next token, then -1;
    accepted: how many the path has; path: its nodes, 0 among them, then -1 (kv_compact moves their
    rows together).  Rows outside cu_seqlens hold nothing in particular.  Graph-capturable; no host
    synchronisation."""
    if _lib.NATIVE is not None:
        done = _lib.NATIVE.verify_tree(logits, ids, parents, cu_seqlens, uniforms, temperature)
        if done is not None:
            return done
    dev, rows, vocab, n_seqs = _check_verify(logits, ids, cu_seqlens, uniforms, temperature)
    _check_int32("parents", parents, 1, dev)
    _require(parents.shape[0] == rows, "logits and parents differ in rows")
    tokens, path = torch.empty_like(ids), torch.empty(rows, dtype=torch.int32, device=dev)
    accepted = torch.empty(n_seqs, dtype=torch.int32, device=dev)
    if n_seqs == 0:
        return tokens, accepted, path
    lib = _lib.load()
    need = lib.ndl_verify_tree_workspace_bytes(rows, n_seqs, vocab)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    with _on(dev):
        rc = lib.ndl_verify_tree(
            tokens.data_ptr(), accepted.data_ptr(), path.data_ptr(), logits.data_ptr(),
            logits.stride(0) if rows > 1 else vocab, _DTYPES[logits.dtype], ids.data_ptr(),
            int(ids.dtype == torch.int64), parents.data_ptr(), cu_seqlens.data_ptr(),
            uniforms.data_ptr(), _ptr(temperature), rows, n_seqs, vocab, ws.data_ptr(), need,
            _stream(dev))
    _lib.check(rc, "ndl_verify_tree")
    return tokens, accepted, path


# ---------------------------------------------------------------- caches that keep some rows

def kv_mass_pool(num_blocks: int, num_kv_heads: int, block_size: int,
                 device=None) -> torch.Tensor:
    """Weights of a pool's rows, float32 [num_blocks, num_kv_heads, block_size], zero: a number for
    each cached token and kv head, found through the block table as its K and V are."""
    return torch.zeros((num_blocks, num_kv_heads, block_size), dtype=torch.float32, device=device)


def _check_mass(mass, nb, hkv, bs, dev) -> None:
    if mass.dtype != torch.float32:
        raise TypeError(f"mass must be float32, got {mass.dtype}")
    if mass.shape != (nb, hkv, bs) or not mass.is_contiguous() or mass.device != dev:
        raise ValueError(f"mass must be a contiguous {[nb, hkv, bs]} tensor on {dev}, got "
                         f"{tuple(mass.shape)}")


def attention_mass_workspace_bytes(num_seqs: int, num_tokens: int, max_seqlen: int, max_keys: int,
                                   num_heads: int, num_kv_heads: int, head_dim: int,
                                   block_size: int = 16) -> int:
    """Bytes of the workspace attention_mass uses on the current GPU, max_keys at most the
    table's."""
    return int(_lib.load().ndl_attention_mass_workspace_bytes(
        num_seqs, num_tokens, max_seqlen, max_keys, num_heads, num_kv_heads, head_dim, block_size))


def attention_mass(q: torch.Tensor, kv_cache: torch.Tensor, block_table: torch.Tensor,
                   context_lens: torch.Tensor, mass: torch.Tensor, scale: float, num_heads: int,
                   num_kv_heads: int, head_dim: int, *, cu_seqlens: Optional[torch.Tensor] = None,
                   max_seqlen: int = 1, max_context_len: int = 0, decay: float = 1.0,
                   out: Optional[torch.Tensor] = None,
                   workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """paged_decode (cu_seqlens None: one token per sequence) or varlen_prefill, which also adds up
    the attention weights of every cached token and kv head, in mass (kv_mass_pool): a cached
    token's number becomes decay times what it was plus its weights in this call, summed over the
    call's tokens and the query heads of the kv head; a new token's (position context_lens[i] and
    on) becomes its weights alone.  kv_select picks the tokens that stay by them.

    q [T, H, D] in bfloat16 or float16, kv_cache a 16-bit pool of the same type in which the tokens'
    K and V are already (kv_append).  For the weights that a prompt's last tokens give, hand over
    their q alone, with context_lens the tokens before them.  max_seqlen bounds a sequence's tokens,
    max_context_len its cached ones (0: not known, the table's width then).  decay 0 forgets what
    was there.  No two sequences may attend one block.  workspace: as decode_workspace gives, of
    attention_mass_workspace_bytes, for one call at a time.  Up to 32 rows (max_seqlen times the group;
    a decode step) it holds their scores for every key of these bounds, 1 GiB at most (past that they
    are made again): give max_context_len where the table is much wider than what is cached."""
    if out is None and workspace is None and _lib.NATIVE is not None:
        out = _lib.NATIVE.attention_mass(q, kv_cache, block_table, cu_seqlens, context_lens, mass,
                                         max_seqlen, max_context_len, scale, num_heads,
                                         num_kv_heads, head_dim, decay)
        if out is not None:
            return out
    if isinstance(kv_cache, Fp8KVCache):
        raise TypeError("attention_mass reads a 16-bit pool, got an Fp8KVCache")
    _check_cache(kv_cache)
    dev = kv_cache.device
    _, nb, hkv, bs, d = kv_cache.shape
    _require(hkv == num_kv_heads and d == head_dim, "kv_cache shape disagrees with head counts")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"q must be bfloat16 or float16, got {q.dtype}")
    _require(q.dtype == kv_cache.dtype, "q dtype must match kv_cache", TypeError)
    qs = _rows("q", q, num_heads, head_dim, dev)
    _check_group(num_heads, num_kv_heads)
    _check_mass(mass, nb, hkv, bs, dev)
    n_seqs, n_tok = _check_table(block_table, nb, dev), q.shape[0]
    _check_int32("context_lens", context_lens, 1, dev)
    _require(context_lens.shape[0] == n_seqs, "context_lens/block_table batch mismatch")
    if cu_seqlens is None:
        _require(n_tok == n_seqs, "q / block_table batch mismatch")
        _require(max_seqlen == 1, "without cu_seqlens every sequence has one token")
    else:
        _check_int32("cu_seqlens", cu_seqlens, 1, dev)
        _require(cu_seqlens.shape[0] == n_seqs + 1, "cu_seqlens must be [num_seqs + 1]")
    out = _check_out(out, n_tok, num_heads, head_dim, q)
    if n_tok == 0 or n_seqs == 0:
        return out
    w = block_table.shape[1]
    _require(w > 0, "block_table has no columns")
    max_seqlen, max_context_len = int(max_seqlen), int(max_context_len)
    _require(max_seqlen > 0, "max_seqlen must be positive")
    _require(max_context_len >= 0, "max_context_len is negative")
    max_keys = min(w * bs, max_context_len + max_seqlen) if max_context_len else w * bs
    lib = _lib.load()
    with _on(dev):
        need = attention_mass_workspace_bytes(n_seqs, n_tok, max_seqlen, max_keys, num_heads,
                                              num_kv_heads, head_dim, bs)
        if workspace is None or workspace.numel() * workspace.element_size() < need \
                or workspace.device != dev:
            workspace = decode_workspace(need, dev)
        rc = lib.ndl_attention_mass(
            out.data_ptr(), mass.data_ptr(), q.data_ptr(), qs, kv_cache.data_ptr(), nb,
            block_table.data_ptr(), block_table.stride(0), w, _ptr(cu_seqlens),
            context_lens.data_ptr(), n_seqs, n_tok, max_seqlen, max_keys, num_heads, num_kv_heads,
            head_dim, bs, _DTYPES[q.dtype], float(scale), float(decay), workspace.data_ptr(), need,
            _stream(dev))
    _lib.check(rc, "ndl_attention_mass")
    return out


def kv_compact(pools, block_table: torch.Tensor, keep: torch.Tensor, counts: torch.Tensor, *,
               first: Optional[torch.Tensor] = None,
               cu_seqlens: Optional[torch.Tensor] = None,
               dst_table: Optional[torch.Tensor] = None,
               mass: Optional[torch.Tensor] = None) -> None:
    """Move the cached rows that stay together, in every layer's pool, both planes, in one launch:
    row first[i] + j of sequence i (first None: j) becomes what row first[i] + keep[j] was, for
    j < counts[i].

    pools: a list of [2, NB, Hkv, bs, D] tensors, or of Fp8KVCache, up to 128 of one shape and type,
    none twice.
    keep int32: [num_seqs, Hkv, K], a list for each kv head (kv_select's), or, with cu_seqlens
    (int32 [num_seqs + 1]), [T], packed, a list for all kv heads alike: verify_tree's path, with
    first the tokens cached before the tree and counts = accepted + 1.  counts, first int32
    [num_seqs].  mass (kv_mass_pool): weights that move with the rows.

    Without dst_table the rows move in place; a list has to ascend, with keep[j] >= j, and no block in
    which rows move may be another sequence's too (a shared prefix before `first` may).  With dst_table
    (int32 [num_seqs, columns]) they go to its blocks, none of which may hold rows that are read or
    belong to two sequences.  Negative entries, positions past a table and invalid block ids move nothing."""
    import ctypes
    pools = list(pools)
    _require(len(pools) > 0, "no pools given")
    fp8 = isinstance(pools[0], Fp8KVCache)
    if not fp8 and _lib.NATIVE is not None and _lib.NATIVE.kv_compact(
            pools, None, block_table, keep, counts, first, cu_seqlens, dst_table, mass):
        return
    _require(all(isinstance(p, Fp8KVCache) == fp8 for p in pools),
             "16-bit and 8-bit pools cannot be mixed", TypeError)
    main = [p.codes if fp8 else p for p in pools]
    if fp8 and _lib.NATIVE is not None and _lib.NATIVE.kv_compact(
            main, [p.scales for p in pools], block_table, keep, counts, first, cu_seqlens,
            dst_table, mass):
        return
    shape, dtype, dev = main[0].shape, main[0].dtype, main[0].device
    for p, x in zip(pools, main):
        _check_fp8_cache(*p) if fp8 else _check_cache(p)
        _require(x.shape == shape and x.device == dev, "pools must share one shape and GPU")
        _require(x.dtype == dtype or fp8, "pools must share one dtype", TypeError)
    _, nb, hkv, bs, d = shape
    row_bytes = d * main[0].element_size()
    _require(row_bytes % 16 == 0, f"rows of {row_bytes} bytes are not whole 16-byte pieces")
    _require(len(pools) <= 128, f"at most 128 pools a call, got {len(pools)}")
    _require(len({x.data_ptr() for x in main}) == len(main), "a pool is given twice")
    n_seqs = _check_table(block_table, nb, dev)
    _check_int32("counts", counts, 1, dev)
    _require(counts.shape[0] == n_seqs, "counts/block_table batch mismatch")
    if first is not None:
        _check_int32("first", first, 1, dev)
        _require(first.shape[0] == n_seqs, "first/block_table batch mismatch")
    if cu_seqlens is None:
        _check_int32("keep", keep, 3, dev)
        _require(tuple(keep.shape[:2]) == (n_seqs, hkv) and keep.is_contiguous(),
                 f"keep must be a contiguous [{n_seqs}, {hkv}, K] tensor (or packed by cu_seqlens)")
    else:
        _check_int32("keep", keep, 1, dev)
        _check_int32("cu_seqlens", cu_seqlens, 1, dev)
        _require(cu_seqlens.shape[0] == n_seqs + 1, "cu_seqlens must be [num_seqs + 1]")
    if dst_table is not None:
        _require(_check_table(dst_table, nb, dev) == n_seqs, "dst_table/block_table batch mismatch")
    if mass is not None:
        _check_mass(mass, nb, hkv, bs, dev)
    if n_seqs == 0 or keep.numel() == 0:
        return
    _require(block_table.shape[1] > 0 and (dst_table is None or dst_table.shape[1] > 0),
             "a block table has no columns")
    arr = ctypes.c_void_p * len(pools)
    dst = (None, 0, 0) if dst_table is None else (dst_table.data_ptr(), dst_table.stride(0),
                                                  dst_table.shape[1])
    with _on(dev):
        rc = _lib.load().ndl_kv_compact(
            arr(*[x.data_ptr() for x in main]),
            arr(*[p.scales.data_ptr() for p in pools]) if fp8 else None, len(pools), _ptr(mass),
            nb, hkv, bs, row_bytes, block_table.data_ptr(), block_table.stride(0),
            block_table.shape[1], *dst, keep.data_ptr(),
            keep.shape[2] if cu_seqlens is None else 0, _ptr(cu_seqlens), keep.numel(),
            _ptr(first), counts.data_ptr(), n_seqs, _stream(dev))
    _lib.check(rc, "ndl_kv_compact")


def kv_select(mass: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor, budget: int, *,
              sinks: int = 0, recent: int = 0):
    """The tokens of each kv head that stay when a cache is cut to `budget`: (keep int32
    [num_seqs, Hkv, budget], their positions, ascending, then -1; kept int32 [num_seqs] =
    min(lens, budget)), for kv_compact.

    mass (kv_mass_pool): the weights, as attention_mass adds them up; lens int32 [num_seqs]: the cached
    tokens.  Of a sequence of more than budget tokens the first `sinks` and the last `recent` stay
    (at most budget together), and of those between the ones with the largest weights, of equal ones
    the first.  A NaN counts as the largest weight."""
    if _lib.NATIVE is not None:
        done = _lib.NATIVE.kv_select(mass, block_table, lens, budget, sinks, recent)
        if done is not None:
            return done
    if mass.dim() != 3:
        raise ValueError(f"mass must be [num_blocks, num_kv_heads, block_size], got "
                         f"{tuple(mass.shape)}")
    _require(mass.is_cuda, "mass must be a GPU tensor")
    nb, hkv, bs = mass.shape
    dev = mass.device
    _check_mass(mass, nb, hkv, bs, dev)
    n_seqs = _check_table(block_table, nb, dev)
    _check_int32("lens", lens, 1, dev)
    _require(lens.shape[0] == n_seqs, "lens/block_table batch mismatch")
    budget, sinks, recent = int(budget), int(sinks), int(recent)
    _require(budget > 0, "budget must be positive")
    _require(sinks >= 0 and recent >= 0 and sinks + recent <= budget,
             f"sinks {sinks} and recent {recent} must be within the budget {budget}")
    keep = torch.empty((n_seqs, hkv, budget), dtype=torch.int32, device=dev)
    kept = torch.empty(n_seqs, dtype=torch.int32, device=dev)
    if n_seqs == 0:
        return keep, kept
    _require(block_table.shape[1] > 0, "block_table has no columns")
    with _on(dev):
        rc = _lib.load().ndl_kv_select(
            keep.data_ptr(), kept.data_ptr(), mass.data_ptr(), nb, hkv, bs, block_table.data_ptr(),
            block_table.stride(0), block_table.shape[1], lens.data_ptr(), n_seqs, budget, sinks,
            recent, _stream(dev))
    _lib.check(rc, "ndl_kv_select")
    return keep, kept
