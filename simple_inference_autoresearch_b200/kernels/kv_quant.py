"""The functions of ``ops`` for a cache entry held in 8 or 4 bits (``cache.QuantizedKVEntry``).

``ops.rope_kv_write``, ``ops.attention`` and ``ops.rope_and_attention`` come here when their cache entry is
such a one; ``ops.read_kv`` is the read-back.  The formats stand at the top of ``csrc/kv_quant.cu``.
"""

from __future__ import annotations

import copy
from typing import Optional

import torch

from . import ops
from .options import DEFAULT, KernelOptions


def is_quantized(kv) -> bool:
    return getattr(kv, "k_scale", None) is not None


def check_entry(kv, n_kv_heads: int, head_dim: int, device) -> None:
    """Raises ``ValueError`` unless the entry's tensors are what the kernels index: shapes, types,
    contiguity, one device."""
    if head_dim % 16 or not 0 < head_dim <= 256:
        raise ValueError(f"a quantised cache takes head_dim in steps of 16 up to 256, got {head_dim}")
    page, pages = int(kv.page_tokens), kv.k.shape[0]
    if kv.k.dtype == torch.int8:
        want, scale_dtype, scale = (pages, n_kv_heads, page, head_dim), torch.float32, (pages, n_kv_heads, page)
    elif kv.k.dtype == torch.uint8:
        want, scale_dtype = (pages, n_kv_heads, page, head_dim // 2), torch.bfloat16
        scale = (pages, n_kv_heads, page, -(-head_dim // 64), 2)
    else:
        raise ValueError(f"a quantised cache holds int8 (8 bits) or uint8 (4 bits), got {kv.k.dtype}")
    for name, t, shape, dtype in (("k", kv.k, want, kv.k.dtype), ("v", kv.v, want, kv.k.dtype),
                                  ("k_scale", kv.k_scale, scale, scale_dtype), ("v_scale", kv.v_scale, scale, scale_dtype)):
        if t.shape != shape or t.dtype != dtype:
            raise ValueError(f"{name} of a cache entry in {kv.bits} bits must be {dtype} of shape {shape}, "
                             f"got {t.dtype} {tuple(t.shape)}")
        if not t.is_contiguous() or t.data_ptr() % 16:
            raise ValueError(f"{name} of a cache entry must be contiguous and 16-byte aligned")
        if t.device != device:
            raise ValueError(f"{name} of the cache entry is on {t.device}, the activations are on {device}")
    if kv.block_table.dtype != torch.int32 or kv.block_table.dim() != 2 or not kv.block_table.is_contiguous():
        raise ValueError("block_table must be a contiguous int32 tensor [slots, pages per sequence]")
    if kv.block_table.device != device:
        raise ValueError(f"block_table is on {kv.block_table.device}, the activations are on {device}")


def check_rows(qkv: torch.Tensor, n_heads: int, n_kv_heads: int, head_dim: int, meta) -> None:
    if n_kv_heads <= 0 or n_heads % n_kv_heads:
        raise ValueError(f"num heads {n_heads} is not a multiple of kv heads {n_kv_heads}")
    if qkv.shape != (meta.n_tokens, (n_heads + 2 * n_kv_heads) * head_dim):
        raise ValueError(f"qkv must be [{meta.n_tokens}, {(n_heads + 2 * n_kv_heads) * head_dim}] for these heads, "
                         f"got {tuple(qkv.shape)}")
    if qkv.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"compute dtype must be bfloat16 or float32, got {qkv.dtype}")
    if not qkv.is_contiguous() or qkv.data_ptr() % 16:
        raise ValueError("qkv must be contiguous and 16-byte aligned")


def check_window(window: Optional[int]) -> None:
    if window is not None and window <= 0:
        raise ValueError(f"an attention window must be positive, got {window}")


def _batch(meta):
    return ops._ptr(meta.slot_ids), ops._ptr(meta.q_start), ops._ptr(meta.base_len)


def rope_kv_write(qkv: torch.Tensor, rotary, kv, meta, n_heads: int, n_kv_heads: int, head_dim: int,
                  write_kv: bool = True, options: KernelOptions = DEFAULT,
                  q_out: Optional[torch.Tensor] = None) -> None:
    inv_freq, rotary_dim, interleaved = ops.rotary_layout(rotary, head_dim)
    check_rows(qkv, n_heads, n_kv_heads, head_dim, meta)
    check_entry(kv, n_kv_heads, head_dim, qkv.device)
    if q_out is None:
        q_out = qkv
    elif q_out.shape != qkv.shape or q_out.dtype != qkv.dtype or not q_out.is_contiguous() or q_out.device != qkv.device:
        raise ValueError(f"q_out must be a contiguous tensor like qkv, {qkv.dtype} {tuple(qkv.shape)}")
    ops._need_cuda(qkv, inv_freq, kv.k)
    ops._check_if_asked(options, kv, meta, qkv.shape[0], write_kv)
    with ops._on_device(qkv):
        ops._launch("kv_quant", "siar_rope_quantize", ops._is_bf16(qkv.dtype), kv.bits, ops._ptr(qkv), ops._ptr(q_out),
                    ops._ptr(inv_freq), ops._ptr(kv.k), ops._ptr(kv.v), ops._ptr(kv.k_scale), ops._ptr(kv.v_scale),
                    ops._ptr(kv.block_table), *_batch(meta), qkv.shape[0], meta.n_seqs, n_heads, n_kv_heads, head_dim,
                    kv.page_tokens, kv.block_table.shape[1], kv.k.shape[0], int(write_kv),
                    ops._ptr(ops.status_word(qkv.device)), ops._stream(), rotary_dim, int(interleaved))


def _read(kv, meta, dtype: torch.dtype, window: Optional[int]):
    """(KVEntry of the batch's keys and values, the batch's row of its block table per sequence)."""
    from ..cache.sequence_cache import KVEntry

    device = kv.k.device
    n_kv_heads, head_dim, page = kv.k.shape[1], kv.head_dim, int(kv.page_tokens)
    if meta.max_kv_len <= 0:
        raise ValueError(f"max_kv_len must be positive, got {meta.max_kv_len}")
    most = min(-(-meta.max_kv_len // page), kv.block_table.shape[1])
    if meta.base_lens is not None and meta.q_lens is not None:
        pages = sum(min(-(-(n + m) // page), most) for n, m in zip(meta.base_lens, meta.q_lens))
    else:                                   # lengths live on the device only: room for the longest everywhere
        pages = meta.n_seqs * most
    k = torch.empty((pages, n_kv_heads, page, head_dim), dtype=dtype, device=device)
    v = torch.empty_like(k)
    ints = torch.empty((meta.n_seqs, kv.block_table.shape[1] + 1), dtype=torch.int32, device=device).view(-1)
    cells = meta.n_seqs * kv.block_table.shape[1]
    table, slots = ints[:cells].view(meta.n_seqs, -1), ints[cells:]
    with ops._on_device(kv.k):
        ops._launch("kv_quant", "siar_read_kv", ops._is_bf16(dtype), kv.bits, ops._ptr(kv.k), ops._ptr(kv.v),
                    ops._ptr(kv.k_scale), ops._ptr(kv.v_scale), ops._ptr(kv.block_table), *_batch(meta), ops._ptr(k),
                    ops._ptr(v), ops._ptr(table), ops._ptr(slots), meta.n_seqs, n_kv_heads, head_dim, page,
                    kv.block_table.shape[1], kv.k.shape[0], pages, meta.max_kv_len, int(window or 0),
                    ops._ptr(ops.status_word(device)), ops._stream())
    return KVEntry(k, v, table, page), slots


def read_kv(kv, meta, dtype: torch.dtype, window: Optional[int] = None, options: KernelOptions = DEFAULT):
    if not is_quantized(kv):
        raise TypeError("read_kv reads a quantised cache entry back; this one holds its values as they are")
    check_window(window)
    ops._is_bf16(dtype)                     # raises for anything but bfloat16 and float32
    check_entry(kv, kv.k.shape[1], kv.head_dim, kv.k.device)
    ops._need_cuda(kv.k)
    ops._check_if_asked(options, kv, meta, meta.n_tokens, False, window)
    return _read(kv, meta, dtype, window)[0]


#: query rows (new tokens x heads of a group) a sequence may bring to the kernel that works on the codes; a
#: longer run reads the cache back once for the prompt kernel instead of walking the codes for every 16 rows
MOST_ROWS = 64


def works_on_codes(kv, meta, dtype: torch.dtype, n_heads: int, n_kv_heads: int, head_dim: int,
                   window: Optional[int] = None, options: KernelOptions = DEFAULT) -> bool:
    """True when attention over this entry runs on the codes themselves (bfloat16, head_dim 64 or 128, pages of
    a multiple of 64, no window, single tokens or short runs); else the cache is read back first."""
    if dtype != torch.bfloat16 or window is not None or head_dim not in (64, 128) or not options.use_mma_attention:
        return False
    if not meta.is_decode and meta.max_q_len * (n_heads // n_kv_heads) > MOST_ROWS:
        return False
    return bool(ops._fn("attention_quant", "siar_attn_quant_supported")(n_heads, n_kv_heads, head_dim, kv.page_tokens,
                                                                        kv.k.shape[0]))


_eager_counters, _captured_counters = {}, {}


def _zeroed_counters(n: int, device, stream: int) -> torch.Tensor:
    """``n`` int32 zeros that a launch uses and leaves zero.  Launches of one stream follow one another and
    share them; a captured graph may be replayed beside anything, so every capture has its own, zeroed by
    the graph itself, shared by the launches that it holds on one stream."""
    fn = ops._fn("attention_quant", "siar_capture_id")
    fn.restype = ops.c_ulonglong
    capture = fn(stream)
    key = (device.index, stream)
    if capture:
        held = _captured_counters.get(key)
        if held is None or held[0] != capture or held[1].numel() < n:
            held = _captured_counters[key] = (capture, torch.zeros(n, dtype=torch.int32, device=device))
        return held[1]
    t = _eager_counters.get(key)
    if t is None or t.numel() < n:
        t = _eager_counters[key] = torch.zeros(n, dtype=torch.int32, device=device)
    return t


def _on_codes(qkv, inv_freq, kv, meta, n_heads, n_kv_heads, head_dim, scale, fused, write_kv) -> torch.Tensor:
    device = qkv.device
    out = torch.empty((qkv.shape[0], n_heads * head_dim), dtype=qkv.dtype, device=device)
    with ops._on_device(qkv):
        blocks = ops._fn("attention_quant", "siar_attn_quant_blocks")(
            kv.bits, meta.n_seqs, n_heads, n_kv_heads, head_dim, meta.max_q_len, meta.max_kv_len, ops._sm_count(device))
        fn = ops._fn("attention_quant", "siar_attn_quant_scratch_floats")
        fn.restype = ops.c_longlong
        scratch = torch.empty(fn(n_heads, n_kv_heads, head_dim, meta.max_q_len, blocks), dtype=torch.float32, device=device)
        stream = ops._stream()
        counters = _zeroed_counters(blocks, device, stream)
        ops._launch("attention_quant", "siar_attn_quant", kv.bits, ops._ptr(qkv), ops._ptr(kv.k), ops._ptr(kv.v),
                    ops._ptr(kv.k_scale), ops._ptr(kv.v_scale), ops._ptr(kv.block_table), *_batch(meta), ops._ptr(inv_freq),
                    ops._ptr(out), ops._ptr(scratch), ops._ptr(counters), blocks, meta.n_seqs, n_heads, n_kv_heads, head_dim,
                    kv.page_tokens, kv.block_table.shape[1], kv.k.shape[0], meta.max_q_len, int(fused), int(write_kv),
                    float(scale), ops._ptr(ops.status_word(device)), stream)
    return out


def attention(qkv: torch.Tensor, kv, meta, n_heads: int, n_kv_heads: int, head_dim: int, scale: float,
              window: Optional[int] = None, options: KernelOptions = DEFAULT) -> torch.Tensor:
    check_window(window)
    check_rows(qkv, n_heads, n_kv_heads, head_dim, meta)
    check_entry(kv, n_kv_heads, head_dim, qkv.device)
    ops._need_cuda(qkv)
    ops._check_if_asked(options, kv, meta, qkv.shape[0], False, window)
    if works_on_codes(kv, meta, qkv.dtype, n_heads, n_kv_heads, head_dim, window, options):
        return _on_codes(qkv, None, kv, meta, n_heads, n_kv_heads, head_dim, scale, False, False)
    pages, slots = _read(kv, meta, qkv.dtype, window)
    of_batch = copy.copy(meta)
    of_batch.slot_ids = slots
    if meta.is_decode and not ops._fn("attention", "siar_attn_decode_fits")(
            ops._is_bf16(qkv.dtype), n_heads, n_kv_heads, head_dim):
        of_batch.is_decode = False          # one row a sequence on the prompt kernel
    return ops.attention(qkv, pages, of_batch, n_heads, n_kv_heads, head_dim, scale, window=window,
                         options=options.but(check_arguments=False) if options.check_arguments else options)


def rope_and_attention(qkv: torch.Tensor, rotary, kv, meta, n_heads: int, n_kv_heads: int, head_dim: int, scale: float,
                       write_kv: bool = True, window: Optional[int] = None,
                       options: KernelOptions = DEFAULT) -> torch.Tensor:
    check_window(window)
    inv_freq, rotary_dim, interleaved = ops.rotary_layout(rotary, head_dim)
    plain_layout = inv_freq is None or (rotary_dim == head_dim and not interleaved)
    if meta.is_decode and plain_layout and options.fuse_decode_rope and works_on_codes(
            kv, meta, qkv.dtype, n_heads, n_kv_heads, head_dim, window, options):
        check_rows(qkv, n_heads, n_kv_heads, head_dim, meta)
        check_entry(kv, n_kv_heads, head_dim, qkv.device)
        ops._need_cuda(qkv, inv_freq)
        ops._check_if_asked(options, kv, meta, qkv.shape[0], write_kv)
        return _on_codes(qkv, inv_freq, kv, meta, n_heads, n_kv_heads, head_dim, scale, True, write_kv)
    q = torch.empty_like(qkv)               # the rotated queries; qkv stays as it is
    rope_kv_write(qkv, rotary, kv, meta, n_heads, n_kv_heads, head_dim, write_kv=write_kv, options=options, q_out=q)
    return attention(q, kv, meta, n_heads, n_kv_heads, head_dim, scale, window=window, options=options)
