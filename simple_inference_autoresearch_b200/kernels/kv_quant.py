"""The functions of ``ops`` for a cache entry held in 8 or 4 bits (``cache.QuantizedKVEntry``).

``ops.rope_kv_write``, ``ops.attention`` and ``ops.rope_and_attention`` come here when their cache entry is
such a one; ``ops.read_kv`` is the read-back.  The formats stand at the top of ``csrc/kv_quant.cu``.  A decode step over
a short cache is shorter than its own call, so arguments are looked at once and their pointers taken with that, and
what a call needs besides its result is one allocation.
"""

from __future__ import annotations

import array
import copy
from typing import Optional, Tuple

import torch

from . import ops
from .options import DEFAULT, KernelOptions


def is_quantized(kv) -> bool:
    return getattr(kv, "k_scale", None) is not None


def extension_units(needs, dtype: torch.dtype, page_tokens: int) -> Tuple[str, ...]:
    """The CUDA units that steps over a quantised cache of these needs (``parts.base.KVNeed``; others are passed over) launch
    from, besides those of the same model over a cache in the compute type."""
    needs = [n for n in needs if getattr(n, "n_kv_heads", None)]
    units = ("kv_quant",) if needs else ()
    if dtype == torch.bfloat16 and page_tokens % 64 == 0 and any(n.head_dim in (64, 128) and n.window is None for n in needs):
        units += ("attention_quant", "attention_quant_tc")
    return units


# ------------------------------------------------------------------ arguments
def check_entry(kv, n_kv_heads: int, head_dim: int, index: int) -> Tuple[int, ...]:
    """Raises ``ValueError`` unless the entry's tensors are what the kernels index: shapes, types, contiguity, all
    on GPU ``index`` (-1: the CPU).  Returns what every kernel takes of an entry first: pointers to codes, scales and
    block table."""
    if head_dim % 16 or not 0 < head_dim <= 256:
        raise ValueError(f"a quantised cache takes head_dim in steps of 16 up to 256, got {head_dim}")
    k, page = kv.k, int(kv.page_tokens)
    code = k.dtype
    rows = (k.shape[0], n_kv_heads, page)
    if code is torch.int8:
        want, scale, scale_dtype = rows + (head_dim,), rows, torch.float32
    elif code is torch.uint8:
        want, scale, scale_dtype = rows + (head_dim // 2,), rows + (-(-head_dim // 64), 2), torch.bfloat16
    else:
        raise ValueError(f"a quantised cache holds int8 (8 bits) or uint8 (4 bits), got {code}")
    pointers = []
    for name, t, shape, dtype in (("k", k, want, code), ("v", kv.v, want, code),
                                  ("k_scale", kv.k_scale, scale, scale_dtype), ("v_scale", kv.v_scale, scale, scale_dtype)):
        if t.shape != shape or t.dtype is not dtype:
            raise ValueError(f"{name} of a cache entry in {kv.bits} bits must be {dtype} of shape {shape}, "
                             f"got {t.dtype} {tuple(t.shape)}")
        at = t.data_ptr()
        if at % 16 or not t.is_contiguous():
            raise ValueError(f"{name} of a cache entry must be contiguous and 16-byte aligned")
        if t.get_device() != index:
            raise ValueError(f"{name} of the cache entry is on {t.device}, not where the call's other tensors are")
        pointers.append(at)
    table = kv.block_table
    if table.dtype is not torch.int32 or table.dim() != 2 or not table.is_contiguous():
        raise ValueError("block_table must be a contiguous int32 tensor [slots, pages per sequence]")
    if table.get_device() != index:
        raise ValueError(f"block_table is on {table.device}, not where the call's other tensors are")
    return (*pointers, table.data_ptr())


def check_rows(qkv: torch.Tensor, n_heads: int, n_kv_heads: int, head_dim: int, meta) -> None:
    if n_kv_heads <= 0 or n_heads % n_kv_heads:
        raise ValueError(f"num heads {n_heads} is not a multiple of kv heads {n_kv_heads}")
    if qkv.shape != (meta.n_tokens, (n_heads + 2 * n_kv_heads) * head_dim):
        raise ValueError(f"qkv must be [{meta.n_tokens}, {(n_heads + 2 * n_kv_heads) * head_dim}] for these heads, "
                         f"got {tuple(qkv.shape)}")
    if qkv.dtype is not torch.bfloat16 and qkv.dtype is not torch.float32:
        raise TypeError(f"compute dtype must be bfloat16 or float32, got {qkv.dtype}")
    if not qkv.is_contiguous() or qkv.data_ptr() % 16:
        raise ValueError("qkv must be contiguous and 16-byte aligned")


def check_batch_tensors(meta, index: int) -> Tuple[int, ...]:
    """Pointers to the batch's slot ids, row starts and lengths, which have to be int32 on GPU ``index``."""
    pointers = []
    for name, n in (("slot_ids", meta.n_seqs), ("q_start", meta.n_seqs + 1), ("base_len", meta.n_seqs)):
        t = getattr(meta, name)
        if t.dtype is not torch.int32 or not t.is_contiguous() or t.numel() < n or t.get_device() != index:
            raise ValueError(f"{name} must be a contiguous int32 tensor of {n} where the call's other tensors are, "
                             f"got {t.dtype} {tuple(t.shape)} on {t.device}")
        pointers.append(t.data_ptr())
    return tuple(pointers)


def check_rotary(rotary, head_dim: int, index: int):
    """``ops.rotary_layout``, with the frequencies where the call's other tensors are."""
    if isinstance(rotary, torch.Tensor) and rotary.dtype is torch.float32 and 2 * rotary.numel() == head_dim:
        inv_freq, rotary_dim, interleaved = rotary, head_dim, False       # the common one, without attribute look-ups that fail
    else:
        inv_freq, rotary_dim, interleaved = ops.rotary_layout(rotary, head_dim)
    if inv_freq is not None and (inv_freq.get_device() != index or not inv_freq.is_contiguous()):
        raise ValueError(f"inv_freq must be contiguous and where the call's other tensors are, got a tensor on {inv_freq.device}")
    return inv_freq, rotary_dim, interleaved


def check_window(window: Optional[int]) -> None:
    if window is not None and window <= 0:
        raise ValueError(f"an attention window must be positive, got {window}")


def _at(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _carve(device, *sizes: int):
    """One allocation for pieces of so many bytes: the tensor to keep while they are in use, and their pointers."""
    at, offsets = 0, []
    for n in sizes:
        offsets.append(at)
        at += -(-n // 256) * 256
    held = torch.empty(at, dtype=torch.uint8, device=device)
    first = held.data_ptr()
    return (held, *(first + o for o in offsets))


# ------------------------------------------------------------------ store and read back
def rope_kv_write(qkv: torch.Tensor, rotary, kv, meta, n_heads: int, n_kv_heads: int, head_dim: int,
                  write_kv: bool = True, options: KernelOptions = DEFAULT,
                  q_out: Optional[torch.Tensor] = None) -> None:
    index = qkv.get_device()
    inv_freq, rotary_dim, interleaved = check_rotary(rotary, head_dim, index)
    check_rows(qkv, n_heads, n_kv_heads, head_dim, meta)
    pools, batch = check_entry(kv, n_kv_heads, head_dim, index), check_batch_tensors(meta, index)
    if q_out is None:
        q_out = qkv
    elif q_out.shape != qkv.shape or q_out.dtype is not qkv.dtype or not q_out.is_contiguous() or q_out.get_device() != index:
        raise ValueError(f"q_out must be a contiguous tensor like qkv, {qkv.dtype} {tuple(qkv.shape)}")
    elif 0 < abs(q_out.data_ptr() - qkv.data_ptr()) < qkv.numel() * qkv.element_size():
        raise ValueError("q_out must be qkv itself or lie apart from it")
    ops._need_cuda(qkv)
    ops._check_if_asked(options, kv, meta, qkv.shape[0], write_kv)
    with ops._on_device(index):
        ops._launch_words("kv_quant", "siar_rope_quantize", int(qkv.dtype is torch.bfloat16), kv.bits, qkv.data_ptr(), q_out.data_ptr(),
                    _at(inv_freq), *pools, *batch, qkv.shape[0], meta.n_seqs, n_heads, n_kv_heads, head_dim,
                    kv.page_tokens, kv.block_table.shape[1], kv.k.shape[0], int(write_kv),
                    ops.status_word(qkv.device).data_ptr(), ops._stream(), rotary_dim, int(interleaved))


def _pages(kv, meta, page: int) -> int:
    """Pages of ``page`` positions that the batch's sequences hold together."""
    most = -(-min(meta.max_kv_len, kv.block_table.shape[1] * kv.page_tokens) // page)
    if meta.base_lens is None or meta.q_lens is None:        # lengths live on the device only: room for the longest everywhere
        return meta.n_seqs * most
    return sum([min(-(-(n + m) // page), most) for n, m in zip(meta.base_lens, meta.q_lens)])


def _read(kv, meta, dtype: torch.dtype, window: Optional[int], pools, batch, with_slots: bool = False):
    """(KVEntry of the batch's keys and values, the row of its block table per sequence)."""
    device, index = kv.k.device, kv.k.get_device()
    n_kv_heads, head_dim, page = kv.k.shape[1], kv.head_dim, int(kv.page_tokens)
    if meta.max_kv_len <= 0:
        raise ValueError(f"max_kv_len must be positive, got {meta.max_kv_len}")
    pages = _pages(kv, meta, page)
    k, v = torch.empty((2, pages, n_kv_heads, page, head_dim), dtype=dtype, device=device).unbind(0)
    table = torch.empty((meta.n_seqs, kv.block_table.shape[1]), dtype=torch.int32, device=device)
    slots = torch.empty(meta.n_seqs, dtype=torch.int32, device=device) if with_slots else None
    with ops._on_device(index):
        ops._launch_words("kv_quant", "siar_read_kv", int(dtype is torch.bfloat16), kv.bits, *pools, *batch, k.data_ptr(),
                    v.data_ptr(), table.data_ptr(), _at(slots), meta.n_seqs, n_kv_heads, head_dim, page,
                    kv.block_table.shape[1], kv.k.shape[0], pages, meta.max_kv_len, int(window or 0),
                    ops.status_word(device).data_ptr(), ops._stream())
    return ops.KVEntry(k, v, table, page), slots


def read_kv(kv, meta, dtype: torch.dtype, window: Optional[int] = None, options: KernelOptions = DEFAULT):
    if not is_quantized(kv):
        raise TypeError("read_kv reads a quantised cache entry back; this one holds its values as they are")
    check_window(window)
    ops._is_bf16(dtype)                     # raises for anything but bfloat16 and float32
    index = kv.k.get_device()
    pools, batch = check_entry(kv, kv.k.shape[1], kv.head_dim, index), check_batch_tensors(meta, index)
    ops._need_cuda(kv.k)
    ops._check_if_asked(options, kv, meta, meta.n_tokens, False, window)
    return _read(kv, meta, dtype, window, pools, batch)[0]


# ------------------------------------------------------------------ attention
#: query rows (new tokens x heads of a group) a sequence may bring to the kernel that works on the codes; a longer run
#: widens the cache once for the tensor-core kernel instead of walking the codes for every 16 rows.  Measured on B200,
#: codes against tiles in us, 32 heads on 8.  Four sequences of 4,000 held positions, 128 dims: 64 rows 33 and 41 (4 bits 41
#: and 43), 96 rows 50 and 43 (64 and 44), 256 rows 86 and 51; 64 dims: 64 rows 25 and 33 (4 bits 27 and 34), 128 rows 32 and 31
#: (35 and 32).  One sequence of 500: 64 rows 20 and 17 (4 bits 24 and 17; 64 dims 19 and 15), of 16,000 44 and 52 (52 and 52; 30
#: and 37)
MOST_ROWS = 64


def works_on_codes(kv, meta, dtype: torch.dtype, n_heads: int, n_kv_heads: int, head_dim: int, scale: float,
                   window: Optional[int] = None, options: KernelOptions = DEFAULT) -> bool:
    """True when attention over this entry runs on the codes themselves (bfloat16, head_dim 64 or 128, pages of
    a multiple of 64, no window): single tokens, short runs, and whatever ``works_on_tiles`` does not take."""
    if dtype != torch.bfloat16 or window is not None or head_dim not in (64, 128) or not options.use_mma_attention:
        return False
    if not _codes_can_be_addressed(kv, n_kv_heads):
        return False
    return meta.is_decode or meta.max_q_len * (n_heads // n_kv_heads) <= MOST_ROWS or not works_on_tiles(
        kv, dtype, n_heads, n_kv_heads, head_dim, scale, window, options)


def _codes_can_be_addressed(kv, n_kv_heads: int) -> bool:
    return kv.page_tokens % 64 == 0 and kv.k.shape[0] * n_kv_heads * kv.page_tokens < 1 << 31


def new_on_codes(kv, meta, n_heads: int, n_kv_heads: int) -> int:
    """In a batch that brings long runs: sequences of up to so many new tokens (0: none) are attended to on the codes all the
    same, each by its own length.  On tiles they would have their whole cache widened, several times the bytes of the codes,
    and take a block of 128 rows for a few.  A launch of its own costs 7 us (runs of several tokens: up to 20, at 16 rows a kv
    head), so it takes keys enough: a long sequence, whose tiles follow one another, or many, each of which costs the tiles about
    256 keys more.  Measured on B200 beside a chunk of 512, all on tiles against two launches (8 bits, 32 heads on 8, 128
    dims; us): one token on 100 keys 25 and 30, on 1,000 34 and 32, on 16,000 100 and 40; eight of them on 100 29 and 30, on 500
    37 and 35, on 4,000 110 and 45; 32 on 100 51 and 33; four new tokens on 2,000 46 and 43, eight times four on 500 37 and 43,
    on 1,000 46 and 46, 32 times four on 100 51 and 41.  64 dims and 4 bits cross at about the same lengths.  Where the batch's lengths are on the device only, nothing is known of them."""
    if meta.q_lens is None or meta.base_lens is None or not _codes_can_be_addressed(kv, n_kv_heads):
        return 0
    most = max(1, MOST_ROWS * n_kv_heads // n_heads)
    short = [(m, c + m) for c, m in zip(meta.base_lens, meta.q_lens) if 0 < m <= most]
    if not short:
        return 0
    worth = 1024 if max(short)[0] == 1 else 2048
    keys = [n for _, n in short]
    return most if max(keys) >= worth or sum(keys) + 256 * len(keys) >= 4 * worth else 0


_workspaces, _captured_workspaces = {}, {}


def _workspace(index: int, stream: int):
    """Pointers to the counters (zeros, which a launch uses and leaves zero) and the scratch of launches on
    one stream of GPU ``index``.  Launches of one stream follow one another and share them; a captured graph may be
    replayed beside anything, so every capture has its own, zeroed by the graph itself, for the launches that
    it holds on one stream.  It is the graph's memory, held here only as long as the capture may ask for it again: up to
    ``end_of_capture``, or the next capture or launch on the stream."""
    key = (index, stream)
    if not torch._C._cuda_isCurrentStreamCapturing():
        if _captured_workspaces:
            _captured_workspaces.pop(key, None)
        held = _workspaces.get(key)
        if held is None:
            held = _workspaces.setdefault(key, _new_workspace(index))      # (one of two threads' is kept)
        return held[:2]
    fn = ops._fn("attention_quant", "siar_capture_id")
    fn.restype = ops.c_ulonglong
    capture = fn(stream)
    held = _captured_workspaces.get(key)
    if held is None or held[-1] != capture:
        held = _captured_workspaces[key] = _new_workspace(index) + (capture,)
    return held[:2]


def end_of_capture() -> None:
    """As the last thing in a capture: its workspace on the current stream is not asked for again."""
    index = torch._C._cuda_getDevice()
    _captured_workspaces.pop((index, torch._C._cuda_getCurrentRawStream(index)), None)


def _new_workspace(index: int):
    sms = ops._sm_count(index)
    sizes = []
    for name in ("siar_attn_quant_counters", "siar_attn_quant_scratch_floats"):
        fn = ops._fn("attention_quant", name)
        fn.restype = ops.c_longlong
        sizes.append(fn(sms))
    counters = torch.zeros(sizes[0], dtype=torch.int32, device=f"cuda:{index}")
    scratch = torch.empty(sizes[1], dtype=torch.float32, device=f"cuda:{index}")
    return counters.data_ptr(), scratch.data_ptr(), counters, scratch


def _queries16(qkv, inv_freq, kv, meta, pools, batch, n_heads, n_kv_heads, head_dim, write_kv, q16: int, factor: int) -> None:
    """Rotates the queries into float16 rows with a factor each, and stores the new keys and values (``write_kv``)."""
    ops._launch_words("kv_quant", "siar_rope_quantize_q16", kv.bits, qkv.data_ptr(), q16, factor, _at(inv_freq), *pools, *batch,
                qkv.shape[0], meta.n_seqs, n_heads, n_kv_heads, head_dim, kv.page_tokens, kv.block_table.shape[1],
                kv.k.shape[0], int(write_kv), ops.status_word(qkv.device).data_ptr(), ops._stream())


def _launch_codes(out, qkv, q16: int, factor: int, inv_freq, kv, meta, pools, batch, n_heads, n_kv_heads, head_dim, scale, fused,
                  write_kv, most_new: int, max_q_len: int, max_kv_len: int) -> None:
    index, stream = qkv.get_device(), ops._stream()
    counters, scratch = _workspace(index, stream)
    ops._launch_words("attention_quant", "siar_attn_quant", kv.bits, qkv.data_ptr(), q16, factor, *pools, *batch,
                _at(inv_freq), out.data_ptr(), counters, scratch, meta.n_seqs, n_heads, n_kv_heads, head_dim,
                kv.page_tokens, kv.block_table.shape[1], kv.k.shape[0], max_q_len, max_kv_len, ops._sm_count(index), int(fused),
                int(bool(write_kv)), most_new, float(scale), ops.status_word(qkv.device).data_ptr(), stream)


def _on_codes(qkv, inv_freq, kv, meta, pools, batch, n_heads, n_kv_heads, head_dim, scale, fused, write_kv) -> torch.Tensor:
    """``fused``: one token a sequence, rotated (``inv_freq``) and stored (``write_kv``) by the attention kernel itself;
    else, where ``write_kv`` is not None, by a kernel in front."""
    device, index, n = qkv.device, qkv.get_device(), qkv.shape[0]
    with ops._on_device(index):
        held, q16, factor = None, 0, 0
        if not fused and write_kv is not None:
            held, q16, factor = _carve(device, n * n_heads * head_dim * 2, n * n_heads * 4)
            _queries16(qkv, inv_freq, kv, meta, pools, batch, n_heads, n_kv_heads, head_dim, write_kv, q16, factor)
        out = torch.empty((n, n_heads * head_dim), dtype=torch.bfloat16, device=device)
        _launch_codes(out, qkv, q16, factor, inv_freq, kv, meta, pools, batch, n_heads, n_kv_heads, head_dim, scale, fused, write_kv,
                      0x7fffffff, meta.max_q_len, meta.max_kv_len)
    return out


def works_on_tiles(kv, dtype: torch.dtype, n_heads: int, n_kv_heads: int, head_dim: int, scale: float,
                   window: Optional[int] = None, options: KernelOptions = DEFAULT) -> bool:
    """True when prompts' attention over this entry runs on float16 tiles on the tensor cores (bfloat16, head_dim 64
    or 128, at most 128 query heads per kv head, pages of a multiple of 64, no window, a positive scale)."""
    return (dtype == torch.bfloat16 and window is None and head_dim in (64, 128) and n_heads // n_kv_heads <= 128
            and kv.page_tokens % 64 == 0 and scale > 0 and options.use_tc_attention and options.use_mma_attention)


def key_parts(blocks: int, longest: int, average: float, row_floats: int, sms: int) -> int:
    """Into how many parts the keys of a block of 128 rows are cut (the rule stands at ``siar_attn_quant_tc_parts``)."""
    return ops._fn("attention_quant_tc", "siar_attn_quant_tc_parts")(blocks, longest, average, row_floats, sms)


def tiles_of(kv, meta, passed_new: int):
    """(new tokens, key tiles of 64) of every sequence that is attended to on tiles, (0, 0) of the others: those of no more than
    ``passed_new`` new tokens."""
    most = -(-min(meta.max_kv_len, kv.block_table.shape[1] * kv.page_tokens) // 64)
    if meta.base_lens is None or meta.q_lens is None:        # lengths live on the device only: room for the longest everywhere
        return [(meta.max_q_len, most)] * meta.n_seqs
    return [(m, min(-(-(n + m) // 64), most)) if m > passed_new else (0, 0) for n, m in zip(meta.base_lens, meta.q_lens)]


#: bytes of float16 tiles that one launch may take, where it has more than one sequence: a batch's tiles are several times its
#: codes, and only those of a launch are held at a time.  One sequence of 131,072 keys of 8 heads of 128 dims takes half of it.
MOST_TILE_BYTES = 1 << 30


def runs_of_tiles(lengths, most_seqs: int, tile_bytes: int):
    """The places of the sequences that have tiles (of ``tile_bytes`` each, keys and values), launch by launch: at most
    ``most_seqs`` of them and MOST_TILE_BYTES, but one at least; about as much in each launch."""
    bytes_of = [(i, t * tile_bytes) for i, (_, t) in enumerate(lengths) if t > 0]
    total = sum([n for _, n in bytes_of])
    share = total / max(1, -(-total // MOST_TILE_BYTES), -(-len(bytes_of) // most_seqs))
    runs, held = [], 0
    for i, n in bytes_of:
        if not runs or len(runs[-1]) == most_seqs or held >= share or held + n > MOST_TILE_BYTES:
            runs.append([])
            held = 0
        runs[-1].append(i)
        held += n
    return runs


def _on_tiles(qkv, inv_freq, kv, meta, pools, batch, n_heads, n_kv_heads, head_dim, scale, write_kv) -> torch.Tensor:
    """Rotates (``inv_freq``) and stores (``write_kv``) the new tokens, widens the cache of the sequences that bring long runs to
    float16 tiles and attends on those; the others (``new_on_codes``) work on the codes."""
    device, index, n, heads = qkv.device, qkv.get_device(), qkv.shape[0], (n_heads, n_kv_heads, head_dim)
    group = n_heads // n_kv_heads
    block_rows = 128 // group * group
    passed = new_on_codes(kv, meta, n_heads, n_kv_heads)
    lengths = tiles_of(kv, meta, passed)
    fn = ops._fn("attention_quant_tc", "siar_attn_quant_tc_most_seqs")
    launches, info_bytes = [], ops._fn("attention_quant_tc", "siar_attn_quant_tc_tile_info_bytes")()
    for ids in runs_of_tiles(lengths, fn(), 2 * n_kv_heads * 64 * head_dim * 2):
        tiles, blocks = [lengths[i][1] for i in ids], [-(-lengths[i][0] * group // block_rows) for i in ids]
        average = sum([w * (t - lengths[i][0] / 128) for i, w, t in zip(ids, blocks, tiles)]) / sum(blocks)     # key tiles a block
        splits = key_parts(n_kv_heads * sum(blocks), max(tiles), average, n * n_heads * (head_dim + 8), ops._sm_count(index))
        launches.append((array.array("i", ids), sum(tiles), max(tiles), max([lengths[i][0] for i in ids]), splits))
    if not launches:
        raise ValueError("q_lens, max_q_len and max_kv_len of the batch do not agree")
    tiles, splits = max([t for _, t, _, _, _ in launches]), max([s for *_, s in launches])
    row_bytes, tile_bytes = n * n_heads * 4, tiles * n_kv_heads * 64 * head_dim * 2
    with ops._on_device(index):
        stream, status = ops._stream(), ops.status_word(device).data_ptr()
        out = torch.empty((n, n_heads * head_dim), dtype=torch.bfloat16, device=device)
        held, q16, factor, k16, v16, info, seq, scratch = _carve(
            device, row_bytes // 2 * head_dim, row_bytes, tile_bytes, tile_bytes, tiles * n_kv_heads * info_bytes,
            max([len(ids) for ids, *_ in launches]) * 8, row_bytes * splits * (head_dim + 8) if splits > 1 else 0)
        _queries16(qkv, inv_freq, kv, meta, pools, batch, *heads, write_kv, q16, factor)
        if passed:
            short = [(m, c + m) for c, m in zip(meta.base_lens, meta.q_lens) if 0 < m <= passed]
            _launch_codes(out, qkv, q16, factor, None, kv, meta, pools, batch, *heads, scale, False, False, passed,
                          max([m for m, _ in short]), max([c for _, c in short]))
        for ids, tiles, most, most_new, splits in launches:
            which = (ids.buffer_info()[0], len(ids))
            ops._launch_words("attention_quant_tc", "siar_widen_tiles", kv.bits, *pools, *batch, k16, v16, info, seq, *which,
                        meta.n_seqs, n_kv_heads, head_dim, kv.page_tokens, kv.block_table.shape[1], kv.k.shape[0], tiles, most * 64,
                        status, stream)
            ops._launch_words("attention_quant_tc", "siar_attn_quant_tc", q16, factor, k16, v16, info, seq, batch[1], batch[2],
                        out.data_ptr(), scratch, *which, n, meta.n_seqs, *heads, tiles, most_new, splits, float(scale), status,
                        stream, kernels=2 if splits > 1 else 1)
    return out


def attention(qkv: torch.Tensor, kv, meta, n_heads: int, n_kv_heads: int, head_dim: int, scale: float,
              window: Optional[int] = None, options: KernelOptions = DEFAULT) -> torch.Tensor:
    check_window(window)
    check_rows(qkv, n_heads, n_kv_heads, head_dim, meta)
    index, heads = qkv.get_device(), (n_heads, n_kv_heads, head_dim)
    pools, batch = check_entry(kv, n_kv_heads, head_dim, index), check_batch_tensors(meta, index)
    ops._need_cuda(qkv)
    ops._check_if_asked(options, kv, meta, qkv.shape[0], False, window)
    if works_on_codes(kv, meta, qkv.dtype, *heads, scale, window, options):
        return _on_codes(qkv, None, kv, meta, pools, batch, *heads, scale, False, None)
    if not meta.is_decode and works_on_tiles(kv, qkv.dtype, *heads, scale, window, options):
        return _on_tiles(qkv, None, kv, meta, pools, batch, *heads, scale, False)
    pages, slots = _read(kv, meta, qkv.dtype, window, pools, batch, with_slots=True)
    of_batch = copy.copy(meta)
    of_batch.slot_ids = slots
    if meta.is_decode and not ops._fn("attention", "siar_attn_decode_fits")(ops._is_bf16(qkv.dtype), *heads):
        of_batch.is_decode = False          # one row a sequence on the prompt kernel
    with ops._on_device(index):
        return ops.attention(qkv, pages, of_batch, *heads, scale, window=window,
                             options=options.but(check_arguments=False) if options.check_arguments else options)


def rope_and_attention(qkv: torch.Tensor, rotary, kv, meta, n_heads: int, n_kv_heads: int, head_dim: int, scale: float,
                       write_kv: bool = True, window: Optional[int] = None,
                       options: KernelOptions = DEFAULT) -> torch.Tensor:
    check_window(window)
    check_rows(qkv, n_heads, n_kv_heads, head_dim, meta)
    index, heads = qkv.get_device(), (n_heads, n_kv_heads, head_dim)
    inv_freq, rotary_dim, interleaved = check_rotary(rotary, head_dim, index)
    if inv_freq is None or (rotary_dim == head_dim and not interleaved):      # paths that rotate and store as well
        codes = works_on_codes(kv, meta, qkv.dtype, *heads, scale, window, options)
        if codes or (not meta.is_decode and works_on_tiles(kv, qkv.dtype, *heads, scale, window, options)):
            pools, batch = check_entry(kv, n_kv_heads, head_dim, index), check_batch_tensors(meta, index)
            ops._need_cuda(qkv)
            ops._check_if_asked(options, kv, meta, qkv.shape[0], write_kv)
            if codes:
                return _on_codes(qkv, inv_freq, kv, meta, pools, batch, *heads, scale,
                                 meta.is_decode and options.fuse_decode_rope, write_kv)
            return _on_tiles(qkv, inv_freq, kv, meta, pools, batch, *heads, scale, write_kv)
    q = torch.empty_like(qkv)               # the rotated queries; qkv stays as it is
    rope_kv_write(qkv, rotary, kv, meta, *heads, write_kv=write_kv, options=options, q_out=q)
    return attention(q, kv, meta, *heads, scale, window=window, options=options)
