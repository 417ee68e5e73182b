"""Plain torch restatements of the functions that work on a cache held in 8 or 4 bits
(``kernels/kv_quant.py``), for the same two uses as ``emulated_kernels.py``: the GPU tests compare with
them, and the CPU tests of the engine's logic swap them in.

The rotation, the scales and the codes are formed in float32 from 64-bit angles, operation by
operation as the kernels state them, so that codes and scales can be compared for equality."""

from __future__ import annotations

import math

import torch

from simple_inference_autoresearch_b200.cache import KVEntry
from tests import emulated_kernels as emu

GROUP = 64


def quantise(x, bits):
    """float32 [..., D] -> (codes, scales) as the cache holds them."""
    finite = torch.isfinite(x)
    if bits == 8:
        s = x.abs().amax(-1) * (1 / 127)                  # the float32 reciprocal, as the kernels
        c = torch.round(x / torch.where(s > 0, s, 1.0)[..., None]).clamp(-127, 127)
        bad = ~finite.all(-1)
        c = torch.where(bad[..., None] | (s <= 0)[..., None], torch.zeros_like(c), c)
        return c.to(torch.int8), torch.where(bad, float("nan"), s)
    codes, scales = [], []
    for at in range(0, x.shape[-1], GROUP):
        g = x[..., at:at + GROUP]
        lo, hi = g.amin(-1), g.amax(-1)
        s = (hi * (1 / 15) - lo * (1 / 15)).to(torch.bfloat16).float()
        m = (lo + 8.0 * s).to(torch.bfloat16).float()
        c = (torch.round((g - m[..., None]) / torch.where(s > 0, s, 1.0)[..., None]) + 8.0).clamp(0, 15)
        bad = ~finite[..., at:at + GROUP].all(-1)
        c = torch.where(bad[..., None] | ~(s > 0)[..., None], torch.full_like(c, 8.0), c)
        codes.append(c)
        nan = torch.tensor(float("nan"))
        scales.append(torch.stack((torch.where(bad, nan, s), torch.where(bad, nan, m)), -1))
    c = torch.cat(codes, -1).to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4), torch.stack(scales, -2).to(torch.bfloat16)


def values(codes, scales, dtype=torch.float64):
    """What codes and scales stand for, [..., D]."""
    if codes.dtype == torch.int8:
        return codes.to(dtype) * scales.to(dtype)[..., None]
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).to(dtype) - 8
    out = torch.empty_like(c)
    for i, at in enumerate(range(0, c.shape[-1], GROUP)):
        out[..., at:at + GROUP] = c[..., at:at + GROUP] * scales[..., i, :1].to(dtype) + scales[..., i, 1:].to(dtype)
    return out


def rotate(x, positions, rotary):
    """x float32 [T, heads, D] rotated by 64-bit angles rounded to a float32 cosine and sine."""
    inv_freq = getattr(rotary, "inv_freq", rotary)
    dim = int(getattr(rotary, "rotary_dim", None) or 2 * inv_freq.numel())
    ang = torch.outer(torch.as_tensor(positions, dtype=torch.float64), inv_freq.cpu().double())
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]
    out = x.clone()
    ia, ib = (slice(0, dim, 2), slice(1, dim, 2)) if getattr(rotary, "interleaved", False) else (
        slice(0, dim // 2), slice(dim // 2, dim))
    a, c = x[..., ia], x[..., ib]
    out[..., ia] = a * cos - c * sin
    out[..., ib] = c * cos + a * sin
    return out


def is_quantized(kv):
    return getattr(kv, "k_scale", None) is not None


def rope_kv_write(qkv, rotary, kv, meta, n_heads, n_kv_heads, head_dim, write_kv=True, options=None, q_out=None):
    if not is_quantized(kv):
        return emu.rope_kv_write(qkv, rotary, kv, meta, n_heads, n_kv_heads, head_dim, write_kv=write_kv)
    pos, seq = emu._positions(meta)
    n = qkv.shape[0]
    x = qkv.view(n, n_heads + 2 * n_kv_heads, head_dim).float()
    qk, v = x[:, :n_heads + n_kv_heads], x[:, n_heads + n_kv_heads:]
    if rotary is not None:
        qk = rotate(qk, pos, rotary)
    (qkv if q_out is None else q_out).view(n, -1, head_dim)[:, :n_heads] = qk[:, :n_heads].to(qkv.dtype)
    if not write_kv:
        return
    slots = meta.slot_ids.tolist()
    for pool, scale, rows in ((kv.k, kv.k_scale, qk[:, n_heads:]), (kv.v, kv.v_scale, v)):
        codes, scales = quantise(rows, kv.bits)
        for t in range(n):
            page = int(kv.block_table[slots[seq[t]], pos[t] // kv.page_tokens])
            if page < 0:
                raise RuntimeError("a kernel reported: a cache write met a position without a page")
            pool[page, :, pos[t] % kv.page_tokens] = codes[t]
            scale[page, :, pos[t] % kv.page_tokens] = scales[t]


def whole(kv, dtype):
    """The entry with every row replaced by its values."""
    return KVEntry(values(kv.k, kv.k_scale).to(dtype), values(kv.v, kv.v_scale).to(dtype), kv.block_table, kv.page_tokens)


def attention(qkv, kv, meta, n_heads, n_kv_heads, head_dim, scale, window=None, options=None):
    if is_quantized(kv):
        kv = whole(kv, torch.float32)
    return emu.attention(qkv, kv, meta, n_heads, n_kv_heads, head_dim, scale, window=window)


def rope_and_attention(qkv, rotary, kv, meta, n_heads, n_kv_heads, head_dim, scale, write_kv=True, window=None,
                       options=None):
    rope_kv_write(qkv, rotary, kv, meta, n_heads, n_kv_heads, head_dim, write_kv=write_kv)
    return attention(qkv, kv, meta, n_heads, n_kv_heads, head_dim, scale, window=window)


def install(monkeypatch):
    from simple_inference_autoresearch_b200.kernels import ops

    emu.install(monkeypatch)
    for name in ("rope_kv_write", "attention", "rope_and_attention"):
        monkeypatch.setattr(ops, name, globals()[name])


class Batch:
    """A batch over a cache entry with random contents, scrambled pages and slots, on the CPU and, by
    ``to``, on a device.  ``stale``: what rows behind the last token hold ("nan" poisons their scales)."""

    def __init__(self, bits, n_heads, n_kv_heads, head_dim, held, new, seed=0, dtype=torch.bfloat16, page=64,
                 spare_slots=2, stale="nan"):
        from simple_inference_autoresearch_b200.cache import QuantizedKVEntry
        g = torch.Generator().manual_seed(seed)
        self.bits, self.heads, self.kv_heads, self.dim = bits, n_heads, n_kv_heads, head_dim
        self.held, self.new, self.page = list(held), list(new), page
        b = len(held)
        per = [-(-(c + n) // page) for c, n in zip(held, new)]
        pages = sum(per) + 2
        order = torch.randperm(pages, generator=g).tolist()
        slots = torch.randperm(b + spare_slots, generator=g)[:b].tolist()
        table = torch.full((b + spare_slots, max(per) + 1), -1, dtype=torch.int32)
        pools = [quantise(torch.randn(pages, n_kv_heads, page, head_dim, generator=g), bits) for _ in range(2)]
        at = 0
        for i, s in enumerate(slots):
            table[s, :per[i]] = torch.tensor(order[at:at + per[i]], dtype=torch.int32)
            if stale == "nan":
                for j in range(held[i], per[i] * page):
                    for _codes, scales in pools:
                        scales[order[at + j // page], :, j % page] = float("nan")
            at += per[i]
        (k, ks), (v, vs) = pools
        self.kv = QuantizedKVEntry(k, v, ks, vs, table, page)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        self.tokens = starts[-1]
        i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
        self.slot_ids, self.q_start, self.base_len = i32(slots), i32(starts), i32(self.held)
        self.qkv = torch.randn(self.tokens, (n_heads + 2 * n_kv_heads) * head_dim, generator=g).to(dtype)

    def meta(self, device="cpu", host_lengths=True, max_kv_len=None):
        from simple_inference_autoresearch_b200.engine.batch import BatchMeta
        return BatchMeta(self.slot_ids.to(device), self.q_start.to(device), self.base_len.to(device), None, None,
                         len(self.held), self.tokens, 0, max(self.new),
                         max_kv_len or max(c + n for c, n in zip(self.held, self.new)), False,
                         q_lens=self.new if host_lengths else None, base_lens=self.held if host_lengths else None)

    def entry(self, device="cpu"):
        from simple_inference_autoresearch_b200.cache import QuantizedKVEntry
        c = self.kv
        return QuantizedKVEntry(*(t.clone().to(device) for t in (c.k, c.v, c.k_scale, c.v_scale, c.block_table)), c.page_tokens)

    def sizes(self):
        return self.heads, self.kv_heads, self.dim


def attention_bounds(batch, q, kv, scale, window=None):
    """float64 attention of queries q [tokens, heads, D] over the entry's values, and what its result in
    ``batch.qkv.dtype`` may be off.  A query element, a key element, a value element and a probability
    are each rounded once (half a step: u = eps / 2 of the dtype), and the result once more:

        a score moves by at most d = 2 u scale sum_i |q_i k_i|, a probability by a factor within
        exp(+-2 d) (its own score and the sum's), and the result by at most
        ((exp(2 d_max) - 1) + 3 u) sum_j p_j |v_j| + u |out|          (float32: + 2^-12 for the sums).

    The kernel that works on the codes (bfloat16) rounds p_j s_j (s_j the value's scale) to 16 bits of the
    largest P of a step of keys: by at most P / (2 x 65500) each, times a code of at most 127 (8 bits, 127 s
    <= max|v|) or 15 (4 bits, 15 s = a run's range <= 2 max|v|), so n keys add at most n p_max max|v| 2^-16;
    and in 4 bits it forms a value as code x s + (mid - 8 s), two sums whose terms are at most 4 max|v|
    together and whose factors (two exponentials of 2^-22, a handful of roundings of 2^-24) are right to
    2^-20 of that: 2^-18 max|v| more, also where the value itself is zero.

    The rms counts those roundings as independent and even within half a step (variance u^2 / 3), and the
    float32 sums too, w = 2^-24: a score is a sum of D terms, the result and its divisor are sums of n terms;
    each addition rounds a partial sum, which is at most the sum of the absolute terms, so they add at most
    D w^2 / 3 (scale sum_i |q_i k_i|)^2 to a score's variance and n w^2 / 3 ((sum_j p_j |v_j|)^2 + out^2) to
    the result's.

    Returns (out, bound elementwise, that rms)."""
    w = 2.0 ** -24
    u = float(torch.finfo(batch.qkv.dtype).eps) / 2
    n, hq, d = q.shape
    g = hq // batch.kv_heads
    k_all, v_all = values(kv.k, kv.k_scale), values(kv.v, kv.v_scale)
    out, bound, var = (torch.zeros(n, hq, d, dtype=torch.float64) for _ in range(3))
    for b, (c, m) in enumerate(zip(batch.held, batch.new)):
        rows = kv.block_table[int(batch.slot_ids[b]), :-(-(c + m) // batch.page)].long()
        first = max(0, c - window + 1) if window else 0
        rows = rows.clamp(min=0)
        k, v = (t[rows].transpose(1, 2).reshape(-1, batch.kv_heads, d)[:c + m] for t in (k_all, v_all))
        t0 = int(batch.q_start[b])
        for i in range(m):
            lo = max(0, c + i + 1 - window) if window else 0
            kk = k[lo:c + i + 1].repeat_interleave(g, 1)
            vv = v[lo:c + i + 1].repeat_interleave(g, 1)
            terms = q[t0 + i].double()[None] * kk
            s = terms.sum(-1) * scale                                   # [keys, heads]
            p = torch.softmax(s, 0)
            dmax = (2 * u * abs(scale) * terms.abs().sum(-1)).amax(0)        # [heads]
            o = (p[..., None] * vv).sum(0)
            pv = (p[..., None] * vv.abs()).sum(0)
            small = 2.0 ** -12 if batch.qkv.dtype == torch.float32 else 0.0
            out[t0 + i] = o
            if batch.qkv.dtype == torch.bfloat16:
                vmax = vv.abs().amax((0, 2))[:, None]
                extra = len(kk) * p.amax(0)[:, None] * vmax * 2.0 ** -16 + vmax * 2.0 ** -18
            else:
                extra = 0.0
            bound[t0 + i] = extra + (torch.expm1(2 * dmax)[:, None] + 3 * u + small * u) * pv + u * o.abs() + 1e-7 * pv
            dvar = (u * scale) ** 2 * 2 / 3 * terms.square().sum(-1) + \
                d * w * w / 3 * (scale * terms.abs().sum(-1)).square()  # of a score
            var[t0 + i] = ((dvar[..., None] + 2 * u * u / 3) * (p[..., None] * (vv - o)).square()).sum(0) + \
                (2 * u * u / 3) * (p[..., None] * vv).square().sum(0) + u * u / 3 * o.square() + \
                len(kk) * w * w / 3 * (pv.square() + o.square())
    return out, bound, math.sqrt(float(var.mean()))
