"""The operators of a quantised key/value cache: their cases, plain forms and 64-bit values.

A cache entry holds keys and values of ``Hkv`` heads in pages of 64 positions, ``[pages, Hkv, 64, D]``, a row
(one position of one head) in whole numbers:

* 8 bits: one float32 ``scale = max|x| / 127`` a row, ``code = rint(x / scale)``, value ``code * scale``;
* 4 bits: for every 64 dims of a row (the last run may be shorter) a bfloat16 ``scale = max(x)/15 - min(x)/15`` and a
  bfloat16 ``mid = min(x) + 8 scale``, ``code = rint((x - mid) / scale) + 8`` within 0..15, value
  ``(code - 8) * scale + mid``; dim 2i sits in the low half of byte i, dim 2i + 1 in the high half.

Three operators work on it, each with the rotary encoding of its new tokens (pairs (i, i + D/2), angle = position x
frequency) in front; keys are held rotated:

* ``store``: new tokens are rotated and quantised into the cache, and the batch's keys and values are read
  back as bfloat16 pages (what a prompt's attention reads);
* ``decode``: one new token a sequence is rotated, stored, and attends to all keys of its sequence;
* ``extend``: several new tokens a sequence (a whole prompt, a chunk of one, a few guessed tokens) do the same, causally.
"""

import math

import torch

own = False

PAGE = 64
GROUP = 64
THETA = 500000.0


# ------------------------------------------------------------------ cases
def listed():
    llama8b = {"heads": 32, "kv_heads": 8, "dim": 128}
    llama3b = {"heads": 24, "kv_heads": 8, "dim": 128}
    llama1b = {"heads": 32, "kv_heads": 8, "dim": 64}
    return [
        # the first steps of one chat: nothing to stream, only the call itself
        {"name": "decode8-first", "kind": "decode", "bits": 8, "batch": 1, "context": 33, "new": 1, **llama8b},
        # the benchmark's batch at its prompt length
        {"name": "decode8-batch", "kind": "decode", "bits": 8, "batch": 8, "context": 2047, "new": 1, **llama8b},
        # one document as long as the configuration allows
        {"name": "decode8-document", "kind": "decode", "bits": 8, "batch": 1, "context": 130017, "new": 1, **llama8b},
        # a full server: many sequences of unequal lengths
        {"name": "decode8-server", "kind": "decode", "bits": 8, "batch": 64, "context": 4500, "new": 1, **llama8b},
        # the same batch as above in 4 bits, three query heads to a kv head
        {"name": "decode4-batch", "kind": "decode", "bits": 4, "batch": 8, "context": 2047, "new": 1, **llama3b},
        # a full server in 4 bits: twice the length in the same memory
        {"name": "decode4-server", "kind": "decode", "bits": 4, "batch": 64, "context": 9000, "new": 1, **llama8b},
        # two documents, small heads
        {"name": "decode4-documents", "kind": "decode", "bits": 4, "batch": 2, "context": 60001, "new": 1, **llama1b},
        # a few prompts of unequal lengths come in
        {"name": "store8-prompts", "kind": "store", "bits": 8, "batch": 5, "context": 0, "new": 2500, **llama8b},
        # short turns added to held conversations, in 4 bits
        {"name": "store4-turns", "kind": "store", "bits": 4, "batch": 7, "context": 700, "new": 45, **llama1b},
        # guessed tokens checked against long contexts
        {"name": "extend8-guesses", "kind": "extend", "bits": 8, "batch": 6, "context": 16000, "new": 4, **llama8b},
        # a prompt, attended to through the 4-bit cache
        {"name": "extend4-prompt", "kind": "extend", "bits": 4, "batch": 1, "context": 0, "new": 2048, **llama8b},
        # the next chunk of a long prompt
        {"name": "extend8-chunk", "kind": "extend", "bits": 8, "batch": 1, "context": 8191, "new": 515, **llama3b},
    ]


HEADS = ((32, 8, 128), (24, 8, 128), (32, 8, 64), (16, 16, 64), (8, 1, 128), (16, 2, 128), (12, 4, 64), (16, 1, 64))


def draw(rng):
    def spread(low, high):
        return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))

    heads, kv_heads, dim = rng.choice(HEADS)
    case = {"kind": rng.choice(("decode", "decode", "decode", "store", "extend")), "bits": rng.choice((8, 4)),
            "heads": heads, "kv_heads": kv_heads, "dim": dim}
    if case["kind"] == "decode":
        context = spread(1, 100000)
        case.update(batch=spread(1, max(1, min(96, 250000 // context))), context=context, new=1)
    elif case["kind"] == "store":
        new = spread(1, 8000)
        case.update(batch=spread(1, max(1, min(16, 12000 // new))), context=rng.choice((0, spread(1, 4000))), new=new)
    else:
        new = spread(2, 1500)
        context = rng.choice((0, spread(1, 20000)))
        batch = max(1, min(8, 3000 // new, 100000 // (new + context)))
        case.update(batch=spread(1, batch), context=context, new=new)
    return case


def lengths(case):
    """(keys held, new tokens) of every sequence: the first has the most, the others spread down to half of it."""
    held, new = [], []
    for b in range(case["batch"]):
        c, n = case["context"], case["new"]
        held.append(c - (b * 7919) % (c // 2 + 1))
        new.append(n - (b * 104729) % (n // 2 + 1) if n > 4 else n)
    return held, new


def work(case):
    held, new = lengths(case)
    hq, hkv, d = case["heads"], case["kv_heads"], case["dim"]
    row = d + 4 if case["bits"] == 8 else d // 2 + 4 * -(-d // GROUP)       # bytes of one held row
    tokens, keys, old = sum(new), sum(held) + sum(new), sum(held)
    qkv, out = tokens * (hq + 2 * hkv) * d * 2, tokens * hq * d * 2
    cache = 2 * hkv * row
    if case["kind"] == "store":
        pages = sum(-(-(c + n) // PAGE) for c, n in zip(held, new)) * PAGE
        return {"bytes": qkv + out + old * cache + tokens * cache + 2 * pages * hkv * d * 2, "flops": 10 * tokens * (hq + 2 * hkv) * d}
    pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(held, new))
    return {"bytes": qkv + out + old * cache + tokens * cache, "flops": 4 * pairs * hq * d}


# ------------------------------------------------------------------ the cache's two formats, in plain torch
def quantise(x, bits):
    """float32 [..., D] -> (codes as the cache holds them, scales as it holds them)."""
    if bits == 8:
        scale = x.abs().amax(-1) / 127.0
        code = torch.round(x / torch.where(scale > 0, scale, torch.ones_like(scale))[..., None])
        return code.clamp(-127, 127).to(torch.int8), scale
    d = x.shape[-1]
    groups = -(-d // GROUP)
    pad = groups * GROUP - d
    g = torch.nn.functional.pad(x, (0, pad), value=float("nan")).unflatten(-1, (groups, GROUP))
    low = torch.where(g.isnan(), torch.full_like(g, float("inf")), g).amin(-1)
    high = torch.where(g.isnan(), torch.full_like(g, float("-inf")), g).amax(-1)
    scale = (high / 15.0 - low / 15.0).to(torch.bfloat16).float()
    mid = (low + 8.0 * scale).to(torch.bfloat16).float()
    code = torch.round((g - mid[..., None]) / torch.where(scale > 0, scale, torch.ones_like(scale))[..., None]) + 8.0
    code = code.nan_to_num(8.0).clamp(0, 15).to(torch.uint8).flatten(-2)[..., :d]
    packed = code[..., 0::2] | (code[..., 1::2] << 4)
    return packed, torch.stack((scale, mid), -1).to(torch.bfloat16)


def values(codes, scales, bits):
    """What codes and scales stand for, float32 [..., D]."""
    if bits == 8:
        return codes.float() * scales[..., None]
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float() - 8.0
    d = code.shape[-1]
    s, m = (scales[..., i].float().repeat_interleave(GROUP, -1)[..., :d] for i in (0, 1))
    return code * s + m


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    held, new = lengths(case)
    b, hq, hkv, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    # keys have channels that stand off zero in every token; values do not
    offset = normal(hkv, 1, d) * (torch.rand((hkv, 1, d), generator=g, device="cuda") < 0.1) * 3.0
    per_seq = [-(-(c + n) // PAGE) for c, n in zip(held, new)]
    total = sum(per_seq) + 3
    pools = {}
    for name, off in (("k", offset), ("v", None)):
        codes, scales = [], []
        for at in range(0, total, 512):                # in pieces: a large pool's floats are many times its codes
            x = normal(min(512, total - at), hkv, PAGE, d)
            c, s = quantise(x + off if off is not None else x, case["bits"])
            codes.append(c)
            scales.append(s)
        pools[name], pools[name + "_scale"] = torch.cat(codes), torch.cat(scales)
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    slots = torch.randperm(b + 2, generator=g, device="cuda")[:b].to(torch.int32)
    table = torch.full((b + 2, max(per_seq)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, (slot, n) in enumerate(zip(slots.tolist(), per_seq)):
        table[slot, :n] = order[at:at + n]
        at += n
    tokens = sum(new)
    qkv = normal(tokens, (hq + 2 * hkv), d)
    qkv[:, hq:hq + hkv] += offset[:, 0]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return {**pools, "case": case, "table": table, "slots": slots, "q_start": ints(starts), "base": ints(held),
            "qkv": qkv.reshape(tokens, -1).to(torch.bfloat16),
            "inv_freq": (1.0 / THETA ** (torch.arange(0, d, 2, dtype=torch.float64) / d)).float().cuda(),
            "held": held, "new": new}


# ------------------------------------------------------------------ one pass
def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    from simple_inference_autoresearch_b200.cache import QuantizedKVEntry
    from simple_inference_autoresearch_b200.engine.batch import BatchMeta
    from simple_inference_autoresearch_b200.kernels import ops

    c = s["case"]
    hq, hkv, d = c["heads"], c["kv_heads"], c["dim"]
    kv = QuantizedKVEntry(s["k"], s["v"], s["k_scale"], s["v_scale"], s["table"], PAGE)
    meta = BatchMeta(s["slots"], s["q_start"], s["base"], None, None, c["batch"], s["qkv"].shape[0], 0, c["new"],
                     c["context"] + c["new"], False, q_lens=s["new"], base_lens=s["held"])
    if c["kind"] == "store":
        q = torch.empty_like(s["qkv"])
        ops.rope_kv_write(s["qkv"], s["inv_freq"], kv, meta, hq, hkv, d, q_out=q)
        pages = ops.read_kv(kv, meta, torch.bfloat16)
        return {"q": q[:, :hq * d], "k": pages.k, "v": pages.v}
    return {"out": ops.rope_and_attention(s["qkv"], s["inv_freq"], kv, meta, hq, hkv, d, 1.0 / math.sqrt(d))}


def _plain(s):
    c = s["case"]
    b, hq, hkv, d, bits = c["batch"], c["heads"], c["kv_heads"], c["dim"], c["bits"]
    base, start = s["base"].long(), s["q_start"].long()
    tokens = s["qkv"].shape[0]
    row = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(start[1:], row, right=True)
    place = row - start[seq]
    pos = base[seq] + place
    # rotary encoding: angles of far positions need more than 32 bits
    angle = pos[:, None].double() * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    x = s["qkv"].float().view(tokens, hq + 2 * hkv, d)
    lo, hi = x[:, :hq + hkv, :d // 2], x[:, :hq + hkv, d // 2:]
    qk = torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), -1)
    q, k, v = qk[:, :hq], qk[:, hq:], x[:, hq + hkv:]
    # the batch's keys and values: the pages its block table names, the new tokens' rows put in
    n_pages = s["table"].shape[1]
    table = s["table"][s["slots"].long()].long()
    page = table[seq, pos // PAGE]
    dense = []
    for name, fresh in (("k", k), ("v", v)):
        codes, scales = quantise(fresh, bits)
        s[name][page, :, pos % PAGE] = codes
        s[name + "_scale"][page, :, pos % PAGE] = scales
        flat = table.clamp(min=0).flatten()
        dense.append(values(s[name][flat], s[name + "_scale"][flat], bits).unflatten(0, (b, n_pages)))
    total = base + (start[1:] - start[:-1])
    if c["kind"] == "store":
        used = torch.arange(n_pages, device="cuda") < ((total + PAGE - 1) // PAGE)[:, None]
        inside = torch.arange(n_pages * PAGE, device="cuda").view(n_pages, 1, PAGE, 1) < total.view(b, 1, 1, 1, 1)
        k, v = (torch.where(inside, t, torch.zeros_like(t))[used].to(torch.bfloat16) for t in dense)
        return {"q": q.reshape(tokens, hq * d).to(torch.bfloat16), "k": k, "v": v}
    # attention, the batch padded to its longest sequence: [b, kv heads, group, new tokens, keys]
    group, most = hq // hkv, c["new"]
    kd, vd = (t.transpose(1, 2).flatten(2, 3) for t in dense)               # [b, kv heads, keys, d]
    qd = torch.zeros(b, most, hq, d, device="cuda")
    qd[seq, place] = q
    qd = qd.view(b, most, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, group * most, d)
    score = (qd @ kd.transpose(2, 3)) / math.sqrt(d)
    last = base[:, None] + torch.arange(most, device="cuda")                # the last key a new token sees
    seen = torch.arange(kd.shape[2], device="cuda") <= last.repeat(1, group)[:, :, None]
    score = score.masked_fill(~seen[:, None], float("-inf"))
    e = torch.exp(score - score.amax(-1, keepdim=True))
    out = (e @ vd) / e.sum(-1, keepdim=True)
    out = out.view(b, hkv, group, most, d).permute(0, 3, 1, 2, 4).reshape(b, most, hq * d)
    return {"out": out[seq, place].to(torch.bfloat16)}


# ------------------------------------------------------------------ 64 bits, sequence by sequence
def exact(case, seed):
    if sum(lengths(case)[1]) * max(lengths(case)[0] + lengths(case)[1]) > 4e7:
        return None
    s = prepare(case, seed)
    hq, hkv, d, bits = case["heads"], case["kv_heads"], case["dim"], case["bits"]
    f64 = torch.float64
    runs = [slice(i, min(d, i + GROUP)) for i in range(0, d, GROUP)]

    def stands_for(x):                      # a row's values after it has gone through the cache
        if bits == 8:
            step = x.abs().amax(-1, keepdim=True) / 127
            return torch.where(step > 0, torch.round(x / step) * step, torch.zeros_like(x))
        y = torch.empty_like(x)
        for r in runs:
            part = x[..., r]
            low, high = part.amin(-1, keepdim=True), part.amax(-1, keepdim=True)
            step = ((high - low) / 15).to(torch.bfloat16).to(f64)
            mid = (low + 8 * step).to(torch.bfloat16).to(f64)
            code = torch.where(step > 0, torch.round((part - mid) / step), torch.zeros_like(part)).clamp(-8, 7)
            y[..., r] = code * step + mid
        return y

    def held_rows(name, table_row, n):      # [n, kv heads, d] of what the cache held before
        need = -(-n // PAGE)
        codes, scales = s[name][table_row[:need].long()], s[name + "_scale"][table_row[:need].long()].to(f64)
        if bits == 8:
            x = codes.to(f64) * scales.unsqueeze(-1)
        else:
            x = torch.empty(codes.shape[:-1] + (d,), dtype=f64, device="cuda")
            x[..., 0::2], x[..., 1::2] = (codes % 16).to(f64), (codes // 16).to(f64)
            for i, r in enumerate(runs):
                x[..., r] = (x[..., r] - 8) * scales[..., i, :1] + scales[..., i, 1:]
        return x.transpose(1, 2).reshape(need * PAGE, hkv, d)[:n]

    qs, ks, vs, outs = [], [], [], []
    at = 0
    for slot, c, n in zip(s["slots"].tolist(), s["held"], s["new"]):
        x = s["qkv"][at:at + n].to(f64).view(n, hq + 2 * hkv, d)
        at += n
        turn = torch.polar(torch.ones(n, d // 2, dtype=f64, device="cuda"),
                           torch.arange(c, c + n, device="cuda").to(f64)[:, None] * s["inv_freq"].to(f64))[:, None]
        z = torch.complex(x[:, :hq + hkv, :d // 2].contiguous(), x[:, :hq + hkv, d // 2:].contiguous()) * turn
        x = torch.cat((torch.cat((z.real, z.imag), -1), x[:, hq + hkv:]), 1)
        k = torch.cat((held_rows("k", s["table"][slot], c), stands_for(x[:, hq:hq + hkv])))
        v = torch.cat((held_rows("v", s["table"][slot], c), stands_for(x[:, hq + hkv:])))
        q = x[:, :hq]
        if case["kind"] == "store":
            pad = -(c + n) % PAGE
            for rows, to in ((k, ks), (v, vs)):
                to.append(torch.nn.functional.pad(rows, (0, 0, 0, 0, 0, pad)).view(-1, PAGE, hkv, d).transpose(1, 2))
            qs.append(q.reshape(n, hq * d))
            continue
        o = torch.empty(n, hq, d, dtype=f64, device="cuda")
        hidden = torch.arange(c + n, device="cuda") > torch.arange(c, c + n, device="cuda")[:, None]
        for h in range(hkv):
            of = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            score = torch.einsum("ngd,kd->ngk", q[:, of], k[:, h]) / math.sqrt(d)
            score = score.masked_fill(hidden[:, None], float("-inf"))
            o[:, of] = torch.einsum("ngk,kd->ngd", torch.softmax(score, -1), v[:, h])
        outs.append(o.reshape(n, hq * d))
    if case["kind"] == "store":
        return {"q": torch.cat(qs), "k": torch.cat(ks), "v": torch.cat(vs)}
    return {"out": torch.cat(outs)}
