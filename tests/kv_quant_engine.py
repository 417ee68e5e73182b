"""An engine over a cache in 8 or 4 bits whose results depend on its attention, and what its steps may be off: shared by the
comparison on the GPU and by the test on the CPU that faults exceed the bounds."""

from __future__ import annotations

import torch

import simple_inference_autoresearch_b200 as siar
from simple_inference_autoresearch_b200.kernels import ops
from tests import emulated_kv_quant as eq
from tests import tiny_configs

#: What the codes in the cache and the logits may be off, on average, between two runs in bfloat16 that differ in the order of
#: sums.  That turns the last bit of bfloat16 roundings (of normed rows, products, probabilities, attention results), so by the
#: second layer rows differ by about that rounding, 2^-8 of their size, and scores of a few units by 2^-8 of themselves, as
#: much again in the probabilities: 2^-6 (rms, of a row's rms) is allowed for both with some room.
#:  * 8 bits: a step is max|x| / 127, with max|x| about 2.8 rms; 0.8 x 2^-6 rms (the mean of |x|) is 0.57 steps;
#:  * 4 bits: a step is range / 15, about 0.3 rms; rows move codes by 0.8 x 2^-6 / 0.3 = 0.04; a scale whose last bit
#:    turns (2^-8 of it) moves the 4 codes an average one lies from the middle by 2^-6, and a mid's, 2^-8 of up to two steps
#:    more; together 0.07;
#:  * logits: the final rows differ by the roundings above and, in 4 bits, by 0.07 steps of 0.3 rms: under 0.05 of their norm.
CODE_BOUND = {"int8": 0.57, "int4": 0.07}
LOGIT_BOUND = 0.05


def folder_of(tmp_path, config):
    """The tiny configuration with query and key weights that give scores of one or two, and an attention result that
    outweighs the embedding and the feed-forward."""
    from safetensors.torch import save_file

    folder = tiny_configs.make_folder(tmp_path, config, seed=5)
    raw, w = tiny_configs.read_folder(folder)
    boost = 8.0 if raw["hidden_size"] < 200 else 4.0
    for name, t in w.items():
        if name.endswith(("q_proj.weight", "k_proj.weight")):
            t *= boost
        if name.endswith("o_proj.weight"):
            t *= 8.0
    save_file(w, str(folder / "model.safetensors"))
    return folder


def run(folder, device, kv_format, **engine_options):
    """(codes of keys and of values of both layers, where the cache holds any; logits of all steps): prompts of unequal
    lengths, a second turn of several tokens, a long chunk beside single tokens, single tokens."""
    raw, _ = tiny_configs.read_folder(folder)
    g = torch.Generator().manual_seed(2)
    tok = lambda n: torch.randint(0, raw["vocab_size"], (n,), generator=g).tolist()  # noqa: E731
    turns = [[tok(n) for n in ns] for ns in ((5, 64, 33), (3, 1, 2), (1, 90, 1), (1, 1, 1), (1, 1, 1))]
    engine = siar.build_engine(siar.load_model(folder, device=device, dtype=torch.bfloat16), max_batch=3, max_seq_len=256,
                               kv_cache=kv_format, **engine_options)
    slots = [engine.open() for _ in range(3)]
    logits = [engine.step([siar.StepEntry(s, t, range(len(t))) for s, t in zip(slots, turn)]).cpu().double() for turn in turns]
    codes = []
    for layer in range(raw["num_hidden_layers"]):
        e = engine.cache.entry(layer)
        for pool in (e.k, e.v):
            p = pool.cpu().int()
            if kv_format == "int4":
                p = torch.stack((p & 15, p >> 4), -1).flatten(-2)
            rows = []
            for s in slots:
                n = engine.cache.length(s)
                rows.append(p[e.block_table[s, :-(-n // 64)].long().cpu()].transpose(1, 2).flatten(0, 1)[:n])
            codes.append(torch.cat(rows))
    return codes, torch.cat(logits)


def distances(a, b):
    """(mean distance of the codes of keys and values, layer by layer; of the logits, relative to their norm)."""
    return [float((x - y).abs().double().mean()) for x, y in zip(a[0], b[0])], float((a[1] - b[1]).norm() / b[1].norm())


def within(kv_format, a, b, times=1.0):
    codes, logits = distances(a, b)
    return max(codes) <= times * CODE_BOUND[kv_format] and logits <= times * LOGIT_BOUND


# ------------------------------------------------------------------ faults, for the restated functions
def _attention_with(change):
    def attention(qkv, kv, meta, n_heads, n_kv_heads, head_dim, scale, window=None, options=None):
        return change(qkv, kv, meta, n_heads, n_kv_heads, head_dim, scale)
    return attention


def _last_keys(qkv, kv, meta, *sizes):
    return eq.emu.attention(qkv, eq.whole(kv, torch.float32), meta, *sizes, window=20)


def _other_kv_head(qkv, kv, meta, *sizes):
    w = eq.whole(kv, torch.float32)
    w.k, w.v = w.k.flip(1), w.v.flip(1)
    return eq.emu.attention(qkv, w, meta, *sizes)


def _no_value_scales(qkv, kv, meta, *sizes):
    w = eq.whole(kv, torch.float32)
    w.v = w.v / w.v.abs().amax(-1, keepdim=True).clamp(min=1e-30)
    return eq.emu.attention(qkv, w, meta, *sizes)


def _unscaled(qkv, kv, meta, n_heads, n_kv_heads, head_dim, scale):
    return eq.emu.attention(qkv, eq.whole(kv, torch.float32), meta, n_heads, n_kv_heads, head_dim, 0.0)


_write = eq.rope_kv_write


def _no_rotation(qkv, rotary, kv, meta, n_heads, n_kv_heads, head_dim, write_kv=True, options=None, q_out=None):
    return _write(qkv, None, kv, meta, n_heads, n_kv_heads, head_dim, write_kv=write_kv, q_out=q_out)


#: name -> what stands in for the restated function of that name
FAULTS = {
    "every key weighs the same": ("attention", _attention_with(_unscaled)),
    "only the last 20 keys": ("attention", _attention_with(_last_keys)),
    "another kv head": ("attention", _attention_with(_other_kv_head)),
    "values without their scales": ("attention", _attention_with(_no_value_scales)),
    "no rotation": ("rope_kv_write", _no_rotation),
}


def restated(monkeypatch, fault=None):
    """Puts the restated functions, one of them at fault, in the place of the kernels."""
    eq.install(monkeypatch)
    if fault is not None:
        name, wrong = FAULTS[fault]
        monkeypatch.setattr(eq, name, wrong)
        monkeypatch.setattr(ops, name, wrong)
