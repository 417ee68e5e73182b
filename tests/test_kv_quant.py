"""A cache held in 8 or 4 bits, without a GPU: storage and accounting, what the functions refuse, and the
engine's logic over it with the plain restatements in place of the kernels."""

import math

import pytest
import torch

import simple_inference_autoresearch_b200 as siar
from simple_inference_autoresearch_b200.cache import CacheError, QuantizedKVEntry, SequenceCache
from simple_inference_autoresearch_b200.kernels import kv_quant, ops
from simple_inference_autoresearch_b200.parts.base import KVNeed, StateNeed
from tests import emulated_kv_quant as eq
from tests import kv_quant_engine, plain_llama, tiny_configs


def cache(kv_format, need=KVNeed(2, 80), **kw):
    return SequenceCache([need, need, StateNeed((3,))], 640, 4, 256, torch.bfloat16, "cpu", kv_format=kv_format, **kw)


@pytest.mark.parametrize("kv_format,row", [("int8", 80 + 4), ("int4", 40 + 2 * 4)])
def test_entries_and_bytes(kv_format, row):
    c = cache(kv_format)
    e = c.entry(0)
    assert isinstance(e, QuantizedKVEntry) and e.bits == int(kv_format[3:]) and e.head_dim == 80
    kv_quant.check_entry(e, 2, 80, -1)
    assert c.entry(1).k.data_ptr() != e.k.data_ptr() and c.entry(2).state.shape == (4, 3)
    assert c.groups[0].bytes() == 2 * 2 * 10 * 2 * 64 * row          # entries, k and v, pages, heads, positions
    assert not eq.values(e.k, e.k_scale).any() or kv_format == "int4"
    s = c.alloc()
    c.reserve([s], [130])
    c.commit([s], [130])
    assert c.groups[0].held_pages(s) == 3
    c.free(s)
    assert c.groups[0].pages.held == 0


def test_what_a_cache_refuses():
    with pytest.raises(CacheError, match="int8, int4"):
        cache("fp8")
    with pytest.raises(CacheError, match="one width"):
        cache("int8", KVNeed(2, 64, v_head_dim=32))
    with pytest.raises(CacheError, match="steps of 16"):
        cache("int4", KVNeed(2, 20))
    with pytest.raises(CacheError, match="steps of 16"):
        cache("int8", KVNeed(2, 272))


@pytest.mark.parametrize("bits", [8, 4])
def test_what_the_functions_refuse(bits):
    b = eq.Batch(bits, 4, 2, 64, [70, 3], [1, 1])
    run = lambda kv=b.kv, qkv=b.qkv, heads=4, **kw: ops.rope_and_attention(  # noqa: E731
        qkv, None, kv, b.meta(), heads, 2, 64, 0.125, **kw)
    with pytest.raises(RuntimeError, match="CUDA device only"):
        run()
    with pytest.raises(RuntimeError, match="CUDA device only"):
        ops.read_kv(b.kv, b.meta(), torch.bfloat16)
    with pytest.raises(ValueError, match="not a multiple"):
        run(heads=5)
    with pytest.raises(ValueError, match="qkv must be"):
        run(qkv=b.qkv[:1])
    with pytest.raises(ValueError, match="contiguous"):
        run(qkv=torch.empty(512, 2, dtype=torch.bfloat16).t())
    with pytest.raises(TypeError, match="bfloat16 or float32"):
        run(qkv=b.qkv.half())
    with pytest.raises(ValueError, match="window"):
        run(window=0)
    with pytest.raises(TypeError, match="bfloat16 or float32"):
        ops.read_kv(b.kv, b.meta(), torch.float16)
    with pytest.raises(ValueError, match="window"):
        ops.read_kv(b.kv, b.meta(), torch.bfloat16, window=-1)
    with pytest.raises(ValueError, match="q_out"):
        ops.rope_kv_write(b.qkv, None, b.kv, b.meta(), 4, 2, 64, q_out=torch.empty(2, 64, dtype=torch.bfloat16))

    def changed(**kw):
        e = b.entry()
        return QuantizedKVEntry(**{**{n: getattr(e, n) for n in ("k", "v", "k_scale", "v_scale", "block_table", "page_tokens")}, **kw})

    for entry, words in ((changed(v=b.kv.v[:1]), "v of a cache entry"), (changed(k=b.kv.k.float()), "int8 .8 bits. or uint8"),
                         (changed(k_scale=b.kv.k_scale.double()), "k_scale"), (changed(v_scale=b.kv.v_scale[:, :1]), "v_scale"),
                         (changed(k=b.kv.k.transpose(1, 2).contiguous().transpose(1, 2)), "contiguous"),
                         (changed(block_table=b.kv.block_table.long()), "block_table"),
                         (changed(block_table=b.kv.block_table.t()), "block_table"), (changed(page_tokens=32), "k of a cache entry")):
        with pytest.raises(ValueError, match=words):
            run(kv=entry)


def test_an_ordinary_entry_has_no_read_back_and_rotates_in_place():
    c = SequenceCache([KVNeed(2, 16)], 64, 1, 64, torch.float32, "cpu")
    b = eq.Batch(8, 4, 2, 16, [0], [1], dtype=torch.float32)
    with pytest.raises(TypeError, match="quantised cache entry"):
        ops.read_kv(c.entry(0), b.meta(), torch.float32)
    with pytest.raises(ValueError, match="q_out"):
        ops.rope_kv_write(b.qkv, None, c.entry(0), b.meta(), 4, 2, 16, q_out=b.qkv)


@pytest.mark.parametrize("bits,step", [(8, 1 / 127), (4, 1 / 7.5)])
def test_the_formats_error_is_half_a_step(bits, step):
    """|value - x| <= half a step (8 bits: max|row| / 127; 4 bits: range / 15 of its run of 64), plus the
    rounding of a 4-bit run's scale and mid to 16 bits: 8 steps x 2^-8 and 2^-8 of |mid|, plus float32's."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(50, 3, 160, generator=g) * 3 + 1
    got = eq.values(*eq.quantise(x, bits))
    if bits == 8:
        s = x.abs().amax(-1, keepdim=True).double() / 127
        bound = s * (0.5 + 2 ** -16)
    else:
        bound = torch.empty_like(got)
        for at in (0, 64, 128):
            r = x[..., at:at + 64].double()
            lo, hi = r.amin(-1, keepdim=True), r.amax(-1, keepdim=True)
            s = (hi - lo) / 15
            bound[..., at:at + 64] = s * (0.5 + 15 * 2 ** -8) + (lo + 8 * s).abs() * 2 ** -8
    assert bool(((got - x.double()).abs() <= bound).all())


@pytest.mark.parametrize("kv_format", ["int8", "int4"])
def test_engine_over_a_quantised_cache(tmp_path, monkeypatch, kv_format):
    """The engine's logic with the restated kernels: unequal batches, early enders and slot reuse give what
    a sequence alone gives, and 8 bits stay near the cache in the compute dtype."""
    eq.install(monkeypatch)
    folder = tiny_configs.make_folder(tmp_path, "A", seed=3)
    loaded = siar.load_model(folder, device="cpu", dtype=torch.float32)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 256, (n,), generator=g).tolist() for n in (3, 17, 66)]
    run = lambda ps, fmt, **kw: siar.build_engine(loaded, max_batch=2, max_seq_len=96, kv_cache=fmt, **kw).generate(  # noqa: E731
        ps, siar.SamplingParams(temperature=0.0), max_new_tokens=4, ignore_eos=True)
    outs = run(prompts, kv_format)
    assert outs == [run([p], kv_format)[0] for p in prompts]
    engine, plain = (siar.build_engine(loaded, max_batch=1, max_seq_len=96, kv_cache=f) for f in (kv_format, None))
    assert isinstance(engine.cache.entry(0), QuantizedKVEntry)
    logits = [e.step([siar.StepEntry(e.open(), prompts[2], [65])]) for e in (engine, plain)]
    # rounding to steps of s gives an rms error of s / sqrt(12); a row of 16 has max / rms about 2, a run's
    # range / rms about 3.6: 2 / 127 / 3.5 = 0.5% and 3.6 / 15 / 3.5 = 7% of the keys and values, which reach
    # the logits through scores and sums; four times that is allowed
    off = float((logits[0] - logits[1]).norm() / logits[1].norm())
    assert 0 < off < (0.02 if kv_format == "int8" else 0.3), off


def test_unknown_kv_cache_is_refused(tmp_path):
    folder = tiny_configs.make_folder(tmp_path, "A", seed=3)
    loaded = siar.load_model(folder, device="cpu", dtype=torch.float32)
    with pytest.raises(CacheError, match="int8, int4"):
        siar.build_engine(loaded, max_seq_len=64, kv_cache="int2")


@pytest.mark.parametrize("name,wrong", [("slot_ids", lambda t: t.long()), ("q_start", lambda t: t[:-1]),
                                        ("base_len", lambda t: torch.stack([t, t], 1)[:, 0])])
def test_batch_tensors_of_another_type_or_shape(name, wrong):
    b = eq.Batch(8, 4, 2, 64, [70, 3], [1, 1])
    for call in (lambda m: ops.rope_and_attention(b.qkv, None, b.kv, m, 4, 2, 64, 0.125),
                 lambda m: ops.rope_kv_write(b.qkv, None, b.kv, m, 4, 2, 64),
                 lambda m: ops.attention(b.qkv, b.kv, m, 4, 2, 64, 0.125), lambda m: ops.read_kv(b.kv, m, torch.bfloat16)):
        meta = b.meta()
        setattr(meta, name, wrong(getattr(meta, name)))
        with pytest.raises(ValueError, match=name):
            call(meta)


def test_frequencies_that_are_not_contiguous():
    b = eq.Batch(8, 4, 2, 64, [70, 3], [1, 1])
    with pytest.raises(ValueError, match="inv_freq"):
        ops.rope_and_attention(b.qkv, torch.ones(64)[::2], b.kv, b.meta(), 4, 2, 64, 0.125)


def test_queries_that_would_go_over_other_rows():
    b = eq.Batch(8, 4, 2, 64, [70, 3], [1, 1])
    room = torch.zeros(3, 512, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="apart"):
        ops.rope_kv_write(room[:2], None, b.kv, b.meta(), 4, 2, 64, q_out=room[1:])


def test_which_sequences_of_a_batch_go_on_the_codes():
    """Short runs beside a long one: by their own length where their keys are many, or the lengths are known at all."""
    def new_on_codes(held, new, heads=8, **kw):
        b = eq.Batch(8, heads, 2, 64, [0] * len(held), [1] * len(held))
        meta = b.meta()
        meta.base_lens, meta.q_lens, meta.max_q_len = held, new, max(new)
        meta.max_kv_len = max(c + n for c, n in zip(held, new))
        for name, value in kw.items():
            setattr(meta, name, value)
        b.kv.block_table = torch.zeros(len(held) + 2, 200, dtype=torch.int32)
        passed = kv_quant.new_on_codes(b.kv, meta, heads, 2)
        return passed, kv_quant.tiles_of(b.kv, meta, passed)

    assert new_on_codes([0, 2000], [512, 1]) == (16, [(512, 8), (0, 0)])
    assert new_on_codes([0, 100], [512, 1]) == (0, [(512, 8), (1, 2)])
    assert new_on_codes([0] + [600] * 8, [512] + [1] * 8) == (16, [(512, 8)] + [(0, 0)] * 8)
    assert new_on_codes([0] + [100] * 8, [512] + [1] * 8) == (0, [(512, 8)] + [(1, 2)] * 8)
    assert new_on_codes([0] + [100] * 16, [512] + [1] * 16) == (16, [(512, 8)] + [(0, 0)] * 16)
    assert new_on_codes([0, 1500, 0], [512, 4, 0]) == (0, [(512, 8), (4, 24), (0, 0)])
    assert new_on_codes([0, 2100, 700], [512, 16, 17]) == (16, [(512, 8), (0, 0), (17, 12)])
    assert new_on_codes([0, 2000], [512, 1], heads=256) == (1, [(512, 8), (0, 0)])
    assert new_on_codes([0, 2000], [512, 1], base_lens=None) == (0, [(512, 32), (512, 32)])


def test_tiles_of_a_launch_are_bounded():
    """Sequences in launches of up to 64 and MOST_TILE_BYTES, one at least, in order, none without tiles, about even."""
    runs, most = kv_quant.runs_of_tiles, kv_quant.MOST_TILE_BYTES
    assert runs([(70, 3)] * 5, 64, 1000) == [[0, 1, 2, 3, 4]]
    assert runs([(70, 3), (0, 0), (90, 3)] * 50, 64, 8) == [[i for i in range(75) if i % 3 != 1], [i for i in range(75, 150) if i % 3 != 1]]
    assert runs([(70, 10)] * 7, 64, most // 30) == [[0, 1, 2], [3, 4, 5], [6]]
    assert runs([(70, 10)] * 8, 64, most // 70) == [[0, 1, 2, 3], [4, 5, 6, 7]]
    assert runs([(70, 1), (70, 40), (70, 1), (70, 28), (0, 0), (70, 1)], 64, most // 30) == [[0], [1], [2, 3], [5]]
    assert runs([(0, 0)], 64, 1) == []
    g = torch.Generator().manual_seed(0)
    for _ in range(200):
        n = int(torch.randint(1, 150, (1,), generator=g))
        lengths = [(1, t) for t in torch.randint(0, 60, (n,), generator=g).tolist()]
        got = runs(lengths, 64, most // 100)
        assert [i for r in got for i in r] == [i for i in range(n) if lengths[i][1]]
        assert all(len(r) <= 64 and (len(r) == 1 or sum(lengths[i][1] for i in r) <= 100) for r in got)


@pytest.mark.parametrize("config,dtype,units", [("A", torch.float32, ["kv_quant"]), ("A", torch.bfloat16, ["kv_quant"]),
                                                ("D", torch.bfloat16, ["kv_quant", "attention_quant", "attention_quant_tc"])])
def test_an_engine_names_the_units_of_its_cache(tmp_path, config, dtype, units):
    loaded = siar.load_model(tiny_configs.make_folder(tmp_path, config, seed=3), device="cpu", dtype=dtype)
    engine = lambda fmt: siar.build_engine(loaded, max_seq_len=64, kv_cache=fmt)  # noqa: E731
    assert engine(None).extension_units() == []
    assert engine("int8").extension_units() == engine("int4").extension_units() == units
    assert kv_quant.extension_units([None, StateNeed((3,))], torch.bfloat16, 64) == ()
    assert kv_quant.extension_units([KVNeed(2, 128, window=9)], torch.bfloat16, 64) == ("kv_quant",)
    assert kv_quant.extension_units([KVNeed(2, 128)], torch.bfloat16, 16) == ("kv_quant",)


@pytest.mark.parametrize("kv_format", ["int8", "int4"])
@pytest.mark.parametrize("config", ["C", "D", "E"])
def test_faults_exceed_the_bounds_of_the_engines_comparison(tmp_path, monkeypatch, kv_format, config):
    """What the comparison on the GPU allows would not hide a fault: planted in the restated functions, each is three times
    beyond it, and a cache that is not quantised (its logits) twice where 4 bits make that much of a difference."""
    folder = kv_quant_engine.folder_of(tmp_path, config)

    def run(fault=None, fmt=kv_format):
        with monkeypatch.context() as m:
            kv_quant_engine.restated(m, fault)
            return kv_quant_engine.run(folder, "cpu", fmt)

    right = run()
    assert kv_quant_engine.distances(run(), right) == ([0.0] * 4, 0.0)
    for fault in kv_quant_engine.FAULTS:
        assert not kv_quant_engine.within(kv_format, run(fault), right, times=3), fault
    if kv_format == "int4":
        plain = run(fmt=None)[1]
        assert float((plain - right[1]).norm() / right[1].norm()) > 2 * kv_quant_engine.LOGIT_BOUND
