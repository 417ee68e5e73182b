"""A cache held in 8 or 4 bits on the GPU: what is stored, what is read back, and the attention over it,
against plain restatements (``emulated_kv_quant.py``)."""

import math

import pytest
import torch

from simple_inference_autoresearch_b200.kernels import ops
from simple_inference_autoresearch_b200.kernels.options import DEFAULT as OPTS
from simple_inference_autoresearch_b200.parts.rope import RotaryParams
from tests import emulated_kv_quant as eq

pytestmark = pytest.mark.gpu
DEV = "cuda"


def freqs(dim, theta=10000.0):
    return (1.0 / theta ** (torch.arange(0, dim, 2, dtype=torch.float64) / dim)).float()


def on_device(rotary):
    if isinstance(rotary, RotaryParams):
        return RotaryParams(rotary.inv_freq.to(DEV), rotary.rotary_dim, rotary.interleaved)
    return None if rotary is None else rotary.to(DEV)


def same(a, b):
    """Equal, NaN where NaN."""
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(0.5), b.nan_to_num(0.5))


SHAPES = [(4, 2, 16), (3, 1, 48), (8, 2, 64), (32, 8, 128), (6, 6, 80), (2, 1, 256)]


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
def test_store_gives_the_plain_codes_and_touches_nothing_else(bits, dtype, heads, kv_heads, dim):
    b = eq.Batch(bits, heads, kv_heads, dim, [0, 63, 130, 5, 100000 % 640], [1, 2, 70, 64, 3], seed=dim + bits, dtype=dtype)
    kv = b.entry(DEV)
    qkv = b.qkv.to(DEV)
    q = torch.full_like(qkv, 7.0)
    inv = freqs(dim)
    ops.rope_kv_write(qkv, inv.to(DEV), kv, b.meta(DEV), *b.sizes(), q_out=q)
    ops.check_status(DEV)
    assert torch.equal(qkv.cpu(), b.qkv)
    want, want_q = b.entry(), torch.full_like(b.qkv, 7.0)
    eq.rope_kv_write(b.qkv, inv, want, b.meta(), *b.sizes(), q_out=want_q)
    assert torch.equal(q.cpu(), want_q)
    for name in ("k", "v", "k_scale", "v_scale"):
        assert same(getattr(kv, name).cpu().float(), getattr(want, name).float()), name
    # in place, and without storing
    again, before = qkv.clone(), kv.k.clone()
    ops.rope_kv_write(again, inv.to(DEV), kv, b.meta(DEV), *b.sizes(), write_kv=False)
    n = heads * dim
    assert torch.equal(again[:, :n].cpu(), want_q[:, :n]) and torch.equal(again[:, n:].cpu(), b.qkv[:, n:])
    assert torch.equal(kv.k, before)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("layout", ["none", "partial", "interleaved", "partial_interleaved"])
def test_store_takes_every_rotary_layout(bits, layout):
    b = eq.Batch(bits, 4, 2, 64, [0, 200], [70, 3], seed=3)
    dim = 32 if "partial" in layout else 64
    rotary = None if layout == "none" else RotaryParams(freqs(dim), dim, "interleaved" in layout)
    kv, qkv, q = b.entry(DEV), b.qkv.to(DEV), torch.zeros_like(b.qkv, device=DEV)
    ops.rope_kv_write(qkv, on_device(rotary), kv, b.meta(DEV), *b.sizes(), q_out=q)
    want, want_q = b.entry(), torch.zeros_like(b.qkv)
    eq.rope_kv_write(b.qkv, rotary, want, b.meta(), *b.sizes(), q_out=want_q)
    assert torch.equal(q.cpu(), want_q)
    for name in ("k", "v", "k_scale", "v_scale"):
        assert same(getattr(kv, name).cpu().float(), getattr(want, name).float()), name


@pytest.mark.parametrize("bits", [8, 4])
def test_far_positions_are_rotated_by_their_exact_angle(bits):
    """Positions near 131,072: a float32 product of position and frequency is off by up to 2^-8 there."""
    page = 64
    b = eq.Batch(bits, 2, 1, 64, [3], [2], seed=9)
    b.base_len[0] = 131061                                  # the table's row is as long as that needs
    table = torch.full((3, 131072 // page), -1, dtype=torch.int32)
    table[int(b.slot_ids[0]), 131061 // page] = 1
    b.kv.block_table, b.held = table, [131061]
    kv, qkv, q = b.entry(DEV), b.qkv.to(DEV), torch.zeros_like(b.qkv, device=DEV)
    ops.rope_kv_write(qkv, freqs(64).to(DEV), kv, b.meta(DEV), *b.sizes(), q_out=q)
    want, want_q = b.entry(), torch.zeros_like(b.qkv)
    eq.rope_kv_write(b.qkv, freqs(64), want, b.meta(), *b.sizes(), q_out=want_q)
    assert torch.equal(q.cpu(), want_q)
    for name in ("k", "v", "k_scale", "v_scale"):
        assert same(getattr(kv, name).cpu().float(), getattr(want, name).float()), name


@pytest.mark.parametrize("bits", [8, 4])
def test_rows_with_special_values(bits):
    """Zeros, a constant, infinities, NaN, the largest and the smallest numbers: a bad row (or run of 64
    dims) reads back as NaN, every other one as its values."""
    b = eq.Batch(bits, 2, 2, 128, [0], [8], seed=4, dtype=torch.float32)
    rows = b.qkv.view(8, 6, 128)
    rows[0, 2:] = 0.0
    rows[1, 2:] = 1.5
    rows[2, 2, 100] = float("inf")
    rows[2, 4, 3] = float("-inf")
    rows[3, 3, 77] = float("nan")
    rows[4, 2:] *= 1e38
    rows[5, 2:] *= 1e-38
    rows[6, 2:] *= 1e-44
    rows[7, 2:, 0] = 1e30
    kv = b.entry(DEV)
    ops.rope_kv_write(b.qkv.to(DEV), None, kv, b.meta(DEV), *b.sizes(), q_out=torch.empty_like(b.qkv, device=DEV))
    want = b.entry()
    eq.rope_kv_write(b.qkv, None, want, b.meta(), *b.sizes(), q_out=torch.empty_like(b.qkv))
    for name in ("k", "v", "k_scale", "v_scale"):
        assert same(getattr(kv, name).cpu().float(), getattr(want, name).float()), name
    got = ops.read_kv(kv, b.meta(DEV), torch.float32)
    ops.check_status(DEV)
    page = int(got.block_table[0, 0])
    ref = eq.values(want.k, want.k_scale, torch.float32)[int(want.block_table[int(b.slot_ids[0]), 0])]
    assert same(got.k[page, :, :8].cpu(), ref[:, :8])
    assert not got.k[page, :, 8:].any()                      # rows behind the last token, stale NaN in the cache
    assert bool(ref[0, 2].isnan().any()) and not bool(ref[1, 2].isnan().any()) and not bool(ref[:, 4:8].isnan().any())


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
def test_read_back_gives_the_values_of_the_batch(bits, dtype, heads, kv_heads, dim):
    held, new = [0, 63, 130, 300, 64], [1, 1, 70, 5, 64]
    b = eq.Batch(bits, heads, kv_heads, dim, held, new, seed=dim, dtype=dtype, stale="random")
    for host in (True, False):
        got = ops.read_kv(b.entry(DEV), b.meta(DEV, host_lengths=host), dtype)
        ops.check_status(DEV)
        assert got.block_table.shape == (5, b.kv.block_table.shape[1])
        k_all, v_all = (eq.values(c, s, torch.float32).to(dtype) for c, s in ((b.kv.k, b.kv.k_scale), (b.kv.v, b.kv.v_scale)))
        at = 0
        for i, (c, n) in enumerate(zip(held, new)):
            pages = -(-(c + n) // 64)
            assert got.block_table[i].tolist() == list(range(at, at + pages)) + [-1] * (b.kv.block_table.shape[1] - pages)
            rows = b.kv.block_table[int(b.slot_ids[i]), :pages].long()
            for pool, whole in ((got.k, k_all), (got.v, v_all)):
                want = whole[rows].transpose(1, 2).reshape(pages * 64, kv_heads, dim).clone()
                want[c + n:] = 0
                assert torch.equal(pool[at:at + pages].transpose(1, 2).reshape(pages * 64, kv_heads, dim).cpu(), want)
            at += pages
        if host:
            assert got.k.shape[0] == at


def check_attention(b, out, q, kv, scale, window=None):
    want, bound, rms = eq.attention_bounds(b, q, kv, scale, window)
    err = (out.cpu().double().view_as(want) - want).abs()
    assert torch.isfinite(out).all()
    assert bool((err <= bound).all()), float((err / bound).max())
    assert float(err.square().mean().sqrt()) <= 4 * rms + 1e-9, (float(err.square().mean().sqrt()), rms)


ATTN = [(4, 2, 16), (3, 1, 48), (8, 2, 64), (16, 16, 64), (32, 8, 128), (6, 2, 128), (16, 1, 128), (8, 1, 64),
        (40, 2, 64), (5, 1, 256)]
STEPS = {
    "first": ([0], [1]),
    "decode": ([0, 1, 63, 64, 65, 200, 1000, 127], [1] * 8),
    "long": ([3001, 17], [1, 1]),
    "run": ([0, 63, 500, 130], [2, 4, 3, 1]),
    "chunk": ([0, 100, 64], [70, 33, 130]),
}


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("step", list(STEPS))
@pytest.mark.parametrize("heads,kv_heads,dim", ATTN)
def test_attention_over_the_quantised_cache(bits, dtype, heads, kv_heads, dim, step):
    """Scale poison behind every sequence's last token (NaN in masked places must not come through)."""
    held, new = STEPS[step]
    b = eq.Batch(bits, heads, kv_heads, dim, held, new, seed=heads + dim, dtype=dtype)
    inv, scale = freqs(dim), 1.0 / math.sqrt(dim)
    kv = b.entry(DEV)
    out = ops.rope_and_attention(b.qkv.to(DEV), inv.to(DEV), kv, b.meta(DEV), *b.sizes(), scale)
    ops.check_status(DEV)
    want = b.entry()
    eq.rope_kv_write(b.qkv.clone(), inv, want, b.meta(), *b.sizes())
    for name in ("k", "v", "k_scale", "v_scale"):
        assert same(getattr(kv, name).cpu().float(), getattr(want, name).float()), name
    pos = [c + i for c, n in zip(held, new) for i in range(n)]
    q = eq.rotate(b.qkv.view(b.tokens, -1, dim)[:, :heads].float(), pos, inv)
    check_attention(b, out, q, want, scale)
    # the same without rotation or storing, on what is in the cache now
    plain = ops.attention(b.qkv.to(DEV), kv, b.meta(DEV), *b.sizes(), scale)
    check_attention(b, plain, b.qkv.view(b.tokens, -1, dim)[:, :heads].float(), want, scale)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("step", ["decode", "run", "chunk"])
def test_attention_with_a_window(bits, step):
    held, new = STEPS[step]
    b = eq.Batch(bits, 4, 2, 64, held, new, seed=2)
    window = 70
    for i, c in enumerate(held):                             # pages in front of the window were given back
        b.kv.block_table[int(b.slot_ids[i]), :max(0, c - window + 1) // 64] = -1
    kv = b.entry(DEV)
    out = ops.rope_and_attention(b.qkv.to(DEV), None, kv, b.meta(DEV), *b.sizes(), 0.125, window=window)
    ops.check_status(DEV)
    want = b.entry()
    eq.rope_kv_write(b.qkv.clone(), None, want, b.meta(), *b.sizes())
    check_attention(b, out, b.qkv.view(b.tokens, -1, 64)[:, :4].float(), want, 0.125, window)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("new", [1, 5, 80])
def test_an_absent_page_is_reported(bits, new):
    for where in ("old", "new"):
        b = eq.Batch(bits, 8, 2, 128, [300, 20], [new, 1], seed=1)
        b.kv.block_table[int(b.slot_ids[0]), 1 if where == "old" else (300 + new - 1) // 64] = -1
        kv = b.entry(DEV)
        before = [t.clone() for t in (kv.k, kv.v)]
        ops.rope_and_attention(b.qkv.to(DEV), None, kv, b.meta(DEV), *b.sizes(), 0.1)
        with pytest.raises(RuntimeError, match="without a page"):
            ops.check_status(DEV)
        if where == "new" and new == 1:                      # the first sequence's token had no place
            for pool, old in zip((kv.k, kv.v), before):
                rows = b.kv.block_table[int(b.slot_ids[1])]
                pool[rows[:1].long()] = old[rows[:1].long()]
                assert torch.equal(pool, old)
    ops.check_status(DEV)


def test_argument_checks_see_the_quantised_entry():
    b = eq.Batch(8, 8, 2, 64, [70], [1], seed=1)
    b.kv.block_table[int(b.slot_ids[0]), 0] = 1000
    with pytest.raises(ValueError, match="no page of the pool"):
        ops.rope_and_attention(b.qkv.to(DEV), None, b.entry(DEV), b.meta(DEV), *b.sizes(), 0.1,
                               options=OPTS.but(check_arguments=True))


# ----------------------------------------------------------------------------- through the engine
@pytest.mark.parametrize("kv_format", ["int8", "int4"])
@pytest.mark.parametrize("config,dtype", [("A", torch.float32), ("C", torch.bfloat16), ("D", torch.bfloat16), ("E", torch.bfloat16)])
def test_engine_steps_against_the_restated_kernels(tmp_path, monkeypatch, kv_format, config, dtype):
    """Prompts of unequal lengths, a second turn of several tokens, single tokens: every step's logits
    against the same engine on the CPU with the restated kernels (same weights; bfloat16 rounds there as
    here up to the order of sums, hence the tolerance the engine's own tests use)."""
    import simple_inference_autoresearch_b200 as siar
    from tests import tiny_configs
    folder = tiny_configs.make_folder(tmp_path, config, seed=5)
    raw, _ = tiny_configs.read_folder(folder)
    g = torch.Generator().manual_seed(2)
    tok = lambda n: torch.randint(0, raw["vocab_size"], (n,), generator=g).tolist()  # noqa: E731
    turns = [[tok(n) for n in ns] for ns in ((5, 64, 33), (3, 1, 2), (1, 1, 1), (1, 1, 1))]

    def logits(device, dt):
        engine = siar.build_engine(siar.load_model(folder, device=device, dtype=dt), max_batch=3, max_seq_len=96, kv_cache=kv_format)
        slots = [engine.open() for _ in range(3)]
        return [engine.step([siar.StepEntry(s, t, range(len(t))) for s, t in zip(slots, turn)]).cpu().double() for turn in turns]

    got = logits(DEV, dtype)
    ops.check_status(DEV)
    with monkeypatch.context() as m:
        eq.install(m)
        want = logits("cpu", torch.float32 if dtype == torch.float32 else dtype)
    for a, w in zip(got, want):
        off = float((a - w).abs().max() / w.abs().max())
        # a key or value next to a rounding border may fall to the other side: one step of its row, in one of
        # thousands of terms, so the 4-bit cache gets its 15 / 127 times coarser step's share on top
        assert off <= (2e-4 if dtype == torch.float32 else 3e-2) * (1 if kv_format == "int8" else 127 / 15), off


@pytest.mark.parametrize("kv_format", ["int8", "int4"])
@pytest.mark.parametrize("config,dtype", [("A", torch.float32), ("C", torch.bfloat16), ("D", torch.bfloat16), ("E", torch.bfloat16)])
def test_captured_steps_draw_what_eager_steps_draw(tmp_path, kv_format, config, dtype):
    import simple_inference_autoresearch_b200 as siar
    from tests import tiny_configs
    folder = tiny_configs.make_folder(tmp_path, config, seed=6)
    raw, _ = tiny_configs.read_folder(folder)
    loaded = siar.load_model(folder, device=DEV, dtype=dtype)
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, raw["vocab_size"], (n,), generator=g).tolist() for n in (3, 40, 21, 9, 60)]
    outs = {}
    for graph in (False, True):
        engine = siar.build_engine(loaded, max_batch=3, max_seq_len=96, use_cuda_graph=graph, kv_cache=kv_format)
        outs[graph] = [engine.generate(prompts, siar.SamplingParams(temperature=0.0), max_new_tokens=n, ignore_eos=True)
                       for n in (12, 5)]
    assert outs[False] == outs[True]


def test_command_line_takes_the_cache_format(capsys):
    from simple_inference_autoresearch_b200 import inference
    for fmt in ("int8", "int4"):
        assert inference.main(["--model", "tiny-a", "--random-weights", "--prompt-len", "9", "--max-new-tokens", "4",
                               "--temperature", "0", "--kv-cache", fmt]) == 0
    assert "new_tokens" in capsys.readouterr().out


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("heads,kv_heads,dim", [(3, 1, 128), (4, 2, 64), (128, 1, 64)])
def test_a_chunk_against_a_long_cache_is_cut_into_parts(bits, heads, kv_heads, dim):
    from simple_inference_autoresearch_b200.kernels import kv_quant
    held, new = ([1700, 3], [70, 90]) if heads < 100 else ([700], [9])
    b = eq.Batch(bits, heads, kv_heads, dim, held, new, seed=7)
    assert kv_quant.key_parts(kv_heads, 28, 20.0, b.tokens * heads * (dim + 8), 148) > 1
    kv, inv = b.entry(DEV), freqs(dim)
    out = ops.rope_and_attention(b.qkv.to(DEV), inv.to(DEV), kv, b.meta(DEV), *b.sizes(), dim ** -0.5)
    ops.check_status(DEV)
    want = b.entry()
    eq.rope_kv_write(b.qkv.clone(), inv, want, b.meta(), *b.sizes())
    pos = [c + i for c, n in zip(held, new) for i in range(n)]
    check_attention(b, out, eq.rotate(b.qkv.view(b.tokens, -1, dim)[:, :heads].float(), pos, inv), want, dim ** -0.5)
    # the batch's lengths known on the device only, a launch sized for more, and other rotary layouts
    again = ops.rope_and_attention(b.qkv.to(DEV), inv.to(DEV), b.entry(DEV), b.meta(DEV, host_lengths=False, max_kv_len=1900),
                                   *b.sizes(), dim ** -0.5)
    check_attention(b, again, eq.rotate(b.qkv.view(b.tokens, -1, dim)[:, :heads].float(), pos, inv), want, dim ** -0.5)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("layout", ["partial", "interleaved"])
def test_attention_behind_other_rotary_layouts(bits, layout):
    for held, new in (([70, 3], [1, 1]), ([70, 3], [2, 3]), ([70, 3], [40, 75])):
        b = eq.Batch(bits, 8, 2, 64, held, new, seed=3)
        rotary = RotaryParams(freqs(32 if layout == "partial" else 64), 32 if layout == "partial" else 64, layout == "interleaved")
        out = ops.rope_and_attention(b.qkv.to(DEV), on_device(rotary), b.entry(DEV), b.meta(DEV), *b.sizes(), 0.125)
        want = b.entry()
        eq.rope_kv_write(b.qkv.clone(), rotary, want, b.meta(), *b.sizes())
        pos = [c + i for c, n in zip(held, new) for i in range(n)]
        check_attention(b, out, eq.rotate(b.qkv.view(b.tokens, -1, 64)[:, :8].float(), pos, rotary), want, 0.125)
    ops.check_status(DEV)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (4, 1, 128), (3, 1, 48)])
@pytest.mark.parametrize("held,new", [([5, 30], [4, 3]), ([5, 90], [70, 40]), ([0, 63], [130, 1])])
def test_numbers_that_are_none_reach_only_the_rows_that_see_them(bits, heads, kv_heads, dim, held, new):
    """A key with an infinity and a value with a NaN among the new tokens: rows in front of them (the mask hides
    them) are as without, rows behind are NaN: every dim for a bad key, the value's row (8 bits) or run of 64 dims
    (4 bits) for a bad value."""
    b = eq.Batch(bits, heads, kv_heads, dim, held, new, seed=5)
    x = b.qkv.view(b.tokens, heads + 2 * kv_heads, dim)
    bad_v, bad_k = 1, int(b.q_start[1]) + new[1] - 1          # the first sequence's second token, the second's last
    clean = b.qkv.clone()
    x[bad_v, heads + kv_heads, 3] = float("nan")              # value of kv head 0
    x[bad_k, heads + kv_heads - 1, 7] = float("inf")          # key of the last kv head
    out = ops.rope_and_attention(b.qkv.to(DEV), None, b.entry(DEV), b.meta(DEV), *b.sizes(), 0.125).cpu().view(b.tokens, heads, dim)
    ops.check_status(DEV)
    group = heads // kv_heads
    bad = torch.zeros(b.tokens, heads, dim, dtype=torch.bool)
    bad[bad_v:new[0], :group, :dim if bits == 8 else 64] = True
    bad[bad_k, heads - group:] = True
    assert torch.equal(out.isnan(), bad)
    b.qkv = clean
    want = b.entry()
    eq.rope_kv_write(clean.clone(), None, want, b.meta(), *b.sizes())
    ref, bound, _ = eq.attention_bounds(b, clean.view(b.tokens, -1, dim)[:, :heads].float(), want, 0.125)
    hidden = torch.ones(b.tokens, heads, dtype=torch.bool)    # rows that see neither
    hidden[bad_v:new[0], :group] = False
    hidden[bad_k, heads - group:] = False
    assert bool(((out.double() - ref).abs() <= bound)[hidden].all())


def attend(b, device_kv, *, scale, meta=None, **kw):
    return ops.rope_and_attention(b.qkv.to(DEV), None, device_kv, meta or b.meta(DEV), *b.sizes(), scale, **kw)


def plain_of(b):
    """The entry with the batch's new tokens stored, and the queries, for a batch without rotation."""
    want = b.entry()
    eq.rope_kv_write(b.qkv.clone(), None, want, b.meta(), *b.sizes())
    return want, b.qkv.view(b.tokens, -1, b.dim)[:, :b.heads].float()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("page", [128, 192])
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 2, 1], [90, 5, 200]])
def test_pages_of_other_sizes(bits, page, new):
    b = eq.Batch(bits, 8, 2, 64, [0, 300, 191], new, seed=page, page=page)
    out = attend(b, b.entry(DEV), scale=0.125)
    ops.check_status(DEV)
    want, q = plain_of(b)
    check_attention(b, out, q, want, 0.125)
    got = ops.read_kv(b.entry(DEV), b.meta(DEV), torch.float32)
    assert got.page_tokens == page and got.k.shape[2] == page
    ops.check_status(DEV)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 1, 64), (4, 2, 128), (3, 1, 32)])
@pytest.mark.parametrize("kind", ["decode", "run", "chunk"])
def test_more_sequences_than_a_warp_has_lanes(bits, heads, kv_heads, dim, kind):
    g = torch.Generator().manual_seed(11)
    held = torch.randint(0, 200, (75,), generator=g).tolist()
    new = [1] * 75 if kind == "decode" else torch.randint(1, 4 if kind == "run" else 12, (75,), generator=g).tolist()
    if kind == "chunk":
        new[40] = 130
    b = eq.Batch(bits, heads, kv_heads, dim, held, new, seed=1, stale="random")
    out = attend(b, b.entry(DEV), scale=dim ** -0.5)
    ops.check_status(DEV)
    want, q = plain_of(b)
    check_attention(b, out, q, want, dim ** -0.5)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("new", [1, 3, 70])
@pytest.mark.parametrize("scale", [0.0, -0.1])
def test_any_scale(bits, new, scale):
    b = eq.Batch(bits, 8, 2, 64, [130, 7], [new, 1], seed=8)
    out = attend(b, b.entry(DEV), scale=scale)
    want, q = plain_of(b)
    check_attention(b, out, q, want, scale)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("new", [1, 4, 40])
@pytest.mark.parametrize("tall", [3, 200])
def test_a_dominant_key_without_a_value(bits, new, tall):
    """Scores of 30 (base e) for key ``tall`` with a value of zeros, 0 for all others with values of 1: the result is
    n e^-30 / (1 + n e^-30), far below the reference that the scores alone would set.  Every number is its code times a
    power of two, so only p (16 bits of the largest of a step, all equal here), the exponential (2^-21 at 30 log2 e,
    whose own rounding is 2^-19 there) and the result (2^-9) round.  Runs of more than 64 rows go over float16 tiles,
    where p is a float16 that starts 2^8 below the largest score's: what is under 2^-24 of that, 2^-32 of the largest,
    is lost, at most 2^-32 a key of values of 1."""
    dim, held = 64, 300
    b = eq.Batch(bits, 2, 1, dim, [held], [new], seed=0, stale="random")
    x = b.qkv.view(new, 4, dim)
    x.zero_()
    x[:, :2, 0] = 1.0
    x[:, 3] = 1.0                                             # new values; new keys are zeros
    k = torch.zeros(b.kv.k.shape[0], 1, 64, dim)
    v = torch.ones_like(k)
    page, at = int(b.kv.block_table[int(b.slot_ids[0]), tall // 64]), tall % 64
    k[page, 0, at, 0] = 15.0 * 16
    k[page, 0, at, 1] = -15.0 * 16                            # (4 bits: the run's range is a multiple of 15)
    v[page, 0, at] = 0.0
    b.kv.k, b.kv.k_scale = eq.quantise(k, bits)
    b.kv.v, b.kv.v_scale = eq.quantise(v, bits)
    top = float(eq.values(b.kv.k, b.kv.k_scale)[page, 0, at, 0])
    scale = 30.0 / top
    out = attend(b, b.entry(DEV), scale=scale).cpu().double().view(new, 2, dim)
    ops.check_status(DEV)
    for i in range(new):
        n = held + i
        want = n * math.exp(-30.0) / (1 + n * math.exp(-30.0))
        lost = n * 2.0 ** -32 if new * 2 > 64 else 0.0
        assert bool(((out[i] - want).abs() <= want * (2 ** -9 + 2 ** -15 + 2 ** -18) + lost).all()), out[i, 0, :3]


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("new", [1, 4, 40])
def test_values_of_very_unequal_rows(bits, new):
    """Rows of values from 2^-40 to 2^40 of one another and rows of zeros; where every value is zero the result is."""
    b = eq.Batch(bits, 4, 2, 128, [200, 66], [new, 1], seed=6)
    powers = torch.randint(-40, 41, b.kv.v_scale.shape[:3], generator=torch.Generator().manual_seed(1)).float().exp2()
    powers[powers < 2.0 ** -30] = 0.0
    s = b.kv.v_scale
    b.kv.v_scale = (s.float() * (powers if bits == 8 else powers[..., None, None])).to(s.dtype)
    out = attend(b, b.entry(DEV), scale=0.05)
    want, q = plain_of(b)
    check_attention(b, out, q, want, 0.05)
    b.kv.v_scale = torch.zeros_like(s)
    b.qkv.view(b.tokens, 8, 128)[:, 6:] = 0.0
    assert not attend(b, b.entry(DEV), scale=0.05).any()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("new", [1, 3, 80])
def test_results_are_the_same_every_time_on_any_stream(bits, new):
    b = eq.Batch(bits, 8, 2, 128, [3000, 17, 900], [new, 1, 2 if new > 1 else 1], seed=4)
    kv = b.entry(DEV)
    first = attend(b, kv, scale=0.09)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for i in range(12):
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            again = attend(b, kv, scale=0.09)
            assert torch.equal(again, first)
        torch.cuda.synchronize()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("new", [1, 3, 80])
def test_two_captured_graphs_run_side_by_side(bits, new):
    """Captured on one stream, replayed on two at once, an eager call beside them: no workspace is shared."""
    batches = [eq.Batch(bits, 8, 2, 128, [4000 + 600 * i, 70], [new, 1], seed=20 + i) for i in range(3)]
    state = [(b.qkv.to(DEV), b.entry(DEV), b.meta(DEV), b.sizes()) for b in batches]
    call = lambda s: ops.rope_and_attention(s[0], None, s[1], s[2], *s[3], 0.09)  # noqa: E731
    want = [call(s) for s in state]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in state[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append([call(s) for _ in range(3)])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        eager = call(state[2])
        torch.cuda.synchronize()
        assert torch.equal(eager, want[2])
        for got, w in zip(outs, want):
            assert all(torch.equal(o, w) for o in got)
    ops.check_status(DEV)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dim", [128, 48])
def test_a_captured_step_replayed_while_the_sequences_grow(bits, dim):
    """One capture, lengths advanced on the device by the graph itself, over page and step borders; as eager steps."""
    steps = 9
    b = eq.Batch(bits, 4, 2, dim, [60, 250, 0], [steps, steps, steps], seed=2, stale="nan")
    g = torch.Generator().manual_seed(9)
    rows = torch.randn(steps, 3, 8 * dim, generator=g).to(torch.bfloat16).to(DEV)
    inv = freqs(dim).to(DEV)
    from simple_inference_autoresearch_b200.engine.batch import BatchMeta
    starts = torch.arange(4, dtype=torch.int32, device=DEV)

    def meta(base):
        return BatchMeta(b.slot_ids.to(DEV), starts, base, None, None, 3, 3, 0, 1, 512, False)

    kv, want = b.entry(DEV), []
    for i in range(steps):
        want.append(ops.rope_and_attention(rows[i], inv, kv, meta((b.base_len + i).to(DEV)), 4, 2, dim, 0.1))
    kv2, base, qkv = b.entry(DEV), b.base_len.to(DEV), rows[0].clone()
    m = meta(base)
    ops.rope_and_attention(qkv, inv, kv2, m, 4, 2, dim, 0.1)               # loads the kernels
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.rope_and_attention(qkv, inv, kv2, m, 4, 2, dim, 0.1)
        ops.advance_lengths(base, starts, 3)
    for i in range(steps):
        qkv.copy_(rows[i])
        graph.replay()
        assert torch.equal(out, want[i]), i
    ops.check_status(DEV)
    for name in ("k", "v", "k_scale", "v_scale"):
        assert same(getattr(kv, name).float(), getattr(kv2, name).float())


def test_offsets_past_32_bits():
    """A pool of 70,000 pages (4.6 GB of codes): the batch's pages are its last ones."""
    pages, heads, dim = 70000, 8, 128
    from simple_inference_autoresearch_b200.cache import QuantizedKVEntry
    b = eq.Batch(8, 8, heads, dim, [100, 63], [1, 1], seed=3)
    small = b.entry(DEV)
    n = small.k.shape[0]
    k, v = (torch.empty(pages, heads, 64, dim, dtype=torch.int8, device=DEV) for _ in range(2))
    ks, vs = (torch.empty(pages, heads, 64, device=DEV) for _ in range(2))
    for big, few in ((k, small.k), (v, small.v), (ks, small.k_scale), (vs, small.v_scale)):
        big[pages - n:] = few
    table = torch.where(small.block_table >= 0, small.block_table + (pages - n), small.block_table)
    big = QuantizedKVEntry(k, v, ks, vs, table, 64)
    assert k.numel() > 1 << 32
    for new in ([1, 1], [2, 1], [27, 1]):
        b.new, b.tokens = new, sum(new)
        b.q_start = torch.tensor([0, new[0], sum(new)], dtype=torch.int32)
        b.qkv = torch.randn(b.tokens, 24 * dim, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
        assert torch.equal(attend(b, big, scale=0.09), attend(b, small, scale=0.09))
        a, c = (ops.read_kv(e, b.meta(DEV), torch.bfloat16) for e in (big, small))
        assert torch.equal(a.k, c.k) and torch.equal(a.v, c.v)
        assert torch.equal(k[pages - n:], small.k) and same(vs[pages - n:], small.v_scale)
    ops.check_status(DEV)


@pytest.mark.parametrize("kv_format", ["int8", "int4"])
def test_layers_with_a_window_over_a_quantised_cache(tmp_path, monkeypatch, kv_format):
    """Layer 0 keeps all keys, the others the last 37: prompt and single tokens far past the window, against the
    restated kernels on the CPU."""
    import simple_inference_autoresearch_b200 as siar
    from simple_inference_autoresearch_b200.architectures.llama import llama_model_spec
    from simple_inference_autoresearch_b200.config.llama import LlamaConfig
    from simple_inference_autoresearch_b200.engine.model import DecoderModel, ModelSpec
    from simple_inference_autoresearch_b200.parts.base import PartSpec
    from tests import tiny_configs
    raw, w = tiny_configs.read_folder(tiny_configs.make_folder(tmp_path, "B", seed=5))
    base = llama_model_spec(LlamaConfig.from_dict(raw))
    layers = list(base.layers)
    for i in (1, 2):
        p = dict(layers[i].params)
        p["mixer"] = PartSpec("gqa_attention", {**p["mixer"].params, "window": 37})
        layers[i] = PartSpec(layers[i].kind, p)
    toks = torch.randint(0, raw["vocab_size"], (150,), generator=torch.Generator().manual_seed(4)).tolist()

    def run(device):
        model = DecoderModel(ModelSpec(**{**base.__dict__, "layers": tuple(layers)}), torch.float32, device)
        model.load({k: v.float().to(device) for k, v in w.items()})
        eng = siar.Engine(model, max_batch=2, max_seq_len=256, use_cuda_graph=False, kv_cache=kv_format)
        a = eng.open()
        outs = [eng.step([siar.StepEntry(a, toks[:90], range(90))])]
        outs += [eng.step([siar.StepEntry(a, [t], [0])]) for t in toks[90:]]
        assert eng.cache.groups[1].held_pages(a) <= 2
        eng.close(a)
        assert all(len(g.pages) == g.pages.n for g in eng.cache.groups)
        return torch.cat(outs).cpu().double()

    got = run(DEV)
    ops.check_status(DEV)
    with monkeypatch.context() as m:
        eq.install(m)
        want = run("cpu")
    off = float((got - want).abs().max() / want.abs().max())
    assert off <= 2e-4 * (1 if kv_format == "int8" else 127 / 15), off      # as in the engine test above


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("new", [1, 4, 40, 300])
@pytest.mark.parametrize("power", [60, 100])
@pytest.mark.parametrize("tall", [2, 290, 4000])
def test_one_very_large_value_among_zeros(bits, new, power, tall):
    """All scores are equal, all values are zeros but those of key ``tall``, 15 x 2^power: the result is that over the number
    of keys.  Every number is its code times a power of two (8 bits: a scale off by 2^-24), the sum of equal p by at most
    2^-23 a key, an exponential and a quotient by 2^-21 each; the result rounds by 2^-9."""
    dim, held = 64, 4100
    b = eq.Batch(bits, 2, 1, dim, [held], [new], seed=0, stale="random")
    x = b.qkv.view(new, 4, dim)
    x.zero_()
    x[:, :2, 0] = 1.0                                         # keys are zeros
    k = torch.zeros(b.kv.k.shape[0], 1, 64, dim)
    v = torch.zeros_like(k)
    page = int(b.kv.block_table[int(b.slot_ids[0]), tall // 64])
    v[page, 0, tall % 64, :] = 15.0 * 2.0 ** power
    v[page, 0, tall % 64, 1::2] *= -1.0                       # (4 bits: a scale that is not zero)
    b.kv.k, b.kv.k_scale = eq.quantise(k, bits)
    b.kv.v, b.kv.v_scale = eq.quantise(v, bits)
    value = eq.values(b.kv.v, b.kv.v_scale)[page, 0, tall % 64]
    out = attend(b, b.entry(DEV), scale=1.0).cpu().double().view(new, 2, dim)
    ops.check_status(DEV)
    for i in range(new):
        n = held + i + 1
        assert bool(((out[i] - value / n).abs() <= (value / n).abs() * (2 ** -9 + n * 2 ** -23 + 2 ** -19)).all()), (i, out[i, 0, :3], value[:3] / n)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.bfloat16, 48), (torch.float32, 64)])
@pytest.mark.parametrize("new", [[1, 1], [3, 2], [70, 0, 9]])
def test_rows_behind_the_last_sequence_stay_as_they_are(bits, dtype, dim, new):
    b = eq.Batch(bits, 4, 2, dim, [65] * len(new), new, seed=9, dtype=dtype)
    want = b.entry()
    q = b.qkv.clone()
    eq.rope_kv_write(q, freqs(dim), want, b.meta(), *b.sizes())
    pad = torch.randn(37, b.qkv.shape[1], generator=torch.Generator().manual_seed(1)).to(dtype)
    padded, kv, meta = torch.cat([b.qkv, pad]).to(DEV), b.entry(DEV), b.meta(DEV)
    meta.n_tokens += 37
    out = ops.rope_and_attention(padded.clone(), freqs(dim).to(DEV), kv, meta, *b.sizes(), 0.1)
    ops.rope_kv_write(padded, freqs(dim).to(DEV), kv, meta, *b.sizes())
    ops.check_status(DEV)
    for name in ("k", "v", "k_scale", "v_scale"):
        assert same(getattr(kv, name).cpu().float(), getattr(want, name).float()), name
    assert torch.equal(padded[b.tokens:].cpu(), pad) and torch.equal(padded[:b.tokens].cpu(), q)
    alone = ops.rope_and_attention(b.qkv.to(DEV), freqs(dim).to(DEV), kv, b.meta(DEV), *b.sizes(), 0.1)
    assert torch.equal(out[:b.tokens], alone)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("new", [1, 3, 80])
def test_threads_that_call_on_one_stream_and_on_their_own(bits, new):
    import threading
    batches = [eq.Batch(bits, 8, 2, 64, [700, 1500, 20 + i], [new] * 3, seed=i) for i in range(4)]
    entries, inv = [b.entry(DEV) for b in batches], freqs(64).to(DEV)
    call = lambda i: ops.rope_and_attention(  # noqa: E731
        batches[i].qkv.to(DEV), inv, entries[i], batches[i].meta(DEV), 8, 2, 64, 0.125)
    want = [call(i) for i in range(4)]
    torch.cuda.synchronize()
    for shared in (True, False):
        stream = torch.cuda.Stream()
        got, errors = [None] * 4, []

        def work(i):
            try:
                with torch.cuda.stream(stream if shared else torch.cuda.Stream()):
                    for _ in range(20):
                        got[i] = call(i)
                    torch.cuda.current_stream().synchronize()
            except Exception as e:  # noqa: BLE001 - reported below
                errors.append(e)

        threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert not errors
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    ops.check_status(DEV)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("new", [[1, 1], [3, 2]])
@pytest.mark.parametrize("dim,channel", [(128, 6), (128, 77), (64, 37)])
@pytest.mark.parametrize("ratio", [30.0, 100.0, 1000.0])
def test_queries_with_one_large_channel(bits, new, dim, channel, ratio):
    """One channel of every query is ``ratio`` times the others, as some channels of real models are; the cache's
    keys are zero there, so the scores are ordinary ones and what counts is how the other channels are held beside the
    large one.  On the codes a query row becomes whole numbers of 16 bits: its largest element a is 32512 of them, so
    each element is off by at most a / 65024, evenly within that (these queries are bfloat16 and not rotated:
    nothing else rounds them).  With d = that rounding of the row, o the result and p the probabilities, to first order

        o' - o = scale sum_i d_i sum_j p_j k_ji (v_j - o),

    so its variance is scale^2 (a / 32512)^2 / 12 sum_i (sum_j p_j k_ji (v_j - o))^2.  The codes' sum p_j s_j is rounded to
    1 / 65500 of a step's largest (variance P^2 / 12 a key, P = p_max / 65500 times a code times its scale: at most
    max|v| in 8 bits, twice that in 4), the result to bfloat16 (at most u^2 / 3 of its square, u = 2^-8).  The rms
    over all results has to be that to half as much again (some 1,000 independent roundings, so a few percent by chance; second
    order: scores move by at most scale sum |k| a / 65024 < 0.2)."""
    heads, kv_heads, held = 8, 2, [700, 320]
    scale, g = dim ** -0.5, heads // kv_heads
    b = eq.Batch(bits, heads, kv_heads, dim, held, new, seed=dim + channel, stale="random")
    gen = torch.Generator().manual_seed(int(ratio) + channel)
    if bits == 8:
        b.kv.k = torch.randint(-127, 128, b.kv.k.shape, generator=gen).to(torch.int8)
        b.kv.k[..., channel] = 0
        b.kv.k_scale = torch.full_like(b.kv.k_scale, 1 / 64)
    else:
        code = torch.randint(0, 16, b.kv.k.shape[:-1] + (dim,), generator=gen).to(torch.uint8)
        code[..., channel] = 8
        b.kv.k = code[..., 0::2] | (code[..., 1::2] << 4)
        b.kv.k_scale[..., 0], b.kv.k_scale[..., 1] = 0.25, 0.0
    x = b.qkv.view(b.tokens, -1, dim)
    x[:, heads:heads + kv_heads] = 0.0                        # the new tokens' keys
    x[:, :heads, channel] = ratio * x[:, :heads, channel].sign()
    out = attend(b, b.entry(DEV), scale=scale).cpu().double().view(b.tokens, heads, dim)
    ops.check_status(DEV)
    want, q = plain_of(b)
    k_all, v_all = eq.values(want.k, want.k_scale), eq.values(want.v, want.v_scale)
    square, expected = [], []
    for i, (c, m) in enumerate(zip(held, new)):
        rows = want.block_table[int(b.slot_ids[i]), :-(-(c + m) // 64)].long()
        k, v = (t[rows].transpose(1, 2).reshape(-1, kv_heads, dim) for t in (k_all, v_all))
        for t in range(m):
            for h in range(heads):
                kk, vv, row = k[:c + t + 1, h // g], v[:c + t + 1, h // g], q[int(b.q_start[i]) + t, h].double()
                p = torch.softmax(scale * (kk @ row), 0)
                o = p @ vv
                step = scale * float(row.abs().max()) / 32512
                by_query = step ** 2 / 12 * ((p[:, None] * kk).T @ (vv - o)).square().sum(0)
                top = float(p.max() * vv.abs().max()) * (1 if bits == 8 else 2) / 65500
                expected.append(by_query + len(kk) * top ** 2 / 12 + 2.0 ** -16 / 3 * o.square())
                square.append((out[int(b.q_start[i]) + t, h] - o).square())
    rms, most = (float(torch.cat(s).mean().sqrt()) for s in (square, expected))
    assert rms <= 1.5 * most, (rms, most)


MIXED = {
    "a chunk and tokens": ([0, 700, 64, 1, 130], [90, 1, 1, 1, 1]),
    "a chunk and long tokens": ([63, 1200, 0, 300], [90, 1, 1, 1]),
    "two long runs": ([500, 10, 0, 64, 2100, 2100], [40, 16, 130, 0, 3, 1]),
}


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (32, 8, 128), (16, 1, 128), (80, 1, 64)])
@pytest.mark.parametrize("batch", list(MIXED))
def test_long_and_short_runs_in_one_batch(bits, heads, kv_heads, dim, batch):
    """Every sequence is attended to by its own length: what a batch of its own kind gives, NaN behind every sequence."""
    held, new = MIXED[batch]
    b = eq.Batch(bits, heads, kv_heads, dim, held, new, seed=heads + dim)
    inv, scale = freqs(dim), dim ** -0.5
    kv = b.entry(DEV)
    out = ops.rope_and_attention(b.qkv.to(DEV), inv.to(DEV), kv, b.meta(DEV), *b.sizes(), scale)
    ops.check_status(DEV)
    want = b.entry()
    eq.rope_kv_write(b.qkv.clone(), inv, want, b.meta(), *b.sizes())
    for name in ("k", "v", "k_scale", "v_scale"):
        assert same(getattr(kv, name).cpu().float(), getattr(want, name).float()), name
    pos = [c + i for c, n in zip(held, new) for i in range(n)]
    check_attention(b, out, eq.rotate(b.qkv.view(b.tokens, -1, dim)[:, :heads].float(), pos, inv), want, scale)
    check_attention(b, ops.attention(b.qkv.to(DEV), kv, b.meta(DEV), *b.sizes(), scale),
                    b.qkv.view(b.tokens, -1, dim)[:, :heads].float(), want, scale)
    again = ops.rope_and_attention(b.qkv.to(DEV), inv.to(DEV), kv, b.meta(DEV, host_lengths=False), *b.sizes(), scale)
    ops.check_status(DEV)
    check_attention(b, again, eq.rotate(b.qkv.view(b.tokens, -1, dim)[:, :heads].float(), pos, inv), want, scale)


@pytest.mark.parametrize("bits", [8, 4])
def test_single_tokens_beside_a_chunk_are_not_widened(bits):
    """24 sequences of 3,000 keys bring one token, one of 100 keys brings 40: besides the result a call takes the float16
    queries and their factors, the tiles of the one sequence (3 of 64 positions, keys and values, 32 bytes beside each), 8 bytes
    a sequence and at most 16 parts of every row;
    256-byte steps of nine pieces and the allocator's 2 MB."""
    heads, kv_heads, dim = 8, 2, 128
    held, new = [100] + [3000] * 24, [40] + [1] * 24
    b = eq.Batch(bits, heads, kv_heads, dim, held, new, seed=1, stale="random")
    kv, qkv, meta = b.entry(DEV), b.qkv.to(DEV), b.meta(DEV)
    ops.rope_and_attention(qkv, None, kv, meta, *b.sizes(), 0.09)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    ops.rope_and_attention(qkv, None, kv, meta, *b.sizes(), 0.09)
    taken = torch.cuda.max_memory_allocated() - before
    rows = b.tokens * heads
    allowed = 2 * rows * dim * 2 + rows * 4 + 2 * 3 * kv_heads * 64 * dim * 2 + 3 * kv_heads * 32 + 25 * 8 + 16 * rows * (dim + 8) * 4
    assert taken <= allowed + 9 * 256 + (2 << 20), (taken, allowed)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("host_lengths", [True, False])
def test_chunks_whose_tiles_are_bounded(bits, host_lengths, monkeypatch):
    """The tiles of at most two sequences at a time: the same results, with the workspace of two."""
    from simple_inference_autoresearch_b200.kernels import kv_quant
    heads, kv_heads, dim = 8, 2, 128
    b = eq.Batch(bits, heads, kv_heads, dim, [1300, 700, 0, 1500, 1200], [70, 40, 90, 40, 70], seed=4)
    kv, qkv, meta = b.entry(DEV), b.qkv.to(DEV), b.meta(DEV, host_lengths=host_lengths)
    whole = attend(b, kv, scale=0.09, meta=meta)
    per_tile = 2 * kv_heads * 64 * dim * 2
    tiles = 25                                                # of the longest sequence
    monkeypatch.setattr(kv_quant, "MOST_TILE_BYTES", 2 * tiles * per_tile)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = ops.rope_and_attention(qkv, None, kv, meta, *b.sizes(), 0.09)
    taken = torch.cuda.max_memory_allocated() - before
    ops.check_status(DEV)
    rows = b.tokens * heads
    allowed = 2 * rows * dim * 2 + rows * 4 + 2 * tiles * (per_tile + kv_heads * 32) + 5 * 8 + 16 * rows * (dim + 8) * 4
    assert taken <= allowed + 9 * 256 + (2 << 20), (taken, allowed)
    want, q = plain_of(b)
    check_attention(b, out, q, want, 0.09)
    check_attention(b, whole, q, want, 0.09)


@pytest.mark.parametrize("kv_format", ["int8", "int4"])
@pytest.mark.parametrize("config,dtype", [("A", torch.float32), ("A", torch.bfloat16), ("D", torch.bfloat16)])
def test_every_unit_of_a_step_is_built_with_the_engine(tmp_path, monkeypatch, kv_format, config, dtype):
    """Whatever a prompt and decode steps load has been asked for by the time the engine stands: nothing is compiled, and no
    missing compiler found, inside a step."""
    import simple_inference_autoresearch_b200 as siar
    from simple_inference_autoresearch_b200.kernels import build
    from tests import tiny_configs
    folder = tiny_configs.make_folder(tmp_path, config, seed=6)
    built, loaded_units = [], []
    real_build, real_load = build.ensure_built, build.load_unit
    monkeypatch.setattr(build, "ensure_built", lambda units: built.extend(units) or real_build(units))
    engine = siar.build_engine(siar.load_model(folder, device=DEV, dtype=dtype), max_batch=2, max_seq_len=128, kv_cache=kv_format)
    asked = set(built)
    monkeypatch.setattr(build, "load_unit", lambda unit: loaded_units.append(unit) or real_load(unit))
    monkeypatch.setattr(ops, "_bound", {})
    engine.generate([list(range(1, 90)), [3, 4]], siar.SamplingParams(temperature=0.0), max_new_tokens=4, ignore_eos=True)
    assert "kv_quant" in loaded_units and set(loaded_units) <= asked, set(loaded_units) - asked


@pytest.mark.parametrize("kv_format", ["int8", "int4"])
def test_a_dropped_engine_leaves_no_workspace_of_its_captures(tmp_path, kv_format):
    """The memory of captured steps' workspaces is the graphs': with the engine it goes back to the device."""
    import gc

    import simple_inference_autoresearch_b200 as siar
    from simple_inference_autoresearch_b200.kernels import kv_quant
    from tests import tiny_configs
    loaded = siar.load_model(tiny_configs.make_folder(tmp_path, "D", seed=6), device=DEV, dtype=torch.bfloat16)
    kv_quant._captured_workspaces.clear()                     # what captures of other tests left

    def held(graph):
        engine = siar.build_engine(loaded, max_batch=2, max_seq_len=96, use_cuda_graph=graph, kv_cache=kv_format)
        out = engine.generate([[5, 6, 7], [8]], siar.SamplingParams(temperature=0.0), max_new_tokens=6, ignore_eos=True)
        out += engine.generate([[5, 6, 7]], siar.SamplingParams(temperature=0.0), max_new_tokens=6, ignore_eos=True)
        del engine
        gc.collect()
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        return out, torch.cuda.memory_allocated(), torch.cuda.memory_reserved()

    held(False)
    eager = held(False)
    assert held(True) == eager and held(True) == eager


def test_captures_on_one_stream_let_go_of_each_others_workspaces():
    """One's own captures, without an engine: an eager call or another capture on the stream lets the last one's go, and every
    graph still gives its result."""
    from simple_inference_autoresearch_b200.kernels import kv_quant
    b = eq.Batch(8, 8, 2, 128, [2000, 70], [1, 1], seed=2)
    kv, qkv, meta = b.entry(DEV), b.qkv.to(DEV), b.meta(DEV)
    call = lambda: ops.rope_and_attention(qkv, None, kv, meta, *b.sizes(), 0.09)  # noqa: E731
    want = call()
    side, graphs = torch.cuda.Stream(), []
    for _ in range(3):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs = [call() for _ in range(2)]
        graphs.append((g, outs))
        assert len([k for k in kv_quant._captured_workspaces if k[1] == side.cuda_stream]) == 1
    with torch.cuda.stream(side):
        assert torch.equal(call(), want)
    assert not [k for k in kv_quant._captured_workspaces if k[1] == side.cuda_stream]
    torch.cuda.synchronize()
    filler = [torch.full((1 << 22,), 7.0, device=DEV) for _ in range(4)]        # what was let go is not the eager pool's to hand out
    for _ in range(3):
        for g, outs in graphs:
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(o, want) for o in outs)
    assert all(bool((f == 7.0).all()) for f in filler)
    ops.check_status(DEV)


WAYS = {"as by default": {}, "rotation and store in front": {"fuse_decode_rope": False},
        "no tcgen05": {"use_tc_attention": False}, "no tensor cores": {"use_mma_attention": False}}


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("step", [*STEPS, "a chunk and long tokens"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (6, 2, 128), (16, 1, 128)])
@pytest.mark.parametrize("way", list(WAYS)[1:])
def test_attention_with_kernels_switched_off(bits, heads, kv_heads, dim, step, way):
    """Every choice that KernelOptions offers over a quantised cache, with the cache it leaves."""
    held, new = {**STEPS, **MIXED}[step]
    b = eq.Batch(bits, heads, kv_heads, dim, held, new, seed=heads + dim)
    inv, scale, options = freqs(dim), dim ** -0.5, OPTS.but(**WAYS[way])
    kv = b.entry(DEV)
    out = ops.rope_and_attention(b.qkv.to(DEV), inv.to(DEV), kv, b.meta(DEV), *b.sizes(), scale, options=options)
    ops.check_status(DEV)
    want = b.entry()
    eq.rope_kv_write(b.qkv.clone(), inv, want, b.meta(), *b.sizes())
    for name in ("k", "v", "k_scale", "v_scale"):
        assert same(getattr(kv, name).cpu().float(), getattr(want, name).float()), name
    pos = [c + i for c, n in zip(held, new) for i in range(n)]
    check_attention(b, out, eq.rotate(b.qkv.view(b.tokens, -1, dim)[:, :heads].float(), pos, inv), want, scale)


@pytest.mark.parametrize("kv_format", ["int8", "int4"])
@pytest.mark.parametrize("config", ["C", "D", "E"])
@pytest.mark.parametrize("way", list(WAYS))
def test_engine_codes_and_logits_against_the_restated_kernels(tmp_path, monkeypatch, kv_format, config, way):
    """A model whose results depend on its attention: the codes that both layers leave in the cache and every step's logits,
    within bounds that planted faults exceed (test_kv_quant.py plants them)."""
    from tests import kv_quant_engine
    folder = kv_quant_engine.folder_of(tmp_path, config)
    got = kv_quant_engine.run(folder, DEV, kv_format, options=OPTS.but(**WAYS[way]))
    ops.check_status(DEV)
    with monkeypatch.context() as m:
        kv_quant_engine.restated(m)
        want = kv_quant_engine.run(folder, "cpu", kv_format)
    assert kv_quant_engine.within(kv_format, got, want), kv_quant_engine.distances(got, want)


@pytest.mark.parametrize("bits", [8, 4])
def test_a_batch_of_both_kinds_captured_padded_and_repeated(bits):
    """Long and short runs in one call: the same from a graph, on another stream and with rows behind the last sequence, which
    the store leaves out."""
    heads, kv_heads, dim = 8, 2, 128
    b = eq.Batch(bits, heads, kv_heads, dim, [2100, 0, 50, 1400], [1, 90, 3, 40], seed=6)
    pad = torch.randn(21, b.qkv.shape[1], generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    kv, inv, meta = b.entry(DEV), freqs(dim).to(DEV), b.meta(DEV)
    padded_meta = b.meta(DEV)
    padded_meta.n_tokens += len(pad)
    qkv, padded = b.qkv.to(DEV), torch.cat([b.qkv, pad]).to(DEV)
    call = lambda x, m: ops.rope_and_attention(x, inv, kv, m, *b.sizes(), 0.09)  # noqa: E731
    first = call(qkv, meta)
    want = b.entry()
    eq.rope_kv_write(b.qkv.clone(), freqs(dim), want, b.meta(), *b.sizes())
    assert torch.equal(call(padded, padded_meta)[:b.tokens], first)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [call(qkv, meta), call(padded, padded_meta)]
    side = torch.cuda.Stream()
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o[:b.tokens], first) for o in outs)
        with torch.cuda.stream(side):
            assert torch.equal(call(qkv, meta), first)
        torch.cuda.synchronize()
    ops.check_status(DEV)
    for name in ("k", "v", "k_scale", "v_scale"):
        assert same(getattr(kv, name).cpu().float(), getattr(want, name).float()), name


def test_host_lengths_that_do_not_agree_are_refused():
    b = eq.Batch(8, 8, 2, 64, [70, 2100], [90, 1], seed=1)
    meta = b.meta(DEV)
    meta.q_lens = [1, 1]
    with pytest.raises(ValueError, match="do not agree"):
        attend(b, b.entry(DEV), scale=0.1, meta=meta)
