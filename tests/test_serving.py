"""Rotary positions and the paged cache without a GPU: refusals, the programs' bytes and
schedules, and the oracle's forms against independent ones."""
import numpy as np
import pytest

import serving_util as SU
from oracle import vmref
from pjrt_amd import graph as G
from pjrt_amd import passes
from pjrt_amd import scheduler as S
from pjrt_amd import vmprogram as V


def run(prog, args, nlanes=8, reuse=True):
    """Both oracle validators on a scheduled program; the lanes' order must not matter."""
    cfg = S.DeviceConfig(nlanes=nlanes)
    if reuse:
        passes.reuse_arena(prog, cfg)
    blob = V.serialize(prog, S.schedule_program(prog, cfg))
    state = V.state_inputs(blob)
    twin = [a.copy() if i in state else a for i, a in enumerate(args)]
    a = vmref.execute(blob, twin)
    b = vmref.execute_schedule(blob, args)
    for x, y in zip(a + [twin[i] for i in state], b + [args[i] for i in state]):
        assert np.array_equal(x.view(np.uint8), y.view(np.uint8))
    assert V.serialize(V.parse(blob)) == blob
    return b


# ---- frequencies and angles ---------------------------------------------------------------

def test_turn_words_against_long_division():
    from decimal import Decimal, getcontext
    getcontext().prec = 60
    pi = Decimal("3.14159265358979323846264338327950288419716939937510582097494")
    for f in (1.0, 0.1, 1e-4, 2.5, 0.0, 1e-12):
        lo, hi = G.turn_words([f])[0]
        want = (Decimal(f) / (2 * pi)) % 1 * (1 << 64)
        assert abs((int(hi) << 32 | int(lo)) - want) <= Decimal("0.5000001")


def test_frequencies_scaled_for_long_contexts():
    plain = G.rotary_frequencies(128, 10000.0)
    assert plain[0] == 1.0 and np.isclose(plain[-1], 10000.0 ** (-126 / 128), rtol=1e-15)
    assert np.allclose(G.rotary_frequencies(128, factor=4.0), plain / 4, rtol=1e-15)
    f = G.rotary_frequencies(128, factor=8.0, original=4096)
    turns = plain * 4096 / (2 * np.pi)
    assert np.array_equal(f[turns >= 32], plain[turns >= 32])
    assert np.allclose(f[turns <= 1], plain[turns <= 1] / 8, rtol=1e-15)
    assert (np.diff(f) < 0).all()
    for bad in (dict(rot=3), dict(rot=0), dict(rot=8, factor=0.5), dict(rot=8, low=2.0, high=2.0)):
        with pytest.raises(G.GraphError):
            G.rotary_frequencies(**bad)


# ---- the oracle against forms of its own ---------------------------------------------------

@pytest.mark.parametrize("inter,norm,rot,inverse", [(False, True, 16, False), (True, False, 8, True), (True, True, 12, False)])
def test_oracle_rotary(inter, norm, rot, inverse):
    rng = np.random.default_rng(rot)
    x = rng.standard_normal((5, 3, 16)).astype(np.float32)
    pos = np.array([0, 3, 70000, -5, 12], np.int32)
    freq = G.rotary_frequencies(rot)
    w = rng.uniform(0.5, 1.5, 16).astype(np.float32) if norm else None
    (got,) = run(SU.rotary_program(x.shape, "f32", freq, norm, inter, 1.5, inverse), [x, pos] + ([w] if norm else []))
    want, mag = SU.rotary_plain(x, pos, freq, inter, 1.5, inverse, w)
    assert (np.abs(got - want) <= 2.0 ** -23 * mag).all()


def test_oracle_rotary_grad_against_differences():
    rng = np.random.default_rng(0)
    x, dy = rng.standard_normal((2, 3, 4, 12))
    pos, w = np.array([2, 5, 11]), rng.uniform(0.5, 1.5, 12)
    fw = G.turn_words(G.rotary_frequencies(8))
    dx, dw = vmref.rotary_grad(dy, x, pos, fw, 8, True, 1.3, w, 1e-3)

    def loss(x, w):
        return (vmref.rotary(x, pos, fw, 8, True, False, 1.3, w, 1e-3) * dy).sum()
    h = 1e-5
    for _ in range(20):
        i = tuple(rng.integers(0, s) for s in x.shape)
        e = np.zeros_like(x)
        e[i] = h
        # central differences: O(h^2) of third derivatives of order 10, and 1e-16 / h of rounding
        assert abs((loss(x + e, w) - loss(x - e, w)) / (2 * h) - dx[i]) < 1e-7
    for k in range(12):
        e = np.zeros(12)
        e[k] = h
        assert abs((loss(x, w + e) - loss(x, w - e)) / (2 * h) - dw[k]) < 1e-7


def test_rotary_grad_program():
    rng = np.random.default_rng(1)
    x, dy = (rng.standard_normal((9, 4, 16)).astype(np.float32) for _ in range(2))
    pos, w = np.arange(9, dtype=np.int32), rng.uniform(0.5, 1.5, 16).astype(np.float32)
    g = G.Graph()
    a = [g.input(x.shape), g.input(x.shape), g.input((9,), "i32"), g.input((16,))]
    g.output(*g.rotary_grad(a[0], a[1], a[2], G.rotary_frequencies(16), weight=a[3]))
    dx, dw = run(g.build(), [dy, x, pos, w])
    want, wdw = vmref.rotary_grad(dy.astype(np.float64), x, pos, G.turn_words(G.rotary_frequencies(16)), 16, False, 1.0, w,
                                  1e-6)
    assert np.allclose(dx, want, rtol=0, atol=2.0 ** -21) and np.allclose(dw, wdw, rtol=0, atol=2.0 ** -18)


@pytest.mark.parametrize("dt,cache,window", [("f32", "f32", 0), ("bf16", "bf16", 5), ("f32", "i8", 3)])
def test_oracle_attention(dt, cache, window):
    c = SU.Case([(1, 9), (3, 3), (0, 4), (4, 11)], 4, 2, 8, 4, dt, cache, pad=2, window=window, seed=1)
    (got,) = run(c.attention_program(), [*c.batch(), *c.state(), c.q])
    want, mag, top = c.attention()
    assert (np.abs(SU.to_f64(got, dt) - want) <= c.attention_tolerance(want, mag, top)).all()
    assert not SU.to_f64(got, dt)[c.cu[-1]:].any()


def test_oracle_attention_is_flash_attention_of_one_sequence():
    c = SU.Case([(6, 6)], 2, 2, 8, 4, "f32", seed=3)
    (got,) = run(c.attention_program(), [*c.batch(), *c.state(), c.q])
    k, v = (c.values(i, 0)[0].transpose(1, 0, 2) for i in range(2))
    want = vmref.attention(c.q.transpose(1, 0, 2), k.transpose(0, 2, 1), v, c.scale, True)
    assert np.allclose(got, want.transpose(1, 0, 2), rtol=0, atol=2e-6)


@pytest.mark.parametrize("cache", ["f32", "i8"])
def test_oracle_append_then_read(cache):
    """Whole sequences read back after an append, bad lengths and pages among them."""
    c = SU.Case([(2, 5), (3, 9), (4, 4), (2, 7)], 2, 2, 8, 4, "f32", cache, pad=1, seed=5, max_pages=3)
    c.lens[1], c.lens[2], c.table[3, 1] = 13, 3, c.N + 5
    before = c.state()
    g = G.Graph()
    b, pc = c.declare(g)
    g.cache_append(pc, b, g.input(c.k.shape), g.input(c.v.shape))
    g.output(*g.cache_read(pc, b, c.T))
    state = c.state()
    kk, vv = run(g.build(), [*c.batch(), *state, c.k, c.v])
    for got, x in ((kk, c.k), (vv, c.v)):
        for r in range(c.T):
            if r in (0, 1):
                step = 0.0 if cache == "f32" else np.abs(x[r]).max(-1, keepdims=True) / 254 * (1 + 1e-6)
                assert (np.abs(got[r] - x[r]) <= step).all()
            else:
                assert not got[r].any()
    # only positions 3 and 4 of sequence 0 were written
    for old, new in zip(before, state):
        changed = {tuple(i[[0, 2]]) for i in np.argwhere((old != new) & ~(np.isnan(old.astype(np.float64)) &
                                                                          np.isnan(new.astype(np.float64))))}
        assert changed <= {(c.table[0, 0], 3), (c.table[0, 1], 0)}


def test_quantised_rows():
    rng = np.random.default_rng(2)
    x = rng.standard_normal(64).astype(np.float32)
    q, s = vmref.quantise_row(x)
    assert np.abs(q).max() == 127 and (np.abs(q * s.astype(np.float64) - x) <= s * (0.5 + 1e-5)).all()
    assert vmref.quantise_row(np.zeros(8))[1] == 0 and not vmref.quantise_row(np.zeros(8))[0].any()
    for bad in (np.inf, np.nan):
        x[3] = bad
        assert np.isnan(vmref.quantise_row(x)[1])


# ---- refusals -------------------------------------------------------------------------------

def test_rotary_refusals():
    g = G.Graph()
    x, pos, f = g.input((4, 2, 16)), g.input((4,), "i32"), G.rotary_frequencies(16)
    w = g.input((16,))
    for call in (
            lambda: g.rotary(g.input((4, 32)), pos, f), lambda: g.rotary(x, g.input((5,), "i32"), f),
            lambda: g.rotary(x, g.input((4,)), f), lambda: g.rotary(x, pos, G.rotary_frequencies(18)),
            lambda: g.rotary(x, pos, []), lambda: g.rotary(x, pos, [np.inf]), lambda: g.rotary(x, pos, f, weight=pos),
            lambda: g.rotary(x, pos, f, weight=w, eps=-1.0), lambda: g.rotary(x, pos, f, weight=g.input((8,))),
            lambda: g.rotary(g.input((4, 2, 16), "i32"), pos, f), lambda: g.rotary(g.input((4, 2, 258)), pos, f),
            lambda: g.rotary(g.input((4, 2, 15)), pos, f[:4]), lambda: g.rotary(g.view(x, (4, 2, 16), (16, 1, 2), 0), pos, f),
            lambda: g.rotary_grad(x, g.input((4, 2, 16), "bf16"), pos, f, weight=w),
            lambda: g.rotary_grad(g.input((4, 1, 16)), x, pos, f, weight=w)):
        with pytest.raises(G.GraphError):
            call()


def test_cache_refusals():
    g = G.Graph()
    for bad in (dict(pages=0), dict(heads=0), dict(page=0), dict(head_dim=12), dict(head_dim=264), dict(dtype="i32"),
                dict(page=1 << 17), dict(pages=1 << 33)):
        with pytest.raises(G.GraphError):
            g.paged_cache(**{**dict(pages=4, heads=2, page=8, head_dim=16, dtype="bf16"), **bad})
    c = g.paged_cache(4, 2, 8, 16, "bf16")
    b = g.paged_batch(3, 5)
    new = g.input((6, 2, 16), "bf16")
    for call in (
            lambda: g.cache_append(c, b, new, g.input((6, 2, 16), "f16")),
            lambda: g.cache_append(c, b, g.input((6, 2, 16)), g.input((6, 2, 16))),
            lambda: g.cache_append(c, b, g.input((6, 4, 16), "bf16"), g.input((6, 4, 16), "bf16")),
            lambda: g.cache_append(c, b, new, g.input((5, 2, 16), "bf16")),
            lambda: g.cache_read(c, b, 0), lambda: g.cache_read(c, b, 4, "i8"),
            lambda: g.paged_attention(g.input((6, 3, 16), "bf16"), c, b, 1.0),
            lambda: g.paged_attention(g.input((6, 4, 8), "bf16"), c, b, 1.0),
            lambda: g.paged_attention(g.input((6, 4, 16)), c, b, 1.0),
            lambda: g.paged_attention(g.input((6, 4, 16), "bf16"), c, b, 0.0),
            lambda: g.paged_attention(g.input((6, 4, 16), "bf16"), c, b, 1.0, window=-1),
            lambda: g.paged_attention(g.input((6, 2 * 129, 16), "bf16"), c, b, 1.0),
            lambda: g.paged_batch(0, 1), lambda: g.output(c.k), lambda: g.alias(c.k, 0, (8,)),
            lambda: g.paged_attention(g.input((6, 4, 16), "bf16"), c,
                                      G.PagedBatch(g.input((3,), "i32"), b.lens, b.table), 1.0)):
        with pytest.raises(G.GraphError):
            call()


# ---- states, phases, schedules ----------------------------------------------------------------

def test_state_buffers_take_no_arena():
    """A pool far larger than an arena can be; its bytes survive the round trip, and a program
    that calls it an output is refused."""
    g = G.Graph()
    b, c = g.paged_batch(1, 4), g.paged_cache(40000, 8, 64, 128, "bf16")
    q = g.input((1, 8, 128), "bf16")
    g.output(g.paged_attention(q, c, b, 0.1))
    prog = g.build()
    assert prog.arena_bytes < 1 << 16
    passes.reuse_arena(prog, S.DeviceConfig(nlanes=8))
    assert prog.arena_bytes < 1 << 16 and prog.buffers[c.k.buf].arena_byte_offset >= prog.arena_bytes
    blob = V.serialize(prog, S.schedule_program(prog, S.DeviceConfig(nlanes=8)))
    assert V.state_inputs(blob) == (3, 4)
    back = V.parse(blob)
    assert [x.state for x in back.buffers] == [x.state for x in prog.buffers]
    back.outputs.append(c.k.buf)
    back.output_shapes.append(c.k.shape)
    for parse in (V.parse, vmref.parse):
        with pytest.raises((V.FormatError, vmref.FormatError)):
            parse(V.serialize(back, back.schedule))


def test_append_runs_before_attention_and_after_the_last_reader():
    g = G.Graph()
    b, c = g.paged_batch(2, 4), g.paged_cache(8, 2, 8, 16, "f32")
    q, k, v = g.input((3, 4, 16)), g.input((3, 2, 16)), g.input((3, 2, 16))
    o1 = g.paged_attention(q, c, b, 0.25)
    g.cache_append(c, b, k, v)
    g.output(o1, g.paged_attention(q, c, b, 0.25))
    sched = S.schedule_program(g.build(), S.DeviceConfig(nlanes=8))
    order, at = [], 0
    for e in sched.lane_streams[0]:
        if e.task == V.ENT_BARRIER:
            at += 1
    assert at == 2                       # attention, append, attention: a barrier between each


def test_layers_share_the_split_scratch_only_apart():
    """Attention over two caches of one phase, and in later phases: the schedule keeps
    every tile once (the lane simulator checks the coverage)."""
    c = SU.Case([(2, 6), (1, 9)], 4, 2, 8, 4, "f32", seed=8)
    g = G.Graph()
    b, c1 = c.declare(g)
    c2 = g.paged_cache(c.N, 2, 4, 8, "f32")
    q = g.input(c.q.shape)
    o1, o2 = g.paged_attention(q, c1, b, c.scale), g.paged_attention(q, c2, b, c.scale)
    g.output(g.add(o1, o2))
    (got,) = run(g.build(), [*c.batch(), *c.state(), *c.state(), c.q])
    want, mag, top = c.attention()
    assert (np.abs(got - 2 * want) <= 4 * c.attention_tolerance(want, mag, top)).all()
