"""Rotary positions and the paged cache on the GPU, against plain forms in 64 bits."""
import numpy as np
import pytest

import gpu_util
import serving_util as SU
from pjrt_amd import graph as G
from pjrt_amd import vmprogram as V
from pjrt_amd.runtime import INVALID_ARGUMENT, VmrtError

pytestmark = pytest.mark.gpu


def compiled(prog, **kw):
    return gpu_util.runtime().compile(prog, **kw)


def check(got, want, tol, what=""):
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.size}, first {[tuple(i) for i in np.argwhere(bad)[:4]]}: " \
                          f"{got[bad][:4]} for {want[bad][:4]}, allowed {np.broadcast_to(tol, bad.shape)[bad][:4]}"


# ---- rotary ----------------------------------------------------------------------------------
# f32 work of one element: two products and a sum of a pair (3 roundings), the sine and
# cosine off by at most 4 steps, the norm's sum of squares (a lane's run and the lanes' tree:
# at most 24 roundings, halved by the root), root, quotient and two products: 32 covers it
ROT_F32 = 32 * 2.0 ** -24


@pytest.mark.parametrize("T,H,hd,rot,dt,inter,norm", [
    (1, 1, 2, 2, "f32", False, False), (1, 16, 128, 128, "bf16", False, True), (3, 5, 64, 64, "f16", True, True),
    (7, 40, 128, 64, "bf16", True, False), (33, 2, 80, 20, "f32", False, True), (130, 9, 96, 24, "bf16", False, True),
    (5, 3, 256, 256, "f32", True, True), (4, 7, 250, 34, "bf16", False, True), (300, 3, 10, 6, "f16", True, True),
    (1025, 8, 128, 128, "bf16", False, True), (2, 67, 32, 32, "f32", False, False), (6, 4, 256, 2, "f16", False, True)])
def test_rotary(T, H, hd, rot, dt, inter, norm):
    rng = np.random.default_rng(T * 1000 + hd)
    x = SU.to_dt(rng.standard_normal((T, H, hd)), dt)
    pos = rng.integers(-50, 100000, T).astype(np.int32)
    freq = G.rotary_frequencies(rot)
    w = rng.uniform(0.5, 1.5, hd).astype(np.float32) if norm else None
    lp = compiled(SU.rotary_program((T, H, hd), dt, freq, norm, inter, magnitude=1.25))
    (got,) = lp(x, pos, *([w] if norm else []))
    want, mag = SU.rotary_plain(SU.to_f64(x, dt), pos, freq, inter, 1.25, weight=w)
    check(SU.to_f64(got, dt), want, SU.U[dt] * np.abs(want) + ROT_F32 * mag)


def test_rotary_far_positions():
    """The whole range of 32-bit positions, negative ones too: angles lose nothing."""
    pos = np.array([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 10 ** 9 + 7, 123456789], np.int32)
    freq = G.rotary_frequencies(64, 500000.0, factor=8.0, original=8192)
    x = np.random.default_rng(1).standard_normal((len(pos), 2, 64)).astype(np.float32)
    (got,) = compiled(SU.rotary_program(x.shape, "f32", freq, False, False))(x, pos)
    words = [(int(h) << 32 | int(l)) for l, h in G.turn_words(freq)]
    turns = np.array([[(int(p) * w) % 2 ** 64 / 2 ** 64 * 2 * np.pi for w in words] for p in pos])
    c, s = np.cos(turns)[:, None], np.sin(turns)[:, None]
    a, b = x[..., :32].astype(np.float64), x[..., 32:].astype(np.float64)
    want = np.concatenate([a * c - b * s, b * c + a * s], -1)
    mag = np.concatenate([np.abs(a) + np.abs(b)] * 2, -1)
    check(got, want, ROT_F32 * mag)


def test_rotary_view_and_inverse():
    """Queries and keys inside the rows of a fused projection, at any offset, and back."""
    rng = np.random.default_rng(5)
    T, hq, hkv, hd = 37, 6, 2, 64
    for dt, off in (("bf16", 0), ("f32", 3), ("f16", 1)):
        width = (hq + 2 * hkv) * hd + 5
        x = SU.to_dt(rng.standard_normal((T, width)), dt)
        pos = np.arange(T, dtype=np.int32)
        freq = G.rotary_frequencies(hd)
        g = G.Graph()
        src, p = g.input((T, width), dt), g.input((T,), "i32")
        y = g.rotary(g.view(src, (T, hkv, hd), (width, hd, 1), hq * hd + off), p, freq)
        g.output(y, g.rotary(y, p, freq, inverse=True))
        got, back = compiled(g.build())(x, pos)
        part = SU.to_f64(x, dt)[:, hq * hd + off:(hq + hkv) * hd + off].reshape(T, hkv, hd)
        want, mag = SU.rotary_plain(part, pos, freq, False)
        check(SU.to_f64(got, dt), want, SU.U[dt] * np.abs(want) + ROT_F32 * mag)
        # two roundings of each of the pair's two terms on the way there and back
        pair = np.abs(part) + np.abs(np.concatenate([part[..., 32:], part[..., :32]], -1))
        check(SU.to_f64(back, dt), part, (3 * SU.U[dt] + 2 * ROT_F32) * 2 * pair)


@pytest.mark.parametrize("T,H,hd,rot,dt,inter", [
    (1, 1, 64, 64, "f32", False), (9, 3, 128, 128, "bf16", False), (50, 5, 80, 20, "f32", True),
    (257, 32, 128, 64, "bf16", True), (64, 2, 250, 250, "f16", False), (1000, 1, 32, 16, "f32", False)])
def test_rotary_grad(T, H, hd, rot, dt, inter):
    rng = np.random.default_rng(T + hd)
    x, dy = (SU.to_dt(rng.standard_normal((T, H, hd)), dt) for _ in range(2))
    pos = rng.integers(0, 5000, T).astype(np.int32)
    w = rng.uniform(0.5, 1.5, hd).astype(np.float32)
    freq = G.rotary_frequencies(rot)
    g = G.Graph()
    ins = [g.input((T, H, hd), dt), g.input((T, H, hd), dt), g.input((T,), "i32"), g.input((hd,), "f32")]
    g.output(*g.rotary_grad(ins[0], ins[1], ins[2], freq, weight=ins[3], interleaved=inter, magnitude=1.1))
    lp = compiled(g.build())
    dx, dw = lp(dy, x, pos, w)
    x64, dy64 = SU.to_f64(x, dt), SU.to_f64(dy, dt)
    dz, mag = SU.rotary_plain(dy64, pos, freq, inter, 1.1, inverse=True)
    r = 1.0 / np.sqrt((x64 ** 2).mean(-1, keepdims=True) + 1e-6)
    u, gz = x64 * r, dz * w
    want = r * (gz - u * (gz * u).mean(-1, keepdims=True))
    big = r * (mag * w + np.abs(u) * (mag * w * np.abs(u)).mean(-1, keepdims=True))
    # twice a rotation's work, and a second sum over the head
    check(SU.to_f64(dx, dt), want, SU.U[dt] * np.abs(want) + 3 * ROT_F32 * big)
    # a sum of T H terms in some tree: at most T H roundings, far fewer in fact; each term as above
    check(dw, (dz * u).sum((0, 1)), (2 * ROT_F32 + np.sqrt(T * H) * 4 * 2.0 ** -24 + 64 * 2.0 ** -24) * (mag * np.abs(u)).sum((0, 1)))
    again, dw2 = lp(dy, x, pos, w)
    assert np.array_equal(again, dx) and np.array_equal(dw2, dw)       # the same order every time


# ---- the cache ---------------------------------------------------------------------------------

CACHES = [
    # seqs (new, length), heads, head dim, page, type, cache
    ([(1, 1)], 1, 8, 1, "f32", "f32"), ([(1, 17), (1, 5), (1, 16)], 3, 64, 16, "bf16", "bf16"),
    ([(5, 21), (0, 9), (70, 70), (1, 40)], 2, 80, 7, "f16", "f16"), ([(300, 411)], 4, 128, 64, "bf16", "i8"),
    ([(2, 3), (9, 100), (33, 33)], 5, 96, 24, "f16", "i8"), ([(4, 4), (3, 1000)], 1, 256, 128, "f32", "i8"),
    ([(1, i + 1) for i in range(130)], 2, 16, 3, "bf16", "i8"), ([(513, 600)], 3, 72, 16, "f32", "f32")]


def slot_of(c, i, p):
    return int(c.table[i, p // c.page]), p % c.page


def append_want(c, k, v):
    """The pools after an append, row by row."""
    from oracle import vmref
    pools, scales = [p.copy() for p in c.pools], [s.copy() for s in c.scales]
    for i in range(len(c.seqs)):
        a, b, length = int(c.cu[i]), int(c.cu[i + 1]), int(c.lens[i])
        if b <= a or length < b - a or length > c.MP * c.page:
            continue
        for r in range(a, b):
            pg, sl = slot_of(c, i, length - (b - r))
            if not 0 <= pg < c.N:
                continue
            for m, x in enumerate((k, v)):
                if c.cache == "i8":
                    for h in range(c.hkv):
                        q, s = vmref.quantise_row(SU.to_f64(x[r, h], c.dt))
                        pools[m][pg, h, sl], scales[m][pg, h, sl] = q, s
                else:
                    pools[m][pg, :, sl] = x[r]
    return pools + scales


def same(a, b):
    """Bit for bit, with NaN equal to NaN of the same pattern."""
    assert a.dtype == b.dtype and a.shape == b.shape
    assert np.array_equal(a.view(np.uint8), b.view(np.uint8)), f"{int((a.view(np.uint8) != b.view(np.uint8)).sum())} bytes"


@pytest.mark.parametrize("case", range(len(CACHES)))
@pytest.mark.parametrize("pad", [0, 3])
def test_cache_append_and_read(case, pad):
    seqs, hkv, hd, page, dt, cache = CACHES[case]
    c = SU.Case(seqs, hkv, hkv, hd, page, dt, cache, pad=pad, seed=case)
    g = G.Graph()
    b, pc = c.declare(g)
    g.cache_append(pc, b, g.input(c.k.shape, dt), g.input(c.v.shape, dt))
    out = "f32" if cache == "i8" else dt
    g.output(*g.cache_read(pc, b, c.T, out))
    state = c.state()
    kk, vv = compiled(g.build())(*c.batch(), *state, c.k, c.v)
    want = append_want(c, c.k, c.v)
    for got, w in zip(state, want):
        same(got, w)
    c.pools, c.scales = want[:2], want[2:]
    for got, m in ((kk, 0), (vv, 1)):
        ref = np.zeros(c.k.shape)
        for i in range(len(seqs)):
            n = int(c.cu[i + 1] - c.cu[i])
            if n:
                x, ok = c.values(m, i)
                ref[c.cu[i]:c.cu[i + 1]] = x[-n:]
        check(SU.to_f64(got, out), ref, (2.0 ** -24 if cache == "i8" else 0.0) * np.abs(ref))


def test_cache_append_special_rows():
    """i8 rows of zeros, with an infinity, with a NaN, at the type's largest value and of
    denormals."""
    c = SU.Case([(6, 6)], 1, 1, 64, 4, "f32", "i8")
    c.k[0] = 0.0
    c.k[1, 0, 5] = np.inf
    c.k[2, 0, 63] = np.nan
    c.k[3] = np.float32(3.4e38)
    c.k[4] = np.float32(1e-42)
    g = G.Graph()
    b, pc = c.declare(g)
    g.cache_append(pc, b, g.input(c.k.shape, "f32"), g.input(c.v.shape, "f32"))
    state = c.state()
    compiled(g.build())(*c.batch(), *state, c.k, c.v)
    want = append_want(c, c.k, c.v)
    for got, w in zip(state[:2], want[:2]):
        same(got, w)
    for got, w in zip(state[2:], want[2:]):
        assert np.array_equal(np.isnan(got), np.isnan(w)) and np.array_equal(got[~np.isnan(w)], w[~np.isnan(w)])


@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cache", ["f32", "f16", "bf16", "i8"])
def test_cache_read_into_other_types(cache, out):
    """Pages of every type read as every type, rounded once (f16's smallest steps are 2^-24;
    an i8 value is a product rounded to f32 first)."""
    dt = "bf16" if cache == "i8" else cache
    c = SU.Case([(5, 30), (1, 9), (70, 100)], 3, 3, 40, 8, dt, cache, pad=1, seed=6)
    g = G.Graph()
    b, pc = c.declare(g)
    g.output(*g.cache_read(pc, b, c.T, out))
    kk, vv = compiled(g.build())(*c.batch(), *c.state())
    for got, m in ((kk, 0), (vv, 1)):
        ref = np.zeros(c.k.shape)
        for i, (n, _) in enumerate(c.seqs):
            ref[c.cu[i]:c.cu[i + 1]] = c.values(m, i)[0][-n:]
        eps = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[out] + (2.0 ** -24 if cache == "i8" else 0.0)
        if out == cache or out == "f32" and cache != "i8":
            eps = 0.0
        check(SU.to_f64(got, out), ref, eps * np.abs(ref) + (2.0 ** -25 if out == "f16" and eps else 0.0))


def test_cache_append_from_views():
    """Keys and values inside the rows of a fused projection."""
    c = SU.Case([(19, 30), (4, 4)], 4, 2, 64, 16, "bf16")
    width = 8 * 64 + 1
    rows = SU.to_dt(np.random.default_rng(3).standard_normal((c.T, width)), "bf16")
    g = G.Graph()
    b, pc = c.declare(g)
    src = g.input(rows.shape, "bf16")
    g.cache_append(pc, b, g.view(src, (c.T, 2, 64), (width, 64, 1), 4 * 64), g.view(src, (c.T, 2, 64), (width, 64, 1), 6 * 64 + 1))
    state = c.state()
    compiled(g.build())(*c.batch(), *state, rows)
    k, v = rows[:, 256:384].reshape(c.T, 2, 64), rows[:, 385:513].reshape(c.T, 2, 64)
    for got, w in zip(state, append_want(c, k, v)):
        same(got, w)


@pytest.mark.parametrize("cache", ["f32", "i8"])
def test_cache_bad_batches(cache):
    """Lengths that do not fit and table entries that are no page: nothing is written
    there, reads give zeros, and every other row is served."""
    c = SU.Case([(4, 9), (6, 20), (5, 5), (3, 8)], 2, 2, 32, 4, "f32", cache, pad=2, seed=2, max_pages=6)
    c.lens[1] = 25                      # more than six pages of four hold
    c.lens[2] = 4                       # less than its new rows
    c.table[3, 1] = c.N                 # one past the last page
    c.table[0, 2] = -7
    g = G.Graph()
    b, pc = c.declare(g)
    g.cache_append(pc, b, g.input(c.k.shape, "f32"), g.input(c.v.shape, "f32"))
    g.output(*g.cache_read(pc, b, c.T, "f32"))
    state = c.state()
    kk, _ = compiled(g.build())(*c.batch(), *state, c.k, c.v)
    want = append_want(c, c.k, c.v)
    for got, w in zip(state, want):
        same(got, w)
    live = np.zeros(c.T, bool)
    live[0:3] = True                    # positions 5..7 of sequence 0; position 8 lies in the entry -7
    assert not kk[~live].any() and kk[live].any(axis=(1, 2)).all()


# ---- attention -----------------------------------------------------------------------------------

ATTEND = [
    # seqs (new, length), hq, hkv, hd, page, dt, cache, pad, window
    ([(1, 1)], 1, 1, 8, 1, "f32", "f32", 0, 0),
    ([(1, 1)], 4, 2, 64, 16, "bf16", "bf16", 0, 0),
    ([(1, 1000)], 12, 12, 64, 16, "bf16", "bf16", 0, 0),
    ([(1, 127), (1, 128), (1, 129), (1, 33)], 8, 2, 128, 16, "bf16", "bf16", 2, 0),
    ([(1, 700 + 37 * i) for i in range(40)], 8, 2, 128, 16, "f16", "f16", 0, 0),
    ([(1, 9000)], 8, 8, 128, 64, "bf16", "bf16", 0, 0),
    ([(1, 9000), (1, 3)], 8, 2, 128, 24, "bf16", "i8", 1, 0),
    ([(3, 50), (8, 8), (1, 600), (0, 77), (17, 300)], 16, 4, 80, 24, "f16", "f16", 5, 0),
    ([(300, 300)], 4, 4, 64, 16, "bf16", "bf16", 0, 0),
    ([(300, 1111)], 8, 2, 128, 64, "bf16", "bf16", 0, 0),
    ([(513, 640), (1, 900), (63, 64), (65, 1000)], 6, 2, 96, 7, "f16", "f16", 3, 0),
    ([(200, 900), (1, 900), (40, 41)], 8, 1, 64, 100, "bf16", "i8", 0, 0),
    ([(200, 900), (1, 900), (40, 41)], 8, 2, 64, 16, "f16", "f16", 0, 128),
    ([(1, 900), (1, 100), (129, 129), (1000, 1500)], 4, 2, 128, 16, "bf16", "bf16", 1, 777),
    ([(150, 500), (1, 129)], 6, 2, 96, 16, "f32", "f32", 2, 0),
    ([(30, 100), (1, 1500)], 4, 4, 128, 32, "f32", "i8", 0, 64),
    ([(5, 60), (1, 300)], 2, 1, 256, 16, "bf16", "bf16", 0, 0),
    ([(20, 90), (1, 300)], 4, 2, 200, 16, "f16", "i8", 0, 50),
    ([(2, 300), (1, 10)], 256, 2, 64, 16, "bf16", "bf16", 0, 0),
    ([(70, 200)], 96, 1, 64, 8, "bf16", "bf16", 0, 0),
    ([(1, 2)] * 300, 2, 1, 64, 16, "bf16", "bf16", 0, 0),
    ([(9, 4000)] * 3, 5, 1, 128, 16, "f16", "f16", 0, 1),
    # f32 on the matrix cores: 16, 32 and 64 rows a block, heads wider than a block, both caches
    ([(1, 2000), (5, 17), (16, 16), (1, 15)], 6, 2, 64, 16, "f32", "f32", 1, 0),
    ([(7, 700), (9, 333), (40, 40)], 8, 4, 96, 16, "f32", "f32", 0, 200),
    ([(1, 5000), (130, 300)], 8, 1, 128, 24, "f32", "f32", 0, 0),
    ([(1, 3000), (20, 500), (3, 3)], 10, 2, 80, 7, "f32", "i8", 2, 0),
    ([(33, 700)], 4, 2, 128, 64, "f32", "i8", 0, 333),
    ([(2, 200)], 70, 1, 64, 16, "f32", "f32", 0, 0),
    ([(1, 300), (4, 90)], 6, 3, 72, 16, "f32", "i8", 0, 0),
    ([(1, 300), (4, 90)], 6, 3, 72, 16, "f32", "f32", 0, 0),
    # items cut into many pieces, on few workers' boundaries and many
    ([(1, 60000)], 2, 1, 64, 64, "bf16", "bf16", 0, 0),
    ([(2, 30000), (1, 31000), (1, 5)], 4, 2, 128, 16, "bf16", "i8", 0, 0),
    ([(100, 20000)], 4, 1, 64, 16, "f16", "f16", 0, 0),
    ([(1, 20000), (3, 4)], 2, 1, 128, 16, "f32", "f32", 0, 0),
]


@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_paged_attention(case):
    seqs, hq, hkv, hd, page, dt, cache, pad, window = ATTEND[case]
    c = SU.Case(seqs, hq, hkv, hd, page, dt, cache, pad, window, seed=case)
    lp = compiled(c.attention_program())
    (got,) = lp(*c.batch(), *c.state(), c.q)
    want, mag, top = c.attention()
    check(SU.to_f64(got, dt), want, c.attention_tolerance(want, mag, top))
    (again,) = lp(*c.batch(), *c.state(), c.q)
    assert np.array_equal(again, got)
    assert not SU.to_f64(got, dt)[c.cu[-1]:].any()


@pytest.mark.parametrize("dt,cache,hd", [("bf16", "bf16", 64), ("f16", "i8", 128), ("f32", "f32", 96), ("bf16", "i8", 64),
                                         ("f32", "i8", 128), ("f32", "f32", 136)])
def test_paged_attention_bad_batches(dt, cache, hd):
    c = SU.Case([(4, 90), (6, 190), (50, 50), (30, 80), (1, 150)], 4, 2, hd, 16, dt, cache, pad=2, seed=7, max_pages=12,
                first=1)
    c.lens[1] = 193                     # more than twelve pages of sixteen hold
    c.lens[2] = 49                      # less than its new rows
    c.table[3, 1] = c.N                 # positions 16..31 are nowhere
    c.table[4, :] = -1                  # nothing to see
    (got,) = compiled(c.attention_program())(*c.batch(), *c.state(), c.q)
    want, mag, top = c.attention()
    check(SU.to_f64(got, dt), want, c.attention_tolerance(want, mag, top))
    out = SU.to_f64(got, dt)
    assert not out[0].any() and not out[c.cu[1]:c.cu[3]].any() and not out[c.cu[4]:].any()


@pytest.mark.parametrize("cache", ["bf16", "i8"])
def test_rows_outside_the_step(cache):
    """A sequence whose rows reach past the step's, or lie before them, is not served: append
    and read skip it, its rows' attention is 0."""
    c = SU.Case([(4, 40), (6, 60), (5, 30)], 2, 2, 64, 16, "bf16", cache, seed=4)
    state = c.state()
    c.cu[0], c.cu[3] = -2, c.T + 3
    g = G.Graph()
    b, pc = c.declare(g)
    g.cache_append(pc, b, g.input(c.k.shape, "bf16"), g.input(c.v.shape, "bf16"))
    g.output(g.paged_attention(g.input(c.q.shape, "bf16"), pc, b, c.scale), *g.cache_read(pc, b, c.T, "f32"))
    before = [x.copy() for x in state]
    out, kk, vv = compiled(g.build())(*c.batch(), *state, c.k, c.v, c.q)
    out, live = SU.to_f64(out, "bf16"), np.zeros(c.T, bool)
    live[4:10] = True
    for x in (out, kk, vv):
        assert not x[~live].any() and x[live].any(axis=(1, 2)).all()
    for i, n in ((0, range(36, 40)), (2, range(25, 30))):
        for p in n:
            pg, sl = slot_of(c, i, p)
            for x, y in zip(state, before):
                same(np.ascontiguousarray(x[pg, :, sl]), np.ascontiguousarray(y[pg, :, sl]))


def test_attentions_of_other_shapes_share_scratch():
    """Attention of several shapes in one program, each cut into pieces: their partials use the
    same memory one after another, in every launch."""
    cases = [SU.Case([(1, 40000)], 2, 1, 64, 64, "bf16", seed=1), SU.Case([(50, 9000), (1, 5000)], 8, 2, 128, 16, "bf16", seed=2),
             SU.Case([(3, 7000)], 10, 5, 96, 16, "f32", seed=3)]
    g = G.Graph()
    ins, outs = [], []
    for c in cases:
        b, pc = c.declare(g)
        q = g.input(c.q.shape, c.dt)
        outs.append(g.paged_attention(q, pc, b, c.scale))
        ins += [*c.batch(), *c.state(), c.q]
    g.output(*outs)
    lp = compiled(g.build())
    first = lp(*ins)
    for c, got in zip(cases, first):
        want, mag, top = c.attention()
        check(SU.to_f64(got, c.dt), want, c.attention_tolerance(want, mag, top))
    for _ in range(3):
        for got, was in zip(lp(*ins), first):
            assert np.array_equal(got, was)


@pytest.mark.parametrize("dt,cache,hd", [("bf16", "bf16", 128), ("f16", "f16", 64), ("f32", "f32", 64), ("bf16", "i8", 128),
                                         ("f32", "i8", 64), ("f32", "f32", 200)])
def test_paged_attention_ignores_what_it_does_not_see(dt, cache, hd):
    """NaN and infinities at positions after a row's own and before its window, inside the
    tiles that other rows need: rows that do not see them are as without them."""
    seqs = [(40, 200), (1, 300), (3, 3)]
    c = SU.Case(seqs, 4, 2, hd, 16, dt, cache, window=100, seed=3)
    clean, (a, m, top) = c.state(), c.attention()
    # sequence 0's last position: its earlier rows do not see it; its position 65: rows from 166 on do not
    for p, bad in ((199, np.nan), (65, np.inf)):
        pg, sl = slot_of(c, 0, p)
        for k in range(2):
            if cache == "i8":
                c.scales[k][pg, :, sl] = bad
            else:
                c.pools[k][pg, :, sl] = SU.to_dt(np.full((2, hd), bad), cache)
    (got,) = compiled(c.attention_program())(*c.batch(), *c.state(), c.q)
    out, tol = SU.to_f64(got, dt), c.attention_tolerance(a, m, top)
    rows = np.r_[6:39, 40:44]            # sequence 0's rows 6.. see positions 67.. and up
    check(out[rows], a[rows], tol[rows])
    assert np.isnan(out[39]).any() and not np.isfinite(out[0:5]).all()


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_paged_attention_rising_scores(dt):
    """Scores that grow by hundreds along the keys and ones that are all very low."""
    for sign in (1.0, -1.0):
        c = SU.Case([(1, 1000), (64, 700), (2, 300)], 4, 2, 64, 16, dt, seed=5)
        q, k = SU.to_f64(c.q, dt), SU.to_f64(c.pools[0], dt)
        q[:] = 0.0
        q[..., 0] = 8.0
        c.q = SU.to_dt(q, dt)
        for i, (_, length) in enumerate(c.seqs):
            for p in range(length):
                pg, sl = slot_of(c, i, p)
                k[pg, :, sl, 0] = sign * p * 0.25
        c.pools[0] = SU.to_dt(k, dt)
        (got,) = compiled(c.attention_program())(*c.batch(), *c.state(), c.q)
        want, mag, top = c.attention()
        check(SU.to_f64(got, dt), want, c.attention_tolerance(want, mag, top))


def test_long_cache_offsets():
    """Pools of more than 2^32 bytes: positions in the first and last pages."""
    rt = gpu_util.runtime()
    N, page, hkv, hd = (1 << 32) // (64 * 8 * 128 * 2) + 40, 64, 8, 128
    T, length = 3, 180
    g = G.Graph()
    b = g.paged_batch(1, 4)
    pc = g.paged_cache(N, hkv, page, hd, "bf16")
    g.cache_append(pc, b, g.input((T, hkv, hd), "bf16"), g.input((T, hkv, hd), "bf16"))
    g.output(g.paged_attention(g.input((T, 16, hd), "bf16"), pc, b, hd ** -0.5))
    lp = rt.compile(g.build())
    rng = np.random.default_rng(1)
    table = np.array([[N - 1, 0, N - 7, 5]], np.int32)
    nb = hkv * page * hd * 2
    pages = [SU.to_dt(rng.standard_normal((4, hkv, page, hd)), "bf16") for _ in range(2)]
    pools = [rt.alloc(N * nb) for _ in range(2)]
    for pool, x in zip(pools, pages):
        for i in range(4):
            rt.h2d(pool.ptr + int(table[0, i]) * nb, np.ascontiguousarray(x[i]).ctypes.data, nb)
    k, v = (SU.to_dt(rng.standard_normal((T, hkv, hd)), "bf16") for _ in range(2))
    q = SU.to_dt(rng.standard_normal((T, 16, hd)), "bf16")
    small = [rt.to_device(x) for x in (np.array([0, T], np.int32), np.array([length], np.int32), table)]
    (out,) = lp.execute(small + pools + [rt.to_device(x) for x in (k, v, q)])
    got = SU.to_f64(out.to_host(np.uint16, (T, 16, hd)), "bf16")
    for x, new in zip(pages, (k, v)):
        for t in range(T):
            p = length - T + t
            x[p // page, :, p % page] = new[t]
    for pool, x in zip(pools, pages):
        back = np.empty((hkv, page, hd), np.uint16)
        for i in range(4):
            rt.d2h(back.ctypes.data, pool.ptr + int(table[0, i]) * nb, nb)
            assert np.array_equal(back, x[i])
    at = np.arange(length)
    kk, vv = (SU.to_f64(x[at // page, :, at % page], "bf16").repeat(2, 1) for x in pages)
    for t in range(T):
        n = length - T + t + 1
        s = np.einsum("jhd,hd->hj", kk[:n], SU.to_f64(q[t], "bf16")) * hd ** -0.5
        w = np.exp(s - s.max(-1, keepdims=True))
        w /= w.sum(-1, keepdims=True)
        want, mag = np.einsum("hj,jhd->hd", w, vv[:n]), np.einsum("hj,jhd->hd", w, np.abs(vv[:n]))
        # half a step of P and of the output; f32 sums of scores up to about 6
        check(got[t], want, 2.0 ** -8 * (2 * mag + np.abs(want)) + 2 * 4000 * 2.0 ** -24 * mag)
    for x in pools:
        x.free()
    lp.close()


def test_state_inputs_are_checked():
    """A state buffer that meets another buffer of the launch, or is not aligned, is refused."""
    rt = gpu_util.runtime()
    c = SU.Case([(2, 5)], 1, 1, 64, 4, "f32")
    g = G.Graph()
    b, pc = c.declare(g)
    g.cache_append(pc, b, g.input(c.k.shape, "f32"), g.input(c.v.shape, "f32"))
    g.output(*g.cache_read(pc, b, c.T, "f32"))
    lp = rt.compile(g.build())
    dev = [rt.to_device(x) for x in [*c.batch(), *c.pools, c.k, c.v]]
    outs = lp.alloc_outputs()
    for at, value in ((3, dev[4].ptr), (3, dev[4].ptr + 16), (4, dev[5].ptr), (3, outs[0].ptr), (3, dev[3].ptr + 4)):
        ins = list(dev)
        ins[at] = value
        with pytest.raises(VmrtError) as e:
            lp.execute(ins, outs)
        assert e.value.code == INVALID_ARGUMENT
    lp.execute(dev, outs)


def step_program(c, freq, layers):
    """Layers of a step: norm and rotation of queries and keys inside the fused rows, keys and
    values into the cache, attention, and the next layer's rows from its output."""
    g = G.Graph()
    hq, hkv, hd = c.hq, c.hkv, c.hd
    width = (hq + 2 * hkv) * hd
    x, pos = g.input((c.T, hq * hd), c.dt), g.input((c.T,), "i32")
    b = g.paged_batch(len(c.seqs), c.MP)
    w = g.input((hd,), "f32")
    for _ in range(layers):
        pc = g.paged_cache(c.N, hkv, c.page, hd, c.cache)
        rows = g.dot(x, g.input((hq * hd, width), c.dt), out_dtype=c.dt)
        q = g.rotary(g.view(rows, (c.T, hq, hd), (width, hd, 1), 0), pos, freq, weight=w)
        k = g.rotary(g.view(rows, (c.T, hkv, hd), (width, hd, 1), hq * hd), pos, freq, weight=w)
        g.cache_append(pc, b, k, g.view(rows, (c.T, hkv, hd), (width, hd, 1), (hq + hkv) * hd))
        x = g.reshape(g.paged_attention(q, pc, b, c.scale, c.window), (c.T, hq * hd))
    g.output(x)
    return g.build()


@pytest.mark.parametrize("cache", ["f32", "i8"])
def test_a_step_of_them_together(cache):
    """Two layers over chunks and single tokens, against the same in 64 bits."""
    c = SU.Case([(1, 40), (9, 30), (1, 7), (17, 17)], 4, 2, 64, 8, "f32", cache, pad=1, seed=11)
    layers, freq = 2, G.rotary_frequencies(64)
    rng = np.random.default_rng(4)
    pos = np.zeros(c.T, np.int32)
    for i, (n, length) in enumerate(c.seqs):
        pos[c.cu[i]:c.cu[i + 1]] = np.arange(length - n, length)
    width = (4 + 4) * 64
    x = rng.standard_normal((c.T, 256)).astype(np.float32)
    w = rng.uniform(0.8, 1.2, 64).astype(np.float32)
    mats = [(rng.standard_normal((256, width)) / 16).astype(np.float32) for _ in range(layers)]
    states = [c.state() for _ in range(layers)]
    args = [x, pos, *c.batch(), w]
    for st, m in zip(states, mats):
        args += st + [m]
    (got,) = compiled(step_program(c, freq, layers))(*args)
    y = x.astype(np.float64)
    first = (c.pools, c.scales)
    for st, m in zip(states, mats):
        rows = y @ m.astype(np.float64)
        q, _ = SU.rotary_plain(rows[:, :256].reshape(c.T, 4, 64), pos, freq, False, weight=w)
        k, _ = SU.rotary_plain(rows[:, 256:384].reshape(c.T, 2, 64), pos, freq, False, weight=w)
        # the pools as the run left them: rounding decides the last step of eight bits
        c.pools, c.scales = st[:2], st[2:]
        n = int(c.cu[-1])
        step = 2.0 ** -20 if cache == "f32" else 1.01 / 127 / 2
        for i in range(len(c.seqs)):
            new = int(c.cu[i + 1] - c.cu[i])
            for m2, ref in ((0, k), (1, rows[:, 384:].reshape(c.T, 2, 64))):
                r = ref[c.cu[i]:c.cu[i + 1]]
                kept = c.values(m2, i)[0][-new:]
                top = np.abs(r).max(-1, keepdims=True)
                assert (np.abs(kept - r) <= (step + 2e-5) * top).all()
        c.q = q
        c.dt = "f32"
        y = np.zeros((c.T, 256))
        q32, c.q = c.q, q
        out, _, _ = c.attention()
        y[:n] = out[:n].reshape(n, 256)
        c.pools, c.scales = first
    # every stage is f32: a few hundred roundings of values of order 1 through two layers
    check(got, y, 3e-4)
