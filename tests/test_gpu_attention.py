"""Rotation, 8-bit cache and attention through the C ABI against the 64-bit restatement (attnref.py).

Bars, derived before the first run (half a rounding step is 2^-24 for f32, 2^-11 for f16, 2^-8 for bf16, relative):
  rotation: the norm's factor collects 8 squares and 12 sums of the squares' tree, a division, an addition, half of that
      through the square root, the root and its reciprocal (10 half steps), two products (2), sine and cosine of an angle
      reduced to a fraction of a turn in fp32 (2^-26 turns = 1.6 half steps of a radian) with 2 of their own and one for
      mscale, two products and a sum (3): below 20 half steps of hypot(a, b) mscale, times sqrt(2): bar 2^-19, plus half a
      step of the output's type;
  cache: fp32 operations rounded one by one: the bytes and scales are equal;
  attention: attnref.attention's bound; for the 16-bit types plus half a step of the probabilities (2^-11 of the largest
      value seen) and of the output.
"""
import numpy as np
import pytest

import attnref
from hipmem import DeviceArray, Stream
from ollama_amd import qmm

pytestmark = pytest.mark.gpu
TYPES = {"f32": (qmm.F32, 2.0 ** -24), "f16": (qmm.F16, 2.0 ** -11), "bf16": (qmm.BF16, 2.0 ** -8)}


@pytest.fixture(scope="module")
def ctx():
    c = qmm.Context(0)
    yield c
    c.close()


class Device:
    """device arrays of one test, freed together"""

    def __init__(self, ctx):
        self.ctx, self.all = ctx, []

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.ctx.sync()
        for a in self.all:
            a.free()

    def __call__(self, a, dtype=None):
        self.all.append(DeviceArray(np.ascontiguousarray(a, dtype)))
        return self.all[-1]

    def values(self, x, kind):
        """x in the type, on the device, and the float32 values it then has"""
        if kind == "bf16":
            bits = attnref.bf16_bits(x)
            return self(bits), attnref.bf16_values(bits)
        y = np.asarray(x, np.float16 if kind == "f16" else np.float32)
        return self(y), y.astype(np.float32)


def host(a, kind):
    y = a.numpy()
    return attnref.bf16_values(y) if kind == "bf16" else y.astype(np.float32)


class Steps:
    """sequences with their page tables, numpy and device side"""

    def __init__(self, rng, n_seqs, max_pages, spare=3):
        self.n_pages = n_seqs * max_pages + spare
        self.pages = rng.permutation(self.n_pages)[: n_seqs * max_pages].reshape(n_seqs, max_pages).astype(np.int32)
        self.kv_len = np.zeros(n_seqs, np.int32)
        self.n_seqs, self.max_pages = n_seqs, max_pages

    def grow(self, counts):
        self.kv_len = (self.kv_len + np.asarray(counts)).astype(np.int32)
        return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)

    def batch(self, dev, row_start):
        self.on_device = [dev(row_start, np.int32), dev(self.kv_len, np.int32), dev(self.pages, np.int32)]
        return qmm.Batch(self.n_seqs, self.max_pages, *[a.ptr for a in self.on_device])


# ---- rotation -----------------------------------------------------------------------------------------------------------
ROPE = [  # rows, heads, kv_heads, dim, rot, halves, norm, kind, mscale
    (1, 32, 8, 128, 128, True, True, "f32", 1.0),
    (1, 1, 0, 8, 8, False, True, "f32", 1.0),
    (3, 5, 5, 64, 64, False, False, "f16", 1.25),
    (7, 28, 4, 80, 32, True, True, "f32", 1.0),
    (2, 3, 1, 96, 96, False, True, "bf16", 0.75),
    (5, 4, 4, 256, 64, True, False, "f32", 1.0),
    (129, 16, 2, 128, 128, True, True, "bf16", 1.0),
    (1000, 24, 8, 72, 72, True, True, "f16", 1.0),
    (4, 6, 2, 40, 0, True, True, "f32", 1.0),
    (600, 64, 8, 200, 152, False, True, "f32", 1.1),
]


def _rope_check(got, want, x, rot, halves, norm_scale, half, mscale):
    pair = np.abs(want) + 0.0
    if rot:
        a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if halves else (slice(0, rot, 2), slice(1, rot, 2))
        size = np.hypot(want[..., a], want[..., b])
        pair[..., a] = pair[..., b] = size
    assert np.all(np.abs(got - want) <= 2.0 ** -19 * pair + half * np.abs(want) * 1.01 + 1e-30 + (2.0 ** -25 if half == 2.0 ** -11 else 0))


@pytest.mark.parametrize("rows,heads,kv_heads,dim,rot,halves,norm,kind,mscale", ROPE)
def test_rotation(ctx, rows, heads, kv_heads, dim, rot, halves, norm, kind, mscale):
    rng = np.random.default_rng(rows * 7 + dim)
    t, half = TYPES[kind]
    freqs = 1e6 ** (-np.arange(rot // 2) / max(rot // 2, 1))
    pos = rng.integers(0, 131072, rows).astype(np.int32)
    pos[0] = 131071
    wq, wk = (1 + 0.3 * rng.standard_normal((2, dim))).astype(np.float32) if norm else (None, None)
    with Device(ctx) as dev:
        # rows of one joined buffer [q | k | 16 more values], rotated in place, and separate outputs
        stride = (heads + kv_heads) * dim + 16
        joined, vals = dev.values(rng.standard_normal((rows, stride)) * 3, kind)
        q, k = vals[:, : heads * dim].reshape(rows, heads, dim), vals[:, heads * dim: stride - 16].reshape(rows, kv_heads, dim)
        dpos, dfreqs = dev(pos), dev(freqs if rot else np.zeros(1))
        dw = [dev(w).ptr if norm else None for w in (wq, wk)]
        h = qmm.QKHeads(t, heads, kv_heads, dim, dfreqs.ptr, rot, qmm.ROPE_HALVES if halves else qmm.ROPE_ADJACENT, mscale, *dw, 1e-5)
        size = 4 if kind == "f32" else 2
        qo, ko = dev.values(np.zeros((rows, heads, dim)), kind)[0], dev.values(np.zeros((rows, max(kv_heads, 1), dim)), kind)[0]
        kp = joined.ptr + heads * dim * size if kv_heads else None
        ctx.qk_norm_rope_device(h, joined.ptr, kp, dpos.ptr, rows, qo.ptr, ko.ptr if kv_heads else None, q_stride=stride, k_stride=stride)
        ctx.qk_norm_rope_device(h, joined.ptr, kp, dpos.ptr, rows, joined.ptr, kp, stride, stride, stride, stride)
        ctx.sync()
        placed = host(joined, kind)
        for got, x, w, at in ((host(qo, kind), q, wq, slice(0, heads * dim)), (host(ko, kind), k, wk, slice(heads * dim, stride - 16))):
            if not x.size:
                continue
            want = attnref.rope(x, pos, freqs, halves, mscale, w, 1e-5)
            _rope_check(got, want, x, rot, halves, 1, half, mscale)
            assert np.array_equal(placed[:, at].reshape(x.shape), got)  # in place: the same bits
        assert np.array_equal(placed[:, stride - 16:], vals[:, stride - 16:])


def test_rotation_host_arrays_and_edges(ctx):
    rng = np.random.default_rng(5)
    freqs, _ = qmm.rope_freqs(64, 10000.0)
    q, k = rng.standard_normal((6, 4, 64)).astype(np.float32), rng.standard_normal((6, 2, 64)).astype(np.float32)
    pos = np.array([0, 1, -3, 2 ** 31 - 1, -2 ** 31, 77], np.int32)
    qo, ko = ctx.qk_norm_rope(q, k, pos, freqs)
    _rope_check(qo, attnref.rope(q, pos, freqs), q, 64, True, 1, 2.0 ** -24, 1.0)
    assert np.array_equal(qo[0], q[0]) and np.array_equal(ko[0], k[0])  # position 0 turns nothing
    assert ctx.qk_norm_rope(q, None, pos, freqs)[1] is None
    assert ctx.qk_norm_rope(q[:0], k[:0], pos[:0], freqs)[0].shape == (0, 4, 64)
    z = np.zeros((1, 2, 64), np.float32)
    assert np.all(ctx.qk_norm_rope(z, None, [3], freqs, q_weight=np.ones(64), eps=1e-6)[0] == 0)
    x = q.copy()
    x[1, 2, 5] = np.nan
    bad = ctx.qk_norm_rope(x, k, pos, freqs, q_weight=np.ones(64))[0]
    assert np.isnan(bad[1, 2]).all() and np.isfinite(np.delete(bad.reshape(24, 64), 6, 0)).all()
    # outputs interleaved in one host buffer: neither copy overwrites the other
    buf = np.full((6, 6 * 64), 9.0, np.float32)
    hd = qmm.QKHeads(qmm.F32, 4, 2, 64, freqs.ctypes.data, 64)
    assert qmm.lib().mi_qmm_qk_norm_rope(ctx._h, hd._p, q.ctypes.data, 256, k.ctypes.data, 128, pos.ctypes.data, 6,
                                         buf.ctypes.data, 384, buf.ctypes.data + 4 * 256, 384, qmm.HOST) == 0
    assert np.array_equal(buf[:, :256].reshape(qo.shape), qo) and np.array_equal(buf[:, 256:].reshape(ko.shape), ko)


def test_rotation_refusals(ctx):
    with Device(ctx) as dev:
        a, pos, freqs = dev(np.zeros(4096, np.float32)), dev(np.zeros(4, np.int32)), dev(np.ones(32))
        h = qmm.QKHeads(qmm.F32, 4, 2, 64, freqs.ptr, 64)
        o = a.ptr + 8192

        def call(q=a.ptr, k=a.ptr + 1024, p=pos.ptr, qo=o, ko=o + 1024, n=4, s=384, os=384, hh=h):
            return qmm.lib().mi_qmm_qk_norm_rope(ctx._h, hh._p, q, s, k, s, p, n, qo, os, ko, os, qmm.DEVICE)

        assert call() == 0
        assert call(q=a.ptr, k=a.ptr + 1024, qo=a.ptr, ko=a.ptr + 1024) == 0
        for bad in (dict(q=None), dict(k=None), dict(p=None), dict(qo=None), dict(ko=None), dict(q=a.ptr + 4), dict(s=382),
                    dict(s=100), dict(os=250), dict(qo=a.ptr + 16), dict(qo=a.ptr + 1024), dict(qo=a.ptr, os=512), dict(ko=o + 512),
                    dict(hh=qmm.QKHeads(qmm.F32, 4, 2, 64, None, 64))):
            assert call(**bad) == qmm.ERR_INVALID, bad
        ctx.sync()


# ---- the cache ----------------------------------------------------------------------------------------------------------
CACHE = [  # seqs, heads, dim, block, kind, rounds of new rows per sequence
    (1, 1, 8, 64, "f32", [[1], [1], [62], [1], [130]]),
    (3, 2, 128, 64, "f32", [[5, 0, 64], [59, 1, 1], [1, 1, 1], [70, 200, 0], [1, 1, 1]]),
    (4, 3, 64, 16, "f16", [[15, 16, 17, 1], [1, 1, 1, 1], [33, 0, 5, 129], [0, 0, 0, 0], [1, 47, 1, 2]]),
    (2, 5, 80, 32, "bf16", [[31, 64], [2, 1], [1, 1], [100, 65]]),
    (2, 2, 256, 16, "f32", [[200, 3], [1, 1], [1, 60]]),
    (2, 1, 184, 32, "f32", [[40, 90], [30, 1], [64, 64]]),
    (70, 1, 64, 32, "f32", [[i % 5 for i in range(70)], [1] * 70, [(i * 7) % 70 for i in range(70)], [1] * 70]),
]


@pytest.mark.parametrize("seqs,heads,dim,block,kind,rounds", CACHE)
def test_cache_holds_the_defined_bytes(ctx, seqs, heads, dim, block, kind, rounds):
    rng = np.random.default_rng(seqs + dim)
    t, _ = TYPES[kind]
    table = -(-max(sum(r[i] for r in rounds) for i in range(seqs)) // 64) + 1
    st = Steps(rng, seqs, table)
    ref = attnref.Cache(st.n_pages, heads, dim, block)
    with Device(ctx) as dev:
        mem = dev(np.zeros(qmm.kv_bytes(st.n_pages, heads, dim, block), np.uint8))
        kv = ctx.kv_create(st.n_pages, heads, dim, block, memory=mem.ptr)
        for i, counts in enumerate(rounds):
            rs = st.grow(counts)
            n = int(rs[-1])
            grow = [1.0, 0.5, 3.0, 10.0, 1.0][i]  # later rounds outgrow some blocks' scales and not others
            pad, extra = 3, 8 * heads  # rows behind the last sequence; strides longer than a row
            k, kv_ = dev.values(rng.standard_normal((n + pad, heads * dim + extra)) * grow, kind)
            v, vv_ = dev.values(rng.standard_normal((n + pad, heads * dim + extra)) * rng.uniform(0.1, 5, (n + pad, 1)), kind)
            b = st.batch(dev, rs)
            ctx.kv_write_device(kv, b, t, k.ptr, v.ptr, n + pad, heads * dim + extra, heads * dim + extra)
            ref.write(rs, st.kv_len, st.pages, kv_[:, : heads * dim].reshape(-1, heads, dim), vv_[:, : heads * dim].reshape(-1, heads, dim))
            ctx.sync()
            got, want = mem.numpy(), ref.memory()
            codes = st.n_pages * heads * 64 * attnref.row_dim(dim)
            assert np.array_equal(got[2 * codes:].view(np.float32), want[2 * codes:].view(np.float32)), f"scales of round {i}"
            touched = attnref.places(dim)
            for j in range(2):  # bytes of real dimensions (the padding is nobody's)
                g_, w_ = (x[j * codes:(j + 1) * codes].reshape(-1, 64 * attnref.row_dim(dim))[:, touched[j].reshape(-1)] for x in (got, want))
                assert np.array_equal(g_, w_), f"{'kv'[j]} codes of round {i}: {np.count_nonzero(g_ != w_)} differ"
        # read everything back, in each type, into rows with gaps and padding behind
        rs = np.concatenate([[0], np.cumsum(st.kv_len)]).astype(np.int32)
        n = int(rs[-1])
        want_k, want_v = ref.read(rs, st.kv_len, st.pages, n)
        for out, (ot, half) in TYPES.items():
            ko, vo = dev.values(np.full((n + 2, heads * dim + 8), 7.0), out)[0], dev.values(np.full((n + 2, heads * dim), 7.0), out)[0]
            ctx.kv_read_device(kv, st.batch(dev, rs), ot, ko.ptr, vo.ptr, n + 2, heads * dim + 8)
            ctx.sync()
            gk, gv = host(ko, out), host(vo, out)
            assert np.all(gk[n:] == 7) and np.all(gv[n:] == 7) and np.all(gk[:, heads * dim:] == 7)
            for g_, w_ in ((gk[:n, : heads * dim], want_k), (gv[:n], want_v)):
                w32 = w_.astype(np.float32).reshape(n, -1)
                if out == "f32":
                    assert np.array_equal(g_, w32)
                else:
                    assert np.array_equal(g_, w32.astype(np.float16).astype(np.float32) if out == "f16" else attnref.bf16_values(attnref.bf16_bits(w32)))
        # a suffix only
        rs2 = np.minimum(st.kv_len, 3).cumsum()
        rs2 = np.concatenate([[0], rs2]).astype(np.int32)
        gk, gv = ctx.kv_read(kv, qmm.Batch.of(rs2, st.kv_len, st.pages), int(rs2[-1]))
        wk, wv = ref.read(rs2, st.kv_len, st.pages, int(rs2[-1]))
        assert np.array_equal(gk, wk.astype(np.float32)) and np.array_equal(gv, wv.astype(np.float32))
        kv.free()


def test_cache_of_values_that_are_not_numbers(ctx):
    """infinities and NaN poison their block and head until it is started anew, nothing else; zeros and subnormals hold"""
    rng = np.random.default_rng(3)
    kv = ctx.kv_create(4, 2, 64, 16)
    ref = attnref.Cache(4, 2, 64, 16)
    pages = [[2, 1]]

    def write(rs, ln, k, v):
        ctx.kv_write(kv, qmm.Batch.of(rs, ln, pages), k, v)
        ref.write(rs, ln, pages, k, v)
        n = ln[0]
        gk, gv = ctx.kv_read(kv, qmm.Batch.of([0, n], [n], pages), n)
        wk, wv = ref.read([0, n], [n], pages, n)
        assert np.array_equal(gk, wk.astype(np.float32), equal_nan=True) and np.array_equal(gv, wv.astype(np.float32), equal_nan=True)
        return gk, gv

    k, v = rng.standard_normal((70, 2, 64)).astype(np.float32), rng.standard_normal((70, 2, 64)).astype(np.float32)
    k[20, 1, 3], v[40, 0, 0], v[66, 1, 1] = np.nan, np.inf, -np.inf
    k[48:64] = 0
    v[0:16] *= np.float32(1e-43)
    v[16:32, 0] *= np.float32(1e38)
    gk, gv = write([0, 70], [70], k, v)
    assert np.isnan(gk[16:32, 1]).all() and np.isfinite(gk[16:32, 0]).all() and np.all(gk[48:64] == 0)
    assert np.isnan(gv[32:48, 0]).all() and np.isnan(gv[64:70, 1]).all()
    one = np.ones((1, 2, 64), np.float32)
    gk, gv = write([0, 1], [71], one, one)
    assert np.isnan(gv[64:71, 1]).all() and np.all(gv[70, 0] != 0)
    gk, gv = write([0, 7], [71], np.ones((7, 2, 64), np.float32), np.ones((7, 2, 64), np.float32))  # the block anew
    assert np.isfinite(gv[64:]).all()
    kv.free()


def test_cache_bad_pages_and_rows_on_the_device(ctx):
    """page numbers that there are not, tables that are too short, lengths and row ranges that do not fit"""
    rng = np.random.default_rng(9)
    with Device(ctx) as dev:
        mem = dev(np.zeros(qmm.kv_bytes(4, 2, 64, 64), np.uint8))
        kv = ctx.kv_create(4, 2, 64, 64, memory=mem.ptr)
        k, kval = dev.values(rng.standard_normal((400, 2, 64)), "f32")
        v, vval = dev.values(rng.standard_normal((400, 2, 64)), "f32")
        pages = dev(np.array([[0, 4], [-1, 1], [2, 3]], np.int32))
        lens, starts = dev(np.array([128, 128, 200], np.int32)), dev(np.array([0, 100, 164, 364], np.int32))
        b = qmm.Batch(3, 2, starts.ptr, lens.ptr, pages.ptr)
        ctx.kv_write_device(kv, b, qmm.F32, k.ptr, v.ptr, 400)
        ctx.sync()
        ref = attnref.Cache(4, 2, 64, 64)
        # what fits: page 0 from sequence 0 (tokens 28..63), page 1 from sequence 1, pages 2 and 3 from sequence 2
        ref.write([0, 36], [64], [[0]], kval[:36], vval[:36])
        ref.write([0, 64], [128], [[0, 1]], kval[100:164], vval[100:164])
        ref.write([0, 128], [128], [[2, 3]], kval[164:292], vval[164:292])
        assert np.array_equal(mem.numpy(), ref.memory())
        ko, vo = dev(np.full((400, 2, 64), 7, np.float32)), dev(np.full((400, 2, 64), 7, np.float32))
        ctx.kv_read_device(kv, b, qmm.F32, ko.ptr, vo.ptr, 400)
        ctx.sync()
        wk = np.full((400, 2, 64), 7.0)
        wk[:364] = np.nan
        wk[:36] = ref.values([0], 64)[0][28:]
        wk[100:164] = ref.values([0, 1], 128)[0][64:]
        wk[164:292] = ref.values([2, 3], 128)[0]
        assert np.array_equal(ko.numpy(), wk.astype(np.float32), equal_nan=True)
        # rows that run backwards or out of the call, lengths below the rows: nothing is touched that is not the sequence's
        before = mem.numpy()
        starts.set(np.array([5, 2, 500, 400], np.int32))
        ctx.kv_write_device(kv, b, qmm.F32, k.ptr, v.ptr, 400)
        starts.set(np.array([-4, 0, 0, 0], np.int32))
        ctx.kv_write_device(kv, b, qmm.F32, k.ptr, v.ptr, 400)
        lens.set(np.array([-5, 0, -2 ** 31], np.int32))
        starts.set(np.array([0, 5, 10, 20], np.int32))
        ctx.kv_write_device(kv, b, qmm.F32, k.ptr, v.ptr, 400)
        ctx.sync()
        assert np.array_equal(mem.numpy(), before)
        kv.free()


# ---- attention ----------------------------------------------------------------------------------------------------------
def _attend(ctx, rng, lens, news, heads, kv_heads, dim, block, kind, window=0, cap=0.0, sinks=False, causal=True, spread=1.0, spare_table=0,
            scale=None):
    t, half = TYPES[kind]
    seqs = len(lens)
    st = Steps(rng, seqs, max(1, -(-max(lens) // 64) + spare_table))
    ref = attnref.Cache(st.n_pages, kv_heads, dim, block)
    scale = scale or dim ** -0.5
    with Device(ctx) as dev:
        mem = dev(np.zeros(qmm.kv_bytes(st.n_pages, kv_heads, dim, block), np.uint8))
        kv = ctx.kv_create(st.n_pages, kv_heads, dim, block, memory=mem.ptr)
        rs = st.grow(lens)
        k = (rng.standard_normal((int(rs[-1]), kv_heads, dim)) * rng.uniform(0.3, 2, (int(rs[-1]), 1, 1))).astype(np.float32)
        v = (rng.standard_normal((int(rs[-1]), kv_heads, dim)) * rng.uniform(0.1, 3, (int(rs[-1]), 1, 1))).astype(np.float32)
        if len(k):
            ctx.kv_write(kv, qmm.Batch.of(rs, st.kv_len, st.pages), k, v)
            ref.write(rs, st.kv_len, st.pages, k, v)
        starts = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        n, pad, gap = int(starts[-1]), 2, 16
        q, qv = dev.values(rng.standard_normal((n + pad, heads * dim + gap)) * spread, kind)
        out = dev.values(np.full((n + pad, heads * dim + gap), 7.0), kind)[0]
        sink = rng.standard_normal(heads).astype(np.float32) * 2 if sinks else None
        how = qmm.Attention(t, heads, scale, window, cap, dev(sink).ptr if sinks else None, causal)
        ctx.attention_device(kv, st.batch(dev, starts), how, q.ptr, n + pad, out.ptr, heads * dim + gap, heads * dim + gap)
        ctx.sync()
        got = host(out, kind)
        assert np.all(got[n:] == 7) and np.all(got[:, heads * dim:] == 7)
        qn = qv[:n, : heads * dim].reshape(n, heads, dim)
        want, bound = attnref.attention(ref, starts, st.kv_len, st.pages, qn, np.float64(np.float32(scale)), window, cap, sink, causal)
        got = got[:n, : heads * dim].reshape(n, heads, dim)
        vmax = max([float(np.abs(ref.values(st.pages[s], int(st.kv_len[s]))[1]).max(initial=0)) for s in range(seqs)])
        bar = bound + (0 if kind == "f32" else vmax * 2.0 ** -10 + half * np.abs(want)) + 2.0 ** -24 * np.abs(want)
        err = np.abs(got - want)
        assert np.all(err <= bar), f"worst {np.max(err / (bar + 1e-30))} of the bar, {np.max(err)} at {np.unravel_index(np.argmax(err), err.shape)}"
        kv.free()
        return got, want


ATTEND = [  # lens, new rows, heads, kv_heads, dim, block, kind, options
    ([1], [1], 1, 1, 8, 64, "f32", {}),
    ([64], [1], 4, 1, 64, 64, "f32", {}),
    ([65, 63, 0, 1, 200], [1, 1, 0, 1, 1], 8, 2, 128, 16, "f32", {}),
    ([300, 5, 64, 129], [3, 5, 0, 17], 6, 2, 80, 32, "f32", {}),
    ([257], [257], 2, 1, 64, 16, "f32", {}),
    ([150, 90], [150, 33], 8, 8, 128, 64, "f16", {}),
    ([150, 90], [100, 90], 21, 3, 96, 32, "bf16", {}),
    ([700, 40], [2, 1], 16, 1, 256, 64, "f32", {}),
    ([129, 70], [129, 9], 4, 2, 256, 32, "f32", {"cap": 30.0}),
    ([400, 400, 20], [1, 60, 20], 8, 1, 64, 64, "f16", {"window": 128, "sinks": True}),
    ([333, 64], [65, 64], 6, 3, 192, 16, "bf16", {"window": 50, "cap": 20.0, "sinks": True}),
    ([200, 64, 10], [40, 64, 3], 4, 4, 72, 64, "f32", {"causal": False}),
    ([200, 64, 10], [40, 64, 3], 4, 2, 128, 64, "f16", {"causal": False, "window": 7}),
    ([500], [500], 5, 1, 128, 32, "f32", {"window": 1}),
    ([100, 100], [1, 100], 32, 1, 40, 64, "f32", {"sinks": True}),
    ([8192, 31, 5000], [1, 1, 2], 16, 2, 128, 32, "f32", {}),
    ([3000], [700], 4, 1, 128, 64, "bf16", {}),
    ([2500, 1], [130, 1], 3, 1, 64, 32, "f32", {"spare_table": 40}),
    ([130] * 70, [i % 3 for i in range(70)], 2, 2, 64, 64, "f32", {}),
    ([640], [300], 8, 2, 256, 64, "f16", {"cap": 50.0}),
    ([350], [130], 2, 2, 128, 64, "f32", {"spread": 40.0}),
    ([350], [130], 2, 2, 128, 64, "f16", {"spread": 1e-5, "scale": 1e4}),
    ([300], [1], 64, 1, 64, 16, "f32", {}),                                       # one token of many heads per key head
    ([8200, 300, 5000, 64], [1, 150, 2, 0], 4, 1, 64, 64, "f32", {}),             # prompts and single tokens, the latter split
    ([4200, 40, 700], [3, 40, 300], 6, 2, 128, 32, "bf16", {"sinks": True}),
    ([4200, 40, 700], [3, 40, 300], 2, 2, 256, 16, "f16", {"window": 200, "cap": 15.0}),
    ([200, 90], [100, 1], 4, 4, 8, 64, "f32", {}),
    ([200, 90], [100, 80], 4, 2, 24, 16, "bf16", {}),
    ([333], [64], 8, 2, 200, 32, "f32", {"cap": 3.0}),
    ([333], [64], 8, 2, 128, 32, "f32", {"scale": -0.2}),
    ([333], [2], 8, 2, 128, 32, "f16", {"scale": -0.2}),
    ([70, 333], [64, 1], 8, 2, 64, 32, "f32", {"scale": 1e-30}),
    ([3000], [100], 1, 1, 256, 64, "f32", {}),
    ([600, 500], [600, 500], 3, 1, 192, 64, "f32", {"sinks": True}),
]


@pytest.mark.parametrize("lens,news,heads,kv_heads,dim,block,kind,options", ATTEND)
def test_attention(ctx, lens, news, heads, kv_heads, dim, block, kind, options):
    _attend(ctx, np.random.default_rng(sum(lens) + dim), lens, news, heads, kv_heads, dim, block, kind, **options)


SPLIT = [  # caches cut over many workgroups: lens, new rows, heads, kv_heads, dim, block, kind, options
    ([33000], [1], 16, 1, 128, 64, "f32", {}),                                       # more splits than a round of the join takes
    ([8100, 5000], [100, 62], 16, 4, 128, 64, "f32", {"sinks": True}),              # ten splits of 128 rows, many values to join
    ([3000] * 3 + [0] * 20, [9, 1, 1] + [0] * 20, 8, 1, 64, 32, "f32", {}),          # one sequence of many more rows than most
    ([3000] * 3 + [0] * 20, [9, 1, 1] + [0] * 20, 8, 1, 256, 16, "bf16", {"cap": 30.0, "sinks": True}),
    ([2100], [17], 8, 2, 80, 64, "f16", {}),                                         # 68 rows: the least that goes by 128
    ([2100], [16], 8, 2, 80, 64, "f16", {"sinks": True}),                            # 64 rows: the most that goes by 16
    ([2100, 70], [17, 16], 8, 2, 80, 32, "f32", {}),                                 # both at once
    ([5000] * 5, [1] * 5, 12, 3, 192, 64, "f32", {"window": 4000}),
    ([i % 90 for i in range(1000)], [min(i % 90, i % 3) for i in range(1000)], 2, 1, 64, 32, "f32", {}),   # many sequences
    ([40] * 257, [i % 2 for i in range(257)], 4, 2, 128, 64, "bf16", {}),
]


@pytest.mark.parametrize("lens,news,heads,kv_heads,dim,block,kind,options", SPLIT)
def test_attention_split_over_workgroups(ctx, lens, news, heads, kv_heads, dim, block, kind, options):
    _attend(ctx, np.random.default_rng(sum(lens) * 3 + heads), lens, news, heads, kv_heads, dim, block, kind, **options)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new", [1, 100])
@pytest.mark.parametrize("block", [16, 64])
def test_attention_of_scales_far_apart(ctx, kind, new, block):
    """keys that grow along the sequence (the maximum leaves every reference behind), values whose scales differ by many
    orders of magnitude from block to block in both directions, blocks of zeros among them"""
    t, half = TYPES[kind]
    rng = np.random.default_rng(block + new)
    n, dim = 700, 64
    k = rng.standard_normal((n, 1, dim)) * np.linspace(0.2, 6, n)[:, None, None]
    v = rng.standard_normal((n, 1, dim))
    for b in range(0, n, 64):
        v[b:b + 64] *= 10.0 ** rng.uniform(-9, 3)
    k[128:192], v[256:320], v[0:64] = 0, 0, 0
    k, v = k.astype(np.float32), v.astype(np.float32)
    ref = attnref.Cache(12, 1, dim, block)
    pages = rng.permutation(12)[:11].reshape(1, 11)
    kv = ctx.kv_create(12, 1, dim, block)
    ctx.kv_write(kv, qmm.Batch.of([0, n], [n], pages), k, v)
    ref.write([0, n], [n], pages, k, v)
    with Device(ctx) as dev:
        for sign in (1.0, -1.0):  # the keys of the end against the rows, and with them
            q, qv = dev.values(rng.standard_normal((new, 3, dim)) + sign * k[-1], kind)
            out = dev.values(np.zeros((new, 3, dim)), kind)[0]
            b = qmm.Batch(1, 11, dev(np.array([0, new], np.int32)).ptr, dev(np.array([n], np.int32)).ptr, dev(pages, np.int32).ptr)
            ctx.attention_device(kv, b, qmm.Attention(t, 3, 0.05), q.ptr, new, out.ptr)
            ctx.sync()
            want, bound = attnref.attention(ref, [0, new], [n], pages, qv, np.float64(np.float32(0.05)))
            # what each row could take from its largest value, weighted: a rounding of a probability is one of its own share
            got = host(out, kind)
            bar = bound + (0 if kind == "f32" else np.abs(v).max() * 2.0 ** -10 + half * np.abs(want)) + 2.0 ** -24 * np.abs(want)
            assert np.all(np.abs(got - want) <= bar)
            if sign < 0:  # rows that turn from the large values to small ones: exact to the small ones' own size
                assert np.isfinite(got).all()
    kv.free()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("news", [(1, 2, 1), (40, 70, 1), (100, 120, 200)])
@pytest.mark.parametrize("dim,block", [(64, 16), (128, 32), (200, 64)])
def test_attention_over_memory_with_earlier_content(ctx, kind, news, dim, block):
    """a cache in memory that is not cleared: codes and scales of any size, infinities and NaN stand behind the last token
    and in tokens that a window has left, and no result changes by a bit"""
    t, half = TYPES[kind]
    rng = np.random.default_rng(dim + sum(news))
    lens, pages = [101, 130, 200], rng.permutation(12).reshape(3, 4).astype(np.int32)
    rs = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    starts = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    k, v = rng.standard_normal((2, 431, 2, dim)).astype(np.float32)
    size, codes = qmm.kv_bytes(12, 2, dim, block), 2 * 12 * 2 * 64 * attnref.row_dim(dim)
    used = rng.integers(0, 256, size).astype(np.uint8)
    scales = rng.choice(np.array([3e38, np.inf, np.nan, 1e30, -1e20, 1e-44, 5e3, -np.inf], np.float32), (size - codes) // 4)
    used[codes:] = scales.view(np.uint8)
    ref = attnref.Cache(12, 2, dim, block)
    ref.write(rs, lens, pages, k, v)
    got = []
    with Device(ctx) as dev:
        q, qv = dev.values(rng.standard_normal((int(starts[-1]), 6, dim)), kind)
        for memory in (np.zeros(size, np.uint8), used):
            kv = ctx.kv_create(12, 2, dim, block, memory=dev(memory).ptr)
            ctx.kv_write(kv, qmm.Batch.of(rs, lens, pages), k, v)
            b = qmm.Batch(3, 4, dev(starts, np.int32).ptr, dev(np.array(lens, np.int32)).ptr, dev(pages).ptr)
            for window, cap in ((0, 0.0), (90, 20.0)):
                out = dev.values(np.zeros((int(starts[-1]), 6, dim)), kind)[0]
                ctx.attention_device(kv, b, qmm.Attention(t, 6, 0.2, window, cap), q.ptr, int(starts[-1]), out.ptr)
                ctx.sync()
                got.append(host(out, kind))
                want, bound = attnref.attention(ref, starts, lens, pages, qv, np.float64(np.float32(0.2)), window, cap)
                bar = bound + (0 if kind == "f32" else np.abs(v).max() * 2.0 ** -10 + half * np.abs(want)) + 2.0 ** -24 * np.abs(want)
                assert np.all(np.abs(got[-1] - want) <= bar)
            kv.free()
    assert np.array_equal(got[0], got[2]) and np.array_equal(got[1], got[3])


def test_attention_of_lengths_behind_the_table(ctx):
    """device lengths beyond the page table, absurd and negative ones: NaN for the rows that see such tokens, zeros for rows
    that see none, and the call ends"""
    rng = np.random.default_rng(6)
    for kind in ("f32", "f16"):
        t, _ = TYPES[kind]
        with Device(ctx) as dev:
            kv = ctx.kv_create(4, 1, 64, 64)
            k = rng.standard_normal((128, 1, 64)).astype(np.float32)
            ctx.kv_write(kv, qmm.Batch.of([0, 128], [128], [[0, 1]]), k, k)
            pages, n = dev(np.array([[0, 1]] * 5, np.int32)), 50
            q = dev.values(rng.standard_normal((5 * n, 2, 64)), kind)[0]
            for window in (0, 30):
                out = dev.values(np.full((5 * n, 2, 64), 7.0), kind)[0]
                lens = dev(np.array([128, 150, 2 ** 31 - 1, -7, -2 ** 31], np.int32))
                b = qmm.Batch(5, 2, dev(np.arange(6) * n, np.int32).ptr, lens.ptr, pages.ptr)
                ctx.attention_device(kv, b, qmm.Attention(t, 2, 0.125, window), q.ptr, 5 * n, out.ptr)
                ctx.sync()
                got = host(out, kind).reshape(5, n, -1)
                assert np.isfinite(got[0]).all() and not (got[0] == 0).all(-1).any()
                assert np.isfinite(got[1, :28]).all() and np.isnan(got[1, 28:]).all()  # row 28 is at position 128
                assert np.isnan(got[2]).all() and np.all(got[3:] == 0)
            kv.free()


def test_attention_rows_that_see_nothing(ctx):
    """more rows than tokens: rows of negative positions see none (device arrays cannot be looked at) and give zeros"""
    rng = np.random.default_rng(2)
    for sinks in (False, True):
        with Device(ctx) as dev:
            kv = ctx.kv_create(2, 2, 64, 64)
            k = rng.standard_normal((3, 2, 64)).astype(np.float32)
            ctx.kv_write(kv, qmm.Batch.of([0, 3], [3], [[1]]), k, k)
            q, out = dev(rng.standard_normal((40, 4, 64)).astype(np.float32)), dev(np.full((40, 4, 64), 7, np.float32))
            st, ln, pg = dev(np.array([0, 20, 40], np.int32)), dev(np.array([3, 0], np.int32)), dev(np.array([[1], [0]], np.int32))
            how = qmm.Attention(qmm.F32, 4, 0.125, sinks=dev(np.zeros(4, np.float32)).ptr if sinks else None)
            ctx.attention_device(kv, qmm.Batch(2, 1, st.ptr, ln.ptr, pg.ptr), how, q.ptr, 40, out.ptr)
            ctx.sync()
            got = out.numpy()
            assert np.all(got[:17] == 0) and np.all(got[20:] == 0) and np.all(np.abs(got[17:20]).max(-1) > 0)
            kv.free()


def test_attention_of_bad_pages_and_poisoned_blocks(ctx):
    """a page that there is not, or a block with NaN, reaches exactly the rows that see it"""
    rng = np.random.default_rng(4)
    for kind in ("f32", "f16"):
        t, _ = TYPES[kind]
        for new in (1, 150):
            with Device(ctx) as dev:
                kv = ctx.kv_create(6, 1, 64, 64)
                ref = attnref.Cache(6, 1, 64, 64)
                pages = np.array([[0, 1, 2], [3, 4, 5]], np.int32)
                k, v = rng.standard_normal((2, 380, 1, 64)).astype(np.float32)
                v[10, 0, 3] = np.nan            # block 0 of sequence 0
                k[190 + 70, 0, 3] = np.inf      # block 1 of sequence 1
                ctx.kv_write(kv, qmm.Batch.of([0, 190, 380], [190, 190], pages), k, v)
                ref.write([0, 190, 380], [190, 190], pages, k, v)
                pages[0, 1] = 99
                st = np.array([0, new, 2 * new], np.int32)
                q, qv = dev.values(rng.standard_normal((2 * new, 3, 64)), kind)
                for window in (0, 40, 1):
                    out = dev.values(np.full((2 * new, 3, 64), 7.0), kind)[0]
                    b = qmm.Batch(2, 3, dev(st).ptr, dev(np.array([190, 190], np.int32)).ptr, dev(pages).ptr)
                    ctx.attention_device(kv, b, qmm.Attention(t, 3, 0.125, window), q.ptr, 2 * new, out.ptr)
                    ctx.sync()
                    want, _ = attnref.attention(ref, st, [190, 190], pages, qv, 0.125, window)
                    got = host(out, kind)
                    assert np.array_equal(np.isnan(got), np.isnan(want)), (kind, new, window)
                    fine = ~np.isnan(want)
                    assert not fine.any() or np.abs(got - want)[fine].max() < 0.02
                kv.free()


def test_attention_host_arrays(ctx):
    rng = np.random.default_rng(12)
    kv = ctx.kv_create(5, 2, 64, 32)
    ref = attnref.Cache(5, 2, 64, 32)
    rs, ln, pg = [0, 100, 130], [100, 30], [[4, 2], [0, 1]]
    k, v = rng.standard_normal((130, 2, 64)).astype(np.float32), rng.standard_normal((130, 2, 64)).astype(np.float32)
    b = qmm.Batch.of(rs, ln, pg)
    ctx.kv_write(kv, b, k, v)
    ref.write(rs, ln, pg, k, v)
    q = rng.standard_normal((133, 4, 64)).astype(np.float32)
    sinks = rng.standard_normal(4)
    got = ctx.attention(kv, b, q, 0.125, window=33, softcap=5.0, sinks=sinks)
    want, bound = attnref.attention(ref, rs, ln, pg, q[:130], 0.125, 33, 5.0, sinks)
    assert np.all(got[130:] == 0) and np.all(np.abs(got[:130] - want) <= bound + 2.0 ** -24 * np.abs(want))
    kv.free()


def test_refusals(ctx):
    kv = ctx.kv_create(4, 2, 64, 32)
    x = np.zeros((10, 2, 64), np.float32)
    q = np.zeros((10, 4, 64), np.float32)
    ok = qmm.Batch.of([0, 10], [10], [[1, 2]])
    ctx.kv_write(kv, ok, x, x)
    bad = [([0, 10], [10], [[4, 2]]), ([0, 10], [10], [[-1, 2]]), ([0, 10], [129], [[1, 2]]), ([0, 10], [9], [[1, 2]]), ([0, 11], [11], [[1, 2]]),
           ([-1, 10], [20], [[1, 2]]), ([5, 3], [10], [[1, 2]]), ([0, 10], [-1], [[1, 2]])]
    for b in bad:
        for call in (lambda b: ctx.kv_write(kv, b, x, x), lambda b: ctx.kv_read(kv, b, 10), lambda b: ctx.attention(kv, b, q, 1.0)):
            with pytest.raises(qmm.QmmError) as e:
                call(qmm.Batch.of(*b))
            assert e.value.code == qmm.ERR_INVALID, b
    with pytest.raises(qmm.QmmError) as e:   # one page of two sequences
        ctx.kv_write(kv, qmm.Batch.of([0, 5, 10], [5, 5], [[1], [1]]), x, x)
    assert "twice" in str(e.value)
    ctx.kv_read(kv, qmm.Batch.of([0, 5, 10], [5, 5], [[1], [1]]), 10)  # reading is fine
    with pytest.raises(qmm.QmmError):
        ctx.attention(kv, ok, np.zeros((10, 3, 64), np.float32), 1.0)
    with pytest.raises(qmm.QmmError):
        ctx.attention(kv, ok, q, 1.0, softcap=-1.0)
    with pytest.raises(qmm.QmmError):
        ctx.attention(kv, ok, q, 1.0, window=-1)
    for bad in ({"scale": np.nan}, {"scale": np.inf}, {"scale": 1.0, "softcap": np.inf}):
        with pytest.raises(qmm.QmmError) as e:
            ctx.attention(kv, ok, q, **bad)
        assert e.value.code == qmm.ERR_INVALID
    with pytest.raises(ValueError):
        ctx.attention(kv, ok, np.zeros((10, 4, 128), np.float32), 1.0)
    L = qmm.lib()
    with Device(ctx) as dev:
        a, o = dev(q), dev(q)
        b, how = qmm.Batch(1, 2, a.ptr, a.ptr, a.ptr), qmm.Attention(qmm.F32, 4, 1.0)
        assert L.mi_qmm_attention(ctx._h, kv._h, b._p, how._p, a.ptr, 256, a.ptr + 1024, 256, 2, qmm.DEVICE) == qmm.ERR_INVALID
        assert L.mi_qmm_attention(ctx._h, kv._h, b._p, how._p, a.ptr + 4, 256, o.ptr, 256, 2, qmm.DEVICE) == qmm.ERR_INVALID
        assert L.mi_qmm_attention(ctx._h, kv._h, b._p, how._p, a.ptr, 250, o.ptr, 256, 2, qmm.DEVICE) == qmm.ERR_INVALID
        assert L.mi_qmm_attention(ctx._h, kv._h, b._p, how._p, a.ptr, 256, None, 256, 2, qmm.DEVICE) == qmm.ERR_INVALID
        assert L.mi_qmm_attention(ctx._h, None, b._p, how._p, a.ptr, 256, o.ptr, 256, 2, qmm.DEVICE) == qmm.ERR_INVALID
        assert L.mi_qmm_attention(ctx._h, kv._h, None, how._p, a.ptr, 256, o.ptr, 256, 2, qmm.DEVICE) == qmm.ERR_INVALID
        nobody = qmm.Batch(1, 0, a.ptr, a.ptr, a.ptr)
        assert L.mi_qmm_attention(ctx._h, kv._h, nobody._p, how._p, a.ptr, 256, o.ptr, 256, 2, qmm.DEVICE) == qmm.ERR_INVALID
        assert L.mi_qmm_kv_read(ctx._h, kv._h, b._p, qmm.F32, a.ptr, 128, a.ptr + 256, 128, 2, qmm.DEVICE) == qmm.ERR_INVALID
        for many in (qmm.Batch(65537, 2, a.ptr, a.ptr, a.ptr), qmm.Batch(1, (1 << 24) + 1, a.ptr, a.ptr, a.ptr)):
            assert L.mi_qmm_attention(ctx._h, kv._h, many._p, how._p, a.ptr, 256, o.ptr, 256, 2, qmm.DEVICE) == qmm.ERR_UNSUPPORTED
        with pytest.raises(qmm.QmmError):
            ctx.attention_device(kv, b, how, a.ptr, 2, o.ptr, q_stride=0)
        none = qmm.Batch(0, 1, None, None, None)
        assert L.mi_qmm_attention(ctx._h, kv._h, none._p, how._p, a.ptr, 256, o.ptr, 256, 2, qmm.DEVICE) == 0
    # pages that a window leaves behind may be gone
    far = qmm.Batch.of([0, 10], [128], [[-1, 2]])
    assert ctx.attention(kv, far, q, 1.0, window=55).shape == q.shape
    with pytest.raises(qmm.QmmError):
        ctx.attention(kv, far, q, 1.0, window=56)
    kv.free()


def test_long_cache_offsets_past_32_bits(ctx):
    """pages whose codes lie beyond 2^32 bytes from the cache's start"""
    rng = np.random.default_rng(8)
    n_pages = 2 ** 32 // (8 * 64 * 256) + 40
    kv = ctx.kv_create(n_pages, 8, 256, 64)
    small = attnref.Cache(2, 8, 256, 64)
    far = [[n_pages - 1, n_pages - 39]]
    k, v = rng.standard_normal((2, 100, 8, 256)).astype(np.float32)
    ctx.kv_write(kv, qmm.Batch.of([0, 100], [100], far), k, v)
    small.write([0, 100], [100], [[1, 0]], k, v)
    gk, gv = ctx.kv_read(kv, qmm.Batch.of([0, 100], [100], far), 100)
    wk, wv = small.read([0, 100], [100], [[1, 0]], 100)
    assert np.array_equal(gk, wk.astype(np.float32)) and np.array_equal(gv, wv.astype(np.float32))
    for new in (1, 100):
        q = rng.standard_normal((new, 16, 256)).astype(np.float32)
        got = ctx.attention(kv, qmm.Batch.of([0, new], [100], far), q, 0.0625)
        want, bound = attnref.attention(small, [0, new], [100], [[1, 0]], q, 0.0625)
        assert np.all(np.abs(got - want) <= bound + 2.0 ** -24 * np.abs(want))
    kv.free()


def test_steps_replayed_from_a_graph(ctx):
    """rotation, write and attention captured once; the sequences move on between the replays, eager calls run in between"""
    rng = np.random.default_rng(21)
    heads, kv_heads, dim, seqs = 8, 2, 64, 3
    own = qmm.Context(0)
    stream = Stream()
    own.set_stream(stream.ptr.value)
    freqs, _ = qmm.rope_freqs(dim, 10000.0)
    try:
        with Device(own) as dev:
            st = Steps(rng, seqs, 40)
            kv = own.kv_create(st.n_pages, kv_heads, dim, 16)
            ref = attnref.Cache(st.n_pages, kv_heads, dim, 16)
            rs = st.grow([700, 63, 5])
            k, v = rng.standard_normal((2, 768, kv_heads, dim)).astype(np.float32)
            own.kv_write(kv, qmm.Batch.of(rs, st.kv_len, st.pages), k, v)
            ref.write(rs, st.kv_len, st.pages, k, v)
            rs = st.grow([1, 1, 1])
            b = st.batch(dev, rs)
            lens = st.on_device[1]
            q, k1, v1, pos = (dev(np.zeros(s, np.float32)) for s in ((3, heads, dim), (3, kv_heads, dim), (3, kv_heads, dim), (3,)))
            pos = dev(np.zeros(3, np.int32))
            out = dev(np.zeros((3, heads, dim), np.float32))
            hd = qmm.QKHeads(qmm.F32, heads, kv_heads, dim, dev(freqs).ptr, dim)
            how = qmm.Attention(qmm.F32, heads, 0.125)

            def step():
                own.qk_norm_rope_device(hd, q.ptr, k1.ptr, pos.ptr, 3, q.ptr, k1.ptr)
                own.kv_write_device(kv, b, qmm.F32, k1.ptr, v1.ptr, 3)
                own.attention_device(kv, b, how, q.ptr, 3, out.ptr)

            def feed():
                x = [rng.standard_normal(a.shape).astype(np.float32) for a in (q, k1, v1)]
                for a, y in zip((q, k1, v1), x):
                    a.set(y)
                lens.set(st.kv_len)
                pos.set(st.kv_len - 1)
                return x

            def check(x):
                kr = k1.numpy()
                _rope_check(kr, attnref.rope(x[1], st.kv_len - 1, freqs), x[1], dim, True, 1, 2.0 ** -24, 1.0)
                ref.write(rs, st.kv_len, st.pages, kr, x[2])
                want, bound = attnref.attention(ref, rs, st.kv_len, st.pages, q.numpy(), 0.125)
                assert np.all(np.abs(out.numpy() - want) <= bound + 2.0 ** -24 * np.abs(want))

            x = feed()
            step()
            stream.sync()
            check(x)
            own.scratch_freeze(True)
            replay = stream.capture(step)
            for i in range(5):
                st.grow([1, 1, 1])
                x = feed()
                out.set(np.zeros(out.shape, np.float32))
                assert replay() == 0
                stream.sync()
                check(x)
                if i % 2:  # eager work between the replays
                    st.grow([1, 1, 1])
                    x = feed()
                    step()
                    stream.sync()
                    check(x)
            big = qmm.Attention(qmm.F32, heads * 16, 0.125)
            qb = dev(np.zeros((3, heads * 16, dim), np.float32))
            ob = dev(np.zeros((3, heads * 16, dim), np.float32))
            with pytest.raises(qmm.QmmError) as e:  # a call whose partial results need more scratch than there is
                for width in (40, 4000):
                    wide = qmm.Batch(seqs, width, b._s.row_start, b._s.kv_len, dev(np.tile(st.pages, (1, width // 40))).ptr)
                    own.attention_device(kv, wide, big, qb.ptr, 3, ob.ptr)
            assert "frozen" in str(e.value)
            own.scratch_freeze(False)
            kv.free()
    finally:
        own.set_stream(None)
        own.close()
        stream.destroy()


def test_prompts_replayed_from_a_graph(ctx):
    """the 128-row way with split tiles at heads of 256, captured: every replay the eager bits, with eager work between"""
    rng = np.random.default_rng(22)
    own = qmm.Context(0)
    stream = Stream()
    own.set_stream(stream.ptr.value)
    try:
        with Device(own) as dev:
            kv = own.kv_create(20, 2, 256, 32)
            pages = rng.permutation(20)[:16].reshape(1, 16).astype(np.int32)
            k, v = rng.standard_normal((2, 1000, 2, 256)).astype(np.float32)
            own.kv_write(kv, qmm.Batch.of([0, 1000], [1000], pages), k, v)
            q, out = dev(rng.standard_normal((90, 4, 256)).astype(np.float32)), dev(np.zeros((90, 4, 256), np.float32))
            b = qmm.Batch(1, 16, dev(np.array([0, 90], np.int32)).ptr, dev(np.array([1000], np.int32)).ptr, dev(pages).ptr)
            how = qmm.Attention(qmm.F32, 4, 0.0625, softcap=20.0)
            step = lambda: own.attention_device(kv, b, how, q.ptr, 90, out.ptr)  # noqa: E731
            step()
            stream.sync()
            replay = stream.capture(step)
            for i in range(4):
                q.set(rng.standard_normal((90, 4, 256)).astype(np.float32))
                step()
                stream.sync()
                want = out.numpy()
                out.set(np.zeros(out.shape, np.float32))
                assert replay() == 0
                stream.sync()
                assert np.array_equal(out.numpy(), want) and np.abs(want).max() > 0
            kv.free()
    finally:
        own.set_stream(None)
        own.close()
        stream.destroy()


def test_two_contexts_on_two_streams(ctx):
    """calls of two contexts at once on one device give what each gives alone"""
    rng = np.random.default_rng(31)
    other = qmm.Context(0)
    try:
        with Device(ctx) as dev:
            runs = []
            for c in (ctx, other):
                kv = c.kv_create(130, 2, 128, 64)
                pages = rng.permutation(130)[:128].reshape(1, 128).astype(np.int32)
                k, v = rng.standard_normal((2, 8000, 2, 128)).astype(np.float32)
                c.kv_write(kv, qmm.Batch.of([0, 8000], [8000], pages), k, v)
                q = rng.standard_normal((4, 8, 128)).astype(np.float32)
                dq, out = dev(q), dev(np.zeros_like(q))
                b = qmm.Batch(1, 128, dev(np.array([0, 4], np.int32)).ptr, dev(np.array([8000], np.int32)).ptr, dev(pages).ptr)
                runs.append((c, kv, b, dq, out, c.attention(kv, qmm.Batch.of([0, 4], [8000], pages), q, 0.09)))
            how = qmm.Attention(qmm.F32, 8, 0.09)
            for _ in range(20):
                for c, kv, b, dq, out, _ in runs:
                    c.attention_device(kv, b, how, dq.ptr, 4, out.ptr)
            for c, *_ in runs:
                c.sync()
            for c, kv, b, dq, out, want in runs:
                assert np.array_equal(out.numpy(), want)
                kv.free()
    finally:
        other.close()


def test_a_layer_of_decoding(ctx):
    """q, k, v products -> norms and rotation -> cache -> attention -> o product, as a model runs them: a prompt, then
    single tokens; every stage against the restatement on what the stage before gave"""
    from ollama_amd import synth

    rng = np.random.default_rng(40)
    hidden, heads, kv_heads, dim = 512, 8, 2, 64
    freqs, ms = qmm.rope_freqs(dim, 10000.0)
    shapes = {"q": heads * dim, "k": kv_heads * dim, "v": kv_heads * dim}
    ws = [ctx.upload(qmm.Q4_K, synth.weights(qmm.Q4_K, m, hidden, seed=i), hidden, m) for i, m in enumerate(shapes.values())]
    wo = ctx.upload(qmm.Q4_K, synth.weights(qmm.Q4_K, hidden, heads * dim, seed=9), heads * dim, hidden)
    g = (1 + 0.1 * rng.standard_normal((2, dim))).astype(np.float32)
    try:
        with Device(ctx) as dev:
            st = Steps(rng, 2, 3)
            kv = ctx.kv_create(st.n_pages, kv_heads, dim, 32)
            ref = attnref.Cache(st.n_pages, kv_heads, dim, 32)
            hd = qmm.QKHeads(qmm.F32, heads, kv_heads, dim, dev(freqs).ptr, dim, mscale=ms, q_weight=dev(g[0]).ptr, k_weight=dev(g[1]).ptr, eps=1e-6)
            how = qmm.Attention(qmm.F32, heads, dim ** -0.5)
            for counts in ([50, 90], [1, 1], [1, 1], [20, 1], [1, 1]):
                rs = st.grow(counts)
                n = int(rs[-1])
                x = rng.standard_normal((n, hidden)).astype(np.float32)
                pos = np.concatenate([np.arange(st.kv_len[s] - counts[s], st.kv_len[s]) for s in range(2)]).astype(np.int32)
                q, k, v, o, y = (dev(np.zeros((n, m), np.float32)) for m in (heads * dim, kv_heads * dim, kv_heads * dim, heads * dim, hidden))
                dx, dp, b = dev(x), dev(pos), st.batch(dev, rs)
                ctx.mulmat_multi_device(ws, dx.ptr, n, [q.ptr, k.ptr, v.ptr])
                ctx.sync()
                q0, k0, v0 = q.numpy().reshape(n, heads, dim), k.numpy().reshape(n, kv_heads, dim), v.numpy().reshape(n, kv_heads, dim)
                ctx.qk_norm_rope_device(hd, q.ptr, k.ptr, dp.ptr, n, q.ptr, k.ptr)
                ctx.kv_write_device(kv, b, qmm.F32, k.ptr, v.ptr, n)
                ctx.attention_device(kv, b, how, q.ptr, n, o.ptr)
                ctx.mulmat_device(wo, o.ptr, n, y.ptr)
                ctx.sync()
                q1, k1 = q.numpy().reshape(q0.shape), k.numpy().reshape(k0.shape)
                _rope_check(q1, attnref.rope(q0, pos, freqs, True, ms, g[0], 1e-6), q0, dim, True, 1, 2.0 ** -24, 1.0)
                _rope_check(k1, attnref.rope(k0, pos, freqs, True, ms, g[1], 1e-6), k0, dim, True, 1, 2.0 ** -24, 1.0)
                ref.write(rs, st.kv_len, st.pages, k1, v0)
                want, bound = attnref.attention(ref, rs, st.kv_len, st.pages, q1, np.float64(np.float32(dim ** -0.5)))
                o1 = o.numpy()
                assert np.all(np.abs(o1.reshape(want.shape) - want) <= bound + 2.0 ** -24 * np.abs(want))
                assert np.array_equal(y.numpy(), ctx.mulmat(wo, o1)) and np.isfinite(y.numpy()).all()
            kv.free()
    finally:
        for w in ws + [wo]:
            w.free()
