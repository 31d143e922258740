"""Attention over the 8-bit cache: the same bits on every call, and the results that the definition gives where cache contents
or arguments are out of the ordinary.  Restatement and bars as in test_gpu_attention.py."""
import threading

import numpy as np
import pytest

import attnref
from ollama_amd import qmm
from test_gpu_attention import TYPES, Device, ctx, host  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim,cap", [(64, 0.0), (128, 0.0), (128, 30.0), (192, 0.0), (256, 0.0), (256, 50.0)])
def test_the_same_bits_on_every_call(ctx, kind, dim, cap):  # noqa: F811
    """prompts of 1500 and 901 rows, forty calls with work of another context beside half of them"""
    t, _ = TYPES[kind]
    rng = np.random.default_rng(dim)
    lens, heads, kv_heads = [1500, 901], 8, 4
    pages = rng.permutation(50)[:48].reshape(2, 24).astype(np.int32)
    rs = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    n = int(rs[-1])
    other = qmm.Context(0)
    try:
        with Device(ctx) as dev:
            kv = ctx.kv_create(50, kv_heads, dim, 64)
            k, v = rng.standard_normal((2, n, kv_heads, dim)).astype(np.float32)
            ctx.kv_write(kv, qmm.Batch.of(rs, lens, pages), k, v)
            b = qmm.Batch(2, 24, dev(rs).ptr, dev(np.array(lens, np.int32)).ptr, dev(pages).ptr)
            q = dev.values(rng.standard_normal((n, heads, dim)), kind)[0]
            how = qmm.Attention(t, heads, dim ** -0.5, softcap=cap)
            outs = [dev.values(np.zeros((n, heads, dim)), kind)[0] for _ in range(4)]
            beside = dev.values(np.zeros((n, heads, dim)), kind)[0]
            for i in range(10):
                for o in outs:
                    ctx.attention_device(kv, b, how, q.ptr, n, o.ptr)
                    if i % 2:
                        other.attention_device(kv, b, how, q.ptr, n, beside.ptr)
                ctx.sync()
                other.sync()
                got = [o.numpy() for o in outs]
                if i == 0:
                    first = got[0]
                    assert np.abs(host(outs[0], kind)).max() > 0.1
                for g in got:
                    assert np.array_equal(g, first), (i, np.count_nonzero(g != first))
            kv.free()
    finally:
        other.close()

def _defined(kind, want, bound, half):
    """the bar of attnref's bound with the half steps of the output's type and of fp32"""
    return bound + (half + 2.0 ** -24) * np.abs(want) + 2.0 ** -25 * (kind == "f16")


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new", [1, 3, 100, 180])
@pytest.mark.parametrize("block", [16, 64])
def test_blocks_of_scale_zero_hold_zeros(ctx, kind, new, block):  # noqa: F811
    """tokens that were never written stand in cleared memory as code -128 under scale 0, or in a caller's as any code: their
    values are 0 and their scores 0, and they take part in the sum"""
    t, half = TYPES[kind]
    rng = np.random.default_rng(new + block)
    dim, heads, kv_heads, n = 64, 4, 2, 300
    pages = rng.permutation(6)[:5].reshape(1, 5)
    size, codes = qmm.kv_bytes(6, kv_heads, dim, block), 2 * 6 * kv_heads * 64 * dim
    ref = attnref.Cache(6, kv_heads, dim, block)
    k, v = rng.standard_normal((2, n, kv_heads, dim)).astype(np.float32)
    with Device(ctx) as dev:
        for cleared in (True, False):
            used = np.zeros(size, np.uint8)
            if not cleared:
                used[:codes] = rng.integers(0, 256, codes)
                for plane, place in zip(range(2), attnref.places(dim)):
                    flat = used[plane * codes // 2:(plane + 1) * codes // 2].reshape(6, kv_heads, 64 * dim)
                    ref.codes[plane][:] = flat[..., place.reshape(-1)].reshape(6, kv_heads, 64, dim).astype(np.int32) - 128
            for s in ref.scales:
                s[:] = 0
            kv = ctx.kv_create(6, kv_heads, dim, block, memory=None if cleared else dev(used).ptr)
            # the second page's, a part of the third's and the last tokens' blocks are written; the rest is not
            for first, last in ((64, 128), (128, 160), (256, 300)):
                b = qmm.Batch.of([0, last - first], [last], pages)
                ctx.kv_write(kv, b, k[first:last], v[first:last])
                ref.write([0, last - first], [last], pages, k[first:last], v[first:last])
            gk, gv = ctx.kv_read(kv, qmm.Batch.of([0, n], [n], pages), n)
            assert np.all(gv[:64] == 0) and np.all(gv[192:256] == 0) and np.all(np.abs(gv[256:300]).max(-1) > 0)
            q, qv = dev.values(rng.standard_normal((new, heads, dim)), kind)
            out = dev.values(np.zeros((new, heads, dim)), kind)[0]
            b = qmm.Batch(1, 5, dev(np.array([0, new], np.int32)).ptr, dev(np.array([n], np.int32)).ptr, dev(pages, np.int32).ptr)
            for window in (0, 90):
                ctx.attention_device(kv, b, qmm.Attention(t, heads, 0.125, window), q.ptr, new, out.ptr)
                ctx.sync()
                want, bound = attnref.attention(ref, [0, new], [n], pages, qv, 0.125, window)
                bar = _defined(kind, want, bound, half) + (np.abs(v).max() * 2.0 ** -11 if kind == "bf16" else 0)
                err = np.abs(host(out, kind) - want)
                assert np.all(err <= bar), (cleared, window, float(np.max(err / bar)))
            kv.free()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new", [1, 150])
@pytest.mark.parametrize("plane", [0, 1])
def test_negative_scales_count_as_no_number(ctx, kind, new, plane):  # noqa: F811
    t, _ = TYPES[kind]
    rng = np.random.default_rng(new)
    with Device(ctx) as dev:
        size, codes = qmm.kv_bytes(4, 1, 64, 64), 2 * 4 * 64 * 64
        mem = dev(np.zeros(size, np.uint8))
        kv = ctx.kv_create(4, 1, 64, 64, memory=mem.ptr)
        k = rng.standard_normal((200, 1, 64)).astype(np.float32)
        ctx.kv_write(kv, qmm.Batch.of([0, 200], [200], [[0, 1, 2, 3]]), k, k)
        b = qmm.Batch(1, 4, dev(np.array([0, new], np.int32)).ptr, dev(np.array([200], np.int32)).ptr, dev(np.arange(4), np.int32).ptr)
        q = dev.values(rng.standard_normal((new, 2, 64)), kind)[0]
        raw = mem.numpy()
        scales = raw[codes:].view(np.float32)
        scales[4 * plane + 1] *= -1  # tokens 64 .. 127
        mem.set(raw)
        for window in (0, 73, 40):
            out = dev.values(np.zeros((new, 2, 64)), kind)[0]
            ctx.attention_device(kv, b, qmm.Attention(t, 2, 0.125, window), q.ptr, new, out.ptr)
            ctx.sync()
            at = np.arange(200 - new, 200)
            sees = (at >= 64) & (at - (window or 1000) + 1 < 128)
            got = host(out, kind)
            assert np.isnan(got[sees]).all() and np.isfinite(got[~sees]).all()
        kv.free()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new", [40, 150])
def test_rows_that_see_nothing_give_zeros_whatever_they_hold(ctx, kind, new):  # noqa: F811
    """rows of negative positions (device arrays), their queries infinities and NaN"""
    t, _ = TYPES[kind]
    rng = np.random.default_rng(new)
    for sinks in (False, True):
        with Device(ctx) as dev:
            kv = ctx.kv_create(2, 2, 64, 64)
            k = rng.standard_normal((3, 2, 64)).astype(np.float32)
            ctx.kv_write(kv, qmm.Batch.of([0, 3], [3], [[1]]), k, k)
            x = rng.standard_normal((new, 4, 64)).astype(np.float32)
            x[0::3, :, 5], x[1::3, :, 9], x[2:new - 3:3, :, 0] = np.nan, np.inf, -np.inf
            x[new - 3:] = 1
            q, out = dev.values(x, kind)[0], dev.values(np.full((new, 4, 64), 7.0), kind)[0]
            how = qmm.Attention(t, 4, 0.125, sinks=dev(np.zeros(4, np.float32)).ptr if sinks else None)
            b = qmm.Batch(1, 1, dev(np.array([0, new], np.int32)).ptr, dev(np.array([3], np.int32)).ptr, dev(np.array([[1]], np.int32)).ptr)
            ctx.attention_device(kv, b, how, q.ptr, new, out.ptr)
            ctx.sync()
            got = host(out, kind)
            assert np.all(got[:new - 3] == 0) and np.all(np.abs(got[new - 3:]).max(-1) > 0) and np.isfinite(got).all()
            kv.free()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("new", [1, 100])
@pytest.mark.parametrize("size", [120, 126, -90, -110])
def test_queries_at_the_ends_of_the_exponents(ctx, kind, new, size):  # noqa: F811
    """queries around 2^size over keys around 2^-size: ordinary scores"""
    t, half = TYPES[kind]
    rng = np.random.default_rng(new)
    n, dim = 200, 64
    k = (rng.uniform(0.5, 1.9, (n, 1, dim)) * rng.choice([-1, 1], (n, 1, dim)) * 2.0 ** -size).astype(np.float32)
    v = rng.standard_normal((n, 1, dim)).astype(np.float32)
    ref = attnref.Cache(4, 1, dim, 64)
    kv = ctx.kv_create(4, 1, dim, 64)
    pages = [[2, 0, 1, 3]]
    ctx.kv_write(kv, qmm.Batch.of([0, n], [n], pages), k, v)
    ref.write([0, n], [n], pages, k, v)
    with Device(ctx) as dev:
        q, qv = dev.values((rng.uniform(0.5, 1.9, (new, 2, dim)) * rng.choice([-1, 1], (new, 2, dim)) * 2.0 ** size).astype(np.float32), kind)
        out = dev.values(np.zeros((new, 2, dim)), kind)[0]
        b = qmm.Batch(1, 4, dev(np.array([0, new], np.int32)).ptr, dev(np.array([n], np.int32)).ptr, dev(pages, np.int32).ptr)
        ctx.attention_device(kv, b, qmm.Attention(t, 2, 0.125), q.ptr, new, out.ptr)
        ctx.sync()
        with np.errstate(over="ignore"):  # its bound adds a least scale of 1e-30, far above these: formed here as there, from the scales
            want, _ = attnref.attention(ref, [0, new], [n], pages, qv, 0.125)
        magnitudes = float(np.abs(qv.astype(np.float64)).sum(-1).max()) * 0.125 * 1.4427 * 256 * float(ref.scales[0].max())
        assert 20 < magnitudes < 120
        d = 2.0 ** -24 * (4 + 32) * magnitudes
        own = np.abs(v).max() * (2 * (2.0 ** d - 1 + 2.0 ** -20) + (2.0 ** -11 if kind == "bf16" else 0))
        assert np.all(np.abs(host(out, kind) - want) <= own + (half + 2.0 ** -24) * np.abs(want))
    kv.free()


@pytest.mark.parametrize("dim", [192, 256])
def test_first_calls_of_several_threads(dim):
    """a context per thread, all at their first prompt of a head size whose kernel asks for its LDS once per device"""
    rng = np.random.default_rng(dim)
    n, kinds = 150, ["f32", "f16"]
    k, v = rng.standard_normal((2, n, 1, dim)).astype(np.float32)
    ref = attnref.Cache(3, 1, dim, 64)
    ref.write([0, n], [n], [[2, 0, 1]], k, v)
    start, got = threading.Barrier(4), {}

    def work(i):
        with qmm.Context(0) as c:
            kv = c.kv_create(3, 1, dim, 64)
            b = qmm.Batch.of([0, n], [n], [[2, 0, 1]])
            c.kv_write(kv, b, k, v)
            q = np.random.default_rng(i).standard_normal((n, 2, dim)).astype(np.float32 if kinds[i % 2] == "f32" else np.float16)
            start.wait(60)
            got[i] = q, c.attention(kv, b, q, 0.0625, softcap=30.0 * (i // 2))
            kv.free()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert sorted(got) == [0, 1, 2, 3]
    for i, (q, out) in got.items():
        want, bound = attnref.attention(ref, [0, n], [n], [[2, 0, 1]], q, 0.0625, cap=30.0 * (i // 2))
        kind = kinds[i % 2]
        assert np.all(np.abs(out.astype(np.float64) - want) <= _defined(kind, want, bound, TYPES[kind][1]))


def test_caps_from_the_smallest_to_the_largest(ctx):  # noqa: F811
    """2^-64 and 2^64 hold; beyond them a score in units of the cap, or the cap itself in units of log2, leaves fp32: refused"""
    rng = np.random.default_rng(1)
    n, dim = 130, 64
    k, v = rng.standard_normal((2, n, 1, dim)).astype(np.float32)
    ref = attnref.Cache(3, 1, dim, 64)
    kv = ctx.kv_create(3, 1, dim, 64)
    b = qmm.Batch.of([0, n], [n], [[2, 0, 1]])
    ctx.kv_write(kv, b, k, v)
    ref.write([0, n], [n], [[2, 0, 1]], k, v)
    for new in (1, n):
        rows = qmm.Batch.of([0, new], [n], [[2, 0, 1]])
        for kind in (np.float32, np.float16):
            q = rng.standard_normal((new, 2, dim)).astype(kind)
            q[0, 0] = 0  # scores of 0 stay 0 under every cap
            for cap in (2.0 ** -64, 1e-6, 1e6, 2.0 ** 64):
                got = ctx.attention(kv, rows, q, 0.125, softcap=cap).astype(np.float64)
                want, bound = attnref.attention(ref, [0, new], [n], [[2, 0, 1]], q, 0.125, cap=cap)
                name = "f32" if kind is np.float32 else "f16"
                assert np.all(np.abs(got - want) <= _defined(name, want, bound, TYPES[name][1])), (new, kind, cap)
            for cap in (3e38, 1e38, 2.0 ** 65, 2.0 ** -65, 1e-39, 1e-45):
                with pytest.raises(qmm.QmmError) as e:
                    ctx.attention(kv, rows, q, 0.125, softcap=cap)
                assert e.value.code == qmm.ERR_UNSUPPORTED
    kv.free()



@pytest.mark.parametrize("new", [1, 4, 70])
@pytest.mark.parametrize("dim", [64, 128])
def test_scores_that_are_small_differences_f16(ctx, new, dim):  # noqa: F811
    """whole-number queries and keys, so that every product and partial sum of a score is a whole number below 2^24 and fp32
    holds it: what a score may lose is its own rounding, not one of the magnitudes that it is the difference of.  The tokens
    are picked so that their scores lie within a few units of each other, far below those magnitudes (300 in log2)."""
    rng = np.random.default_rng(new + dim)
    n, heads, block = 192, 4, 64
    pages = rng.permutation(4)[:3].reshape(1, 3)
    q = np.zeros((new, heads, dim), np.float16)
    k = np.zeros((n, heads, dim), np.float32)
    for h in range(heads):
        q[:, h] = rng.integers(-255, 256, dim)
        codes = rng.integers(-127, 128, (400000, dim))
        codes[:, 7] = 127  # every block's scale is 1 to a rounding
        score = codes @ q[0, h].astype(np.int64)
        k[:, h] = codes[rng.permutation(np.argsort(np.abs(score - 2 * score.std()))[:n])]
    v = rng.standard_normal((n, heads, dim)).astype(np.float32)
    ref = attnref.Cache(4, heads, dim, block)
    kv = ctx.kv_create(4, heads, dim, block)
    b = qmm.Batch.of([0, n], [n], pages)
    ctx.kv_write(kv, b, k, v)
    ref.write([0, n], [n], pages, k, v)
    assert np.array_equal(ref.codes[0][pages[0]].transpose(0, 2, 1, 3).reshape(n, heads, dim), k)
    magnitudes = np.abs(q[0].astype(np.float64)).sum(-1).max() * 64 * 1.4427
    scale = np.float32(300 / magnitudes)
    got = ctx.attention(kv, qmm.Batch.of([0, new], [n], pages), q, float(scale)).astype(np.float64)
    want, _ = attnref.attention(ref, [0, new], [n], pages, q, np.float64(scale))
    # scores in units of log2 up to |z|: the product with its factor, the factor's own three roundings, the difference to the
    # maximum: 5 half steps of |z|; the weights' and sums' own 2^-20 on top, half a step of f16 and one of its subnormals
    z = max(np.abs(k[:, h].astype(np.float64) @ q[0, h].astype(np.float64)).max() for h in range(heads)) * float(scale) * 1.4427
    bar = np.abs(v).max() * 2 * (2.0 ** (5 * 2.0 ** -24 * z) - 1 + 2.0 ** -20) + 2.0 ** -11 * np.abs(want) + 2.0 ** -25
    err = np.abs(got - want)
    assert np.all(err <= bar), float(np.max(err / bar))
    kv.free()


@pytest.mark.parametrize("new", [1, 4, 100])
@pytest.mark.parametrize("dim", [64, 256])
def test_f16_takes_probabilities_of_22_bits(ctx, new, dim):  # noqa: F811
    """no term for a rounding of the probabilities to 11 bits: attnref's bound and the output's half step, where scores are of
    one dimension (a bound of 1e-5) and six values of either sign cancel (the half step is small too).  Probabilities of 11
    bits are off by 7 to 21 of these bars."""
    rng = np.random.default_rng(new + dim)
    half = TYPES["f16"][1]
    n, heads, kv_heads, window = 200, 8, 2, 6
    k, v = np.zeros((n, kv_heads, dim), np.float32), rng.choice([-1, 1], (n, kv_heads, dim)) * rng.uniform(0.7, 1, (n, 1, 1))
    k[..., 0] = rng.uniform(-1, 1, (n, kv_heads))
    q = np.zeros((new, heads, dim), np.float16)
    q[..., 0] = rng.uniform(0.5, 1.5, (new, heads))
    ref = attnref.Cache(4, kv_heads, dim, 16)
    kv = ctx.kv_create(4, kv_heads, dim, 16)
    pages = [[2, 0, 1, 3]]
    ctx.kv_write(kv, qmm.Batch.of([0, n], [n], pages), k, v.astype(np.float32))
    ref.write([0, n], [n], pages, k, v.astype(np.float32))
    got = ctx.attention(kv, qmm.Batch.of([0, new], [n], pages), q, 1.0, window).astype(np.float64)
    want, bound = attnref.attention(ref, [0, new], [n], pages, q, 1.0, window)
    assert bound.max() < 2e-5 and (np.abs(want) < 2.0 ** -5).any()
    assert np.all(np.abs(got - want) <= _defined("f16", want, bound, half))
    kv.free()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new", [1, 100])
@pytest.mark.parametrize("block", [16, 64])
@pytest.mark.parametrize("gap", [6, 16, 20])
def test_small_values_beside_large_ones_without_weight(ctx, kind, new, block, gap):  # noqa: F811
    """one block in two holds values 2^gap larger under scores so low that it has no weight: the result has the small values'
    size.  A share is rounded at 2^-34 of the largest value scale that a tile sees, or is less than that itself; what is lost
    of a row is at most the sum over its tokens, times 127 codes."""
    t, half = TYPES[kind]
    rng = np.random.default_rng(new + block + gap)
    n, dim, heads = 400, 64, 2
    big = np.arange(n) // block % 2 == 1
    k = rng.standard_normal((n, 1, dim)) * 0.05
    k[:, 0, 0] = np.where(big, -8.0, 8.0)
    k[:, 0, 1] = rng.standard_normal(n)
    v = rng.standard_normal((n, 1, dim)) * np.where(big, 2.0 ** gap, 1.0)[:, None, None]
    k, v = k.astype(np.float32), v.astype(np.float32)
    pages = rng.permutation(8)[:7].reshape(1, 7)
    ref = attnref.Cache(8, 1, dim, block)
    kv = ctx.kv_create(8, 1, dim, block)
    ctx.kv_write(kv, qmm.Batch.of([0, n], [n], pages), k, v)
    ref.write([0, n], [n], pages, k, v)
    with Device(ctx) as dev:
        x = rng.standard_normal((new, heads, dim)) * 0.1
        x[..., 0], x[..., 1] = 16, 6  # scores of -128 and of 128 +- 18: the large values' weights are below e^-200
        q, qv = dev.values(x, kind)
        out = dev.values(np.zeros((new, heads, dim)), kind)[0]
        b = qmm.Batch(1, 7, dev(np.array([0, new], np.int32)).ptr, dev(np.array([n], np.int32)).ptr, dev(pages, np.int32).ptr)
        ctx.attention_device(kv, b, qmm.Attention(t, heads, 1.0), q.ptr, new, out.ptr)
        ctx.sync()
        want, _ = attnref.attention(ref, [0, new], [n], pages, qv, 1.0)
        step = 2.0 ** -33 * float(ref.scales[1].max())  # the kernel's reference is a power of two, up to twice the largest scale
        kk = ref.values(pages[0], n)[0][:, 0]
        z = np.einsum("nhd,md->nhm", qv.astype(np.float64), kk)
        z[:, :, big] = -np.inf
        z = np.where(np.arange(n)[None, None, :] <= np.arange(n - new, n)[:, None, None], z, -np.inf)
        w = np.exp(z - z.max(-1, keepdims=True))
        w /= w.sum(-1, keepdims=True)
        scales = np.repeat(np.concatenate([ref.scales[1][p, 0] for p in pages[0]]), block)[:n].astype(np.float64)
        lost = 127 * np.minimum(step, w * scales).sum(-1)[..., None]
        # scores: 6e-6 of the magnitudes that make them (subnormal key codes; bf16), 64 half steps of them otherwise; a
        # probability's own 2^-12 (bf16); the output's half step
        small = float(np.abs(v[~big]).max())
        d = (8e-6 if kind == "bf16" else 2.0 ** -18) * 1.4427 * (128 + 18 + 12)
        own = small * (2 * (2.0 ** d - 1 + 2.0 ** -20) + (2.0 ** -11 if kind == "bf16" else 0))
        err, bar = np.abs(host(out, kind) - want), lost + own + (half + 2.0 ** -24) * np.abs(want) + 2.0 ** -25 * (kind == "f16")
        assert np.sqrt(np.mean(want ** 2)) > 5 * bar.max()  # the bar would see the small values lost
        assert np.all(err <= bar), (float(np.max(err / bar)), float(lost.max()), own)
    kv.free()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,new", [(200, 1), (200, 150), (9000, 1), (9000, 20)])
def test_sinks_from_the_lowest_to_the_largest(ctx, kind, n, new):  # noqa: F811
    """minus infinity and the lowest numbers: as without a sink; the largest and infinity take all the weight: zeros"""
    t, half = TYPES[kind]
    rng = np.random.default_rng(n + new)
    table = -(-n // 64)
    pages = rng.permutation(table).reshape(1, table)
    k, v = rng.standard_normal((2, n, 1, 64)).astype(np.float32)
    sinks = np.array([-np.inf, -3e38, -1e4, 0.5, 1e4, 3e38, np.inf, np.nan], np.float32)
    kv = ctx.kv_create(table, 1, 64, 64)
    ctx.kv_write(kv, qmm.Batch.of([0, n], [n], pages), k, v)
    with Device(ctx) as dev:
        q = dev.values(rng.standard_normal((new, 8, 64)), kind)[0]
        b = qmm.Batch(1, table, dev(np.array([0, new], np.int32)).ptr, dev(np.array([n], np.int32)).ptr, dev(pages, np.int32).ptr)
        got = []
        for s in (None, dev(sinks).ptr):
            out = dev.values(np.zeros((new, 8, 64)), kind)[0]
            ctx.attention_device(kv, b, qmm.Attention(t, 8, 0.125, sinks=s), q.ptr, new, out.ptr)
            ctx.sync()
            got.append(host(out, kind))
        assert np.array_equal(got[0][:, :3], got[1][:, :3]) and np.isfinite(got[1][:, :7]).all()
        # the sink of 0.5 takes 1.6 / 9000 = 2^-12.4 of the weight there, less than half a step of the 16-bit types: the rounded
        # result is smaller or the same, never larger
        assert np.all(np.abs(got[1][:, 3]) <= np.abs(got[0][:, 3])) and np.all(got[1][:, 4:7] == 0)
        assert np.isnan(got[1][:, 7]).all()
    kv.free()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("new", [3, 40, 150])
def test_the_largest_window_is_none(ctx, causal, new):  # noqa: F811
    """rows of negative positions among them: position less window stays in range, and the bits are those without a window"""
    rng = np.random.default_rng(new)
    kv = ctx.kv_create(3, 1, 64, 64)
    n = 130
    k, v = rng.standard_normal((2, n, 1, 64)).astype(np.float32)
    ctx.kv_write(kv, qmm.Batch.of([0, n], [n], [[2, 0, 1]]), k, v)
    with Device(ctx) as dev:
        q = dev.values(rng.standard_normal((2 * new, 2, 64)), "f32")[0]
        lens = dev(np.array([2, n], np.int32))
        b = qmm.Batch(2, 3, dev(np.array([0, new, 2 * new], np.int32)).ptr, lens.ptr, dev(np.array([[2, 0, 1]] * 2, np.int32)).ptr)
        got = []
        for window in (0, 2 ** 31 - 1, 2 ** 31 - 200):
            out = dev.values(np.full((2 * new, 2, 64), 7.0), "f32")[0]
            ctx.attention_device(kv, b, qmm.Attention(qmm.F32, 2, 0.125, window, causal=causal), q.ptr, 2 * new, out.ptr)
            ctx.sync()
            got.append(out.numpy())
        assert np.isfinite(got[0]).all() and np.abs(got[0][new:]).max() > 0.01
        assert not causal or np.all(got[0][: new - 2] == 0)
        assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])
    kv.free()
