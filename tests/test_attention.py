"""Rotation, cache and attention without a GPU: the restatement that the GPU tests compare with is pinned here by closed
forms, the frequency table by the published rules, and calls that no device is needed to refuse are refused."""
import ctypes

import numpy as np
import pytest

import attnref
from ollama_amd import qmm


def test_places_are_a_permutation_and_match_the_stated_order():
    for dim in (8, 64, 80, 128, 200, 256):
        dp = attnref.row_dim(dim)
        for place in attnref.places(dim):
            assert place.shape == (64, dim) and len(np.unique(place)) == 64 * dim and place.min() >= 0 and place.max() < 64 * dp
    key, value = attnref.places(128)
    assert key[0, 0] == 0 and key[0, 15] == 15 and key[1, 0] == 16 and key[0, 16] == 256 and key[0, 64] == 1024 and key[16, 0] == 2048
    assert value[0, 0] == 0 and value[3, 0] == 3 and value[16, 0] == 4 and value[63, 0] == 3 * 256 + 15 and value[0, 1] == 16 and value[0, 16] == 1024


def test_restated_rotation_closed_forms():
    freqs = np.array([1.0, 0.25])
    x = np.array([[[1.0, 2.0, 3.0, 4.0, 5.0, 6.0]]])
    assert np.allclose(attnref.rope(x, [0], freqs), x)
    y = attnref.rope(x, [2], freqs)[0, 0]  # pairs (0, 2) and (1, 3)
    assert np.allclose(y[[0, 2]], [np.cos(2) - 3 * np.sin(2), np.sin(2) + 3 * np.cos(2)]) and np.allclose(y[4:], [5, 6])
    y = attnref.rope(x, [4], freqs, halves=False)[0, 0]  # pairs (0, 1) and (2, 3)
    assert np.allclose(y[2:4], [3 * np.cos(1) - 4 * np.sin(1), 3 * np.sin(1) + 4 * np.cos(1)])
    y = attnref.rope(np.full((1, 1, 8), 3.0), [7], np.zeros(0), weight=np.arange(8.0))
    assert np.allclose(y[0, 0], np.arange(8.0))
    # scores depend on the difference of positions only
    rng = np.random.default_rng(0)
    f = 10000.0 ** (-np.arange(32) / 32)
    q, k = rng.standard_normal((2, 1, 1, 64))
    dots = [float((attnref.rope(q, [p + 11], f) * attnref.rope(k, [p], f)).sum()) for p in (0, 5, 1000)]
    assert np.allclose(dots, dots[0])


def test_restated_cache_closed_forms():
    c = attnref.Cache(3, 1, 8, 16)
    k = np.zeros((20, 1, 8), np.float32)
    k[:, 0, 0] = np.arange(1, 21)
    c.write([0, 20], [20], [[2, 0]], k, -k)
    assert c.scales[0][2, 0, 0] == np.float32(16 * attnref.PER127) and c.scales[0][2, 0, 1] == np.float32(20 * attnref.PER127)
    assert c.codes[0][2, 0, 15, 0] == 127 and c.codes[1][2, 0, 15, 0] == -127 and c.codes[0][2, 0, 19, 0] == 127
    c.write([0, 1], [21], [[2, 0]], np.full((1, 1, 8), 40, np.float32), np.zeros((1, 1, 8), np.float32))
    assert c.scales[0][2, 0, 1] == np.float32(40 * attnref.PER127) and c.codes[0][2, 0, 20, 0] == 127
    assert c.codes[0][2, 0, 19, 0] == 64  # 127 / 2 to even
    assert c.scales[1][2, 0, 1] == np.float32(20 * attnref.PER127)
    kk, _ = c.read([0, 3], [21], [[2, 0]], 4)
    assert np.allclose(kk[:3, 0, 0], [19, 20, 40], rtol=0.02) and np.all(kk[3] == 0)


def test_restated_attention_closed_forms():
    c = attnref.Cache(2, 1, 8, 64)
    k, v = np.zeros((3, 1, 8), np.float32), np.zeros((3, 1, 8), np.float32)
    v[:, 0, 0] = [127, 64, 1]
    c.write([0, 3], [3], [[1]], k, v)
    q = np.ones((3, 2, 8))
    out, _ = attnref.attention(c, [0, 3], [3], [[1]], q, 1.0)
    assert np.allclose(out[:, :, 0].T, [127, 95.5, 64])
    out, _ = attnref.attention(c, [0, 3], [3], [[1]], q, 1.0, window=1)
    assert np.allclose(out[:, 0, 0], [127, 64, 1])
    out, _ = attnref.attention(c, [0, 3], [3], [[1]], q, 1.0, causal=False, sinks=[0.0, -np.inf])
    assert np.allclose(out[:, 0, 0], 48) and np.allclose(out[:, 1, 0], 64)


def test_rope_freqs():
    f, m = qmm.rope_freqs(64, 10000.0)
    assert m == 1.0 and np.allclose(f, 10000.0 ** (-np.arange(32) / 32), rtol=1e-15)
    f2, m = qmm.rope_freqs(64, 10000.0, freq_scale=0.25, attn_factor=1.5)
    assert m == 1.5 and np.allclose(f2, f / 4, rtol=1e-15)
    fac = np.linspace(1, 8, 32).astype(np.float32)
    assert np.allclose(qmm.rope_freqs(64, 10000.0, factors=fac)[0], f / fac, rtol=1e-15)
    # YaRN: frequencies that turn often stay, those that hardly turn are scaled, in between monotonously
    y, m = qmm.rope_freqs(128, 150000.0, freq_scale=1 / 32, ext_factor=1.0, beta_fast=32, beta_slow=1, n_ctx_orig=4096)
    p = 150000.0 ** (-np.arange(64) / 64)
    turns = 4096 * p / (2 * np.pi)
    assert np.allclose(y[turns > 40], p[turns > 40], rtol=1e-12) and np.allclose(y[turns < 0.8], p[turns < 0.8] / 32, rtol=1e-12)
    ratio = y / p
    assert np.all(np.diff(ratio) <= 1e-12) and np.any((ratio > 0.1) & (ratio < 0.9)) and abs(m - (1 + 0.1 * np.log(32))) < 1e-6
    for bad in (dict(n_rot=63, base=1e4), dict(n_rot=0, base=1e4), dict(n_rot=64, base=1.0), dict(n_rot=64, base=1e4, freq_scale=0.0),
                dict(n_rot=64, base=1e4, ext_factor=1.0)):
        with pytest.raises(qmm.QmmError) as e:
            qmm.rope_freqs(**bad)
        assert e.value.code == qmm.ERR_INVALID
    with pytest.raises(ValueError):
        qmm.rope_freqs(64, 1e4, factors=np.ones(3))


def test_cache_sizes():
    assert qmm.kv_bytes(10, 8, 128, 64) == 10 * 8 * (2 * 64 * 128 + 8)
    assert qmm.kv_bytes(3, 5, 80, 16) == 3 * 5 * (2 * 64 * 128 + 32)
    assert len(attnref.Cache(3, 5, 80, 16).memory()) == qmm.kv_bytes(3, 5, 80, 16)
    for bad in ((0, 8, 128, 64), (1, 0, 128, 64), (1, 8, 12, 64), (1, 8, 264, 64), (1, 8, 128, 8), (1, 8, 128, 128), (1 << 31, 1, 8, 64)):
        assert qmm.kv_bytes(*bad) == -1
    assert qmm.kv_bytes((1 << 31) - 1, 65535, 256, 16) > 1 << 60  # no overflow on the way


def test_struct_layouts():
    """the offsets a C compiler gives the structs of include/mi_qmm.h on a 64-bit machine"""
    h, b, a = qmm._QKHeads, qmm._Batch, qmm._Attn
    assert ctypes.sizeof(h) == 56 and [getattr(h, f).offset for f, _ in h._fields_] == [0, 4, 8, 12, 16, 20, 24, 28, 32, 40, 48]
    assert ctypes.sizeof(b) == 32 and [getattr(b, f).offset for f, _ in b._fields_] == [0, 4, 8, 16, 24]
    assert ctypes.sizeof(a) == 32 and [getattr(a, f).offset for f, _ in a._fields_] == [0, 4, 8, 12, 16, 20, 24]


def test_refusals_without_a_device():
    L = qmm.lib()
    out = ctypes.c_void_p()
    heads = qmm.QKHeads(qmm.F32, 4, 2, 64, None, 0)
    batch, how = qmm.Batch(1, 1, None, None, None), qmm.Attention(qmm.F32, 4, 1.0)
    rope = lambda h, n=1, loc=qmm.DEVICE: L.mi_qmm_qk_norm_rope(None, h._p if h else None, None, 256, None, 128, None, n, None, 256, None, 128, loc)  # noqa: E731
    assert rope(None) == qmm.ERR_INVALID and "heads" in qmm.last_error()
    assert rope(heads) == qmm.ERR_INVALID and "ctx is NULL" in qmm.last_error()
    assert rope(heads, n=-1) == qmm.ERR_INVALID and rope(heads, loc=5) == qmm.ERR_INVALID
    for bad, code in (((qmm.Q8_0, 4, 2, 64, None, 0), qmm.ERR_UNSUPPORTED), ((qmm.F32, 0, 2, 64, None, 0), qmm.ERR_INVALID),
                      ((qmm.F32, 4, -1, 64, None, 0), qmm.ERR_INVALID), ((qmm.F32, 4, 2, 60, None, 0), qmm.ERR_UNSUPPORTED),
                      ((qmm.F32, 4, 2, 512, None, 0), qmm.ERR_UNSUPPORTED), ((qmm.F32, 4, 2, 64, None, 72), qmm.ERR_UNSUPPORTED),
                      ((qmm.F32, 4, 2, 64, None, 20), qmm.ERR_UNSUPPORTED), ((qmm.F32, 4, 2, 64, None, 0, 7), qmm.ERR_INVALID)):
        assert rope(qmm.QKHeads(*bad)) == code, bad
    assert rope(qmm.QKHeads(qmm.F32, 4, 2, 64, None, 0, eps=-1.0)) == qmm.ERR_INVALID
    assert L.mi_qmm_kv_create(None, 1, 1, 64, 64, None, None) == qmm.ERR_INVALID
    assert L.mi_qmm_kv_create(None, 1, 1, 64, 48, None, ctypes.byref(out)) == qmm.ERR_UNSUPPORTED
    assert L.mi_qmm_kv_create(None, 1, 1, 64, 64, 100, ctypes.byref(out)) == qmm.ERR_INVALID and "aligned" in qmm.last_error()
    assert L.mi_qmm_kv_create(None, 1, 1, 64, 64, None, ctypes.byref(out)) == qmm.ERR_INVALID and not out.value
    L.mi_qmm_kv_free(None)
    for call in (L.mi_qmm_kv_write, L.mi_qmm_kv_read):
        assert call(None, None, batch._p, qmm.Q4_K, None, 64, None, 64, 1, qmm.DEVICE) == qmm.ERR_UNSUPPORTED
        assert call(None, None, batch._p, qmm.F32, None, 64, None, 64, -1, qmm.DEVICE) == qmm.ERR_INVALID
        assert call(None, None, batch._p, qmm.F32, None, 64, None, 64, 1 << 25, qmm.DEVICE) == qmm.ERR_UNSUPPORTED
        assert call(None, None, batch._p, qmm.F32, None, 64, None, 64, 1, qmm.DEVICE) == qmm.ERR_INVALID
    assert L.mi_qmm_attention(None, None, batch._p, None, None, 64, None, 64, 1, qmm.DEVICE) == qmm.ERR_INVALID
    assert L.mi_qmm_attention(None, None, batch._p, how._p, None, 64, None, 64, 1, qmm.DEVICE) == qmm.ERR_INVALID and "ctx" in qmm.last_error()


def test_python_side_shape_checks():
    with pytest.raises(ValueError):
        qmm.Batch.of([0, 1], [1, 1], [[0]])
    with pytest.raises(ValueError):
        qmm.Batch.of([0, 1], [1], [0])
    b = qmm.Batch.of([0, 1], [1], [[0, 5]])
    assert b._s.n_seqs == 1 and b._s.max_pages == 2
    with pytest.raises(TypeError):
        qmm._value_type(np.zeros(1))


def test_batches_of_the_wrong_side_are_refused():
    """host addresses never reach a kernel, device addresses never the host's checks"""
    kv = qmm.KVCache(None, 1, 1, 8, 64)
    ctx = qmm.Context.__new__(qmm.Context)
    ctx._h = None
    host, device = qmm.Batch.of([0, 1], [1], [[0]]), qmm.Batch(1, 1, 4096, 4096, 4096)
    x, how = np.zeros((1, 1, 8), np.float32), qmm.Attention(qmm.F32, 1, 1.0)
    for call in (lambda: ctx.kv_write(kv, device, x, x), lambda: ctx.kv_read(kv, device, 1), lambda: ctx.attention(kv, device, x, 1.0),
                 lambda: ctx.kv_write_device(kv, host, qmm.F32, 4096, 4096, 1), lambda: ctx.kv_read_device(kv, host, qmm.F32, 4096, 4096, 1),
                 lambda: ctx.attention_device(kv, host, how, 4096, 1, 4096)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ctx.kv_write(kv, host, x, x), lambda: ctx.attention_device(kv, device, how, 4096, 1, 4096)):
        with pytest.raises(qmm.QmmError):  # these come as far as the missing context
            call()


def test_rope_freqs_of_no_numbers_are_refused():
    """an infinite frequency would turn position 0 into NaN; nothing is written"""
    for bad in (dict(base=np.inf), dict(base=np.nan), dict(freq_scale=np.inf), dict(freq_scale=np.nan), dict(attn_factor=np.nan),
                dict(ext_factor=np.nan, n_ctx_orig=4096), dict(factors=[1, 0, 1, 1]), dict(factors=[1, 1, 1, -2]), dict(factors=[np.nan, 1, 1, 1]),
                dict(factors=[1, np.inf, 1, 1])):
        with pytest.raises(qmm.QmmError) as e:
            qmm.rope_freqs(8, **{"base": 1e4, **bad})
        assert e.value.code == qmm.ERR_INVALID, bad
    f, m = qmm.rope_freqs(8, 1e4, factors=[1, 2, 4, 1e30])
    assert np.isfinite(f).all() and (f > 0).all() and m == 1.0
