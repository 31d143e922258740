"""Attention over the 8-bit cache: the same bits on every call, and the results that the definition gives where cache contents
or arguments are out of the ordinary.  Restatement and bars as in test_gpu_attention.py."""
import numpy as np
import pytest

import attnref
from hipmem import DeviceArray
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
