"""The 4-bit cache without a GPU: its sizes, the layout as a bijection, and the codes of the plain form."""
import numpy as np
import pytest

import kv4_cases as kc


def test_bytes(lb):
    assert lb.kv4_bytes(3, 64, 4, 256) == 3 * 4 * 4 * 18 * 256
    assert lb.kv4_bytes(64, 1 << 20, 32, 256) == 64 * 32 * (1 << 16) * 18 * 256  # beyond 32 bits
    for shape in ((0, 64, 4, 256), (1, 63, 4, 256), (1, 0, 4, 256), (1, 64, 0, 256), (1, 64, 33, 256), (1, 64, 4, 96), (1 << 20, 64, 4, 256), (1, (1 << 20) + 16, 4, 64)):
        assert lb.kv4_bytes(*shape) == 0, shape


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_layout_is_a_bijection(dim):
    row, f = np.arange(16)[:, None], np.arange(dim)[None]
    seen = np.zeros((kc.block_bytes(dim), 2), int)
    for place in (kc.key_byte, kc.value_byte):
        np.add.at(seen, (place(dim, row, f), f % 2 + 0 * row), 1)
    for part in range(2):
        for r in range(16):
            for g in range(dim // 64):
                for o in range(4):
                    seen[kc.pair_byte(dim, part, r, g) + o] += 1
    assert (seen == 1).all()


def test_codes_are_the_nearest():
    rng = np.random.default_rng(3)
    x = rng.standard_normal((50, 2, 128)) * 10.0 ** rng.uniform(-3, 3, (50, 2, 1))
    x[0] = 2.5  # a constant group: scale 0, its value exact in fp16
    code, scale, lowest = kc.quantise(x)
    v = kc.values(code, scale, lowest)
    assert (v[0] == 2.5).all()
    every = lowest[..., None, None] + scale[..., None, None] * np.arange(16)
    best = np.abs(every - x.reshape(*code.shape)[..., None]).min(-1).reshape(x.shape)
    assert np.allclose(np.abs(v - x), best, rtol=0, atol=1e-12)


def test_a_call_without_a_context_is_refused(lb):
    import ctypes as C
    cache, batch = lb.Kv4Cache(16, 1, 16, 1, 64), lb.Kv4Batch(0, 16, 0, 1, 1)
    L = lb.lib()
    assert L.lb_kv4_append(None, C.byref(cache), C.byref(batch), 16, 16, 0, 0, 0, 0, 1e7, 1e-6) == lb.LB_ERR_INVALID
    assert L.lb_kv4_read(None, C.byref(cache), C.byref(batch), 16, 16, 0) == lb.LB_ERR_INVALID
    assert L.lb_kv4_attention(None, C.byref(cache), C.byref(batch), 16, 0, 0, 0, 0, 0, 16, 1, 1, 0, 1e7, 1e-6) == lb.LB_ERR_INVALID
