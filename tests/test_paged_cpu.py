"""The paged cache's oracle against cases worked out by hand, and what its entry points refuse without a device."""
import ctypes as C

import numpy as np

import vkllama_b200 as vk
from oracle import paged as P


def test_pages_come_and_go():
    table = np.zeros((2, 3), np.uint32)
    table[0, 0] = 7
    got = P.resize(4, [3, 0], [6, 5], table, [5, 1, 2, 9], 9)
    lengths, table, pool, m, starts = got
    assert table.tolist() == [[7, 9, 0], [2, 1, 0]] and pool == [5] and starts.tolist() == [0, 3, 8]
    assert m[0].tolist() == [31, 36, 37, 8, 9, 10, 11, 4, P.NO_SLOT] and m[1].tolist() == [3, 4, 5, 0, 1, 2, 3, 4, 0]
    back = P.resize(4, lengths, [3, 0], table, pool, 0)  # the inverse
    assert back[2] == [5, 1, 2, 9] and back[4].tolist() == [0, 0, 0]
    # what one gives back another can take in the same call
    both = P.resize(4, lengths, [0, 12], table, pool, 9)
    assert both[2] == [5, 9] and both[1][1].tolist() == [2, 1, 7]
    assert P.resize(4, [0, 0], [8, 13], table, [5, 1, 2, 9, 3], 21) is None  # pool
    assert P.resize(4, [0], [13], table[:1], list(range(9)), 13) is None     # table
    assert P.resize(4, [0], [9], table[:1], list(range(9)), 8) is None       # rows


def test_attention_of_the_oracle():
    rng = np.random.default_rng(3)
    k, v, q = rng.standard_normal((1, 5, 8)), rng.standard_normal((1, 5, 8)), rng.standard_normal((2, 2, 8))
    out, mass, size = P.attention(q, [0, 4], k, v, window=2)
    assert np.allclose(out[0], v[0, 0]) and np.allclose(mass[0], np.abs(v[0, 0]))
    for h in range(2):
        s = np.exp(k[0, 3:] @ q[1, h] / np.sqrt(8))
        assert np.allclose(out[1, h], (s[:, None] * v[0, 3:]).sum(0) / s.sum())
    assert P.attention(q[:1], [-1], k, v)[0].max() == 0  # a sequence of nothing


def test_rotation_of_the_oracle():
    x = np.random.default_rng(4).standard_normal((3, 2, 6))
    y = P.rotate(x, [0, 1, 1000], 100.0)
    assert (y[0] == x[0]).all() and np.allclose(np.hypot(y[..., 0::2], y[..., 1::2]), np.hypot(x[..., 0::2], x[..., 1::2]))
    z = (x[2, 1, 2] + 1j * x[2, 1, 3]) * np.exp(1j * 1000 * 100.0 ** (-2 / 6))
    assert np.allclose(y[2, 1, 2:4], [z.real, z.imag])


def test_null_arguments_are_refused():
    L, out = vk.load_library(), C.c_void_p()
    assert L.vkl_paged_tables_create(None, None, 16, C.byref(out)) == 3
    assert L.vkl_update_paged_kvcache_create(None, None, 128, 16, 10000.0, vk.FP16, C.byref(out)) == 3
    assert L.vkl_paged_attention_create(None, None, 8, 8, 128, 16, 0.0, 0, vk.FP16, C.byref(out)) == 3
    assert L.vkl_paged_tables_create(None, None, 16, None) == 3
    assert L.vkl_paged_tables_run(None, None, None, None, None, 0, C.byref(out), C.byref(out)) == 3
    assert L.vkl_update_paged_kvcache_run(None, None, None, None, None, None, None, C.byref(out)) == 3
    assert L.vkl_paged_attention_run(None, None, None, None, None, None, None, C.byref(out)) == 3
    assert b"null" in L.vkl_last_error()
