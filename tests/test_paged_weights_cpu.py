"""The bounds that attention over a paged cache is held to, against results that lack something: they must not pass."""
import numpy as np
import pytest

import vkllama_b200 as vk
from oracle import paged as P
from paged_weights import LONG_STEPS, Cache, Sink, draw, near, references, to_values, tolerance


@pytest.mark.parametrize("dtype", [vk.FP16, vk.BF16])
@pytest.mark.parametrize("kernel,n,dim", [("token", 300, 128), ("token", 4000, 64), ("token", 70001, 64), ("tensor", 3000, 128), ("rows", 900, 200)])
def test_a_missing_tile_does_not_pass(dtype, kernel, n, dim):
    """Sixteen positions that count as if they were not there, as where a part of a pair gets lost."""
    if dtype == vk.BF16 and n > 4000:  # half a step is 2^-8, a position's weight 2^-16
        pytest.skip("bfloat16 outputs have 8 bits: sixteen of 70,000 positions do not show")
    rng = np.random.default_rng(n + dim)
    c = Cache(rng, [n], 1, dim, 16, dtype)
    q = to_values(draw(rng, (1, 2 * dim), dtype), dtype).reshape(1, 2, dim)
    want, mass, size, den, biggest = references(c, 0, q, [n - 1])
    tol = tolerance(want, mass, size, den, dtype, dim, n, biggest, kernel, LONG_STEPS if n > 4000 else None)
    for first in (0, n // 2 // 16 * 16, n - 16):
        keep = np.r_[0:first, first + 16:n]
        k, v = to_values(c.seq_k[0][:, keep], dtype), to_values(c.seq_v[0][:, keep], dtype)
        assert (np.abs(P.attention(q, [n - 17], k, v)[0] - want) > tol).any(), first


@pytest.mark.parametrize("kernel", ["token", "rows", "tensor"])
@pytest.mark.parametrize("gap", [14.0, 17.0, 18.0, 20.0])
def test_small_weights_that_vanish_do_not_pass(kernel, gap):
    """Weights rounded to the steps of fp16 as they are, without a power of two."""
    n, dim = 4000, 64
    rng = np.random.default_rng(3)
    c = Sink(rng, [n], 1, dim, 16, vk.FP16, gap)
    k, v = (to_values(s[0], vk.FP16)[0] for s in (c.seq_k, c.seq_v))
    q = to_values(c.queries(1, 1, dim, vk.FP16), vk.FP16).reshape(1, 1, dim)
    p = np.exp(k @ q[0, 0] - gap)
    hi = p.astype(np.float16).astype(float)
    lo = (p - hi).astype(np.float16).astype(float) if kernel == "token" else 0
    with pytest.raises(AssertionError):
        near(((hi + lo) @ v / p.sum())[None, None], c, 0, q, [n - 1], kernel, scale=1.0)
    near((p @ v / p.sum())[None, None], c, 0, q, [n - 1], kernel, scale=1.0)
