"""Sequences in which one position outweighs all others, and a bound for attention that leaves its small weights room for nothing but
what their own formats cost."""
import numpy as np

import vkllama_b200 as vk
from oracle import paged as P
from paged_util import HALF_STEP, TINY, Cache, draw, tensor, to_bits, to_values

# The kernels hold a probability relative to a reference that is at most the row's largest, times a power of two, in 16 bits: in fp16 steps
# end at 2^-24, so that each is off by up to 2^-25 over that power, however small it is.
FLOOR = {"token": 2.0 ** -39, "rows": 2.0 ** -39, "tensor": 2.0 ** -36}
# One pair alone is cut over all CTAs and their warps: 70,001 positions into 1,184 parts of four products, which meet eight, sixteen and ten at a time.
LONG_STEPS = 40


def tolerance(want, mass, size, den, dtype, dim, tokens, biggest, kernel, steps=None):
    """One rounding of the output. Scores: dim exact products, sums in fp32, each of them off by 2^-24 of what they add up to; twice that (and 2^-17: three
    roundings of exponents below 2^6, 2^-18 ln 2 each, and exp2 itself) relative on a probability, numerator and denominator. Sums of
    probabilities times values go 16 positions at a time, each cut off at 2^-23 of what is there: `steps` of them one after the other, joins among
    them. Probabilities: one 16-bit number, or (one token) two of them, 2^-16 and 2^-22; and in fp16 FLOOR of each position, of a row whose
    weights add up to den."""
    steps = tokens / 16 if steps is None else steps
    p = {"token": {vk.FP16: 2.0 ** -22, vk.BF16: 2.0 ** -16}[dtype]}.get(kernel, HALF_STEP[dtype])
    rel = 4 * (dim + 4) * 2.0 ** -24 * size + 2.0 ** -17 + steps * 2.0 ** -23 + p
    return HALF_STEP[dtype] * np.abs(want) * (1 + 2.0 ** -6) + rel * mass + TINY[dtype] + (dtype == vk.FP16) * tokens * FLOOR[kernel] * biggest / den


def references(cache, i, q, pos, window=0, scale=None):
    """(output, its tolerance's parts) of rows q of sequence i."""
    k, v = (to_values(s[i], cache.dtype) for s in (cache.seq_k, cache.seq_v))
    return (*P.attention(q, pos, k, v, window, scale), P.weights_sum(q, pos, k, window, scale), np.abs(v).max(initial=0))


def near(got, cache, i, q, pos, kernel, window=0, scale=None, what="", steps=None):
    want, mass, size, den, biggest = references(cache, i, q, pos, window, scale)
    tol = tolerance(want, mass, size, den, cache.dtype, cache.dim, max(pos) + 1, biggest, kernel, steps)
    off = np.abs(got - want) / tol
    worst = np.unravel_index(np.argmax(off), off.shape)
    assert off[worst] <= 1, "%s: %r: %g instead of %g, tolerance %g" % (what, worst, got[worst], want[worst], tol[worst])


class Sink(Cache):
    """A position of each sequence has a score `gap` above the others', which are equal but for `spread`, with a scale of 1 and the queries below. Its value is
    `value`; the others' have one sign, so that what is lost does not cancel."""

    def __init__(self, rng, lengths, kv, dim, page, dtype, gap, value=0.0, at=0, spread=0.0):
        super().__init__(rng, lengths, kv, dim, page, dtype)
        for i, n in enumerate(lengths):
            if not n:
                continue
            x = np.zeros((kv, n, dim))
            x[:, :, 0] = rng.standard_normal((kv, n)) * spread
            x[:, min(at, n - 1), 0] = gap
            self.seq_k[i] = to_bits(x, dtype)
            y = 1 + rng.random((kv, n, dim))
            y[:, min(at, n - 1)] = value
            self.seq_v[i] = to_bits(y, dtype)
            self.put(self.k, i, self.seq_k[i])
            self.put(self.v, i, self.seq_v[i])

    @staticmethod
    def queries(rows, heads, dim, dtype):
        q = np.zeros((rows, heads, dim))
        q[..., 0] = 1
        return to_bits(q.reshape(rows, -1), dtype)


__all__ = ["FLOOR", "LONG_STEPS", "Sink", "tensor", "near", "references", "tolerance", "draw", "to_bits", "to_values", "Cache"]
