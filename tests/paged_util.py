"""What the tests of the paged cache share: values in 16 bits, caches with pages in a random order, tolerances."""
import numpy as np

import vkllama_b200 as vk
from oracle import paged as P

HALF_STEP = {vk.FP16: 2.0 ** -11, vk.BF16: 2.0 ** -8}  # most that a rounding is off, relative
TINY = {vk.FP16: 2.0 ** -25, vk.BF16: 2.0 ** -133}     # and below the normal numbers


def to_bits(x, dtype):
    x = np.asarray(x, np.float32)
    if dtype == vk.FP16:
        return x.astype(np.float16).view(np.uint16)
    u = np.ascontiguousarray(x).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7fc0), r)


def to_values(bits, dtype):
    if dtype == vk.FP16:
        return bits.view(np.float16).astype(np.float64)
    return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def draw(rng, shape, dtype, std=1.0):
    return to_bits(rng.standard_normal(shape) * std, dtype)


def tensor(cmd, dev, a, dtype=vk.UINT32):
    a = np.ascontiguousarray(a)
    shape = (1,) * (3 - a.ndim) + a.shape
    t = vk.Tensor(*shape, dev, dtype)
    if a.size:
        cmd.upload(a, t)
    return t


class Cache:
    """Keys and values of n sequences in pages; what no sequence holds, and what lies behind a sequence's last token, is NaN."""

    def __init__(self, rng, lengths, kv, dim, page, dtype, spare=3, std=1.0):
        self.page, self.kv, self.dim, self.dtype, self.lengths = page, kv, dim, dtype, list(lengths)
        need = [-(-l // page) for l in lengths]
        order = rng.permutation(sum(need) + spare).astype(np.uint32)
        self.pages = len(order)
        self.table = np.full((len(lengths), max(need + [1]) + 1), 0xdeadbeef, np.uint32)  # entries behind a sequence are not read
        nan = 0x7e00 if dtype == vk.FP16 else 0x7fc0
        self.k, self.v = (np.full((self.pages, kv, page, dim), nan, np.uint16) for _ in range(2))
        self.seq_k, self.seq_v = [], []
        at = 0
        for i, l in enumerate(lengths):
            self.table[i, :need[i]] = order[at:at + need[i]]
            at += need[i]
            for c, s in ((self.k, self.seq_k), (self.v, self.seq_v)):
                x = draw(rng, (kv, l, dim), dtype, std)
                s.append(x)
                self.put(c, i, x)

    def put(self, c, i, x):
        j = np.arange(x.shape[1])
        if len(j):
            c[self.table[i, j // self.page], :, j % self.page] = x.transpose(1, 0, 2)

    def up(self, cmd, dev):
        flat = (self.pages, self.kv * self.page, self.dim)
        return (tensor(cmd, dev, self.k.reshape(flat), self.dtype), tensor(cmd, dev, self.v.reshape(flat), self.dtype), tensor(cmd, dev, self.table),
                tensor(cmd, dev, np.array(self.lengths, np.uint32)))


def check(got, want, mass, size, dtype, dim, tokens, biggest, rounded_p, what=""):
    """One rounding of the output; scores: dim products and sums in fp32, each off by 2^-24 of what they add up to, twice that (and 2^-20
    for exp2 and the sums) relative on a probability, numerator and denominator; probabilities as 16-bit numbers where
    rounded_p, else as two of them (2^-16 of each for bfloat16, the least half's half step)."""
    assert (np.isnan(got) == np.isnan(want)).all(), what
    prob = 4 * (dim + 4) * 2.0 ** -24 * size + 2.0 ** -19
    prob = prob + (HALF_STEP[dtype] if rounded_p else 2.0 ** -16)
    tol = HALF_STEP[dtype] * np.abs(want) * (1 + 2.0 ** -6) + prob * mass + tokens * TINY[vk.FP16] * biggest * (dtype == vk.FP16) + TINY[dtype]
    off = np.abs(got - want)
    off = np.where(np.isnan(want), 0.0, off)
    worst = np.unravel_index(np.argmax(off / np.where(np.isnan(tol), 1, tol)), off.shape)
    assert off[worst] <= tol[worst], "%s: %r: %g instead of %g, tolerance %g" % (what, worst, got[worst], want[worst], tol[worst])


def attend(cache, i, q, pos, window=0, scale=None):
    """oracle attention of sequence i, with the cache's values."""
    k, v = (to_values(s[i], cache.dtype) for s in (cache.seq_k, cache.seq_v))
    return P.attention(q, pos, k, v, window, scale)
