"""Attention over a paged cache where one position outweighs thousands of others that make up the output, and where a lost tile would show."""
import numpy as np
import pytest

import vkllama_b200 as vk
from paged_weights import LONG_STEPS, Cache, Sink, draw, near, tensor, to_bits, to_values, tolerance

pytestmark = pytest.mark.gpu
GAPS = [14.0, 17.0, 18.0, 20.0]


def attention(dev, c, q, heads, scale=0.0, window=0, starts=None):
    """Rows q, by one call."""
    cmd = vk.Command(dev)
    with cmd:
        k, v, table, lens = c.up(cmd, dev)
        op = vk.PagedAttention(dev, cmd, heads, c.kv, c.dim, c.page, scale, window, c.dtype).init()
        args = () if starts is None else (tensor(cmd, dev, np.array(starts, np.uint32)),)
        got = cmd.download(op(tensor(cmd, dev, q, c.dtype), k, v, table, lens, *args))
    return to_values(got, c.dtype).reshape(-1, heads, c.dim)


@pytest.mark.parametrize("gap", GAPS)
@pytest.mark.parametrize("lengths,heads,kv,dim,at,value", [
    ([4000], 2, 1, 64, 0, 0.0), ([4000], 16, 1, 128, 3999, 0.0), ([300, 20, 150], 8, 1, 128, 0, 0.05), ([2000, 1], 24, 1, 256, 1000, 0.0), ([700] * 150, 4, 4, 64, 5, 0.0),
    ([3000, 900], 8, 8, 192, 0, 0.0)])
def test_one_token_that_a_position_outweighs(dev, gap, lengths, heads, kv, dim, at, value):
    """Pairs that a warp has whole, and parts that warps and CTAs join."""
    for spread in (0.0, 0.5):
        c = Sink(np.random.default_rng(len(lengths) + dim), lengths, kv, dim, 16, vk.FP16, gap, value, at, spread)
        q = c.queries(len(lengths), heads, dim, vk.FP16)
        got, q = attention(dev, c, q, heads, 1.0), to_values(q, vk.FP16).reshape(-1, heads, dim)
        for i in sorted({0, len(lengths) // 2, len(lengths) - 1}):
            near(got[i:i + 1], c, i, q[i:i + 1], [lengths[i] - 1], "token", scale=1.0, what="sequence %d" % i)


def rows(dev, c, past, new, heads, kernel, scale=1.0, window=0, q=None):
    starts = np.concatenate([[0], np.cumsum(new)])
    bits = c.queries(starts[-1], heads, c.dim, c.dtype) if q is None else q
    got = attention(dev, c, bits, heads, scale, window, starts)
    q = to_values(bits, c.dtype).reshape(-1, heads, c.dim)
    for i in sorted({0, len(new) // 2, len(new) - 1}):
        mine = sorted({int(starts[i]), int(starts[i]) + new[i] // 2, int(starts[i + 1]) - 1})
        near(got[mine], c, i, q[mine], [past[i] + r - int(starts[i]) for r in mine], kernel, window, scale or None, "sequence %d" % i)


@pytest.mark.parametrize("gap", GAPS)
@pytest.mark.parametrize("past,new,heads,kv,dim,page", [
    ([4000], [3], 4, 1, 200, 16), ([100, 50, 0], [9, 20, 60], 1, 1, 64, 16), ([60] * 40, [6] * 40, 4, 2, 128, 24), ([0, 1000], [300, 2], 2, 2, 136, 5)])
def test_rows_that_a_position_outweighs(dev, gap, past, new, heads, kv, dim, page):
    for at in (0, 20):
        c = Sink(np.random.default_rng(dim), [a + b for a, b in zip(past, new)], kv, dim, page, vk.FP16, gap, 0.0, at)
        rows(dev, c, past, new, heads, "rows")


@pytest.mark.parametrize("gap", GAPS)
@pytest.mark.parametrize("past,new,heads,kv,dim,page", [
    ([4000], [3], 4, 1, 128, 16), ([200], [600], 1, 1, 64, 16), ([700] * 20, [40] * 20, 8, 8, 64, 16), ([1000, 0], [130, 140], 6, 2, 96, 5)])
def test_rows_on_the_tensor_cores_that_a_position_outweighs(dev, gap, past, new, heads, kv, dim, page):
    """Positions in slices and whole, the position that outweighs the others in the first tile and in a later one."""
    for at in (0, 130):
        c = Sink(np.random.default_rng(dim), [a + b for a, b in zip(past, new)], kv, dim, page, vk.FP16, gap, 0.0, at)
        rows(dev, c, past, new, heads, "tensor")


@pytest.mark.parametrize("dtype", [vk.FP16, vk.BF16])
def test_long_sequences_lack_no_tile(dev, dtype):
    """The sequences of test_paged_weights_cpu.py, whose bounds sixteen positions do not fit into."""
    for n, dim in ((300, 128), (4000, 64), (70001, 64)):
        c = Cache(np.random.default_rng(n + dim), [n], 1, dim, 16, dtype)
        q = draw(np.random.default_rng(1), (1, 2 * dim), dtype)
        near(attention(dev, c, q, 2), c, 0, to_values(q, dtype).reshape(1, 2, dim), [n - 1], "token", steps=LONG_STEPS if n > 4000 else None)
    for past, new, heads, dim, kernel in ((2999, 1, 3, 128, "tensor"), (2700, 300, 2, 128, "tensor"), (898, 2, 2, 200, "rows")):
        c = Cache(np.random.default_rng(dim), [past + new], 1, dim, 16, dtype)
        rows(dev, c, [past], [new], heads, kernel, 0.0, q=draw(np.random.default_rng(2), (new, heads * dim), dtype))


@pytest.mark.parametrize("dtype", [vk.FP16, vk.BF16])
@pytest.mark.parametrize("tokens,kv,dim,kernel,window", [(1 << 20, 160, 64, "tensor", 0), (1 << 21, 8, 64, "tensor", 0), (150000, 150, 128, "tensor", 0), (400000, 150, 80, "tensor", 300000), (1 << 20, 20, 136, "rows", 0)])
def test_sums_over_many_positions(dev, dtype, tokens, kv, dim, kernel, window):
    """Values of one sign, weights that grow along the way: what the matrix units cut off their sums adds up. Two pages, again and again; positions of a CTA
    of its own, and in slices of many tiles."""
    page, rows = 128, 3
    rng, cmd = np.random.default_rng(dim), vk.Command(dev)
    k, v = 0.3 * rng.standard_normal((2, kv, page, dim)), 1 + rng.random((2, kv, page, dim))
    k[1, :, :, 0] += 4  # the second page's scores are higher
    k, v = to_bits(k, dtype), to_bits(v, dtype)
    q = 0.3 * rng.standard_normal((rows, kv, dim))
    q[:, :, 0] = np.sqrt(dim)
    q = to_bits(q, dtype)
    width = -(-tokens // page)
    table = np.repeat(np.array([0, 1], np.uint32), [width // 3, width - width // 3])
    with cmd:
        op = vk.PagedAttention(dev, cmd, kv, kv, dim, page, 0.0, window, dtype).init()
        args = [tensor(cmd, dev, a.reshape(2, kv * page, dim), dtype) for a in (k, v)]
        args += [tensor(cmd, dev, a.astype(np.uint32)) for a in (table[None], np.array([tokens]), np.array([0, rows]))]
        got = to_values(cmd.download(op(tensor(cmd, dev, q.reshape(rows, -1), dtype), *args)), dtype).reshape(rows, kv, dim)
    k, v, q = (to_values(a, dtype) for a in (k, v, q))
    for r in range(rows):
        last = tokens - rows + r
        j = np.arange(max(0, last + 1 - window) if window else 0, last + 1)
        times = np.bincount(table[j // page].astype(int) * page + j % page, minlength=2 * page).reshape(2, 1, page)
        s = np.einsum("pkjd,kd->pkj", k, q[r]) / np.sqrt(dim)
        w = times * np.exp(s - s.max((0, 2), keepdims=True))
        mass = np.einsum("pkj,pkjd->kd", w, v) / w.sum((0, 2))[:, None]  # all values are positive: also the output
        size = (np.einsum("pkjd,kd->pkj", np.abs(k), np.abs(q[r])) / np.sqrt(dim)).max((0, 2))[:, None]
        den = w.sum((0, 2))[:, None]
        tol = tolerance(mass, mass, size, den, dtype, dim, tokens, 2.0, kernel, steps=2048 + tokens / 32768)
        assert (np.abs(got[r] - mass) <= tol).all(), (r, np.abs((got[r] - mass) / tol).max(), ((got[r] - mass) / mass).mean())


@pytest.mark.parametrize("dtype", [vk.FP16, vk.BF16])
@pytest.mark.parametrize("dim,kv", [(64, 150), (128, 4), (136, 4)])
def test_infinite_and_missing_numbers_behind_many_positions(dev, dtype, dim, kv):
    """Before sums are put aside and behind; by rows that see them and by ones that do not."""
    page, width, rows = 128, 1200, 2  # a page of ordinary values again and again, one with an infinity, a last one that ends with NaN
    rng, cmd = np.random.default_rng(27), vk.Command(dev)
    k, v = (draw(rng, (3, kv, page, dim), dtype) for _ in range(2))
    inf, nan = (0x7c00, 0x7e00) if dtype == vk.FP16 else (0x7f80, 0x7fc0)
    v[1, :, 5, 3], v[2, :, page - 1, 7] = inf, nan
    table = np.zeros((1, width), np.uint32)
    table[0, 1], table[0, -1] = 1, 2
    q = draw(rng, (rows, kv * dim), dtype)
    with cmd:
        args = [tensor(cmd, dev, a.reshape(3, kv * page, dim), dtype) for a in (k, v)]
        args += [tensor(cmd, dev, np.array(a, np.uint32)) for a in (table, [width * page], [0, rows])]
        got = cmd.download(vk.PagedAttention(dev, cmd, kv, kv, dim, page, dtype=dtype).init()(tensor(cmd, dev, q, dtype), *args))
    got = to_values(got, dtype).reshape(rows, kv, dim)
    assert np.isposinf(got[:, :, 3]).all() and np.isfinite(got[0, :, 7]).all() and np.isnan(got[1, :, 7]).all()
    assert np.isfinite(np.delete(got, [3, 7], 2)).all() and np.abs(np.delete(got, [3, 7], 2)).max() < 5
