"""Operators of a paged key-value cache against their definitions in 64 bits (oracle/paged.py)."""
import ctypes as C

import numpy as np
import pytest

import vkllama_b200 as vk
from oracle import paged as P
from paged_util import HALF_STEP, TINY, Cache, attend, check, draw, tensor, to_bits, to_values

pytestmark = pytest.mark.gpu
DTYPES = [vk.FP16, vk.BF16]


def code_of(call):
    with pytest.raises(vk.VklError) as e:
        call()
    return e.value.code


# ---- tables ------------------------------------------------------------------------------------------------------------
class Server:
    """Sequences on the device beside the oracle's."""

    def __init__(self, dev, n, width, page, pages, seed=0):
        self.dev, self.page, self.cmd = dev, page, vk.Command(dev)
        rng = np.random.default_rng(seed)
        self.pool, self.lengths, self.table = [int(x) for x in rng.permutation(pages)], np.zeros(n, np.uint32), np.zeros((n, width), np.uint32)
        with self.cmd:
            self.t = [tensor(self.cmd, dev, a) for a in (self.lengths, self.table, np.array([pages] + self.pool, np.uint32))]
            self.op = vk.PagedTables(dev, self.cmd, page).init()

    def step(self, target, rows):
        """Returns what the wait raised, the map and the starts."""
        cmd, failed = self.cmd, None
        cmd.begin()
        want = tensor(cmd, self.dev, np.array(target, np.uint32))
        m, s = self.op(self.t[0], want, self.t[1], self.t[2], rows)
        got = [cmd.download(x) for x in ((m, s) if rows else (s, s))] + [cmd.download(x) for x in self.t]
        cmd.end()
        try:
            cmd.submit_and_wait()
        except vk.VklError as e:
            failed = e.code
        should = P.resize(self.page, self.lengths, target, self.table, self.pool, rows)
        if should is None:
            assert failed is not None
            self.agrees(got)
            assert (got[1] == 0).all() and (not rows or (got[0][0, 0] == P.NO_SLOT).all() and (got[0][0, 1] == 0).all())
            return failed
        assert failed is None
        self.lengths, self.table, self.pool, m, s = should
        self.agrees(got)
        assert (got[1].ravel() == s).all() and (not rows or (got[0][0] == m).all())

    def agrees(self, got):
        assert (got[2].ravel() == self.lengths).all() and (got[3][0] == self.table).all()
        assert got[4].ravel()[0] == len(self.pool) and (got[4].ravel()[1:len(self.pool) + 1] == self.pool).all()


@pytest.mark.parametrize("n,page,most", [(1, 16, 100), (1, 1, 9), (5, 24, 700), (33, 16, 300), (513, 4, 40), (1500, 8, 60), (300, 16, 1000)])
def test_tables_follow_the_oracle_as_sequences_come_and_go(dev, n, page, most):
    rng = np.random.default_rng(n)
    width = -(-most // page)
    s = Server(dev, n, width, page, n * width, n)
    s.step(rng.integers(0, most + 1, n), n * most)
    for turn in range(6):
        kind = rng.integers(0, 4, n)
        target = np.where(kind == 0, 0, np.where(kind == 1, s.lengths, np.where(kind == 2, np.minimum(s.lengths + 1, most), rng.integers(0, most + 1, n))))
        s.step(target, int(np.maximum(0, target.astype(int) - s.lengths).sum()) + turn % 2 * 7)
    s.step(np.minimum(s.lengths + 1, most), n)  # a step of every sequence
    s.step(np.zeros(n, int), 0)
    assert len(s.pool) == n * width


def test_a_batch_of_the_most_sequences(dev):
    s = Server(dev, 8192, 2, 16, 9000, 1)
    rng = np.random.default_rng(1)
    s.step(np.where(np.arange(8192) % 11 == 0, 17, rng.integers(0, 17, 8192)), 120000)
    s.step(s.lengths // 2, 0)
    cmd = vk.Command(dev)
    with cmd:
        op = vk.PagedTables(dev, cmd, 16).init()
        t = [tensor(cmd, dev, np.zeros(x, np.uint32)) for x in (8193, 8193, (8193, 2), 5)]
        assert code_of(lambda: op(t[0], t[1], t[2], t[3], 1)) == 11


def test_taking_and_giving_back_leaves_the_pool_as_it_was(dev):
    s = Server(dev, 40, 20, 16, 500, 2)
    rng = np.random.default_rng(2)
    s.step(rng.integers(1, 200, 40), 8000)
    before, lengths = list(s.pool), s.lengths.copy()
    s.step(s.lengths + rng.integers(0, 50, 40).astype(np.uint32), 2500)
    s.step(lengths, 0)
    assert s.pool == before


def test_calls_that_cannot_be_carried_out_change_nothing(dev):
    s = Server(dev, 3, 4, 16, 8, 3)
    s.step([20, 0, 33], 60)               # 5 pages of 8
    assert s.step([20, 64, 33], 64) == 8  # 4 more
    assert s.step([20, 65, 0], 65) == 11  # 5 in a row of 4
    assert s.step([21, 5, 33], 5) == 11   # 6 new tokens
    s.step([0, 64, 33], 64)               # the pages that the first gives back are taken by the second
    assert s.step([1, 64, 64], 32) == 8
    # a pool that claims more pages than it has room for
    with s.cmd:
        s.cmd.upload(np.array([9] + [0] * 8, np.uint32), s.t[2])
    s.cmd.begin()
    s.op(s.t[0], s.t[0], s.t[1], s.t[2], 0)
    s.cmd.end()
    assert code_of(s.cmd.submit_and_wait) == 9


def test_a_length_beyond_every_table_is_refused_on_the_device(dev):
    s = Server(dev, 2, 4, 16, 8, 4)
    for bad in (0x80000000, 0xffffffff, 65):
        assert s.step([bad, 1], 100) == 11


# ---- update ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,heads,kv,dim,page,theta,wide", [(1, 4, 4, 128, 16, 1e4, 0), (37, 8, 2, 64, 24, 5e5, 0), (5, 3, 3, 80, 1, 1e4, 16), (2, 40, 8, 256, 32, 1e4, 8),
                                                              (9, 0, 5, 8, 7, 1e4, 0), (64, 6, 1, 72, 16, 0.0, 24), (3, 160, 40, 128, 16, 1e4, 0)])
def test_rows_go_to_their_slots(dev, dtype, rows, heads, kv, dim, page, theta, wide):
    rng = np.random.default_rng(rows * dim)
    pages = rows // page + 3
    slots = rng.permutation(pages * page)[:rows].astype(np.uint32)
    pos = rng.integers(0, 3_000_000, rows).astype(np.uint32)
    pos[0] = 0
    if rows > 4:
        slots[rng.integers(0, rows, 2)] = P.NO_SLOT
    cmd = vk.Command(dev)
    old = [draw(rng, (pages, kv * page, dim), dtype) for _ in range(2)]
    x = [draw(rng, (rows, h * dim + wide), dtype) for h in (heads, kv, kv)]
    with cmd:
        caches = [tensor(cmd, dev, a, dtype) for a in old]
        q, k, v = ((tensor(cmd, dev, a, dtype).view(1, rows, a.shape[1] - wide) if a.shape[1] > wide else None) for a in x)
        m = tensor(cmd, dev, np.stack([slots, pos]))
        op = vk.UpdatePagedKVCache(dev, cmd, dim, page, theta, dtype).init()
        got_q = op(caches[0], caches[1], k, v, m, q)
        got = [cmd.download(c) for c in caches] + ([cmd.download(got_q)] if heads else [])
    q, k, v = (to_values(a[:, :a.shape[1] - wide], dtype).reshape(rows, -1, dim) for a in x)
    turn = (lambda a: P.rotate(a, pos, float(np.float32(theta)))) if theta else (lambda a: a)

    def near(got, want, x):
        # one rounding; the angle is off by 2^-25 of a turn times 2 pi and sine and cosine by 2^-23, products and sum by 2^-24 each
        big = np.abs(x).reshape(x.shape[:-1] + (dim // 2, 2)).sum(-1).repeat(2, -1)
        tol = HALF_STEP[dtype] * np.abs(want) * 1.001 + TINY[dtype] + 2.0 ** -20 * big * bool(theta)
        assert (np.abs(got - want) <= tol).all()

    if heads:
        near(to_values(got[2], dtype).reshape(rows, heads, dim), turn(q), q)
    for c, new, was in ((got[0], turn(k), old[0]), (got[1], v, old[1])):
        c, kept = c.reshape(pages, kv, page, dim), was.reshape(pages, kv, page, dim).copy()
        for r in range(rows):
            if slots[r] != P.NO_SLOT:
                at = c[slots[r] // page, :, slots[r] % page]
                near(to_values(at, dtype), new[r], (k if new is not v else v)[r])
                kept[slots[r] // page, :, slots[r] % page] = at
        assert (c == kept).all()  # nothing else was written
    if not theta:
        assert all((got[1].reshape(pages, kv, page, dim)[s // page, :, s % page] == x[2][r, :kv * dim].reshape(kv, dim)).all() for r, s in enumerate(slots) if s != P.NO_SLOT)


def test_slots_beyond_the_cache_are_reported_and_not_written(dev):
    cmd, rng = vk.Command(dev), np.random.default_rng(5)
    old = draw(rng, (4, 2 * 16, 64), vk.FP16)
    x = draw(rng, (3, 128), vk.FP16)
    cmd.begin()
    kc, vc, k = tensor(cmd, dev, old, vk.FP16), tensor(cmd, dev, old, vk.FP16), tensor(cmd, dev, x, vk.FP16)
    op = vk.UpdatePagedKVCache(dev, cmd, 64, 16, 0.0).init()
    op(kc, vc, k, k, tensor(cmd, dev, np.array([[64, 5, 0xfffffff0], [0, 1, 2]], np.uint32)))
    got = cmd.download(kc).reshape(4, 2, 16, 64)
    cmd.end()
    assert code_of(cmd.submit_and_wait) == 11
    want = old.reshape(4, 2, 16, 64).copy()
    want[0, :, 5] = x[1].reshape(2, 64)
    assert (got == want).all()


# ---- attention of one token --------------------------------------------------------------------------------------------
def token(dev, lengths, heads, kv, dim, page, dtype, window=0, scale=None, wide=0, std=1.0, seed=0, cache=None):
    rng = np.random.default_rng(seed + dim + len(lengths))
    cache = cache or Cache(rng, lengths, kv, dim, page, dtype, std=std)
    n, cmd = len(lengths), vk.Command(dev)
    bits = draw(rng, (n, heads * dim + wide), dtype, std)
    with cmd:
        k, v, table, lens = cache.up(cmd, dev)
        q = tensor(cmd, dev, bits, dtype).view(1, n, heads * dim)
        op = vk.PagedAttention(dev, cmd, heads, kv, dim, page, scale or 0.0, window, dtype).init()
        first = cmd.download(op(q, k, v, table, lens))
        again = cmd.download(op(q, k, v, table, lens))
    assert (first == again).all()  # the same bits, whichever CTA joins the parts
    got = to_values(first, dtype).reshape(n, heads, dim)
    q = to_values(bits[:, :heads * dim], dtype).reshape(n, heads, dim)
    for i, l in enumerate(lengths):
        want, mass, size = attend(cache, i, q[i:i + 1], [l - 1], window, scale)
        big = np.abs(to_values(cache.seq_v[i], dtype)).max(initial=0)
        check(got[i:i + 1], want, mass, size, dtype, dim, l, big, False, "sequence %d of %d" % (i, l))
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,heads,kv,dim,page,window", [
    ([1], 1, 1, 8, 1, 0), ([300], 32, 32, 128, 16, 0), ([17, 0, 1, 16, 15, 33, 0], 4, 4, 128, 16, 0), ([5000], 8, 1, 128, 64, 0), ([0, 0], 4, 2, 64, 16, 0),
    ([1200, 3, 801, 640], 12, 4, 64, 8, 0), ([257, 1, 900], 40, 5, 80, 24, 100), ([100, 2000, 31], 12, 1, 128, 16, 0), ([1500, 700], 16, 1, 72, 32, 33),
    ([900, 20], 24, 1, 256, 16, 0), ([63, 64, 65, 1000], 6, 2, 192, 5, 0), ([2500], 40, 1, 128, 16, 1000), ([40, 41, 42], 48, 2, 96, 16, 7),
    ([3000, 40, 0, 900], 16, 1, 256, 16, 0), ([700, 20], 11, 1, 136, 24, 100), ([4000], 48, 3, 64, 16, 0)])
def test_one_token_per_sequence(dev, dtype, lengths, heads, kv, dim, page, window):
    token(dev, lengths, heads, kv, dim, page, dtype, window, wide=16 if len(lengths) > 2 else 0)


@pytest.mark.parametrize("n,most,heads,kv,dim", [(700, 40, 4, 4, 64), (90, 500, 8, 8, 128), (300, 3, 4, 1, 128), (40, 300, 20, 2, 128), (40, 300, 5, 5, 200), (5, 9000, 2, 2, 128)])
def test_batches_of_many_lengths(dev, n, most, heads, kv, dim):
    """Shares cut sequences anywhere, warps and CTAs join parts."""
    lengths = [int(x) for x in np.random.default_rng(n).integers(0, most, n)]
    token(dev, lengths, heads, kv, dim, 16, vk.BF16 if n % 3 else vk.FP16)


def test_one_long_sequence(dev):
    token(dev, [70001], 2, 1, 64, 32, vk.FP16)
    token(dev, [33000], 4, 1, 128, 16, vk.BF16, scale=0.3)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_far_apart(dev, dtype):
    """Running maxima that jump, probabilities that vanish."""
    token(dev, [777, 50], 8, 2, 128, 16, dtype, std=4.0)
    token(dev, [777], 4, 4, 128, 16, dtype, scale=-1.0)


@pytest.mark.parametrize("heads,dim,long", [(4, 64, 0), (12, 64, 0), (4, 128, 5000), (16, 200, 0), (20, 128, 3000)])
def test_infinite_and_missing_numbers_where_a_token_sees_them(dev, heads, dim, long):
    """Also where the weight is far below 16 bits, in whole pairs, in parts that warps and CTAs join."""
    rng = np.random.default_rng(6)
    n = 100 + long
    c = Cache(rng, [n, n, n, n], 1, dim, 16, vk.FP16)
    q = draw(rng, (4, heads * dim), vk.FP16, 0.1)
    q[3] = to_bits(np.ones(heads * dim), vk.FP16)
    c.seq_v[0][0, 40, 3] = c.seq_v[3][0, 50, 7] = 0x7c00
    c.seq_v[1][0, 99, 5] = 0x7e00
    c.seq_k[3][0, 50] = to_bits(np.full(dim, -40 / np.sqrt(dim)), vk.FP16)  # a score of -40
    for i in (0, 1, 3):
        c.put(c.v, i, c.seq_v[i])
        c.put(c.k, i, c.seq_k[i])
    cmd = vk.Command(dev)
    with cmd:
        k, v, table, lens = c.up(cmd, dev)
        out = vk.PagedAttention(dev, cmd, heads, 1, dim, 16).init()(tensor(cmd, dev, q, vk.FP16), k, v, table, lens)
        got = to_values(cmd.download(out), vk.FP16).reshape(4, heads, dim)
    for i, d, ok in ((0, 3, np.isposinf), (1, 5, np.isnan), (3, 7, np.isposinf)):
        assert ok(got[i, :, d]).all() and np.isfinite(np.delete(got[i], d, 1)).all(), i
    assert np.isfinite(got[2]).all()


# ---- attention of several rows -----------------------------------------------------------------------------------------
def prompt(dev, past, new, heads, kv, dim, page, dtype, window=0, wide=0, behind=0, std=1.0, cache=None, finite=True, scale=None):
    rng = np.random.default_rng(sum(new) + dim)
    lengths = [a + b for a, b in zip(past, new)]
    cache = cache or Cache(rng, lengths, kv, dim, page, dtype, std=std)
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.uint32)
    rows, cmd = int(starts[-1]) + behind, vk.Command(dev)
    bits = draw(rng, (rows, heads * dim + wide), dtype, std)
    mark = np.full((1, rows, heads * dim), 0x1234, np.uint16)
    with cmd:
        k, v, table, lens = cache.up(cmd, dev)
        q = tensor(cmd, dev, bits, dtype).view(1, rows, heads * dim)
        op, starts_t = vk.PagedAttention(dev, cmd, heads, kv, dim, page, scale or 0.0, window, dtype).init(), tensor(cmd, dev, starts)
        out = op(q, k, v, table, lens, starts_t)
        cmd.upload(mark, out)
        first = cmd.download(op(q, k, v, table, lens, starts_t))
    assert (first[0, starts[-1]:] == 0x1234).all()  # rows behind the last sequence
    got, q = (to_values(a, dtype).reshape(rows, heads, dim) for a in (first, bits[:, :heads * dim]))
    for i, l in enumerate(lengths):
        mine = slice(starts[i], starts[i + 1])
        want, mass, size = attend(cache, i, q[mine], list(range(past[i], l)), window, scale)
        if new[i] and finite:
            big = np.abs(to_values(cache.seq_v[i], dtype)).max(initial=0)
            check(got[mine], want, mass, size, dtype, dim, l, big, True, "sequence %d, %d behind %d" % (i, new[i], past[i]))
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("past,new,heads,kv,dim,page,window", [
    ([0], [1], 1, 1, 8, 1, 0), ([0], [130], 4, 4, 128, 16, 0), ([0, 5, 0], [63, 0, 65], 2, 2, 64, 16, 0), ([300, 0, 17, 1000], [1, 1, 7, 64], 8, 2, 128, 16, 0),
    ([100], [200], 3, 1, 80, 24, 50), ([0, 40], [70, 30], 5, 1, 256, 8, 0), ([513], [129], 12, 1, 128, 32, 0), ([0, 0], [33, 200], 4, 2, 192, 16, 16),
    ([700], [260], 2, 2, 72, 7, 129), ([5], [300], 16, 1, 128, 128, 0)])
def test_several_rows_per_sequence(dev, dtype, past, new, heads, kv, dim, page, window):
    prompt(dev, past, new, heads, kv, dim, page, dtype, window, wide=8 if len(new) > 1 else 0, behind=len(new) % 3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("past,new,heads,kv,dim,page,window,scale", [
    ([0], [257], 1, 1, 128, 8, 0, -0.05), ([129, 0], [128, 300], 2, 2, 64, 5, 0, 0.3), ([1000], [140], 2, 1, 96, 64, 300, None), ([50, 60, 70], [200, 1, 129], 4, 4, 40, 32, 1, None),
    ([383], [385], 1, 1, 16, 16, 0, None), ([0, 100], [120, 140], 6, 2, 120, 48, 90, 0.02)])
def test_whole_tiles_of_rows(dev, dtype, past, new, heads, kv, dim, page, window, scale):
    """Tiles of 128 rows and positions: borders on and beside them, pages that boxes of rows divide and ones that they do not, windows smaller
    than a tile, turned scores."""
    prompt(dev, past, new, heads, kv, dim, page, dtype, window, scale=scale, behind=1)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_call_with_sequences_for_either_kernel(dev, dtype):
    """A few rows behind many positions and behind few, prompts short and long: two launches share the sequences, and a third joins the parts of the
    one whose positions are split."""
    before = vk.kernel_launches()
    prompt(dev, [2000, 0, 600, 0, 510, 511, 0, 30], [3, 40, 1, 130, 1, 1, 0, 66], 2, 2, 64, 16, dtype, behind=2)
    assert vk.kernel_launches() - before == 6
    prompt(dev, [700, 3, 900], [2, 2, 7], 12, 2, 128, 8, dtype, window=600)
    prompt(dev, [700, 3, 900], [2, 2, 7], 4, 2, 200, 8, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("past,new,heads,kv,dim,page,window", [
    ([5000], [5], 8, 2, 128, 16, 0), ([3000, 10, 700, 0], [3, 20, 1, 0], 4, 1, 64, 32, 0), ([2500], [200], 4, 2, 128, 16, 0), ([4000], [130], 2, 2, 80, 24, 1500),
    ([2000], [300], 1, 1, 96, 5, 0), ([1100, 1100], [64, 2], 6, 2, 40, 64, 600), ([20000], [1], 5, 1, 128, 16, 0), ([1023], [1], 128, 1, 64, 128, 0), ([1022, 1024], [257, 255], 1, 1, 16, 8, 0)])
def test_positions_are_split_where_there_are_few_rows(dev, dtype, past, new, heads, kv, dim, page, window):
    """Slices of four tiles and more, sequences with one slice beside ones with many, windows that begin inside one."""
    prompt(dev, past, new, heads, kv, dim, page, dtype, window, behind=3, wide=8)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,dim,page,window,least", [(8, 128, 16, 0, 0), (2, 64, 24, 0, 0), (6, 96, 5, 300, 0), (8, 40, 128, 129, 200)])
def test_drafts_of_many_sequences(dev, dtype, heads, dim, page, window, least):
    """A few rows behind none, one and more tiles of positions, more sequences than SMs."""
    rng = np.random.default_rng(14)
    past = [0, 127, 128, 255, 256, 383, 384, 1000] + [int(x) for x in rng.integers(least, 1200, 72)]
    prompt(dev, [max(x, least) for x in past], [int(x) for x in rng.integers(0 if least else 1, 8, 80)], heads, 2, dim, page, dtype, window, behind=1)


@pytest.mark.parametrize("dim", [64, 128])
def test_infinite_and_missing_numbers_in_a_slice(dev, dim):
    for dtype in DTYPES:
        inf, nan = (0x7c00, 0x7e00) if dtype == vk.FP16 else (0x7f80, 0x7fc0)
        for window in (0, 1000):
            c = Cache(np.random.default_rng(12), [4000, 60], 1, dim, 16, dtype)
            c.seq_v[0][0, 700, 3], c.seq_v[0][0, 3500, 5], c.seq_v[0][0, 3998, 7], c.seq_k[1][0, 59] = nan, inf, nan, inf
            for i in (0, 1):
                c.put(c.v, i, c.seq_v[i])
                c.put(c.k, i, c.seq_k[i])
            got = prompt(dev, [3996, 56], [4, 4], 3, 1, dim, 16, dtype, window, cache=c, finite=False)
            for r in range(4):  # positions 3996 ...
                assert np.isnan(got[r, :, 3]).all() == (not window) and np.isposinf(got[r, :, 5]).all() and np.isnan(got[r, :, 7]).all() == (r >= 2)
                assert np.isfinite(np.delete(got[r], [3, 5, 7], 1)).all()
            assert np.isfinite(got[4:7]).all() and not np.isfinite(got[7]).any()
            n = 80  # and in many sequences
            c = Cache(np.random.default_rng(13), [500] * n, 2, dim, 16, dtype)
            for i in range(1, n, 2):
                c.seq_v[i][:, 100, 3], c.seq_v[i][:, 200, dim - 1] = nan, inf
                c.put(c.v, i, c.seq_v[i])
            got = prompt(dev, [496] * n, [4] * n, 4, 2, dim, 16, dtype, cache=c, finite=False).reshape(n, 4, 4, dim)
            assert np.isfinite(got[::2]).all() and np.isnan(got[1::2, :, :, 3]).all() and np.isposinf(got[1::2, :, :, dim - 1]).all()
            assert np.isfinite(np.delete(got[1::2], [3, dim - 1], 3)).all()


def test_many_short_prompts_and_a_long_one(dev):
    rng = np.random.default_rng(8)
    new = [int(x) for x in rng.integers(0, 40, 150)] + [700]
    prompt(dev, [int(x) for x in rng.integers(0, 60, 151)], new, 4, 2, 64, 16, vk.FP16, behind=5)
    prompt(dev, [0], [900], 8, 4, 128, 16, vk.BF16, std=3.0)


@pytest.mark.parametrize("dim", [64, 128, 200])
def test_numbers_that_a_row_does_not_see_do_not_reach_it(dev, dim):
    """Infinities and NaN in later positions of the same tile, and before the window."""
    for dtype in DTYPES:
        for window in (0, 20):
            rng = np.random.default_rng(9)
            c = Cache(rng, [150], 1, dim, 16, dtype)
            c.seq_v[0][0, 70], c.seq_v[0][0, 120, ::3] = (0x7e00, 0x7c00) if dtype == vk.FP16 else (0x7fc0, 0x7f80)
            c.seq_k[0][0, 130] = 0x7c00 if dtype == vk.FP16 else 0x7f80
            c.put(c.v, 0, c.seq_v[0])
            c.put(c.k, 0, c.seq_k[0])
            got = prompt(dev, [0], [150], 2, 1, dim, 16, dtype, window, cache=c, finite=False)
            seen = lambda j, r: r >= j and (not window or j > r - window)  # noqa: E731
            for r in range(150):
                assert np.isnan(got[r]).all() == (seen(70, r) or seen(130, r)), r
                if not seen(70, r) and not seen(130, r):
                    assert np.isposinf(got[r, :, ::3]).all() == seen(120, r) and np.isfinite(np.delete(got[r], np.arange(0, dim, 3), 1)).all()
            # and rows that see none of them are right
            assert np.abs(got[60, 0]).max() < 10


def test_a_cta_goes_on_behind_rows_that_are_computed_again(dev):
    """More tiles than SMs; the other sequences' rows are the same bits as without infinities and NaN beside them."""
    n, new = 60, 130
    for bad in (0x7c00, 0x7e00):
        c = Cache(np.random.default_rng(13), [new] * n, 4, 64, 16, vk.FP16)
        clean = prompt(dev, [0] * n, [new] * n, 4, 4, 64, 16, vk.FP16, cache=c, finite=False)
        for i in range(1, n, 2):
            c.seq_v[i][:, 0, 5] = bad
            c.put(c.v, i, c.seq_v[i])
        got = prompt(dev, [0] * n, [new] * n, 4, 4, 64, 16, vk.FP16, cache=c, finite=False).reshape(n, new, 4, 64)
        clean = clean.reshape(n, new, 4, 64)
        assert np.array_equal(got[::2], clean[::2]) and np.isfinite(clean).all()
        assert not np.isfinite(got[1::2, :, :, 5]).any() and np.isfinite(np.delete(got[1::2], 5, 3)).all()


# ---- what is refused ---------------------------------------------------------------------------------------------------
def test_bad_pages_and_lengths_are_reported(dev):
    """The kernels check pages against the cache, lengths against the table, starts against both, and read nothing outside."""
    rng = np.random.default_rng(10)
    for bad in ("page", "length", "starts", "order"):
        for many in (False, True):
            if bad in ("starts", "order") and not many:
                continue
            c, cmd = Cache(rng, [40, 50], 2, 64, 16, vk.FP16), vk.Command(dev)
            if bad == "page":
                c.table[1, 2] = c.pages
            if bad == "length":
                c.lengths[0] = c.table.shape[1] * 16 + 1
            starts = {"starts": [0, 41, 60], "order": [0, 30, 20]}.get(bad, [0, 10, 20])
            cmd.begin()
            k, v, table, lens = c.up(cmd, dev)
            if bad == "length":
                table = tensor(cmd, dev, np.zeros_like(c.table))
            op = vk.PagedAttention(dev, cmd, 4, 2, 64, 16).init()
            op(tensor(cmd, dev, draw(rng, (60 if many else 2, 256), vk.FP16), vk.FP16), k, v, table, lens, tensor(cmd, dev, np.array(starts, np.uint32)) if many else None)
            cmd.end()
            assert code_of(cmd.submit_and_wait) == (3 if many and bad != "page" else 11), (bad, many)
            cmd.begin()  # and the next call is well
            cmd.end()
            cmd.submit_and_wait()


def test_refusals(dev):
    cmd = vk.Command(dev)
    cmd.begin()
    T = lambda c, h, w, d=vk.FP16: vk.Tensor(c, h, w, dev, d)  # noqa: E731
    U = lambda *s: T(*s, vk.UINT32)  # noqa: E731
    for page in (0, -1, (1 << 20) + 1):
        assert code_of(vk.PagedTables(dev, cmd, page).init) == 3
        assert code_of(vk.UpdatePagedKVCache(dev, cmd, 64, page).init) == 3
        assert code_of(vk.PagedAttention(dev, cmd, 4, 4, 64, page).init) == 3
    for dim in (0, 4, 12, 264, -8):
        assert code_of(vk.UpdatePagedKVCache(dev, cmd, dim, 16).init) == 3
        assert code_of(vk.PagedAttention(dev, cmd, 4, 4, dim, 16).init) == 3
    for theta in (-1.0, 0.5, float("nan"), float("inf")):
        assert code_of(vk.UpdatePagedKVCache(dev, cmd, 64, 16, theta).init) == 3
    for heads, kv in ((4, 3), (0, 1), (4, 0), (2, 4), (-4, 2)):
        assert code_of(vk.PagedAttention(dev, cmd, heads, kv, 64, 16).init) == 3
    for scale in (float("inf"), float("nan"), 1e-30, -1e30):
        assert code_of(vk.PagedAttention(dev, cmd, 4, 4, 64, 16, scale).init) == 3
    assert code_of(vk.PagedAttention(dev, cmd, 4, 4, 64, 16, 0.0, -1).init) == 3
    for dtype in (vk.FP32, vk.Q8_0, vk.INT8, vk.UINT32):
        assert code_of(vk.PagedAttention(dev, cmd, 4, 4, 64, 16, dtype=dtype).init) == 3
        assert code_of(vk.UpdatePagedKVCache(dev, cmd, 64, 16, dtype=dtype).init) == 3
    tables, update, att = vk.PagedTables(dev, cmd, 16), vk.UpdatePagedKVCache(dev, cmd, 64, 16), vk.PagedAttention(dev, cmd, 4, 2, 64, 16)
    n, cache = 3, T(5, 32, 64)
    # init() was not called
    assert code_of(lambda: tables(U(1, 1, n), U(1, 1, n), U(1, n, 4), U(1, 1, 6), 3)) == 9
    assert code_of(lambda: att(T(1, n, 256), cache, cache, U(1, n, 4), U(1, 1, n))) == 9
    for op in (tables, update, att):
        op.init()
        op.init()
    good = (U(1, 1, n), U(1, 1, n), U(1, n, 4), U(1, 1, 6))
    for i, other in ((0, U(1, 1, n + 1)), (1, U(1, n, 1)), (2, U(2, n, 4)), (3, U(1, 1, 0)), (0, T(1, 1, n)), (3, T(1, 1, 6, vk.FP32)), (1, None)):
        assert code_of(lambda: tables(*(other if j == i else a for j, a in enumerate(good)), 3)) == 3
    assert code_of(lambda: tables(*good[:2], U(1, n, 8).view(1, n, 4), good[3], 3)) == 12
    k, m, q = T(1, n, 128), U(1, 2, n), T(1, n, 256)
    good = (cache, T(5, 32, 64), k, T(1, n, 128), m, q)
    wrong = [(0, T(5, 16, 64)), (1, T(4, 32, 64)), (2, T(1, n, 100)), (2, T(1, n, 0)), (3, T(1, n + 1, 128)), (4, U(1, 3, n)), (4, U(1, 2, n + 1)), (5, T(1, n, 100)), (5, T(1, n + 1, 256)),
             (0, T(5, 32, 64, vk.BF16)), (2, T(1, n, 128, vk.BF16)), (4, T(1, 2, n)), (2, None), (0, None), (4, None)]
    for i, other in wrong:
        assert code_of(lambda: update(*(other if j == i else a for j, a in enumerate(good)))) == 3, i
    assert code_of(lambda: update(cache, cache, T(1, n, 132).view(1, n, 128), k, m)) == 12  # rows that start at 8 bytes
    good = (q, cache, T(5, 32, 64), U(1, n, 4), U(1, 1, n), U(1, 1, n + 1))
    wrong = [(0, T(1, n, 128)), (0, T(2, n, 256)), (1, T(5, 64, 64)), (2, T(5, 32, 72)), (3, U(2, n, 4)), (4, U(1, 1, n + 1)), (5, U(1, 1, n)), (0, T(1, n, 256, vk.BF16)), (3, T(1, n, 4)),
             (0, None), (2, None), (3, None), (4, None)]
    for i, other in wrong:
        assert code_of(lambda: att(*(other if j == i else a for j, a in enumerate(good)))) == 3, i
    assert code_of(lambda: att(T(1, n + 1, 256), *good[1:5])) == 3  # a query without a sequence
    assert code_of(lambda: att(T(1, n, 260).view(1, n, 256), *good[1:5])) == 12
    out = att(q, *good[1:5])
    assert code_of(lambda: att(out, *good[1:5])) == 3  # its own output
    assert code_of(lambda: update(cache, cache, k, k, m)) == 3  # one cache for both
    far = vk.PagedAttention(dev, cmd, 4, 2, 64, 1 << 20).init()
    assert code_of(lambda: far(q, T(1, 2 << 20, 64), T(1, 2 << 20, 64), U(1, n, 2048), U(1, 1, n))) == 11
    assert cmd.L.vkl_paged_attention_run(tables.h, q.h, cache.h, cache.h, good[3].h, good[4].h, None, C.byref(C.c_void_p())) == 3  # another kind of op
    cmd.end()
    try:
        cmd.submit_and_wait()  # the tensors above hold what they hold
    except vk.VklError:
        pass
    cmd.begin()
    # nothing to do is no error
    assert update(cache, good[2], T(1, 0, 128), T(1, 0, 128), U(1, 2, 0), T(1, 0, 256)).shape() == (1, 0, 256)
    assert att(T(1, 0, 256), cache, good[2], U(1, 0, 4), U(1, 1, 0)).shape() == (1, 0, 256)
    assert tables(U(1, 1, 0), U(1, 1, 0), U(1, 0, 4), U(1, 1, 6), 0)[1].shape() == (1, 1, 1)
    cmd.end()
    cmd.submit_and_wait()


# ---- together ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
def test_sequences_are_served_from_one_cache(dev, dtype):
    """Prompts arrive, tokens follow, a draft is taken back, a sequence ends and another takes its pages: every pass's rows against
    the oracle's attention over all that was ever written."""
    heads, kv, dim, page, n, width, pages = 4, 2, 64, 16, 4, 12, 30
    rng, cmd = np.random.default_rng(11), vk.Command(dev)
    lengths, pool, table = np.zeros(n, np.uint32), list(range(pages)), np.zeros((n, width), np.uint32)
    said = [(np.zeros((kv, 0, dim)), np.zeros((kv, 0, dim))) for _ in range(n)]
    with cmd:
        t_len, t_table, t_pool = tensor(cmd, dev, lengths), tensor(cmd, dev, table), tensor(cmd, dev, np.array([pages] + pool, np.uint32))
        kc, vc = (tensor(cmd, dev, np.full((pages, kv * page, dim), 0x7fff, np.uint16), dtype) for _ in range(2))  # NaN
        tables, update, att = (vk.PagedTables(dev, cmd, page).init(), vk.UpdatePagedKVCache(dev, cmd, dim, page, 1e4, dtype).init(),
                               vk.PagedAttention(dev, cmd, heads, kv, dim, page, dtype=dtype).init())
    targets = [[70, 0, 33, 0], [71, 5, 34, 0], [72, 6, 35, 1], [72, 10, 35, 1], [72, 7, 35, 1], [73, 8, 0, 2], [74, 9, 150, 3], [74, 9, 151, 4], [75, 10, 152, 5]]
    for target in targets:
        new = [max(0, t - int(l)) for t, l in zip(target, lengths)]
        rows = sum(new) + 2  # a padded batch
        x = [draw(rng, (rows, h * dim), dtype) for h in (heads, kv, kv)]
        single = all(a == 1 for a in new)
        cmd.begin()
        q, k, v = (tensor(cmd, dev, a, dtype) for a in x)
        m, starts = tables(t_len, tensor(cmd, dev, np.array(target, np.uint32)), t_table, t_pool, rows)
        turned = update(kc, vc, k, v, m, q)
        outs = [cmd.download(att(turned, kc, vc, t_table, t_len, starts))]
        if single:  # the one-token form says the same
            outs.append(cmd.download(vk.PagedAttention(dev, cmd, heads, kv, dim, page, dtype=dtype).init()(turned.view(1, n, heads * dim), kc, vc, t_table, t_len)))
        cmd.end()
        cmd.submit_and_wait()
        q, k, v = (to_values(a, dtype).reshape(rows, -1, dim) for a in x)
        r = 0
        for i in range(n):
            at = np.arange(int(lengths[i]), int(lengths[i]) + new[i])
            fresh = slice(r, r + new[i])
            turn = lambda a: to_values(to_bits(P.rotate(a[fresh], at, 1e4), dtype), dtype)  # noqa: E731
            keep = min(int(lengths[i]), target[i])
            said[i] = tuple(np.concatenate([s[:, :keep], b.transpose(1, 0, 2)], 1) for s, b in zip(said[i], (turn(k), v[fresh])))
            want, mass, size = P.attention(turn(q), at, *said[i])
            for got in outs:
                # a rotated value that lies between two 16-bit numbers may have been rounded the other way: a step of each operand
                slack = 4 * 2 * HALF_STEP[dtype] * size
                got = to_values(got, dtype).reshape(-1, heads, dim)[fresh]
                if new[i]:
                    check(got, want, mass * (1 + slack / HALF_STEP[dtype]), size, dtype, dim, target[i], 5.0, True, str(target))
            r += new[i]
        lengths = np.array(target, np.uint32)


def test_a_captured_step_follows_what_is_in_its_tensors(dev):
    torch = pytest.importorskip("torch")
    rng, cmd = np.random.default_rng(12), vk.Command(dev)
    heads, kv, dim, page, n = 8, 2, 128, 16, 5
    c = Cache(rng, [1500, 3, 700, 64, 1], kv, dim, page, vk.FP16)
    bits = draw(rng, (n, heads * dim), vk.FP16)
    with cmd:
        k, v, table, lens = c.up(cmd, dev)
        q = tensor(cmd, dev, bits, vk.FP16)
        op = vk.PagedAttention(dev, cmd, heads, kv, dim, page).init()
        out = op(q, k, v, table, lens)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.ExternalStream(cmd.stream())
    cmd.begin()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        op(q, k, v, table, lens)
    cmd.end()
    for lengths in ([1500, 3, 700, 64, 1], [40, 3, 699, 0, 1], [1499, 2, 5, 64, 0]):
        with cmd:
            cmd.upload(np.array(lengths, np.uint32), lens)
            cmd.upload(np.zeros((1, n, heads * dim), np.uint16), out)
        with torch.cuda.stream(stream):
            graph.replay()
        stream.synchronize()
        with cmd:
            got = cmd.download(out)
        with cmd:
            direct = cmd.download(op(q, k, v, table, lens))
        assert (got == direct).all()
        value = to_values(got, vk.FP16).reshape(n, heads, dim)
        for i, l in enumerate(lengths):
            want, mass, size = attend(c, i, to_values(bits, vk.FP16).reshape(n, heads, dim)[i:i + 1], [l - 1])
            check(value[i:i + 1], want, mass, size, vk.FP16, dim, l, 5.0, False)
    del graph


def test_captured_calls_of_several_shapes(dev):
    """Each shape's graph keeps its outputs and workspace when the op goes on to others, whose workspace is larger."""
    torch = pytest.importorskip("torch")
    rng, cmd = np.random.default_rng(15), vk.Command(dev)
    heads, kv, dim, page = 4, 1, 64, 16
    op, kept = vk.PagedAttention(dev, cmd, heads, kv, dim, page).init(), []
    stream = torch.cuda.ExternalStream(cmd.stream())
    for past, new in (([3000], [2]), ([2500, 3000, 40], [3, 300, 1]), ([3000, 3000], [500, 400])):
        c = Cache(rng, [a + b for a, b in zip(past, new)], kv, dim, page, vk.FP16)
        starts = np.concatenate([[0], np.cumsum(new)]).astype(np.uint32)
        with cmd:
            k, v, table, lens = c.up(cmd, dev)
            args = (tensor(cmd, dev, draw(rng, (int(starts[-1]), heads * dim), vk.FP16), vk.FP16), k, v, table, lens, tensor(cmd, dev, starts))
            out = op(*args)
            want = cmd.download(out)
        graph = torch.cuda.CUDAGraph()
        cmd.begin()
        with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
            assert op(*args) is out
        cmd.end()
        kept.append((graph, out, want, args))
    held = [vk.Tensor(1, 1, 1 << x, dev, vk.FP32) for x in range(4, 22)]  # takes what has been given up
    with cmd:
        for t in held:
            cmd.upload(np.full(t.shape(), 7, np.float32), t)
    for graph, out, want, _ in kept + kept[::-1]:
        with cmd:
            cmd.upload(np.zeros_like(want), out)
        with torch.cuda.stream(stream):
            graph.replay()
        stream.synchronize()
        with cmd:
            assert (cmd.download(out) == want).all()
    with cmd:
        assert all((cmd.download(t) == 7).all() for t in held)
    kept.clear()


def test_two_commands_at_once(dev):
    """Ops of their own on streams of their own do not share workspace."""
    rng = np.random.default_rng(13)
    c = Cache(rng, [4000, 2500], 2, 128, 16, vk.FP16)
    cmds, outs = [vk.Command(dev) for _ in range(2)], []
    bits = draw(rng, (2, 8 * 128), vk.FP16)
    ready = []
    for cmd in cmds:
        with cmd:
            ready.append((vk.PagedAttention(dev, cmd, 8, 2, 128, 16).init(), tensor(cmd, dev, bits, vk.FP16), *c.up(cmd, dev)))
    for cmd in cmds:
        cmd.begin()
    for _ in range(20):
        for cmd, (op, *args) in zip(cmds, ready):
            outs.append(cmd.download(op(*args)))
    for cmd in cmds:
        cmd.end()
    for cmd in cmds:
        cmd.submit_and_wait()
    assert all((o == outs[0]).all() for o in outs)


def test_time_of_the_last_run(dev):
    """Op::time() as of the other ops: 0 before a run, microseconds of the device after the wait."""
    rng, cmd = np.random.default_rng(14), vk.Command(dev)
    c = Cache(rng, [30000], 2, 128, 16, vk.FP16)
    with cmd:
        k, v, table, lens = c.up(cmd, dev)
        q, op = tensor(cmd, dev, draw(rng, (1, 256), vk.FP16), vk.FP16), vk.PagedAttention(dev, cmd, 2, 2, 128, 16).init()
        assert op.time() == 0
    for _ in range(3):
        with cmd:
            op(q, k, v, table, lens)
        assert 2 <= op.time() < 1000


@pytest.mark.parametrize("dtype,dim,page", [(vk.FP16, 128, 256), (vk.BF16, 256, 24)])
def test_caches_beyond_32_bits(dev, dtype, dim, page):
    """Pages whose first value lies past 2^32 values (and past 2^32 bytes) of the cache; slots past 2^24."""
    rng, cmd = np.random.default_rng(15), vk.Command(dev)
    rows = 2 ** 32 // dim + 40 * page
    pages, new = rows // page, 150
    table = np.arange(pages - 1, pages - 1 - 2 * (-(-new // page) + 1), -2, dtype=np.uint32)[None]  # the last ones, every other
    pos = np.arange(new)
    slots = (table[0, pos // page].astype(np.uint64) * page + pos % page).astype(np.uint32)
    assert (int(table[0, 0]) * page + 1) * dim > 2 ** 32
    x = [draw(rng, (new, h * dim), dtype) for h in (2, 1, 1)]
    with cmd:
        kc, vc = (vk.Tensor(pages, page, dim, dev, dtype) for _ in range(2))
        q, k, v = (tensor(cmd, dev, a, dtype) for a in x)
        vk.UpdatePagedKVCache(dev, cmd, dim, page, 0.0, dtype).init()(kc, vc, k, v, tensor(cmd, dev, np.stack([slots, pos]).astype(np.uint32)))
        op, t = vk.PagedAttention(dev, cmd, 2, 1, dim, page, dtype=dtype).init(), tensor(cmd, dev, table)
        many = cmd.download(op(q, kc, vc, t, tensor(cmd, dev, np.array([new], np.uint32)), tensor(cmd, dev, np.array([0, new], np.uint32))))
        one = cmd.download(op(tensor(cmd, dev, x[0][-1:], dtype), kc, vc, t, tensor(cmd, dev, np.array([new], np.uint32))))
    q, k, v = (to_values(a, dtype).reshape(new, -1, dim) for a in x)
    want, mass, size = P.attention(q, pos, k.transpose(1, 0, 2), v.transpose(1, 0, 2))
    check(to_values(many, dtype).reshape(new, 2, dim), want, mass, size, dtype, dim, new, 5.0, True)
    check(to_values(one, dtype).reshape(1, 2, dim), want[-1:], mass[-1:], size[-1:], dtype, dim, new, 5.0, False)
