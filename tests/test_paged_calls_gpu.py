"""Calls on the operators of a paged cache as programs make them: times while other work is queued, captures, tables for long contexts, refusals."""
import numpy as np
import pytest

import vkllama_b200 as vk
from paged_util import Cache, attend, check, draw, tensor, to_values

pytestmark = pytest.mark.gpu


def code_of(call):
    with pytest.raises(vk.VklError) as e:
        call()
    return e.value.code


def test_items_of_millions_of_positions(dev):
    """Two rows each behind four million positions, which are one page again and again: half of a CTA's softmax warps have nothing to do as long as that takes. More
    items than SMs, so that none is split."""
    n, heads, dim, page, width = 19, 8, 64, 128, 1 << 15
    rng, cmd = np.random.default_rng(23), vk.Command(dev)
    c = Cache(rng, [page], heads, dim, page, vk.FP16)
    bits = draw(rng, (2 * n, heads * dim), vk.FP16)
    with cmd:
        k, v, _, _ = c.up(cmd, dev)
        table = tensor(cmd, dev, np.full((n, width), c.table[0, 0], np.uint32))
        lens, starts = tensor(cmd, dev, np.full(n, width * page, np.uint32)), tensor(cmd, dev, np.arange(n + 1, dtype=np.uint32) * 2)
        op = vk.PagedAttention(dev, cmd, heads, heads, dim, page).init()
        got = to_values(cmd.download(op(tensor(cmd, dev, bits, vk.FP16), k, v, table, lens, starts)), vk.FP16).reshape(2 * n, heads, dim)
    q = to_values(bits, vk.FP16).reshape(2 * n, heads, dim)
    want, mass, size = attend(c, 0, q, [page - 1] * (2 * n))  # the one position of four million that the first row does not see counts 2^-22
    # as tests/paged_weights.py: 2^11 products one after the other, each cut off at 2^-23 of their sum, and 2^7 such sums rounded
    tol = 2.0 ** -11 * np.abs(want) + (4 * (dim + 4) * 2.0 ** -24 * size + 2.0 ** -11 + 2.0 ** -17 + 2.0 ** -12 + 2.0 ** -17 + 2.0 ** -20) * mass
    assert (np.abs(got - want) <= tol).all()


def test_time_of_a_run_that_is_over_while_others_are_queued(dev):
    """As of the other ops: what counts is the op's own last run."""
    rng, cmd = np.random.default_rng(20), vk.Command(dev)
    c = Cache(rng, [60000], 2, 128, 16, vk.FP16)
    with cmd:
        k, v, table, lens = c.up(cmd, dev)
        q = tensor(cmd, dev, draw(rng, (1, 256), vk.FP16), vk.FP16)
        op, other = (vk.PagedAttention(dev, cmd, 2, 2, 128, 16).init() for _ in range(2))
        op(q, k, v, table, lens)
    took = op.time()
    assert 2 <= took < 1000
    cmd.begin()
    for _ in range(2000):
        other(q, k, v, table, lens)
    assert op.time() == took
    assert code_of(other.time) == 9  # its own has not finished
    op(q, k, v, table, lens)
    assert code_of(op.time) == 9
    cmd.end()
    cmd.submit_and_wait()
    assert 2 <= op.time() < 1000 and 2 <= other.time() < 1000


def test_time_when_the_command_is_gone(dev):
    rng, cmd = np.random.default_rng(20), vk.Command(dev)
    c = Cache(rng, [30000], 2, 128, 16, vk.FP16)
    with cmd:
        k, v, table, lens = c.up(cmd, dev)
        q, op = tensor(cmd, dev, draw(rng, (1, 256), vk.FP16), vk.FP16), vk.PagedAttention(dev, cmd, 2, 2, 128, 16).init()
        op(q, k, v, table, lens)
    cmd.begin()
    op(q, k, v, table, lens)  # its end waits for this
    cmd.end()
    cmd.close()
    assert 2 <= op.time() < 1000


def test_a_shape_that_is_captured_first(dev):
    """Its workspace is zero for the first direct call too, which comes before any replay."""
    torch = pytest.importorskip("torch")
    rng, cmd = np.random.default_rng(21), vk.Command(dev)
    heads, kv, dim, page, past, new = 8, 1, 64, 16, (6000, 100), 40  # the second one's positions are not split
    c = Cache(rng, [a + new for a in past], kv, dim, page, vk.FP16)
    bits = draw(rng, (2 * new, heads * dim), vk.FP16)
    with cmd:
        k, v, table, lens = c.up(cmd, dev)
        args = (tensor(cmd, dev, bits, vk.FP16), k, v, table, lens, tensor(cmd, dev, np.array([0, new, 2 * new], np.uint32)))
        used = [vk.Tensor(1, 1, 1 << x, dev, vk.FP32) for x in range(14, 24)]  # memory that the workspace may get
        for t in used:
            cmd.upload(np.full(t.shape(), 7, np.float32), t)
        op = vk.PagedAttention(dev, cmd, heads, kv, dim, page).init()
    del used, t
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.ExternalStream(cmd.stream())
    cmd.begin()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="relaxed"):
        out = op(*args)
    cmd.end()
    with cmd:
        direct = cmd.download(op(*args))
    with torch.cuda.stream(stream):
        graph.replay()
    stream.synchronize()
    with cmd:
        assert (cmd.download(out) == direct).all()
    q, got = (to_values(a, vk.FP16).reshape(2, new, heads, dim) for a in (bits, direct))
    for i in range(2):
        want, mass, size = attend(c, i, q[i], list(range(past[i], past[i] + new)))
        check(got[i], want, mass, size, vk.FP16, dim, past[i] + new, 5.0, True, str(i))
    del graph

@pytest.mark.parametrize("heads", [32, 300])
def test_tables_that_could_hold_more_than_is_counted(dev, heads):
    """2300 sequences with room for a million tokens each: lengths decide. Beyond 2^31 tiles the call is refused on the device and writes nothing."""
    n, page, width, dim, kv = 2300, 64, 16384, 8, 32 if heads == 32 else 30
    rng, cmd = np.random.default_rng(22), vk.Command(dev)
    c = Cache(rng, [int(x) for x in rng.integers(0, 40, n)], kv, dim, page, vk.FP16, spare=1)
    c.table = np.pad(c.table, ((0, 0), (0, width - c.table.shape[1])))
    bits = draw(rng, (n, heads * dim), vk.FP16)
    with cmd:
        k, v, table, lens = c.up(cmd, dev)
        q = tensor(cmd, dev, bits, vk.FP16)
        op = vk.PagedAttention(dev, cmd, heads, kv, dim, page).init()
        got = cmd.download(op(q, k, v, table, lens))
    q_ = to_values(bits, vk.FP16).reshape(n, heads, dim)
    for i in range(0, n, 17):
        l = c.lengths[i]
        want, mass, size = attend(c, i, q_[i:i + 1], [l - 1])
        check(to_values(got, vk.FP16).reshape(n, heads, dim)[i:i + 1], want, mass, size, vk.FP16, dim, l, 5.0, False, str(i))
    cmd.begin()
    assert n * kv * width * page // 32 > 2 ** 31
    out = op(q, k, v, table, tensor(cmd, dev, np.full(n, width * page, np.uint32)))
    cmd.end()
    assert code_of(cmd.submit_and_wait) == 11
    with cmd:
        assert (cmd.download(out) == got).all()
        assert (cmd.download(op(q, k, v, table, lens)) == got).all()


def test_an_update_on_its_own_output(dev):
    """Queries are turned in their place; keys and values that other threads would store over meanwhile are refused."""
    rng, cmd = np.random.default_rng(24), vk.Command(dev)
    rows, dim, page = 40, 64, 16
    x, m = draw(rng, (rows, 4 * dim), vk.FP16), np.stack([np.arange(rows), np.arange(rows)]).astype(np.uint32)
    with cmd:
        kc, vc = (tensor(cmd, dev, np.zeros((3, 4 * page, dim), np.uint16), vk.FP16) for _ in range(2))
        q, k, mt = tensor(cmd, dev, x, vk.FP16), tensor(cmd, dev, x, vk.FP16), tensor(cmd, dev, m)
        op, other = (vk.UpdatePagedKVCache(dev, cmd, dim, page).init() for _ in range(2))
        out = op(kc, vc, k, k, mt, q)
        once = cmd.download(out)
        want = cmd.download(other(kc, vc, k, k, mt, tensor(cmd, dev, once[0], vk.FP16)))
        assert op(kc, vc, k, k, mt, out) is out and (cmd.download(out) == want).all()
        assert code_of(lambda: op(kc, vc, out, k, mt, q)) == 3
        assert code_of(lambda: op(kc, vc, k, out, mt, q)) == 3
        assert code_of(lambda: op(kc, vc, out.view(1, rows, 4 * dim), k, mt, out)) == 3
        assert op(kc, vc, out, out, mt) is None  # nothing is stored there
        got = cmd.download(vc).reshape(3, 4, page, dim)
    at = np.arange(rows)
    assert (got[at // page, :, at % page].reshape(rows, -1) == want[0]).all()


@pytest.mark.parametrize("bad", ["page", "length", "short", "order"])
@pytest.mark.parametrize("page", [16, 5])
@pytest.mark.parametrize("lengths,new,launches", [([300, 200, 260], [100, 80, 90], 1), ([300, 140, 260, 40], [2, 3, 1, 5], 2), ([3000, 2500, 40], [5, 4, 2], 3)])
def test_bad_rows_of_several_kernels(dev, bad, page, lengths, new, launches):
    """The tcgen05 kernel alone, both kernels, split positions: what is wrong with the second sequence is reported, the others' rows are right, and so is the
    next call."""
    heads, kv, dim, dtype = 4, 2, 64, vk.BF16
    rng, cmd = np.random.default_rng(25), vk.Command(dev)
    c = Cache(rng, lengths, kv, dim, page, dtype)
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.uint32)
    bits = draw(rng, (starts[-1], heads * dim), dtype)
    q_ = to_values(bits, dtype).reshape(-1, heads, dim)
    with cmd:
        k, v, table, lens = c.up(cmd, dev)
        q, good = tensor(cmd, dev, bits, dtype), tensor(cmd, dev, starts)
        op = vk.PagedAttention(dev, cmd, heads, kv, dim, page, dtype=dtype).init()
    wrong_table, wrong_lengths, wrong_starts = c.table.copy(), np.array(lengths, np.uint32), starts.copy()
    if bad == "page":
        wrong_table[1, 3], wrong_table[1, 7] = c.pages, 0xffffffff
    elif bad == "length":
        wrong_lengths[1] = c.table.shape[1] * page + 1
    elif bad == "short":
        wrong_lengths[1] = new[1] - 1
    else:
        wrong_starts[2] = 0
    for first in (True, False):
        before = vk.kernel_launches()
        cmd.begin()
        if first:
            wrong = [tensor(cmd, dev, a) for a in (wrong_table, wrong_lengths, wrong_starts)]
            got = cmd.download(op(q, k, v, *wrong))
        else:
            got = cmd.download(op(q, k, v, table, lens, good))
        cmd.end()
        assert vk.kernel_launches() - before == launches
        if first:
            assert code_of(cmd.submit_and_wait) == (11 if bad == "page" else 3)
        else:
            cmd.submit_and_wait()
        got = to_values(got, dtype).reshape(-1, heads, dim)
        for i, l in enumerate(lengths):
            if first and (i == 1 or bad == "order"):  # rows of the others are the second's too there
                continue
            mine = slice(starts[i], starts[i + 1])
            want, mass, size = attend(c, i, q_[mine], list(range(l - new[i], l)))
            check(got[mine], want, mass, size, dtype, dim, l, 5.0, True, str(i))


@pytest.mark.parametrize("heads,kv,dim", [(12, 1, 128), (4, 2, 64), (16, 1, 200)])
def test_bad_pages_of_single_tokens(dev, heads, kv, dim):
    """In a sequence that several CTAs share, up to eight heads a key head and beyond."""
    rng, cmd, page = np.random.default_rng(26), vk.Command(dev), 16
    c = Cache(rng, [3000, 50, 4000], kv, dim, page, vk.FP16)
    bits = draw(rng, (3, heads * dim), vk.FP16)
    q_ = to_values(bits, vk.FP16).reshape(3, heads, dim)
    wrong = c.table.copy()
    wrong[0, 11], wrong[0, 150] = 0xffffffff, c.pages
    with cmd:
        k, v, table, lens = c.up(cmd, dev)
        q, bad = tensor(cmd, dev, bits, vk.FP16), tensor(cmd, dev, wrong)
        op = vk.PagedAttention(dev, cmd, heads, kv, dim, page).init()
    for t, which in ((bad, (1, 2)), (table, (0, 1, 2))):
        cmd.begin()
        got = to_values(cmd.download(op(q, k, v, t, lens)), vk.FP16).reshape(3, heads, dim)
        cmd.end()
        if t is bad:
            assert code_of(cmd.submit_and_wait) == 11
        else:
            cmd.submit_and_wait()
        for i in which:
            want, mass, size = attend(c, i, q_[i:i + 1], [c.lengths[i] - 1])
            check(got[i:i + 1], want, mass, size, vk.FP16, dim, c.lengths[i], 5.0, False, str(i))
