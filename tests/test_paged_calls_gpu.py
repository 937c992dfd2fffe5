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
    # as tests/paged_weights.py: 2^18 products one after the other, each cut off at 2^-23 of their sum
    tol = 2.0 ** -11 * np.abs(want) + (4 * (dim + 4) * 2.0 ** -24 * size + 2.0 ** -11 + 2.0 ** -17 + 2.0 ** -5 + 2.0 ** -14) * mass
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
