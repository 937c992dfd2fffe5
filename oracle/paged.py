"""Operators of a paged key-value cache, restated in numpy float64 from their definitions: one function per operator, one sequence or
token after the other. Caches are [pages, kv_heads, page, dim]."""
import numpy as np

NO_SLOT = 0xffffffff


def resize(page, lengths, target, table, pool, rows):
    """Pages and slots of sequences that go from lengths to target. pool: list of free pages, the next one to be taken last. Returns
    (lengths, table, pool, map, starts), or None where the pool, the table or the rows do not suffice."""
    up = lambda t: -(-int(t) // page)  # noqa: E731
    table, pool = table.copy(), list(pool)
    fresh = [max(0, int(t) - int(l)) for l, t in zip(lengths, target)]
    need = sum(max(0, up(t) - up(l)) for l, t in zip(lengths, target))
    back = [table[i, j] for i, (l, t) in enumerate(zip(lengths, target)) for j in range(up(t), up(l))]
    if need > len(pool) + len(back) or max(up(t) for t in target) > table.shape[1] or sum(fresh) > rows:
        return None
    pool += back[::-1]
    slots, pos, starts = [], [], [0]
    for i, (l, t) in enumerate(zip(lengths, target)):
        for j in range(up(l), up(t)):
            table[i, j] = pool.pop()
        for p in range(int(l), int(l) + fresh[i]):
            slots.append(int(table[i, p // page]) * page + p % page)
            pos.append(p)
        starts.append(starts[-1] + fresh[i])
    behind = rows - len(slots)
    return (np.array(target, np.uint32), table, pool, np.array([slots + [NO_SLOT] * behind, pos + [0] * behind], np.uint32).reshape(2, rows),
            np.array(starts, np.uint32))


def rotate(x, pos, theta):
    """x [rows, heads, dim]: neighbouring pairs turned by pos * theta^(-2k / dim)."""
    dim = x.shape[-1]
    angle = np.asarray(pos, np.float64)[:, None, None] * theta ** (-np.arange(0, dim, 2) / dim)
    a, b = x[..., 0::2], x[..., 1::2]
    y = np.empty(x.shape)
    y[..., 0::2] = a * np.cos(angle) - b * np.sin(angle)
    y[..., 1::2] = a * np.sin(angle) + b * np.cos(angle)
    return y


def attention(q, pos, keys, values, window=0, scale=None):
    """q [rows, heads, dim] at positions pos, keys and values [kv_heads, tokens, dim] of their sequence. Returns the output, the
    output of |values|, and the most that the products of a row's score add up to in magnitude."""
    rows, heads, dim = q.shape
    per, scale = heads // keys.shape[0], dim ** -0.5 if scale is None else scale
    out, mass, size = np.zeros((3, rows, heads, dim))
    for r in range(rows):
        lo = max(0, pos[r] + 1 - window) if window else 0
        if pos[r] < 0:
            continue
        for h in range(heads):
            k, v = keys[h // per, lo:pos[r] + 1], values[h // per, lo:pos[r] + 1]
            s = scale * (k @ q[r, h])
            p = np.exp(s - s.max())
            p /= p.sum()
            with np.errstate(invalid="ignore"):
                out[r, h], mass[r, h] = p @ v, p @ np.abs(v)
            size[r, h] = abs(scale) * (np.abs(k) @ np.abs(q[r, h])).max()
    return out, mass, size


def weights_sum(q, pos, keys, window=0, scale=None):
    """Of attention's rows: the sum of exp(score - largest score)."""
    rows, heads, dim = q.shape
    per, scale = heads // keys.shape[0], dim ** -0.5 if scale is None else scale
    den = np.ones((rows, heads, 1))
    for r in range(rows):
        lo = max(0, pos[r] + 1 - window) if window else 0
        for h in range(heads if pos[r] >= 0 else 0):
            s = scale * (keys[h // per, lo:pos[r] + 1] @ q[r, h])
            den[r, h] = np.exp(s - s.max()).sum()
    return den
