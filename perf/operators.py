"""Operators of a paged key-value cache, as a program that serves several sequences uses them.

A cache is [pages, kv_heads * page, dim] (head g's row r of a page is row g * page + r); a sequence's pages are a row of a table.
  tables  PagedTables: sequences grow (pages are taken from a pool, the new rows get slots), then shrink to where they were
  update  UpdatePagedKVCache: new queries and keys are rotated by their positions, keys and values written to their slots
  token   PagedAttention, one new token per sequence
  prompt  PagedAttention, several new rows per sequence behind what is cached

`own` chooses between the operators' plain form in elementary torch and the framework's calls.
"""
import math
import random

import torch

own = False

_KIND = {"f16": torch.float16, "bf16": torch.bfloat16}
THETA = 10000.0


def _case(op, dtype, n, heads, kv, dim, page, past, new, window=0, pattern=1, name=None):
    """past, new: (least, most) tokens of a sequence that are cached, that are new."""
    c = {"name": name} if name else {}
    c.update(op=op, dtype=dtype, n=n, heads=heads, kv=kv, dim=dim, page=page, past_lo=past[0], past_hi=past[1], new_lo=new[0],
             new_hi=new[1], window=window, pattern=pattern)
    return c


def listed():
    return [
        # a decode step of 64 sequences: most stay inside their last page; the tokens are then taken back (a draft that was turned down)
        _case("tables", "f16", 64, 32, 32, 128, 16, (1, 4000), (1, 1), name="tables-step"),
        # 256 requests arrive at once, prompts of one token to 2048, and are finished
        _case("tables", "f16", 256, 32, 32, 128, 16, (0, 0), (1, 2048), name="tables-admit"),
        # the decode step's new rows, Llama-2-7B's heads
        _case("update", "f16", 24, 32, 32, 128, 16, (1, 4000), (1, 1), name="update-step"),
        # a batch of prompts, grouped heads
        _case("update", "bf16", 9, 32, 8, 128, 16, (0, 700), (33, 2048), name="update-prompts"),
        # one conversation, a few hundred tokens in: nothing but latency
        _case("token", "f16", 1, 32, 32, 128, 16, (300, 300), (1, 1), name="token-one"),
        # a served batch of Llama-2-7B, ragged lengths up to its context
        _case("token", "f16", 32, 32, 32, 128, 16, (1, 4000), (1, 1), name="token-batch"),
        # a larger batch, four query heads per key head
        _case("token", "bf16", 64, 32, 8, 128, 32, (1, 8000), (1, 1), name="token-grouped"),
        # one very long document
        _case("token", "bf16", 1, 32, 8, 128, 64, (131071, 131071), (1, 1), name="token-long"),
        # odd sizes: pages that are no power of two, heads of 80, a window that begins inside a page
        _case("token", "f16", 17, 40, 5, 80, 24, (5, 5000), (1, 1), window=1000, name="token-window"),
        # a few short prompts, some of a token
        _case("prompt", "f16", 8, 32, 32, 128, 16, (0, 0), (1, 150), name="prompt-short"),
        # one long prompt
        _case("prompt", "f16", 1, 32, 32, 128, 16, (0, 0), (4096, 4096), name="prompt-long"),
        # chunks of prompts behind what earlier chunks left, grouped heads
        _case("prompt", "bf16", 4, 32, 8, 128, 32, (1000, 6000), (300, 512), name="prompt-chunks"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "update", "update", "token", "token", "token", "prompt", "prompt"])
    ratio = rng.choice([1, 1, 2, 4, 5, 8, 12, 16])
    kv = _spread(rng, 1, max(1, 40 // ratio))
    dim = rng.choice([32, 64, 72, 80, 96, 128, 128, 128, 192, 256])
    page = rng.choice([4, 8, 16, 16, 24, 32, 64, 128])
    dtype, pattern = rng.choice(["f16", "bf16"]), rng.randrange(1 << 20)
    if op == "tables":
        hi = _spread(rng, 1, 2000)
        return _case(op, dtype, _spread(rng, 1, 256), ratio * kv, kv, dim, page, (0, _spread(rng, 1, 2000)), (rng.choice([1, hi]), hi), pattern=pattern)
    if op == "update":
        hi = _spread(rng, 1, 1000)
        n = _spread(rng, 1, min(64, max(1, 9000 // hi)))
        return _case(op, dtype, n, ratio * kv, kv, dim, page, (0, _spread(rng, 1, 3000)), (rng.choice([1, hi]), hi), pattern=pattern)
    window = rng.choice([0, 0, 0, _spread(rng, 16, 2000)])
    if op == "token":
        most = _spread(rng, 16, 60000)
        n = _spread(rng, 1, min(200, max(1, 400_000_000 // (4 * kv * dim * most))))
        return _case(op, dtype, n, ratio * kv, kv, dim, page, (rng.choice([0, most]), most), (1, 1), window, pattern)
    new = _spread(rng, 2, 1500)
    past = rng.choice([0, _spread(rng, 1, 3000)])
    n = _spread(rng, 1, min(16, max(1, 20_000_000 // (new * (new + past)))))
    return _case(op, dtype, n, ratio * kv, kv, dim, page, (0, past), (rng.choice([1, new]), new), window, pattern)


def _lengths(case):
    """Cached and new tokens of every sequence, by the case alone."""
    rng = random.Random(case["pattern"])
    past = [rng.randint(case["past_lo"], case["past_hi"]) for _ in range(case["n"])]
    return past, [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["n"])]


def work(case):
    past, new = _lengths(case)
    rows, pages = sum(new), lambda t: -(-t // case["page"])  # noqa: E731
    q, kv = case["heads"] * case["dim"], case["kv"] * case["dim"]
    if case["op"] == "tables":
        fresh = sum(pages(p + t) - pages(p) for p, t in zip(past, new))
        # both ways: lengths and targets read, lengths written; growing writes rows' slots and positions, starts and pages, shrinking the pool
        return {"bytes": 2 * 12 * case["n"] + 4 * (case["n"] + 1) + 8 * rows + 2 * 8 * fresh, "flops": 0}
    if case["op"] == "update":
        return {"bytes": 2 * 2 * rows * (q + 2 * kv) + 8 * rows, "flops": 3 * rows * (q + kv)}
    w = case["window"] or 1 << 40
    seen = sum(min(p + t, w + t - 1) for p, t in zip(past, new))  # cached rows that some new row sees
    pairs = sum(min(p + i + 1, w) for p, t in zip(past, new) for i in range(t))
    return {"bytes": 2 * 2 * rows * q + 2 * 2 * seen * kv + 4 * sum(pages(p + t) for p, t in zip(past, new)), "flops": 4 * pairs * q}


def _inputs(case, seed):
    """What both forms get, on the GPU: tensors of torch."""
    past, new = _lengths(case)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    n, page = case["n"], case["page"]
    rows, total = sum(new), [p + t for p, t in zip(past, new)]
    most = max(1, max(-(-t // page) for t in total)) + 2
    held = sum(-(-t // page) for t in total)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    s = {"past": ints(past), "total": ints(total)}
    order = torch.randperm(held + 3, generator=g, device="cuda").to(torch.int32)  # pages as a server's past has mixed them
    grows = case["op"] == "tables"  # these hold pages for what is cached only; the others for all
    have = ints([-(-t // page) for t in (past if grows else total)])
    before = torch.cumsum(have, 0) - have
    j = torch.arange(most, device="cuda")
    at = (before[:, None] + j[None, :]).clamp(max=held + 2)
    s["table"] = torch.where(j[None, :] < have[:, None], order[at], 0).to(torch.int32)
    if grows:
        taken = sum(-(-p // page) for p in past)
        s["pool"] = torch.cat([ints([held + 3 - taken]), order[taken:], ints([0] * taken)])
        return s
    fresh = ints(new)
    s["starts"] = torch.cat([ints([0]), torch.cumsum(fresh, 0).to(torch.int32)])
    seq = torch.repeat_interleave(torch.arange(n, device="cuda"), fresh)
    pos = s["past"][seq] + torch.arange(rows, device="cuda") - s["starts"][seq]
    slot = s["table"][seq, pos // page] * page + pos % page
    s["map"] = torch.stack([slot, pos]).to(torch.int32)
    kind = _KIND[case["dtype"]]
    draws = lambda *shape: torch.randn(shape, generator=g, device="cuda", dtype=kind)  # noqa: E731
    s["q"] = draws(rows, case["heads"] * case["dim"])
    if case["op"] == "update":
        s["k"], s["v"] = draws(rows, case["kv"] * case["dim"]), draws(rows, case["kv"] * case["dim"])
    s["kcache"], s["vcache"] = (draws(held + 3, case["kv"] * page, case["dim"]) for _ in range(2))
    return s


# ---- the framework's side ----------------------------------------------------------------------------------------------
_session = {}


class _Raw:
    """A library tensor's memory, for torch.as_tensor."""

    def __init__(self, ptr, shape, kind):
        self.__cuda_array_interface__ = {"data": (ptr, False), "shape": shape, "typestr": kind, "version": 3}


def _seen(t, dtype):
    """A torch tensor over a library tensor's memory."""
    shape = tuple(t.shape())
    raw = torch.as_tensor(_Raw(t.device_ptr(), shape, "<i4" if dtype == torch.int32 else "<i2"), device="cuda")
    return raw if dtype == torch.int32 else raw.view(dtype)


def _library():
    """The program's device and its command, which records from the first call on."""
    import vkllama_b200 as vk
    if not _session:
        _session["dev"] = vk.Device(0)
        _session["cmd"] = vk.Command(_session["dev"])
        _session["cmd"].begin()
    return vk, _session["dev"], _session["cmd"]


def _held(t):
    """A library tensor with t's values, rows of up to three dimensions."""
    vk, dev, _ = _library()
    shape = (1,) * (3 - t.dim()) + tuple(t.shape)
    mine = vk.Tensor(*shape, dev, {torch.int32: vk.UINT32, torch.float16: vk.FP16, torch.bfloat16: vk.BF16}[t.dtype])
    _seen(mine, t.dtype).copy_(t.view(shape))
    return mine


def _result(s, t, dtype):
    """An output's memory; operators keep theirs, so the views are kept too."""
    key = (t.device_ptr(), tuple(t.shape()))
    if key not in s["views"]:
        s["views"][key] = _seen(t, dtype)
    return s["views"][key]


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        vk, dev, cmd = _library()
        kind = vk.FP16 if case["dtype"] == "f16" else vk.BF16
        mine = {k: _held(t) for k, t in s.items()}
        state = {k: _seen(mine[k], s[k].dtype) for k in ("table", "past", "pool", "kcache", "vcache") if k in s}
        s = {"mine": mine, "views": {}, **state}
        if case["op"] == "tables":
            mine["back"] = _held(s["past"].view(-1))
            s["grow"], s["shrink"] = (vk.PagedTables(dev, cmd, case["page"]).init() for _ in range(2))
        elif case["op"] == "update":
            s["run"] = vk.UpdatePagedKVCache(dev, cmd, case["dim"], case["page"], THETA, kind).init()
        else:
            s["run"] = vk.PagedAttention(dev, cmd, case["heads"], case["kv"], case["dim"], case["page"], 0.0, case["window"], kind).init()
    elif case["op"] == "tables":
        s["back"] = s["past"].clone()
    return {**s, "case": case, "rows": sum(_lengths(case)[1])}


def run(s):
    op = s["case"]["op"]
    if own:
        m, kind = s["mine"], _KIND[s["case"]["dtype"]]
        if op == "tables":
            slots, starts = s["grow"](m["past"], m["total"], m["table"], m["pool"], s["rows"])
            s["shrink"](m["past"], m["back"], m["table"], m["pool"], 0)
            got = {"map": _result(s, slots, torch.int32), "starts": _result(s, starts, torch.int32)}
            return {**got, **{k: s[k] for k in ("past", "table", "pool")}}
        if op == "update":
            q = s["run"](m["kcache"], m["vcache"], m["k"], m["v"], m["map"], m["q"])
            return {"q": _result(s, q, kind), "kcache": s["kcache"], "vcache": s["vcache"]}
        return {"out": _result(s, s["run"](m["q"], m["kcache"], m["vcache"], m["table"], m["total"], m["starts"] if op == "prompt" else None), kind)}
    if op == "tables":
        slots, starts = _resize(s, s["total"], s["rows"])
        _resize(s, s["back"], 0)
        return {"map": slots[None], "starts": starts[None, None], "past": s["past"][None, None], "table": s["table"][None], "pool": s["pool"][None, None]}
    if op == "update":
        return {"q": _plain_update(s)[None], "kcache": s["kcache"], "vcache": s["vcache"]}
    return {"out": (_plain_token if op == "token" else _plain_prompt)(s)[None]}


# ---- plain forms -------------------------------------------------------------------------------------------------------
def _resize(s, target, rows):
    page, table, pool, past = s["case"]["page"], s["table"], s["pool"], s["past"]
    have, want = (past + page - 1) // page, (target + page - 1) // page
    give, need = (have - want).clamp(min=0), (want - have).clamp(min=0)
    j = torch.arange(table.shape[1], device="cuda")[None]
    # pages given back, the last sequence's last page first
    nth = (torch.cumsum(give, 0) - give)[:, None] + j - want[:, None]
    given = (j >= want[:, None]) & (j < have[:, None])
    count = pool[0] + give.sum()
    stack = torch.cat([pool, pool[:1]])  # and a place for what is not given
    stack[torch.where(given, count - nth, pool.shape[0])] = table
    # pages taken from the end of the pool
    nth = (torch.cumsum(need, 0) - need)[:, None] + j - have[:, None]
    taken = (j >= have[:, None]) & (j < want[:, None])
    table.copy_(torch.where(taken, stack[torch.where(taken, count - nth, 0)], table))
    pool.copy_(stack[:-1])
    pool[0] = count - need.sum()
    starts = torch.nn.functional.pad(torch.cumsum((target - past).clamp(min=0), 0), (1, 0))
    r = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(starts[1:], r, right=True).clamp(max=past.shape[0] - 1)
    pos = torch.where(r < starts[-1], past[seq] + r - starts[seq], 0)
    slot = torch.where(r < starts[-1], table[seq, pos // page] * page + pos % page, -1)
    past.copy_(target)
    return torch.stack([slot, pos]).to(torch.int32), starts.to(torch.int32)


def _turned(x, pos, dim):
    """Neighbouring pairs turned by position * THETA^(-2k / dim); the angle in 64 bits, for far positions."""
    freq = THETA ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
    angle = pos.double()[:, None] * freq[None]
    c, n = angle.cos().float()[:, None], angle.sin().float()[:, None]
    p = x.float().view(x.shape[0], -1, dim // 2, 2)
    return torch.stack([p[..., 0] * c - p[..., 1] * n, p[..., 0] * n + p[..., 1] * c], -1).view(x.shape).to(x.dtype)


def _plain_update(s):
    c = s["case"]
    slot, pos = s["map"][0].long(), s["map"][1]
    at, row = slot // c["page"], slot % c["page"]
    pages = lambda t: t.view(t.shape[0], c["kv"], c["page"], c["dim"])  # noqa: E731
    heads = torch.arange(c["kv"], device="cuda")[None]
    pages(s["kcache"])[at[:, None], heads, row[:, None]] = _turned(s["k"], pos, c["dim"]).view(-1, c["kv"], c["dim"])
    pages(s["vcache"])[at[:, None], heads, row[:, None]] = s["v"].view(-1, c["kv"], c["dim"])
    return _turned(s["q"], pos, c["dim"])


def _cached(s):
    """Keys and values of every sequence in 32 bits, [n, kv, longest, dim], and which positions exist."""
    c = s["case"]
    j = torch.arange(c["past_hi"] + c["new_hi"], device="cuda")
    there = j[None] < s["total"][:, None]
    at = s["table"].long()[:, (j // c["page"]).clamp(max=s["table"].shape[1] - 1)]
    rows = lambda t: t.view(t.shape[0], c["kv"], c["page"], c["dim"])[at, :, (j % c["page"])[None]]  # noqa: E731
    get = lambda t: torch.where(there[..., None, None], rows(t), 0).float().transpose(1, 2)  # noqa: E731
    return get(s["kcache"]), get(s["vcache"]), j


def _plain_token(s):
    c = s["case"]
    k, v, j = _cached(s)
    q = s["q"].float().view(c["n"], c["kv"], -1, c["dim"])
    score = (q @ k.transpose(-1, -2)) * c["dim"] ** -0.5
    last = s["total"][:, None] - 1
    sees = (j[None] <= last) & (j[None] > last - (c["window"] or 1 << 30))
    p = (score.masked_fill(~sees[:, None, None], -math.inf)).softmax(-1)
    return (p @ v).view(c["n"], -1).to(s["q"].dtype)


def _plain_prompt(s):
    c = s["case"]
    k, v, j = _cached(s)
    t = torch.arange(c["new_hi"], device="cuda")
    rows = (s["starts"][:-1, None] + t[None]).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float()[rows].view(c["n"], -1, c["kv"], c["heads"] // c["kv"], c["dim"]).permute(0, 2, 3, 1, 4)
    score = (q.flatten(2, 3) @ k.transpose(-1, -2)).unflatten(2, (-1, c["new_hi"])) * c["dim"] ** -0.5
    pos = s["past"][:, None, None] + t[None, :, None]
    sees = (j[None, None] <= pos) & (j[None, None] > pos - (c["window"] or 1 << 30))
    p = score.masked_fill_(~sees[:, None, None], -math.inf).softmax(-1)
    out = (p.flatten(2, 3) @ v).unflatten(2, (-1, c["new_hi"])).permute(0, 3, 1, 2, 4)
    row = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(s["starts"][1:].contiguous(), row.to(torch.int32), right=True)
    return out[seq, row - s["starts"][seq]].reshape(row.shape[0], -1).to(s["q"].dtype)


# ---- in 64 bits --------------------------------------------------------------------------------------------------------
def exact(case, seed):
    """From the definition, one sequence after the other; nothing for the tables, which are whole numbers."""
    if case["op"] == "tables":
        return None
    s, (past, new) = _inputs(case, seed), _lengths(case)
    page, kv, dim, group = case["page"], case["kv"], case["dim"], case["heads"] // case["kv"]
    if case["op"] == "update":
        k, v = s["kcache"].double(), s["vcache"].double()
        z = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.outer(s["map"][1].double(), torch.exp(
            -math.log(THETA) * torch.arange(dim // 2, device="cuda", dtype=torch.float64) * 2 / dim)))
        turn = lambda x: torch.view_as_real(torch.view_as_complex(x.double().reshape(x.shape[0], -1, dim // 2, 2)) * z[:, None]).reshape(x.shape[0], -1, dim)  # noqa: E731
        slot = s["map"][0].long()
        for h in range(kv):
            at = slot // page * (kv * page) + h * page + slot % page
            k.view(-1, dim)[at] = turn(s["k"])[:, h]
            v.view(-1, dim)[at] = s["v"].double().view(-1, kv, dim)[:, h]
        return {"q": turn(s["q"]).reshape(1, -1, case["heads"] * dim), "kcache": k, "vcache": v}
    out = torch.zeros(1, sum(new), case["heads"], dim, dtype=torch.float64, device="cuda")
    first = 0
    for i in range(case["n"]):
        length = past[i] + new[i]
        at = s["table"][i, : -(-length // page)].long()
        mine = lambda t: t[at].view(-1, kv, page, dim).transpose(0, 1).reshape(kv, -1, dim)[:, :length]  # noqa: E731
        keys, values, j = mine(s["kcache"]), mine(s["vcache"]), torch.arange(length, device="cuda")
        for r in range(0, new[i], 256):
            rows = slice(first + r, first + min(new[i], r + 256))
            pos = past[i] + torch.arange(r, min(new[i], r + 256), device="cuda")[:, None]
            hidden = (j > pos) | (j <= pos - (case["window"] or length + 1))
            for h in range(case["heads"]):
                score = s["q"][rows, h * dim:(h + 1) * dim].double() @ keys[h // group].double().T / math.sqrt(dim)
                e = torch.exp(score.masked_fill(hidden, -math.inf) - score.masked_fill(hidden, -math.inf).amax(1, keepdim=True))
                out[0, rows, h] = e @ values[h // group].double() / e.sum(1, keepdim=True)
        first += new[i]
    return {"out": out.view(1, -1, case["heads"] * dim)}
