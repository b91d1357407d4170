"""The operators of many streams over one paged K/V cache, as they are measured: attention of one new token over the cache, causal attention of
packed prompts, and the cache's own operations (append, take back, fork, compact).

`own` false: their plain form in elementary torch operations.  `own` true: the calls of include/mi355x_kernels.h through whisper.cpp_amd/kernels_api.py.

A cache is two pools of pages (page_size keys of every K/V head), a table with a row of page numbers for each sequence (-1: none), the sequences'
lengths, and for each page the number of rows that hold it (0: free).  Key j of sequence s lies in page table[s][j / page_size], at j % page_size."""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one stream's step on the smallest decoder in use here (base.en: 8 heads of 64, a full text context of 448): latency alone
        dict(name="paged: one stream", op="paged", n=1, heads=8, kv_heads=8, dim=64, page=16, low=448, high=448, window=0, type="f16", io="f32", order="head", shape=1),
        # cross-attention of 32 merged streams (large-v3: 20 heads of 64, 1500 audio positions each), F32 activations as its graphs have them
        dict(name="paged: 32 streams", op="paged", n=32, heads=20, kv_heads=20, dim=64, page=64, low=1500, high=1500, window=0, type="f16", io="f32", order="head", shape=2),
        # a batch of conversations of very different lengths on a decoder with four query heads to a K/V head
        dict(name="paged: ragged, grouped", op="paged", n=64, heads=32, kv_heads=8, dim=128, page=16, low=1, high=8192, window=0, type="bf16", io="bf16", order="key", shape=3),
        # two very long documents: few rows, so the work has to be split over the cache's length
        dict(name="paged: long", op="paged", n=2, heads=64, kv_heads=8, dim=128, page=64, low=100001, high=131072, window=0, type="bf16", io="bf16", order="head", shape=4),
        # four short prompts (start-of-transcript tokens with a little context) on base.en's heads: latency alone
        dict(name="packed: short prompts", op="packed", n=4, heads=8, kv_heads=8, dim=64, low=4, high=48, past=0, page=0, window=0, type="f16", io="f16", order="head", shape=5),
        # prompts of very different lengths in one call, large-v3's heads, up to its audio context's length
        dict(name="packed: ragged", op="packed", n=24, heads=20, kv_heads=20, dim=64, low=1, high=1500, past=0, page=0, window=0, type="f16", io="f16", order="head", shape=6),
        # one long prompt on a decoder with grouped heads: matrix products all over
        dict(name="packed: long, grouped", op="packed", n=1, heads=32, kv_heads=8, dim=128, low=8192, high=8192, past=0, page=0, window=0, type="bf16", io="bf16", order="head", shape=7),
        # the next piece of four prompts whose earlier part lies in the cache, with a sliding window
        dict(name="packed: piece over a cache", op="packed", n=4, heads=32, kv_heads=8, dim=128, low=129, high=512, past=4001, page=16, window=2048, type="f16", io="f16", order="key", shape=8),
        # a decoder step's new keys and values for 32 streams of large-v3, after the last guess of each was taken back
        dict(name="cache: append a token", op="append", n=32, kv_heads=20, dim=64, page=16, low=1, high=447, new_low=1, new_high=1, type="f16", io="f32", order="head", shape=9),
        # the keys and values of 16 prompts of different lengths, put behind what their sequences hold
        dict(name="cache: append prompts", op="append", n=16, kv_heads=8, dim=128, page=64, low=1, high=1000, new_low=100, new_high=4096, type="bf16", io="bf16", order="head", shape=10),
        # beam search: 64 streams with five beams each take over the rows of the beams that they continue
        dict(name="cache: fork beams", op="fork", n=320, kv_heads=20, dim=64, page=16, low=4, high=448, type="f16", order="head", shape=11),
        # a fragmented cache moved to a new pool: half a gigabyte of keys and values in scattered pages
        dict(name="cache: compact", op="compact", n=48, kv_heads=8, dim=128, page=64, low=64, high=8192, type="f16", order="head", shape=12),
    ]


def _between(rng, a, b):
    """A whole number from a to b, spread over their logarithm."""
    return min(b, max(a, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))


def draw(rng):
    while True:
        op = rng.choice(("paged", "paged", "packed", "packed", "append", "fork", "compact"))
        c = dict(op=op, dim=rng.choice((64, 128)), page=rng.choice((8, 16, 32, 64, 128)), type=rng.choice(("f16", "bf16")), order=rng.choice(("head", "key")), shape=rng.randrange(1 << 20))
        c["kv_heads"] = rng.choice((1, 2, 4, 5, 6, 8, 12, 20))
        if op in ("paged", "packed"):
            c["heads"] = c["kv_heads"] * rng.choice((1, 1, 2, 3, 4, 7, 8))
            c["window"] = rng.choice((0, 0, 0, _between(rng, 16, 4096)))
            c["io"] = rng.choice((c["type"], c["type"], "f32")) if op == "paged" else c["type"]
        if op == "paged":
            c["n"], c["high"] = _between(rng, 1, 128), _between(rng, 16, 131072)
            c["low"] = rng.choice((1, c["high"], max(1, c["high"] // 2)))
        elif op == "packed":
            c["n"], c["high"] = _between(rng, 1, 64), _between(rng, 4, 8192)
            c["low"] = rng.choice((1, c["high"], max(1, c["high"] // 2)))
            c["past"] = rng.choice((0, _between(rng, 16, 8192)))
            c["page"] = c["page"] if c["past"] else 0
        elif op == "append":
            c["io"] = rng.choice((c["type"], "f32"))
            c["n"], c["high"], c["low"] = _between(rng, 1, 256), _between(rng, 16, 4096), 1
            c["new_low"], c["new_high"] = rng.choice(((1, 1), (1, _between(rng, 2, 4096))))
        elif op == "fork":
            c["n"], c["high"], c["low"] = 2 * _between(rng, 1, 200), _between(rng, 16, 8192), 1
        else:
            c["n"], c["high"], c["low"] = _between(rng, 2, 128), _between(rng, 64, 8192), 1
        keys = c["high"] + c.get("new_high", 0) + c.get("past", 0)  # a padded form's cost: what it holds of the keys, and of the scores
        cells = c["n"] * c.get("heads", 0) * keys * (c["high"] if op == "packed" else 1)
        if c["n"] * keys * c["kv_heads"] * c["dim"] <= 1 << 28 and cells <= 1 << 31 and work(c)["flops"] <= 1 << 39:
            return c


def _lengths(rng, n, low, high):
    return [high] + [_between(rng, low, high) for _ in range(n - 1)]


def _shape(case):
    """What a case alone says of its sequences: keys held (`old`) and new rows (`new`) of each."""
    rng, n = random.Random(case["shape"]), case["n"]
    if case["op"] == "packed":
        new = _lengths(rng, n, case["low"], case["high"])
        return [rng.randint(case["past"] // 2, case["past"]) if case["past"] else 0 for _ in range(n)], new
    old = _lengths(rng, n, case["low"], case["high"])
    rng.shuffle(old)
    return old, _lengths(rng, n, case["new_low"], case["new_high"]) if case["op"] == "append" else [0] * n


def _pages(keys, page):
    return -(-keys // page)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pool(case, pages, gen):
    """A pool of random pages as [page, head, key, dim], whichever of heads and keys comes first in memory."""
    a, b = (case["kv_heads"], case["page"]) if case["order"] == "head" else (case["page"], case["kv_heads"])
    t = torch.randn(pages, a, b, case["dim"], device="cuda", dtype=TYPES[case["type"]], generator=gen)
    return t if case["order"] == "head" else t.transpose(1, 2)


def _rows(case, rows, heads, gen):
    return torch.randn(rows, heads, case["dim"], device="cuda", dtype=TYPES[case["io"]], generator=gen)


def _tables(case, keys, pages, rng):
    """Scattered pages for sequences of `keys` keys, out of `pages` pages: the table and the pages' counts.  In the caches that are changed every
    fourth sequence goes on from the one before it: as a copy of its row, or (append) from an earlier place in it."""
    page, n = case["page"], case["n"]
    share = range(3, n, 4) if case["op"] in ("append", "compact") else ()
    for i in share:
        keys[i] = keys[i - 1] if case["op"] == "compact" else min(keys[i], (_pages(keys[i - 1], page) - 1) * page)
    spread = list(range(pages))
    rng.shuffle(spread)
    width = max(_pages(a + b, page) for a, b in zip(keys, _shape(case)[1])) if case["op"] == "append" else max(_pages(a, page) for a in keys)
    table, ref = np.full((n, width), -1, dtype=np.int32), np.zeros(pages, dtype=np.int32)
    for i in range(n):
        held = _pages(keys[i], page)
        table[i, :held] = table[i - 1, :held] if i in share else [spread.pop() for _ in range(held)]
    np.add.at(ref, table[table >= 0], 1)
    return table, ref


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    op, n, page, (old, new) = case["op"], case["n"], case["page"], _shape(case)
    at, order = np.concatenate([[0], np.cumsum(new)]), rng.sample(range(n), n)
    s = dict(case=case, op=op, scale=case["dim"] ** -0.5, n=n, rows=int(at[-1]), most_new=max(new), most=max(new), memory=[])
    if page:
        keys = list(old)
        if op == "packed":  # the new rows' own keys are in the cache already, behind what was there
            for i, row in enumerate(order):
                keys[row] = old[i] + new[i]
        total = sum(_pages(a + b, page) for a, b in zip(keys, new if op == "append" else [0] * n)) + n + 3  # and one for each row that copies its last
        table, ref = _tables(case, keys, total * 2 if op == "compact" else total, rng)
        s.update(k=_pool(case, ref.size, gen), v=_pool(case, ref.size, gen), table=_ints(table), len=_ints(keys), ref=_ints(ref), most=max(keys), status=_ints([0]))
        s["seq"] = _ints(order)
    if op == "paged":
        s["q"] = _rows(case, n, case["heads"], gen)
        s["out"] = torch.zeros_like(s["q"])
    elif op == "packed":
        s["cu"], s["q"] = _ints(at), _rows(case, s["rows"] + 3, case["heads"], gen)  # three rows behind the last sequence, as in a padded batch
        s["out"] = torch.zeros_like(s["q"])
        if not page:
            s["k"], s["v"] = _rows(case, s["rows"] + 3, case["kv_heads"], gen), _rows(case, s["rows"] + 3, case["kv_heads"], gen)
    elif op == "append":
        s["seq"], s["keep"], s["cu"] = _ints(list(range(n))), s["len"].clone(), _ints(at)
        s["nk"], s["nv"] = _rows(case, s["rows"], case["kv_heads"], gen), _rows(case, s["rows"], case["kv_heads"], gen)
    elif op == "fork":  # the first half of the rows are the beams that are gone on from, the second half takes them over
        s["src"] = _ints([rng.randrange(n // 2) for _ in range(n // 2)])
        s["dst"] = _ints(rng.sample(range(n // 2, n), n // 2))
    elif op == "compact":
        used = int(np.count_nonzero(ref))
        s["k2"], s["v2"] = torch.zeros_like(s["k"][:used]), torch.zeros_like(s["v"][:used])
        s.update(table2=torch.full_like(s["table"], -1), len2=torch.zeros_like(s["len"]), ref2=torch.zeros(used, dtype=torch.int32, device="cuda"))
    if own:
        s["call"] = _plan(s)
    return s


# ---- the plain forms --------------------------------------------------------------------------------------------------------------------------


def _attend(q, k, v, allowed, scale):
    """softmax(scale q k^T) v over the allowed keys in 32 bits; a row that is allowed nothing is zero.  q [.., rows, dim], k and v [.., keys, dim]."""
    x = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).masked_fill_(~allowed, -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = x.sum(-1, keepdim=True)
    return torch.matmul(x, v) / torch.where(total == 0, 1.0, total)


def _gathered(s, rows, keys):
    """The first `keys` keys and values (or a few more, up to the page's end) of the sequences of `rows`, in 32 bits, as [row, head, key, dim]."""
    pages = s["table"][rows][:, : _pages(keys, s["case"]["page"])].long().clamp_min(0)
    n, p = pages.shape
    return (x[pages].float().permute(0, 2, 1, 3, 4).reshape(n, x.shape[1], p * x.shape[2], x.shape[3]) for x in (s["k"], s["v"]))


def _plain_paged(s):
    c, rows = s["case"], s["seq"].long()
    k, v = _gathered(s, rows, s["most"])
    q = s["q"].float().reshape(s["n"], c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"])
    at, length = torch.arange(k.shape[2], device="cuda"), s["len"][rows].view(-1, 1, 1, 1)
    allowed = (at < length) & ((at >= length - c["window"]) if c["window"] else True)
    s["out"].copy_(_attend(q, k, v, allowed, s["scale"]).reshape(s["q"].shape))
    return s["out"]


def _plain_packed(s):
    c, n = s["case"], s["n"]
    group = c["heads"] // c["kv_heads"]
    cu = s["cu"].long()
    count, lane = cu[1:] - cu[:-1], torch.arange(s["most_new"], device="cuda")
    index = (cu[:-1, None] + lane).clamp_max(s["rows"] - 1)
    if c["page"]:
        rows = s["seq"].long()
        k, v = _gathered(s, rows, s["most"])
        length = s["len"][rows].long()
    else:
        k, v = (x[index].float().transpose(1, 2) for x in (s["k"], s["v"]))
        length = count
    q = s["q"][index].float().reshape(n, s["most_new"], c["kv_heads"], group, c["dim"]).permute(0, 2, 3, 1, 4).reshape(n, c["kv_heads"], group * s["most_new"], c["dim"])
    last = (length - count)[:, None] + lane  # the last key that a row may see
    at = torch.arange(k.shape[2], device="cuda")
    allowed = (at <= last[..., None]) & ((at > last[..., None] - c["window"]) if c["window"] else True)
    out = _attend(q, k, v, allowed.repeat(1, group, 1)[:, None], s["scale"])
    out = out.reshape(n, c["kv_heads"], group, s["most_new"], c["dim"]).permute(0, 3, 1, 2, 4).reshape(n, s["most_new"], c["heads"], c["dim"])
    r = torch.arange(s["rows"], device="cuda")
    e = torch.searchsorted(cu, r, right=True) - 1
    s["out"][: s["rows"]] = out[e, r - cu[e]].to(s["out"].dtype)
    return s["out"]


def _held(s):
    return {"k": s["k"], "v": s["v"], "table": s["table"], "len": s["len"], "ref": s["ref"]}


def _count(ref, pages, by):
    ref.index_add_(0, pages.clamp_min(0).reshape(-1), torch.where(pages >= 0, by, 0).to(torch.int32).reshape(-1))


def _plain_append(s):
    page, seq, cu = s["case"]["page"], s["seq"].long(), s["cu"].long()
    table, length, ref = s["table"], s["len"], s["ref"]
    column = torch.arange(table.shape[1], device="cuda")
    # pages behind the kept length go
    keep = torch.minimum(s["keep"], length[seq]).long()
    held = table[seq].long()
    gone = column >= ((keep + page - 1) // page)[:, None]
    _count(ref, torch.where(gone, held, -1), -1)
    held = torch.where(gone, -1, held)
    # pages for the new rows, lowest free ones first; a last page that other rows hold too is copied first
    new = cu[1:] - cu[:-1]
    first, end = (keep + page - 1) // page, (keep + new + page - 1) // page
    last = held.gather(1, (first - 1).clamp_min(0)[:, None])[:, 0]
    copied = (keep % page > 0) & (new > 0) & (ref[last.clamp_min(0)] > 1)
    fresh = (column >= (first - copied.long())[:, None]) & (column < end[:, None])
    free = torch.sort((ref != 0).int(), stable=True).indices
    rank = fresh.reshape(-1).long().cumsum(0).reshape(fresh.shape) - 1
    taken = torch.where(fresh, free[rank.clamp(0, free.numel() - 1)], held)
    _count(ref, torch.where(copied, last, -1), -1)
    _count(ref, torch.where(fresh, taken, -1), 1)
    table[seq] = taken.to(torch.int32)
    length[seq] = (keep + new).to(torch.int32)
    to = taken.gather(1, (first - 1).clamp_min(0)[:, None])[:, 0]
    row = torch.arange(s["rows"], device="cuda")
    entry = torch.searchsorted(cu, row, right=True) - 1
    at = keep[entry] + row - cu[entry]
    where, slot = taken[entry, at // page], at % page
    inside = copied[:, None] & (torch.arange(page, device="cuda") < (keep % page)[:, None])
    for pool, rows in ((s["k"], s["nk"]), (s["v"], s["nv"])):
        pool[to.clamp_min(0)] = torch.where(inside[:, None, :, None], pool[last.clamp_min(0)], pool[to.clamp_min(0)])
        pool[where, :, slot] = rows.to(pool.dtype)
    return _held(s)


def _plain_fork(s):
    src, dst = s["src"].long(), s["dst"].long()
    _count(s["ref"], s["table"][dst].long(), -1)
    s["table"][dst] = s["table"][src]
    s["len"][dst] = s["len"][src]
    _count(s["ref"], s["table"][dst].long(), 1)
    return {"table": s["table"], "len": s["len"], "ref": s["ref"]}


def _plain_compact(s):
    used = s["ref"] > 0
    rank = used.long().cumsum(0) - 1
    pages = torch.sort((~used).int(), stable=True).indices[: s["k2"].shape[0]]
    s["k2"].copy_(s["k"][pages])
    s["v2"].copy_(s["v"][pages])
    s["ref2"].copy_(s["ref"][pages])
    s["table2"].copy_(torch.where(s["table"] >= 0, rank[s["table"].clamp_min(0).long()], -1))
    s["len2"].copy_(s["len"])
    return {"k": s["k2"], "v": s["v2"], "table": s["table2"], "len": s["len2"], "ref": s["ref2"]}


# ---- the framework's calls --------------------------------------------------------------------------------------------------------------------


_context = None


def _framework():
    global _context
    import __graft_entry__

    __graft_entry__.load_package()
    from whisper_cpp_amd import kernels_api as ka

    if _context is None:
        _context = ka.Ctx(0)
    return ka, _context


def _cache(ka, s, k, v, table, length, ref):
    work = torch.empty(ka.kv_work_bytes(table.shape[0], ref.numel()), dtype=torch.uint8, device="cuda")
    s["memory"].append(work)
    return ka.kv_cache(k, v, table, length, ref, s["status"], work)


def _plan(s):
    """What a program keeps between calls: the context, the cache's description and the operators' arguments."""
    ka, ctx = _framework()
    c = s["case"]
    cache = _cache(ka, s, s["k"], s["v"], s["table"], s["len"], s["ref"]) if c["page"] else None
    if s["op"] == "paged":
        work = torch.empty(ka.attn_paged_work_bytes(cache, s["n"], c["heads"], s["most"]), dtype=torch.uint8, device="cuda")
        s["memory"].append(work)
        return ctx.attn_paged_call(cache, s["q"], s["out"], seq=s["seq"], scale=s["scale"], window=c["window"], max_len=s["most"], work=work)
    if s["op"] == "packed":
        if c["page"]:
            return ctx.attn_packed_call(s["q"], s["out"], s["cu"], cache=cache, seq=s["seq"], scale=s["scale"], causal=True, window=c["window"], max_q=s["most_new"])
        return ctx.attn_packed_call(s["q"], s["out"], s["cu"], k=s["k"], v=s["v"], scale=s["scale"], causal=True, window=c["window"], max_q=s["most_new"])
    if s["op"] == "append":
        back, add = ctx.kv_truncate_call(cache, s["seq"], s["keep"]), ctx.kv_append_call(cache, s["seq"], s["cu"], s["nk"], s["nv"])
        return back, add
    if s["op"] == "fork":
        return ctx.kv_fork_call(cache, s["src"], s["dst"])
    return ctx.kv_compact_call(cache, _cache(ka, s, s["k2"], s["v2"], s["table2"], s["len2"], s["ref2"]))


def _own(s):
    op = s["op"]
    if op == "append":
        s["call"][0]()
        s["call"][1]()
        return _held(s)
    s["call"]()
    if op in ("paged", "packed"):
        return s["out"]
    if op == "fork":
        return {"table": s["table"], "len": s["len"], "ref": s["ref"]}
    return {"k": s["k2"], "v": s["v2"], "table": s["table2"], "len": s["len2"], "ref": s["ref2"]}


def run(state):
    if own:
        return _own(state)
    return {"paged": _plain_paged, "packed": _plain_packed, "append": _plain_append, "fork": _plain_fork, "compact": _plain_compact}[state["op"]](state)


def work(case):
    old, new = _shape(case)
    size = {"f32": 4, "f16": 2, "bf16": 2}
    row = 2 * case["kv_heads"] * case["dim"] * size[case["type"]]  # a key and its value
    if case["op"] == "paged":
        seen = sum(min(x, case["window"]) if case["window"] else x for x in old)
        return {"bytes": seen * row + 2 * case["n"] * case["heads"] * case["dim"] * size[case["io"]], "flops": 4 * seen * case["heads"] * case["dim"]}
    if case["op"] == "packed":
        span = lambda a, b: sum(min(a + i + 1, case["window"] or a + i + 1) for i in range(b))  # noqa: E731
        keys = sum(min(a + b, (case["window"] or a + b) + b - 1) for a, b in zip(old, new))
        return {"bytes": keys * row + 2 * sum(new) * case["heads"] * case["dim"] * size[case["io"]], "flops": 4 * case["heads"] * case["dim"] * sum(map(span, old, new))}
    if case["op"] == "append":
        return {"bytes": sum(new) * (row + 2 * case["kv_heads"] * case["dim"] * size[case["io"]]), "flops": 0}
    if case["op"] == "fork":
        return {"bytes": 4 * 5 * sum(_pages(x, case["page"]) for x in old[: case["n"] // 2]), "flops": 0}
    return {"bytes": 2 * row * case["page"] * sum(_pages(x, case["page"]) for i, x in enumerate(old) if i % 4 != 3), "flops": 0}


# ---- the definition, in 64 bits ---------------------------------------------------------------------------------------------------------------


def _exact_rows(q, k, v, see, scale):
    """One head's rows q [rows, dim] over keys [keys, dim]; `see` [rows, keys]."""
    x = (q @ k.T) * scale
    x = torch.where(see, x, -math.inf)
    top = x.max(1, keepdim=True).values
    w = torch.where(see, torch.exp(x - torch.where(torch.isinf(top), 0.0, top)), 0.0)
    z = w.sum(1, keepdim=True)
    return torch.where(z > 0, (w @ v) / torch.where(z > 0, z, 1.0), 0.0)


def exact(case, seed):
    global own
    mine, own = own, False  # the inputs alone, without a plan
    try:
        s = prepare(case, seed)
    finally:
        own = mine
    op, n, page = case["op"], case["n"], case["page"]
    table, length, ref = (s[x].cpu().numpy().copy() if x in s else None for x in ("table", "len", "ref"))
    if op in ("paged", "packed"):
        out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
        cu, group = (s["cu"].tolist() if op == "packed" else list(range(n + 1))), case["heads"] // case["kv_heads"]
        for i in range(n):
            a, b = cu[i], cu[i + 1]
            if page:
                r = int(s["seq"][i])
                keys = int(length[r])
                pages = torch.from_numpy(table[r][: _pages(keys, page)].astype(np.int64)).cuda()
            else:
                keys = b - a
            here, rows = torch.arange(keys, device="cuda"), torch.arange(b - a, device="cuda")[:, None] + keys - (b - a)
            see = here <= rows
            if case["window"]:
                see &= here > rows - case["window"]
            for h in range(case["kv_heads"]):
                if page:
                    k, v = (x[pages, h].reshape(-1, case["dim"])[:keys].double() for x in (s["k"], s["v"]))
                else:
                    k, v = (x[a:b, h].double() for x in (s["k"], s["v"]))
                for g in range(h * group, (h + 1) * group):
                    out[a:b, g] = _exact_rows(s["q"][a:b, g].double(), k, v, see, s["scale"])
        return out
    if op == "fork":
        before = table.copy(), length.copy()
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            table[b], length[b] = before[0][a], before[1][a]
        return {"table": _ints(table), "len": _ints(length), "ref": _ints(np.bincount(table[table >= 0], minlength=ref.size))}
    if op == "compact":
        pages = np.flatnonzero(ref)
        name = {int(p): i for i, p in enumerate(pages)}
        moved = np.array([[name.get(int(p), -1) for p in row] for row in table], dtype=np.int32)
        return {"k": s["k"][torch.from_numpy(pages).cuda()].double(), "v": s["v"][torch.from_numpy(pages).cuda()].double(), "table": _ints(moved), "len": _ints(length), "ref": _ints(ref[pages])}
    pools, cu = [s["k"].double(), s["v"].double()], s["cu"].tolist()
    free, was = [int(p) for p in np.flatnonzero(ref == 0)], ref.copy()
    for i in range(n):  # the free pages of the start are handed out in the sequences' order
        a, b, keys = cu[i], cu[i + 1], int(length[i])
        if keys % page and was[table[i][keys // page]] > 1 and b > a:
            p = free.pop(0)
            for pool in pools:
                pool[p, :, : keys % page] = pool[table[i][keys // page], :, : keys % page]
            ref[table[i][keys // page]] -= 1
            table[i][keys // page], ref[p] = p, 1
        for j in range(_pages(keys, page), _pages(keys + b - a, page)):
            table[i][j] = free.pop(0)
            ref[table[i][j]] += 1
        at = np.arange(keys, keys + b - a)
        where, slot = torch.from_numpy(table[i][at // page].astype(np.int64)).cuda(), torch.from_numpy(at % page).cuda()
        for pool, rows in zip(pools, (s["nk"], s["nv"])):
            pool[where, :, slot] = rows[a:b].double()
        length[i] = keys + b - a
    return {"k": pools[0], "v": pools[1], "table": _ints(table), "len": _ints(length), "ref": _ints(ref)}
