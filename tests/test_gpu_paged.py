"""The paged K/V cache, attention of one token over it and attention of packed prompts (mi355x_kv_*, mi355x_attn_paged, mi355x_attn_packed), through the C ABI.

The cache's bookkeeping is compared exactly with a restatement in plain Python; the attentions with the definition in 64 bits.  Tolerances are worst-case
bounds from the inputs of each case, with u(t) half a step of type t (f16 2^-11, bf16 2^-8, f32 2^-24):
  * a score is a sum of D products in F32: off by at most e = (D + 8) * 2^-24 * scale * max_j sum_d |q_d k_jd| (and, where q is rounded to the cache's
    type first, by u(cache) * scale * max_j sum_d |q_d k_jd| more), so a weight by the factor exp(2 e) (its own score and the maximum's), which in
    the quotient counts twice: expm1(4 e);
  * a weight rounded to the cache's type is off by u(cache); exp2 and the sums of L weights and products in F32 by (L + 32) * 2^-24 at most;
  * all of these scale values of at most max|v|; the result is rounded to its own type: u(out) * |o|."""
import ctypes as C
import math
import random

import numpy as np
import pytest

from conftest import has_gpu

pytestmark = pytest.mark.gpu

U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


@pytest.fixture(scope="module")
def gpu():
    import torch
    assert torch.cuda.is_available(), "these tests need an MI355X"
    from whisper_cpp_amd import kernels_api as ka
    ctx = ka.Ctx(0)
    yield ctx, ka, torch
    ctx.close()


def dt(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


class Pool:
    """A cache on the GPU and its restatement: lists of page numbers, and the keys that each sequence should hold"""

    def __init__(self, gpu, n_seq=6, n_pages=40, max_pages=12, page=16, heads=2, dim=64, kind="f16", order="head", seed=0, fill=float("nan")):
        self.ctx, self.ka, self.torch = gpu
        torch = self.torch
        self.page, self.heads, self.dim, self.kind, self.n_pages, self.max_pages = page, heads, dim, kind, n_pages, max_pages
        shape = (n_pages, heads, page, dim) if order == "head" else (n_pages, page, heads, dim)
        pool = [torch.full(shape, fill, dtype=dt(torch, kind), device="cuda") for _ in range(2)]      # memory that nothing has been written to yet: NaN
        self.k, self.v = pool if order == "head" else [x.transpose(1, 2) for x in pool]
        self.table = torch.full((n_seq, max_pages), 77, dtype=torch.int32, device="cuda")
        self.len, self.ref = torch.full((n_seq,), 5, dtype=torch.int32, device="cuda"), torch.full((n_pages,), 9, dtype=torch.int32, device="cuda")
        self.status = torch.full((1,), 64, dtype=torch.int32, device="cuda")
        self.work = torch.empty(self.ka.kv_work_bytes(n_seq, n_pages), dtype=torch.uint8, device="cuda")
        self.c = self.ka.kv_cache(self.k, self.v, self.table, self.len, self.ref, self.status, self.work)
        torch.cuda.synchronize()
        self.run(self.ctx.kv_reset_call(self.c))
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        # the restatement
        self.rows, self.count = [[] for _ in range(n_seq)], [0] * n_pages
        self.keys = [[] for _ in range(n_seq)]                       # of each sequence, key by key: (page written to, k, v) in 64 bits
        self.content = {}                                            # (page, slot) -> (k [heads, dim], v), on the CPU in the cache's type

    def run(self, call):
        self.torch.cuda.synchronize()
        call()
        self.ctx.sync()

    def ints(self, values):
        return self.torch.tensor(values, dtype=self.torch.int32, device="cuda")

    def append(self, entries, kind="f32", pad=0, layout="plain"):
        """entries: [(sequence, rows)]; returns what the restatement expects of the status"""
        torch = self.torch
        n = sum(r for _, r in entries) + pad
        k, v = (torch.randn(n, self.heads, self.dim, generator=self.gen, device="cuda").to(dt(torch, kind)) for _ in range(2))
        if layout == "wide":                                         # rows of a larger projection: heads apart, rows further apart
            k, v = (torch.cat([x, x], 2).repeat(1, 2, 1)[:, : self.heads, : self.dim] for x in (k, v))
        cu = np.concatenate([[0], np.cumsum([r for _, r in entries])])
        self.run(self.ctx.kv_append_call(self.c, self.ints([s for s, _ in entries]), self.ints(cu.tolist()), k, v))
        return self._append(entries, k.to(dt(torch, self.kind)).cpu(), v.to(dt(torch, self.kind)).cpu(), cu)

    def _append(self, entries, k, v, cu):
        page, free, taken, todo = self.page, [p for p in range(self.n_pages) if self.count[p] == 0], 0, []
        live = [s for s, _ in entries if s >= 0]
        if any(s >= len(self.rows) for s in live) or len(set(live)) < len(live):
            return self.ka.KV_BAD_ARG
        for (s, r) in entries:
            if s >= 0 and (len(self.keys[s]) + r) > self.max_pages * page:
                return self.ka.KV_ROW_FULL
        for i, (s, r) in enumerate(entries):
            if s < 0:
                continue
            old = len(self.keys[s])
            copy = r > 0 and old % page > 0 and self.count[self.rows[s][-1]] > 1
            new = -(-(old + r) // page) - -(-old // page)
            todo.append((i, s, r, old, copy, free[taken : taken + new + copy]))
            taken += new + copy
        if taken > len(free):
            return self.ka.KV_OUT_OF_PAGES
        for i, s, r, old, copy, pages in todo:
            if copy:
                was, now = self.rows[s][-1], pages.pop(0)
                for j in range(old % page):
                    self.content[now, j] = self.content[was, j]
                self.count[was] -= 1
                self.count[now] = 1
                self.rows[s][-1] = now
            for p in pages:
                self.rows[s].append(p)
                self.count[p] = 1
            for j in range(r):
                x = (k[cu[i] + j], v[cu[i] + j])
                self.content[self.rows[s][(old + j) // page], (old + j) % page] = x
                self.keys[s].append(x)
        return 0

    def truncate(self, entries):
        self.run(self.ctx.kv_truncate_call(self.c, self.ints([s for s, _ in entries]), self.ints([x for _, x in entries])))
        for s, keep in entries:
            if 0 <= s < len(self.rows) and keep >= 0:
                self.keys[s] = self.keys[s][:keep]
                for p in self.rows[s][-(-len(self.keys[s]) // self.page) :]:
                    self.count[p] -= 1
                self.rows[s] = self.rows[s][: -(-len(self.keys[s]) // self.page)]

    def fork(self, pairs):
        self.run(self.ctx.kv_fork_call(self.c, self.ints([s for s, _ in pairs]), self.ints([d for _, d in pairs])))
        before = [list(r) for r in self.rows], [list(x) for x in self.keys]
        for s, d in pairs:
            if d >= 0:
                self.rows[d], self.keys[d] = (list(before[0][s]), list(before[1][s])) if s >= 0 else ([], [])
        self.count = [sum(p in r for r in self.rows) for p in range(self.n_pages)]

    def check(self, status=0, contents=True):
        torch = self.torch
        torch.cuda.synchronize()
        want = [r + [-1] * (self.max_pages - len(r)) for r in self.rows]
        assert int(self.status) == status
        assert self.len.tolist() == [len(x) for x in self.keys]
        assert self.table.tolist() == want
        assert self.ref.tolist() == self.count
        if contents:                                                 # every key where it belongs, and nothing anywhere else
            for pool, which in ((self.k, 0), (self.v, 1)):
                got = pool.cpu()
                held = torch.zeros(self.n_pages, self.page, dtype=torch.bool)
                for s, x in enumerate(self.keys):
                    for j, kv in enumerate(x):
                        p, slot = self.rows[s][j // self.page], j % self.page
                        held[p, slot] = True
                        assert torch.equal(got[p, :, slot], kv[which]), (s, j)
                written = torch.zeros_like(held)
                for p, slot in self.content:
                    written[p, slot] = True
                assert got.transpose(1, 2)[~written].isnan().all()   # slots that no call named are as they were
        self.status.zero_()


# ---- the cache ----------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("kind,io,order,dim,heads,page", [("f16", "f32", "head", 64, 3, 16), ("bf16", "f32", "key", 128, 2, 8), ("f16", "f16", "key", 64, 5, 1),
                                                          ("bf16", "bf16", "head", 128, 1, 64), ("f16", "bf16", "head", 64, 2, 4), ("bf16", "f16", "key", 64, 20, 32)])
def test_append_truncate_and_fork_keep_table_counts_and_keys_as_restated(gpu, kind, io, order, dim, heads, page):
    p = Pool(gpu, page=page, heads=heads, dim=dim, kind=kind, order=order)
    p.check()
    assert p.append([(0, 3 * page - 1), (2, 0), (4, 1)], io) == 0
    p.check()
    assert p.append([(4, 2), (-1, 5), (1, page), (0, 2)], io, pad=3, layout="wide") == 0       # a row of padding, rows behind the last entry, a strided input
    p.check()
    p.fork([(0, 3), (4, 5), (4, 2), (-1, 1)])                        # shared pages; row 1 emptied
    p.check()
    assert p.append([(3, 1), (0, 2), (5, 1)], io) == 0               # sequences that share a partly filled page go their own ways
    p.check()
    p.fork([(3, 0), (0, 3), (2, 2), (5, -1)])                        # rows change places; one onto itself
    p.check()
    p.truncate([(0, page + 1), (3, 0), (5, 100), (-1, 0)])
    p.check()
    p.truncate([(0, 3), (0, 1), (0, 2)])                             # one sequence three times: the smallest holds
    p.check()
    assert p.append([(3, 2 * page + 1), (0, page)], io) == 0         # pages given back are taken again, lowest first
    p.check()


def test_many_rows_and_many_sequences_at_once(gpu):
    rng = random.Random(3)
    n = 1500                                                         # more entries than threads of the workgroup that hands pages out
    p = Pool(gpu, n_seq=n, n_pages=9000, max_pages=5, page=4, heads=1, dim=64)
    order = rng.sample(range(n), n)
    assert p.append([(s, rng.randint(0, 9)) for s in order], "f16") == 0
    p.check(contents=False)
    pairs = [(s, d) for s, d in zip(rng.sample(range(n), n), rng.sample(range(n), n))]
    p.fork(pairs)
    p.check(contents=False)
    assert p.append([(s, rng.randint(0, 5)) for s in order], "f16") == 0
    p.check()


def test_a_call_that_cannot_be_done_says_why_and_changes_nothing(gpu):
    ctx, ka, torch = gpu
    p = Pool(gpu, n_pages=10, max_pages=6, page=4)
    assert p.append([(0, 9), (1, 4)]) == 0
    p.check()
    assert p.append([(2, 1), (3, 24)]) == ka.KV_OUT_OF_PAGES         # 4 pages are held, 7 more wanted, 6 free: not even entry 0 is done
    p.check(ka.KV_OUT_OF_PAGES)
    assert p.append([(2, 1), (0, 16)]) == ka.KV_ROW_FULL
    p.check(ka.KV_ROW_FULL)
    assert p.append([(2, 1), (2, 1)]) == ka.KV_BAD_ARG
    p.check(ka.KV_BAD_ARG)
    assert p.append([(2, 1), (6, 1)]) == ka.KV_BAD_ARG
    p.check(ka.KV_BAD_ARG)
    k = torch.randn(4, 2, 64, device="cuda")
    for cu in ([0, 3, 2], [0, 2, 5], [-1, 1, 2]):                    # offsets that fall, leave the rows, start before them
        p.run(ctx.kv_append_call(p.c, p.ints([2, 3]), p.ints(cu), k, k))
        p.check(ka.KV_BAD_ARG)
    for src, dst in (([0, 1], [2, 2]), ([0, 6], [2, 3]), ([0, 1], [2, 6])):
        p.run(ctx.kv_fork_call(p.c, p.ints(src), p.ints(dst)))
        p.check(ka.KV_BAD_ARG)
    p.run(ctx.kv_truncate_call(p.c, p.ints([6, 0]), p.ints([0, -1])))
    p.check(ka.KV_BAD_ARG)
    assert p.append([(2, 24)]) == 0                                  # the last free page is used up ...
    p.check()
    assert p.append([(0, 0), (1, 0)]) == 0                           # ... and calls without a need go on working
    p.check()


@pytest.mark.parametrize("order,order2,dim,page", [("head", "head", 64, 16), ("key", "head", 128, 4), ("head", "key", 64, 1)])
def test_compact_moves_the_held_pages_and_renames_them(gpu, order, order2, dim, page):
    ctx, ka, torch = gpu
    p = Pool(gpu, n_pages=60, page=page, dim=dim, order=order, heads=3)
    for i in range(3):
        assert p.append([(s, 2 * page - s % 2) for s in range(6)]) == 0
        p.truncate([(i, 0)])
    p.fork([(4, 0), (5, 1)])
    assert p.append([(0, 1), (4, 1)]) == 0
    p.check()
    used = [x for x in range(60) if p.count[x]]
    for n_pages, wide in ((len(used), 0), (len(used) + 7, 3), (len(used) - 1, 0)):
        q = Pool(gpu, n_pages=n_pages, max_pages=12 + wide, page=page, dim=dim, order=order2, heads=3)
        p.run(ctx.kv_compact_call(p.c, q.c))
        p.check()                                                    # the old cache is as it was
        if n_pages < len(used):
            q.check(ka.KV_OUT_OF_PAGES)                              # the new one too, and says why
            continue
        name = {x: i for i, x in enumerate(used)}
        q.rows, q.keys = [[name[x] for x in r] for r in p.rows], [list(x) for x in p.keys]
        q.count = [p.count[x] for x in used] + [0] * (n_pages - len(used))
        q.content = {(i, j): None for i in range(len(used)) for j in range(page)}            # whole pages move, unused slots among them
        q.check()
        full = 0 if n_pages > len(used) else ka.KV_OUT_OF_PAGES
        assert q.append([(2, 1), (0, 2)]) == full                    # and it is a cache to go on with, if it has room
        q.check(full)


@pytest.mark.parametrize("n_pages,page,heads,dim", [(4500, 1, 1, 64), (2048, 1, 2, 128), (2049, 2, 1, 64), (40, 64, 20, 128)])
def test_compact_of_many_pages_or_large_ones(gpu, n_pages, page, heads, dim):
    """on both sides of the sizes from which the ranks have a launch of their own"""
    ctx, ka, torch = gpu
    p = Pool(gpu, n_seq=3, n_pages=n_pages, max_pages=n_pages // 2, page=page, heads=heads, dim=dim)
    third = n_pages // 3 * page
    assert p.append([(0, third), (1, third - 1), (2, third // 2)]) == 0
    p.truncate([(0, third // 3), (1, 0)])
    assert p.append([(1, third // 4)]) == 0
    used = [x for x in range(n_pages) if p.count[x]]
    name = {x: i for i, x in enumerate(used)}
    for room in (len(used), len(used) + 300):
        q = Pool(gpu, n_seq=3, n_pages=room, max_pages=n_pages // 2 + 1, page=page, heads=heads, dim=dim)
        p.run(ctx.kv_compact_call(p.c, q.c))
        q.rows, q.keys = [[name[x] for x in r] for r in p.rows], [list(x) for x in p.keys]
        q.count = [p.count[x] for x in used] + [0] * (room - len(used))
        q.content = {(i, j): None for i in range(len(used)) for j in range(page)}
        q.check()


# ---- attention ----------------------------------------------------------------------------------------------------------------


def expect(torch, q, k, v, see, scale, kind, q_kind, out_kind, round_q, round_w):
    """(64-bit result, allowed error) of rows q [H, D] over k, v [L, Hkv, D]; see [L]"""
    H, D = q.shape
    G = H // k.shape[1]
    q, k, v = q.double(), k.double()[see], v.double()[see]
    if len(k) == 0:
        return torch.zeros(H, D, dtype=torch.float64), torch.zeros(H, D, dtype=torch.float64)
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)      # [L, H, D]
    x = torch.einsum("hd,lhd->hl", q, k) * scale
    w = torch.softmax(x, 1)
    o = torch.einsum("hl,lhd->hd", w, v)
    size = (torch.einsum("hd,lhd->hl", q.abs(), k.abs()) * abs(scale)).amax(1)
    e = size * ((D + 8) * U["f32"] + (U[kind] if round_q else 0.0))
    per = torch.expm1(4 * e) + (2 * U[kind] if round_w else 0.0) + (len(k) + 32) * U["f32"]
    return o, per[:, None] * v.abs().amax(0) .amax(-1, keepdim=True) + U[out_kind] * o.abs() + 1e-30


def same(torch, got, o, tol):
    got = got.double().cpu()
    for f in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(f(got), f(o)), (f.__name__, int(f(got).sum()), int(f(o).sum()), o.numel())
    fine = o.isfinite()
    off = ((got - o).abs() - tol)[fine]
    assert off.numel() == 0 or float(off.max()) <= 0, (float((got - o).abs()[fine].max()), float(off.max()))


LENGTHS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 255, 257, 300]


@pytest.mark.parametrize("kind,q_kind,out_kind", [("f16", "f32", "f32"), ("bf16", "f32", "f32"), ("f16", "f16", "f16"), ("bf16", "bf16", "bf16"), ("bf16", "f16", "f32"), ("f16", "f16", "bf16")])
@pytest.mark.parametrize("dim,kv_heads,heads,page,order,window", [(64, 2, 2, 16, "head", 0), (128, 2, 8, 32, "key", 0), (64, 1, 7, 1, "key", 40), (128, 1, 20, 8, "head", 33), (64, 3, 48, 64, "head", 1),
                                                                  (128, 4, 4, 128, "key", 500)])
def test_attention_of_one_token(gpu, kind, q_kind, out_kind, dim, kv_heads, heads, page, order, window):
    """every length around tile, page and window borders, an order of sequences of the caller's, an entry of -1, pages with NaN behind the sequences' ends"""
    ctx, ka, torch = gpu
    rng = random.Random(dim + heads + page)
    need = sum(-(-x // page) for x in LENGTHS) + 5
    p = Pool(gpu, n_seq=len(LENGTHS), n_pages=need, max_pages=-(-300 // page), page=page, heads=kv_heads, dim=dim, kind=kind, order=order)
    lens = list(LENGTHS)
    rng.shuffle(lens)
    assert p.append([(s, x) for s, x in enumerate(lens)], kind) == 0
    seq = rng.sample(range(len(lens)), len(lens)) + [-1, 3]
    gen = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(len(seq), heads, dim, generator=gen, device="cuda").mul_(2).to(dt(torch, q_kind))
    scale = 1 / math.sqrt(dim)
    for max_len in (0, 300, 1):                                      # what the caller says of the lengths never changes what is computed
        out = torch.full((len(seq), heads, dim), 7.0, device="cuda").to(dt(torch, out_kind))
        work = torch.empty(max(16, ka.attn_paged_work_bytes(p.c, len(seq), heads, max_len)), dtype=torch.uint8, device="cuda")
        p.run(ctx.attn_paged_call(p.c, q, out, seq=p.ints(seq), scale=scale, window=window, max_len=max_len, work=work))
        p.check(contents=False)
        for i, s in enumerate(seq):
            keys = p.keys[s] if s >= 0 else []
            k, v = (torch.stack([x[w] for x in keys]) if keys else torch.zeros(0, kv_heads, dim) for w in (0, 1))
            see = torch.arange(len(keys)) >= (len(keys) - window if window else 0)
            o, tol = expect(torch, q[i].cpu(), k, v, see, scale, kind, q_kind, out_kind, False, q_kind == kind)
            same(torch, out[i], o, tol)


@pytest.mark.parametrize("n,length,kv_heads,heads,dim,kind", [(1, 5003, 1, 1, 64, "f16"), (2, 40001, 2, 8, 128, "bf16"), (5, 3001, 8, 64, 128, "f16")])
def test_attention_of_one_token_split_over_a_long_cache_and_joined(gpu, n, length, kv_heads, heads, dim, kind):
    ctx, ka, torch = gpu
    page, gen = 32, torch.Generator(device="cuda").manual_seed(4)
    lens = [length, 0, 1, length // 2, 700][:n]
    held = [-(-x // page) for x in lens]
    k, v = (torch.randn(sum(held), kv_heads, page, dim, generator=gen, device="cuda").to(dt(torch, kind)) for _ in range(2))
    pages = torch.randperm(sum(held), generator=torch.Generator().manual_seed(1)).int()
    table = torch.full((n, max(held)), -1, dtype=torch.int32)
    at = 0
    for s, h in enumerate(held):
        table[s, :h] = pages[at : at + h]
        at += h
    zero = lambda m: torch.zeros(m, dtype=torch.int32, device="cuda")  # noqa: E731
    work, status, dtab, dlen, ref = torch.empty(ka.kv_work_bytes(n, sum(held)), dtype=torch.uint8, device="cuda"), zero(1), table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), zero(sum(held))
    c = ka.kv_cache(k, v, dtab, dlen, ref, status, work)
    q = torch.randn(n, heads, dim, generator=gen, device="cuda")
    q[0] *= 6                                                        # a few keys far above the others: weights over many powers of two
    scale, rows = 1 / math.sqrt(dim), []
    space = torch.empty(ka.attn_paged_work_bytes(c, n, heads, length), dtype=torch.uint8, device="cuda")
    assert space.numel() > 0
    for rep in range(2):
        out = torch.full_like(q, 3.0)
        torch.cuda.synchronize()
        ctx.attn_paged_call(c, q, out, scale=scale, max_len=length, work=space)()
        ctx.sync()
        rows.append(out)
    assert torch.equal(rows[0], rows[1])                             # nothing depends on which share ends first
    for s in range(n):
        flat = [x.cpu()[table[s, : held[s]].long()].transpose(1, 2).reshape(-1, kv_heads, dim)[: lens[s]] for x in (k, v)]
        o, tol = expect(torch, q[s].cpu(), *flat, torch.ones(lens[s], dtype=torch.bool), scale, kind, "f32", "f32", False, False)
        same(torch, rows[0][s], o, tol)


@pytest.mark.parametrize("kind,q_kind,dim,kv_heads,heads,page,window", [("f16", "f16", 64, 1, 3, 16, 0), ("bf16", "f32", 128, 2, 4, 64, 0), ("bf16", "bf16", 128, 1, 17, 8, 700)])
def test_many_queries_of_very_different_lengths_share_the_runs_of_the_split(gpu, kind, q_kind, dim, kv_heads, heads, page, window):
    """hundreds of queries, most of them short, some empty or left out, a few long: runs that hold several, that begin and end inside one"""
    ctx, ka, torch = gpu
    rng, gen, n = random.Random(7), torch.Generator(device="cuda").manual_seed(4), 200
    lens = [rng.choice((0, 1, 5, 31, 32, 33, 100, 300)) for _ in range(n)]
    for i, x in zip(rng.sample(range(n), 5), (2900, 4100, 1500, 1025, 4097)):
        lens[i] = x
    held = [-(-x // page) for x in lens]
    k, v = (torch.randn(sum(held), kv_heads, page, dim, generator=gen, device="cuda").to(dt(torch, kind)) for _ in range(2))
    table, at = torch.full((n, max(held)), -1, dtype=torch.int32), 0
    for s, h in enumerate(held):
        table[s, :h] = torch.arange(at, at + h)
        at += h
    zero = lambda m: torch.zeros(m, dtype=torch.int32, device="cuda")  # noqa: E731
    work, status, dtab, dlen, ref = torch.empty(ka.kv_work_bytes(n, sum(held)), dtype=torch.uint8, device="cuda"), zero(1), table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), zero(sum(held))
    c = ka.kv_cache(k, v, dtab, dlen, ref, status, work)
    seq = rng.sample(range(n), n) + [-1, 0, 0, n + 5]
    q = torch.randn(len(seq), heads, dim, generator=gen, device="cuda").to(dt(torch, q_kind))
    out, space, scale = torch.full_like(q, 3.0), torch.full((ka.attn_paged_work_bytes(c, len(seq), heads),), 255, dtype=torch.uint8, device="cuda"), 1 / math.sqrt(dim)
    assert space.numel() > 0
    dseq = torch.tensor(seq, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    ctx.attn_paged_call(c, q, out, seq=dseq, scale=scale, window=window, work=space)()
    ctx.sync()
    assert int(status) == 0
    for i in sorted(rng.sample(range(len(seq)), 60) + [j for j, s in enumerate(seq) if not 0 <= s < n or lens[s] > 1000]):
        s = seq[i] if 0 <= seq[i] < n else None
        L = lens[s] if s is not None else 0
        flat = [x.cpu()[table[s, : held[s]].long()].transpose(1, 2).reshape(-1, kv_heads, dim)[:L] if L else torch.zeros(0, kv_heads, dim) for x in (k, v)]
        o, tol = expect(torch, q[i].cpu(), *flat, torch.arange(L) >= (L - window if window else 0), scale, kind, q_kind, q_kind, False, q_kind == kind)
        same(torch, out[i], o, tol)


def packed_case(gpu, kind, q_kind, out_kind, dim, kv_heads, heads, q_lens, k_lens=None, window=0, causal=True, page=0, order="head", spoil=None, max_q=0, scale=None):
    """one call of the packed attention over rows of its own (page 0) or over a cache, against the definition.  `spoil`: {(sequence, key): (k, v)}"""
    ctx, ka, torch = gpu
    gen, n = torch.Generator(device="cuda").manual_seed(9), len(q_lens)
    ks = k_lens or q_lens
    cu = np.concatenate([[0], np.cumsum(q_lens)]).tolist()
    scale = 1 / math.sqrt(dim) if scale is None else scale
    q = torch.randn(cu[-1] + 2, heads, dim, generator=gen, device="cuda").mul_(2).to(dt(torch, q_kind))
    out = torch.full((cu[-1] + 2, heads, dim), 7.0, device="cuda").to(dt(torch, out_kind))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    if page:
        p = Pool(gpu, n_seq=n + 1, n_pages=sum(-(-x // page) for x in ks) + 2, max_pages=max(-(-x // page) for x in ks) + 1, page=page, heads=kv_heads, dim=dim, kind=kind, order=order)
        row = random.Random(2).sample(range(n + 1), n)
        assert p.append([(row[i], ks[i]) for i in range(n)], kind) == 0
        kv = [[torch.stack([x[w] for x in p.keys[r]]) if p.keys[r] else torch.zeros(0, kv_heads, dim) for w in (0, 1)] for r in row]
        for (s, j), (a, b) in (spoil or {}).items():
            at = p.rows[row[s]][j // page], slice(None), j % page
            p.k[at], p.v[at] = a, b
            kv[s][0][j], kv[s][1][j] = a, b
        call = ctx.attn_packed_call(q, out, ints(cu), cache=p.c, seq=ints(row), scale=scale, causal=causal, window=window, max_q=max_q)
    else:
        ck = np.concatenate([[0], np.cumsum(ks)]).tolist()
        k, v = (torch.randn(ck[-1] + 1, kv_heads, 2 * dim if order == "key" else dim, generator=gen, device="cuda").to(dt(torch, kind))[..., :dim] for _ in range(2))
        for (s, j), (a, b) in (spoil or {}).items():
            k[ck[s] + j], v[ck[s] + j] = a, b
        k[ck[-1]:], v[ck[-1]:] = float("nan"), float("nan")
        kv = [[x[ck[i] : ck[i + 1]].cpu() for x in (k, v)] for i in range(n)]
        call = ctx.attn_packed_call(q, out, ints(cu), k=k, v=v, cu_k=ints(ck) if k_lens else None, scale=scale, causal=causal, window=window, max_q=max_q)
    torch.cuda.synchronize()
    call()
    ctx.sync()
    assert torch.equal(out[cu[-1] :].float(), torch.full_like(out[cu[-1] :], 7.0).float())       # rows behind the last sequence
    for i in range(n):
        L, Q = ks[i], q_lens[i]
        rows = range(Q) if Q < 40 else sorted(set(list(range(6)) + list(range(Q - 6, Q)) + random.Random(i).sample(range(Q), 12)))
        for r in rows:
            j = torch.arange(L)
            see = j <= L - Q + r if causal else j >= 0
            if window:
                see = see & (j > L - Q + r - window)
            o, tol = expect(torch, q[cu[i] + r].cpu(), kv[i][0], kv[i][1], see, scale, kind, q_kind, out_kind, q_kind != kind, True)
            try:
                same(torch, out[cu[i] + r], o, tol)
            except AssertionError as e:
                raise AssertionError(f"sequence {i} row {r} of {Q}, {L} keys: {e}")


@pytest.mark.parametrize("kind,q_kind,out_kind", [("f16", "f16", "f16"), ("bf16", "bf16", "bf16"), ("f16", "f32", "f32"), ("bf16", "f16", "f32")])
@pytest.mark.parametrize("dim,kv_heads,heads,window,order", [(64, 2, 2, 0, "head"), (128, 1, 4, 0, "key"), (64, 1, 3, 20, "head"), (128, 2, 14, 100, "head"), (64, 1, 128, 0, "head")])
def test_attention_of_packed_prompts(gpu, kind, q_kind, out_kind, dim, kv_heads, heads, window, order):
    packed_case(gpu, kind, q_kind, out_kind, dim, kv_heads, heads, [1, 0, 5, 64, 17, 130, 63, 0, 257], window=window, order=order)


@pytest.mark.parametrize("dim,kv_heads,heads,page,order,causal,window", [(64, 2, 4, 16, "head", True, 0), (128, 1, 8, 4, "key", True, 50), (128, 2, 2, 64, "head", True, 0), (64, 1, 5, 32, "key", False, 0),
                                                                         (64, 2, 2, 8, "head", False, 30)])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_attention_of_prompt_pieces_over_the_cache(gpu, kind, dim, kv_heads, heads, page, order, causal, window):
    """fewer rows than keys (the rest is the past), as many, more (the first rows see nothing), none of either"""
    packed_case(gpu, kind, kind, kind, dim, kv_heads, heads, [3, 1, 70, 9, 0, 40, 4], [200, 1, 70, 3, 33, 0, 131], page=page, order=order, causal=causal, window=window)


@pytest.mark.parametrize("page", [0, 16])
@pytest.mark.parametrize("heads,dim,q_lens,k_lens", [(128, 64, [200, 3], [200, 3]), (65, 64, [130], [190]), (128, 128, [1, 0, 0, 0], [1500, 2, 0, 30]), (96, 128, [40, 30], [300, 290])])
def test_more_heads_to_a_group_than_half_a_workgroup_has_rows(gpu, heads, dim, q_lens, k_lens, page):
    """a row tile of 64 cannot hold one query of such a group, at lengths where smaller groups would get it"""
    packed_case(gpu, "f16", "f16", "f16", dim, 1, heads, q_lens, k_lens, page=page)
    packed_case(gpu, "bf16", "f32", "f32", dim, 1, heads, q_lens, k_lens, page=page, window=100)


@pytest.mark.parametrize("max_q", [0, 1, 12, 64, 4000])
@pytest.mark.parametrize("dim,heads", [(64, 1), (128, 4)])
def test_what_the_caller_says_of_the_rows_never_changes_what_is_computed(gpu, dim, heads, max_q):
    packed_case(gpu, "f16", "f16", "f16", dim, 1, heads, [4, 1, 12, 70], [700, 1, 300, 70], max_q=max_q)
    packed_case(gpu, "f16", "f16", "f16", dim, 1, heads, [4, 1, 12, 70], [700, 1, 300, 70], max_q=max_q, page=16)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("page,max_q", [(0, 0), (16, 0), (0, 8), (16, 8)])
def test_infinities_and_nan_reach_only_the_rows_that_see_them(gpu, kind, page, max_q):
    inf, nan = float("inf"), float("nan")
    q = [100, 90] if max_q == 0 else [8, 5]
    ks = [100, 90] if max_q == 0 else [308, 290]                     # (few rows over many keys have a kernel of their own)
    late = ks[0] - 3                                                 # seen by the last three rows alone
    packed_case(gpu, kind, kind, kind, 64, 1, 2, q, ks, page=page, max_q=max_q, spoil={(0, late): (0.5, nan), (1, ks[1] - 1): (0.25, inf)})
    packed_case(gpu, kind, kind, kind, 128, 1, 1, q, ks, page=page, max_q=max_q, spoil={(0, late): (0.0, inf), (0, late + 1): (0.0, -inf), (1, ks[1] - 1): (nan, 1.0)})
    packed_case(gpu, kind, kind, kind, 64, 2, 2, q, ks, page=page, max_q=max_q, window=2, spoil={(0, late - 2): (nan, nan), (1, ks[1] - 4): (1.0, -inf)})


@pytest.mark.parametrize("kind,dim,page", [("f16", 64, 16), ("bf16", 128, 64)])
@pytest.mark.parametrize("keys,window", [(75, 0), (75, 20), (1501, 0), (1501, 1100)])
def test_infinities_in_the_first_and_last_key_of_one_token_stay_what_they_are(gpu, kind, dim, page, keys, window):
    """keys outside the span stand for none of its values, at both ends of a tile"""
    ctx, ka, torch = gpu
    p = Pool(gpu, n_seq=1, n_pages=-(-keys // page), max_pages=-(-keys // page), page=page, heads=2, dim=dim, kind=kind)
    assert p.append([(0, keys)], kind) == 0
    q = torch.randn(1, 4, dim, generator=p.gen, device="cuda").to(dt(torch, kind))
    work = torch.empty(max(16, ka.attn_paged_work_bytes(p.c, 1, 4, 0)), dtype=torch.uint8, device="cuda")
    clean, out = torch.empty(1, 4, dim, device="cuda"), torch.empty(1, 4, dim, device="cuda")
    p.run(ctx.attn_paged_call(p.c, q, clean, scale=dim ** -0.5, window=window, work=work))
    first, last = keys - window if window else 0, keys - 1
    for key, d, x in ((last, 3, float("inf")), (last, 4, float("-inf")), (first, 5, float("inf")), (first, 6, float("-inf"))):
        p.v[p.rows[0][key // page], :, key % page, d] = x
    p.run(ctx.attn_paged_call(p.c, q, out, scale=dim ** -0.5, window=window, work=work))
    assert out[..., [3, 5]].isposinf().all() and out[..., [4, 6]].isneginf().all()
    clean[..., 3:7] = out[..., 3:7] = 0.0
    assert torch.equal(out, clean)


@pytest.mark.parametrize("kind,io", [("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("dim,heads,rows,keys,max_q", [(64, 2, 1, 200, 1), (64, 2, 1, 1501, 1), (128, 2, 1, 3001, 1),              # one token: whole, split
                                                       (64, 2, 8, 1201, 8), (128, 2, 8, 1201, 8),                                 # packed: few rows
                                                       (64, 2, 8, 120, 0), (128, 2, 8, 200, 0), (64, 2, 40, 300, 0), (128, 2, 40, 300, 0), (128, 2, 100, 400, 0), (128, 16, 2200, 2300, 0)])
def test_an_infinity_stays_one_however_small_its_weight(gpu, kind, io, dim, heads, rows, keys, max_q):
    """infinities in tiles that every row sees whole, in keys whose weights are far below the smallest number of the cache's type, or of any: the exact weight is none
    of 0, so the value's infinity is the result's; a NaN and two opposite ones make a NaN; all other dims have their values"""
    ctx, ka, torch = gpu
    page = 16
    p = Pool(gpu, n_seq=1, n_pages=-(-keys // page), max_pages=-(-keys // page), page=page, heads=heads, dim=dim, kind=kind)
    assert p.append([(0, keys)], kind) == 0
    q = torch.full((rows, heads, dim), dim ** -0.5, device="cuda").to(dt(torch, io))
    scale, inf = dim ** -0.5, float("inf")
    at = lambda key: (p.rows[0][key // page], slice(None), key % page)  # noqa: E731
    p.k.mul_(0.5)
    low = [40, 41, 42, 64, 71]                                       # 60 and 400 below the others' scores (they are of about 0.5)
    for key, depth in zip(low, (60.0, 400.0, 60.0, 60.0, 400.0)):
        p.k[at(key)] = -depth / dim ** 0.5 / scale / dim ** 0.5
    top = keys - rows - 5
    p.k[at(top)] = 250.0 / dim ** 0.5 / scale / dim ** 0.5 if keys > 1000 else 0.5      # a maximum that comes late and leaves nothing of the others

    def run():
        out = torch.empty(rows, heads, dim, device="cuda")
        if max_q == 1:
            work = torch.empty(max(16, ka.attn_paged_work_bytes(p.c, 1, heads, 0)), dtype=torch.uint8, device="cuda")
            p.run(ctx.attn_paged_call(p.c, q, out, scale=scale, work=work))
            return [out]
        p.run(ctx.attn_packed_call(q, out, p.ints([0, rows]), cache=p.c, scale=scale, max_q=max_q))
        flat = [x.transpose(1, 2).reshape(-1, heads, dim)[:keys].contiguous() if p.rows[0] == list(range(len(p.rows[0]))) else None for x in (p.k, p.v)]
        out2 = torch.empty_like(out)
        p.run(ctx.attn_packed_call(q, out2, p.ints([0, rows]), k=flat[0], v=flat[1], cu_k=p.ints([0, keys]), scale=scale, max_q=max_q))
        return [out, out2]

    clean = run()
    size = float(p.v[: -(-keys // page)].float().nan_to_num(0.0).abs().max())
    for d, (a, x) in enumerate(((0, inf), (1, -inf), (1, inf), (3, -inf), (4, inf), (2, float("nan")), (0, inf), (3, inf))):
        p.v[at(low[a])][..., d] = x
    p.v[at(low[4])][..., 6] = -inf                                   # with +inf in key 40: NaN
    for out, was in zip(run(), clean):
        assert out[..., [0, 2, 4, 7]].isposinf().all() and out[..., [1, 3]].isneginf().all() and out[..., [5, 6]].isnan().all()
        assert float((out[..., 8:] - was[..., 8:]).abs().max()) <= (keys + 32) * U["f32"] * size


@pytest.mark.parametrize("kind,io", [("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("bf16", "f16")])
@pytest.mark.parametrize("dim,keys,page", [(64, 200, 16), (128, 300, 64), (64, 2501, 16), (128, 3001, 64)])
def test_infinities_of_values_under_one_token(gpu, kind, io, dim, keys, page):
    """of ordinary weights, however many terms these are split into"""
    ctx, ka, torch = gpu
    p = Pool(gpu, n_seq=1, n_pages=-(-keys // page), max_pages=-(-keys // page), page=page, heads=2, dim=dim, kind=kind)
    assert p.append([(0, keys)], kind) == 0
    q = torch.randn(1, 4, dim, generator=p.gen, device="cuda").to(dt(torch, io))
    work = torch.empty(max(16, ka.attn_paged_work_bytes(p.c, 1, 4, 0)), dtype=torch.uint8, device="cuda")
    clean, out = torch.empty(1, 4, dim, device="cuda"), torch.empty(1, 4, dim, device="cuda")
    p.run(ctx.attn_paged_call(p.c, q, clean, scale=1 / dim, work=work))
    inf = float("inf")
    for key, d, x in ((33, 3, inf), (50, 4, -inf), (70, 7, float("nan")), (90, 3, inf), (90, 9, -inf), (150, 9, inf)):
        p.v[p.rows[0][key // page], :, key % page, d] = x
    p.run(ctx.attn_paged_call(p.c, q, out, scale=1 / dim, work=work))
    assert out[..., 3].isposinf().all() and out[..., 4].isneginf().all() and out[..., [7, 9]].isnan().all()
    rest = [d for d in range(dim) if d not in (3, 4, 7, 9)]
    assert torch.equal(out[..., rest], clean[..., rest])


@pytest.mark.parametrize("kind,io", [("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("bf16", "f16")])
@pytest.mark.parametrize("dim,keys,page", [(64, 200, 16), (128, 300, 64), (64, 2501, 16), (128, 3001, 64)])
def test_infinities_of_keys_under_one_token(gpu, kind, io, dim, keys, page):
    """a key whose score is -inf weighs nothing, one of +inf or NaN makes the row a NaN, however many terms the query is split into"""
    ctx, ka, torch = gpu
    p = Pool(gpu, n_seq=1, n_pages=-(-keys // page), max_pages=-(-keys // page), page=page, heads=2, dim=dim, kind=kind)
    assert p.append([(0, keys)], kind) == 0
    q = torch.randn(1, 4, dim, generator=p.gen, device="cuda").abs_().add_(0.01).to(dt(torch, io))
    at = lambda key: (p.rows[0][key // page], slice(None), key % page)  # noqa: E731
    work = torch.empty(max(16, ka.attn_paged_work_bytes(p.c, 1, 4, 0)), dtype=torch.uint8, device="cuda")

    def run():
        out = torch.empty(1, 4, dim, device="cuda")
        p.run(ctx.attn_paged_call(p.c, q, out, scale=1 / dim, work=work))
        return out

    for key in (0, 45, 100, keys - 1):
        p.k[at(key)][..., 5] = float("-inf")
        p.v[at(key)] = 1e4                                           # weighs nothing
    flat = [x[: -(-keys // page)].transpose(1, 2).reshape(-1, 2, dim)[:keys].cpu() for x in (p.k, p.v)]
    see = torch.tensor([j not in (0, 45, 100, keys - 1) for j in range(keys)])
    o, tol = expect(torch, q[0].cpu(), *flat, see, 1 / dim, kind, io, "f32", False, io == kind)
    same(torch, run()[0], o, tol)
    for x in (float("inf"), float("nan")):
        p.k[at(60)][..., 8] = x
        assert run().isnan().all()


@pytest.mark.parametrize("kind,dim,page", [("f16", 64, 4), ("bf16", 128, 16), ("f16", 128, 32)])
@pytest.mark.parametrize("max_q,rows", [(0, 70), (0, 1), (8, 3)])
def test_pages_before_the_window_may_be_gone(gpu, kind, dim, page, max_q, rows):
    """columns of the table that lie wholly before the window hold no page: not an error, in either attention; one that a row sees is"""
    ctx, ka, torch = gpu
    keys, window = 401, 90
    p = Pool(gpu, n_seq=1, n_pages=-(-keys // page), max_pages=-(-keys // page), page=page, heads=2, dim=dim, kind=kind)
    assert p.append([(0, keys)], kind) == 0
    q = torch.randn(rows, 4, dim, generator=p.gen, device="cuda").to(dt(torch, kind))
    whole, out = torch.empty(rows, 4, dim, device="cuda"), torch.empty(rows, 4, dim, device="cuda")
    packed = lambda to: ctx.attn_packed_call(q, to, p.ints([0, rows]), cache=p.c, scale=0.1, window=window, max_q=max_q)  # noqa: E731
    paged = lambda to: ctx.attn_paged_call(p.c, q[:1], to[:1], scale=0.1, window=window)  # noqa: E731
    first = keys - rows - window + 1                                 # of the keys that the first row of the packed call sees
    for call, seen in ((packed, first), (paged, keys - window)):
        p.run(call(whole))
        gone = seen // page
        assert gone > 0
        p.table[0, :gone] = -1
        p.run(call(out))
        assert int(p.status) == 0
        assert torch.equal(out[:1] if call is paged else out, whole[:1] if call is paged else whole)
        p.table[0, gone] = -1
        p.run(call(out))
        assert int(p.status) == ka.KV_BAD_ARG
        p.status.zero_()
        p.table[0] = p.ints(p.rows[0])


@pytest.mark.parametrize("page,max_q,ks", [(0, 0, [3, 40]), (16, 0, [3, 40]), (0, 8, [3, 600]), (16, 8, [3, 600])])
@pytest.mark.parametrize("causal", [True, False])
def test_a_window_beyond_every_length_is_none(gpu, page, max_q, ks, causal):
    packed_case(gpu, "f16", "f16", "f16", 64, 1, 2, [8, 8], ks, page=page, max_q=max_q, causal=causal, window=2**31 - 1)


def test_the_largest_and_smallest_values_of_the_type(gpu):
    """keys and values at the type's ends: scores of +-6e4 * |q| * scale do not overflow F32, one weight takes it all"""
    ctx, ka, torch = gpu
    top = {"f16": 65504.0, "bf16": 1e30}
    for kind in ("f16", "bf16"):
        p = Pool(gpu, n_seq=1, n_pages=4, max_pages=4, page=16, heads=1, dim=64, kind=kind)
        assert p.append([(0, 40)], kind) == 0
        k, v = (x.reshape(-1, 64)[:40] for x in (p.k, p.v))          # pages 0, 1, 2 in order
        k[7], k[20], v[7], v[9] = top[kind] * 1e-3, -top[kind] * 1e-3, top[kind], 1e-7
        q = torch.zeros(1, 1, 64, device="cuda")
        q[..., 0] = 1.0
        out = torch.empty(1, 1, 64, device="cuda")
        p.run(ctx.attn_paged_call(p.c, q, out, scale=1.0))
        assert torch.equal(out[0, 0], v[7].float())                  # exp of the runner-up underflows to nothing
        q[..., 0] = -1.0
        p.run(ctx.attn_paged_call(p.c, q, out, scale=1.0))
        assert torch.equal(out[0, 0], v[20].float())
        p.run(ctx.attn_paged_call(p.c, q, out, scale=0.0))           # equal weights
        want = v.double().mean(0)
        assert float(((out[0, 0].double() - want).abs() / want.abs().clamp_min(v.double().abs().mean(0) * 1e-2)).max()) < 100 * 40 * U["f32"]


def equal_best_keys(torch, p, lens, kind, best, rng):
    """Fills the keys of sequences 0 .. of `p` (already appended): `best` of them are the same key, the others zeros, so that scores are sums of one product and the best
    ones are equal in any precision; returns (the queries' two values, the best keys' numbers, values [L, dim] of each sequence, all on the CPU)."""
    a, b = (torch.tensor([x], dtype=torch.float64).to(dt(torch, kind)).item() for x in (rng.uniform(1, 2), rng.uniform(1, 2)))
    at, values = [], []
    for s, L in enumerate(lens):
        keys = sorted(rng.sample(range(L), best))
        for j in range(L):
            x = p.rows[s][j // p.page], 0, j % p.page
            p.k[x] = 0.0
            if j in keys:
                p.k[x[0], 0, x[2], 0] = a
        at.append(keys)
        values.append(torch.stack([x[1][0] for x in p.keys[s]]).double())
    return a, b, at, values


@pytest.mark.parametrize("kind,q_kind", [("f16", "f32"), ("f16", "f16"), ("bf16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("bits", range(18, 44, 2))
def test_scores_up_to_the_ends_of_the_range(gpu, kind, q_kind, bits):
    """Scores of about 2^bits in every way that the attentions run: a few equal best keys share the weight, whatever the products with the scale are rounded by.
    The best weights are the same number w, so that the result is the mean of their values up to the sums' and the quotient's rounding: 8 * 2^-24 of the largest
    value, with w rounded to the cache's type once (the same for all: 2 u(kind) of the largest value in the quotient), and the result's own rounding."""
    ctx, ka, torch = gpu
    rng = random.Random(bits)
    lens, best = [70, 300, 33], 3
    p = Pool(gpu, n_seq=3, n_pages=32, max_pages=20, page=16, heads=1, dim=64, kind=kind, seed=bits)
    assert p.append(list(enumerate(lens)), kind) == 0
    a, b, at, values = equal_best_keys(torch, p, lens, kind, best, rng)
    scale, small = 2.0 ** bits * rng.uniform(1, 2) / (a * b), 2 * U[kind] + 8 * U["f32"]

    def hold(out, s):
        want = values[s][at[s]].mean(0)
        tol = small * values[s][at[s]].abs().amax() + U["f32"] * want.abs()
        assert float(((out.double().cpu() - want).abs() - tol).max()) <= 0, (s, out[:4], want[:4])

    q = torch.zeros(3, 2, 64, device="cuda")
    q[:, 0, 0], q[:, 1, 0] = b, b * 0.75                             # the second head's scores: other roundings of the same keys
    q = q.to(dt(torch, q_kind))
    out = torch.empty(3, 2, 64, device="cuda")
    p.run(ctx.attn_paged_call(p.c, q, out, scale=scale))
    for s in range(3):
        hold(out[s, 0], s)
        hold(out[s, 1], s)
    for max_q, rows in ((8, 2), (0, 2), (0, 100)):                   # few rows, the packed kernel's small and its larger row tiles; not causal, so that all rows see all keys
        for n in (1, 2, 3):
            qr = torch.zeros(n * rows, 2, 64, device="cuda")
            qr[:, 0, 0], qr[:, 1, 0] = b, b * 0.75
            out = torch.empty(n * rows, 2, 64, device="cuda")
            p.run(ctx.attn_packed_call(qr.to(dt(torch, q_kind)), out, p.ints([i * rows for i in range(n + 1)]), cache=p.c, scale=scale, causal=False, max_q=max_q))
            for i in range(n):
                for r in sorted({0, rows // 2, rows - 1}):
                    hold(out[i * rows + r, 0], i)
                    hold(out[i * rows + r, 1], i)


def test_scores_near_the_lowest_number_of_all(gpu):
    """every score is -3.3e38: below any start that a running maximum could have but the lowest number itself"""
    ctx, ka, torch = gpu
    p = Pool(gpu, n_seq=1, n_pages=4, max_pages=4, page=16, heads=1, dim=64, kind="bf16")
    assert p.append([(0, 50)], "bf16") == 0
    k, v = (x.reshape(-1, 64)[:50] for x in (p.k, p.v))
    k.zero_()
    k[:, 0] = 2.0 ** 120
    q = torch.zeros(1, 1, 64, device="cuda")
    q[..., 0] = -1.0
    out, want = torch.empty(1, 1, 64, device="cuda"), v.double().mean(0)
    tol = 50 * U["f32"] * v.double().abs().amax()                    # equal weights: powers of two, so the sums' and the quotient's rounding alone
    for scale in (3.3e38 / 2.0 ** 120 / 1.4426950408889634, 3.39e38 / 2.0 ** 120 / 1.4426950408889634):
        p.run(ctx.attn_paged_call(p.c, q, out, scale=scale))
        assert float((out[0, 0].double() - want).abs().max()) <= tol
        p.run(ctx.attn_packed_call(q, out, p.ints([0, 1]), cache=p.c, scale=scale))
        assert float((out[0, 0].double() - want).abs().max()) <= tol


def test_calls_among_the_programs_own_work_on_the_contexts_stream(gpu):
    """projections that make the rows, the calls, and a product that reads the result, one after the other on ctx.stream with no wait between them"""
    ctx, ka, torch = gpu
    p, n, heads, dim = Pool(gpu, heads=2, dim=64, kind="f16"), 60, 2, 64
    gen = torch.Generator(device="cuda").manual_seed(5)
    x, w = torch.randn(n, 4096, generator=gen, device="cuda"), [torch.randn(4096, heads * dim, generator=gen, device="cuda") / 64 for _ in range(3)]
    late, w_o = torch.randn(4096, 4096, generator=gen, device="cuda") / 64, torch.randn(heads * dim, 32, generator=gen, device="cuda")
    rows, out = [torch.zeros(n, heads, dim, device="cuda") for _ in range(3)], torch.zeros(n, heads, dim, device="cuda")
    seq, cu, keep = p.ints([1, 4]), p.ints([0, 25, n]), p.ints([0, 0])
    calls = [ctx.kv_truncate_call(p.c, seq, keep), ctx.kv_append_call(p.c, seq, cu, rows[1], rows[2]), ctx.attn_packed_call(rows[0], out, cu, cache=p.c, seq=seq, scale=0.125)]

    def step(wait):
        y = x
        for _ in range(20):                                          # milliseconds before the rows are there
            y = torch.mm(y, late)
        for r, m in zip(rows, w):
            torch.mm(y, m, out=r.view(n, heads * dim))
        wait()
        for call in calls:
            call()
        wait()
        return torch.mm(out.view(n, heads * dim), w_o)

    want = step(torch.cuda.synchronize)
    for r in rows:
        r.zero_()
    out.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.ExternalStream(ctx.stream)):
        got = [step(lambda: None) for _ in range(3)]
    torch.cuda.synchronize()
    assert want.abs().max() > 0 and all(torch.equal(g, want) for g in got)
    p.status.zero_()


@pytest.mark.parametrize("n,rows,max_q", [(1, 5, 8), (3, 5, 8), (100, 2, 4), (1, 90, 0), (3, 90, 0), (100, 70, 0)])
@pytest.mark.parametrize("dim,heads", [(64, 2), (128, 4)])
@pytest.mark.parametrize("before", [1, 40, 700])
def test_rows_before_the_first_sequence(gpu, n, rows, max_q, dim, heads, before):
    """offsets that do not begin at 0: the rows before them belong to no sequence, are left as they are, and nothing else changes"""
    ctx, ka, torch = gpu
    p = Pool(gpu, n_seq=n, n_pages=n * 20, max_pages=20, page=16, heads=1, dim=dim, kind="f16")
    lens = [300 + i % 7 for i in range(n)]
    step = -(-n // 25)
    for i in range(0, n, step):
        assert p.append([(s, lens[s]) for s in range(i, min(i + step, n))], "f16") == 0
    q = torch.randn(n * rows, heads, dim, generator=p.gen, device="cuda").half()
    late = torch.cat([torch.full((before, heads, dim), float("nan"), device="cuda").half(), q])
    cu, cu_late = [i * rows for i in range(n + 1)], [before + i * rows for i in range(n + 1)]
    kv = torch.randn(before + n * rows, 1, dim, generator=p.gen, device="cuda").half()
    for own in (False, True):
        out, out_late = torch.full_like(q, 7.0), torch.full_like(late, 7.0)
        on, on_late = (dict(k=kv[before:], v=kv[before:]), dict(k=kv, v=kv)) if own else (dict(cache=p.c), dict(cache=p.c))
        p.run(ctx.attn_packed_call(q, out, p.ints(cu), scale=0.1, max_q=max_q, **on))
        p.run(ctx.attn_packed_call(late, out_late, p.ints(cu_late), scale=0.1, max_q=max_q, **on_late))
        assert (out_late[:before] == 7.0).all()
        # the choice of a kernel goes by the rows of the call: both are within the bounds of the file's head of the same result
        pool = kv if own else p.k[p.ref > 0].nan_to_num(0.0)
        e = (dim + 8) * U["f32"] * 0.1 * float(q.float().abs().sum(2).max() * pool.float().abs().max())
        per = math.expm1(4 * e) + 2 * U["f16"] + (max(rows, 306) + 32) * U["f32"]
        size = float(kv.float().abs().max() if own else p.v[p.ref > 0].float().nan_to_num(0.0).abs().max())
        assert bool(((out_late[before:].float() - out.float()).abs() <= 2 * (per * size + U["f16"] * out.float().abs())).all())


@pytest.mark.parametrize("before,counts", [(3, [2, 0, 1]), (300, [200, 5, 0]), (5000, [1, 0, 600])])
def test_rows_before_the_first_entry_of_an_append(gpu, before, counts):
    ctx, ka, torch = gpu
    a, b = (Pool(gpu, n_seq=3, n_pages=80, max_pages=60, page=16, heads=2, dim=64, kind="f16") for _ in range(2))
    k, v = (torch.randn(before + sum(counts), 2, 64, generator=a.gen, device="cuda") for _ in range(2))
    cu = np.concatenate([[0], np.cumsum(counts)])
    a.run(ctx.kv_append_call(a.c, a.ints([2, 0, 1]), a.ints(cu.tolist()), k[before:], v[before:]))
    b.run(ctx.kv_append_call(b.c, b.ints([2, 0, 1]), b.ints((cu + before).tolist()), k, v))
    for x in ("table", "len", "ref", "status"):
        assert torch.equal(getattr(a, x), getattr(b, x)), x
    assert a.len.tolist() == [counts[1], counts[2], counts[0]] and int(a.status) == 0
    for x in ("k", "v"):                                             # (memory that nothing was written to is NaN)
        assert torch.equal(getattr(a, x).nan_to_num(9.0), getattr(b, x).nan_to_num(9.0)), x


@pytest.mark.parametrize("max_q,rows", [(0, 5), (8, 5), (0, 90)])
def test_what_the_attentions_make_of_lists_and_lengths_out_of_range(gpu, max_q, rows):
    """a sequence that is none holds no keys, a length beyond the row is the row's end, offsets that fall or leave the rows write nothing outside them; no status"""
    ctx, ka, torch = gpu
    p = Pool(gpu, n_seq=3, n_pages=70, max_pages=20, page=16, heads=1, dim=64, kind="f16")
    assert p.append([(0, 320), (1, 100)], "f16") == 0
    q = torch.randn(6 * rows + 4, 2, 64, generator=p.gen, device="cuda").half()
    full = lambda: torch.full((6 * rows + 4, 2, 64), 7.0, device="cuda")  # noqa: E731
    packed = lambda out, cu, seq: p.run(ctx.attn_packed_call(q, out, p.ints(cu), cache=p.c, seq=p.ints(seq), scale=0.1, max_q=max_q))  # noqa: E731
    cu = [i * rows for i in range(7)]
    want, out, one, one_out = full(), full(), full()[:6], full()[:6]
    paged = lambda to, seq: p.run(ctx.attn_paged_call(p.c, q[:6], to, seq=p.ints(seq), scale=0.1))  # noqa: E731
    packed(want, cu, [0, 2, 0, 2, 1, 2])
    paged(one, [0, 2, 0, 2, 1, 2])
    assert (want[rows : 2 * rows] == 0).all()                        # sequence 2 is empty
    p.len[0], p.len[2] = 2 ** 31 - 1, -5
    packed(out, cu, [0, 3, 0, -9, 1, 2])                             # (in 0 the row is full: 320 keys)
    paged(one_out, [0, 3, 0, -9, 1, 2])
    assert torch.equal(out, want) and torch.equal(one_out, one)
    for wrong in ([0, rows, 2 * rows, rows, 4 * rows, 5 * rows, 6 * rows], [-3, rows, 2 * rows, 3 * rows, 4 * rows, 5 * rows, 6 * rows], cu[:-1] + [2 ** 31 - 1], [5 * rows] * 3 + [0] * 4):
        out = full()
        packed(out, wrong, [0, 1, 0, 1, 0, 1])
        assert (out[6 * rows :] == 7).all()
    assert int(p.status) == 0


def expect_rows(torch, q, k, v, see, scale, kind, out_kind, round_q):
    """expect() for rows q [R, H, D] at once, on the GPU in 64 bits; see [R, L].  Values that are not finite are counted apart: what a row does not see is not in its result"""
    (R, H, D), (L, Hkv) = q.shape, k.shape[:2]
    G = H // Hkv
    q, k, v = (x.double().permute(1, 0, 2).contiguous() for x in (q, k, v))          # [heads, rows, D]
    q = q.reshape(Hkv, G * R, D)                                     # head h is G h' + g: rows (g, r) of K/V head h'
    seen = see.repeat(G, 1)
    kt = k.transpose(1, 2).contiguous()
    x = torch.where(seen, torch.matmul(q, kt) * scale, -math.inf)
    w = torch.where(seen, torch.softmax(x, 2), 0.0) if L else x
    w = torch.where(seen.any(1)[:, None], w, 0.0)
    o = torch.matmul(w, v.nan_to_num(0.0, 0.0, 0.0))
    size = torch.where(seen, torch.matmul(q.abs(), kt.abs()) * abs(scale), 0.0).amax(2) if L else torch.zeros(Hkv, G * R, device=q.device).double()
    e = size * ((D + 8) * U["f32"] + (U[kind] if round_q else 0.0))
    per = torch.expm1(4 * e) + 2 * U[kind] + (L + 32) * U["f32"]
    top = v.nan_to_num(0.0, 0.0, 0.0).abs().amax((1, 2)) if L else torch.zeros(Hkv, device=q.device).double()
    tol = (per * top[:, None])[..., None] + U[out_kind] * o.abs() + 1e-30
    has = [torch.matmul(seen.double(), f(v).double()) > 0 for f in (torch.isposinf, torch.isneginf, torch.isnan)]
    o = torch.where(has[0], math.inf, o)
    o = torch.where(has[1], -math.inf, o)
    o = torch.where(has[2] | (has[0] & has[1]), math.nan, o)
    back = lambda y: y.reshape(H, R, D).permute(1, 0, 2)  # noqa: E731
    return back(o), back(tol)


# of each form of the packed attention: dims, K/V heads, heads, rows and keys of the sequences (None: as many), the caller's bound of the rows
FORMS = {
    "k_attn_paged 64": (64, 2, 4, [5, 8, 0, 1], [700, 300, 40, 290], 8),
    "k_attn_paged 128": (128, 1, 5, [7, 1, 3], [800, 3, 420], 8),
    "4, 1 64": (64, 2, 6, [50, 0, 3, 60], None, 0),
    "4, 1 64 many": (64, 1, 32, [1500, 2501, 33, 100], None, 0),
    "4, 2 64": (64, 2, 2, [300, 129, 1], [420, 129, 500], 0),
    "4, 1 128": (128, 2, 6, [100, 0, 3, 77], None, 0),
    "4, 1 128 many": (128, 4, 32, [700, 513, 1, 768, 200], None, 0),
    "4, 2 128": (128, 3, 3, [40, 64, 3], [300, 700, 64], 0),
    "8, 2 128": (128, 2, 4, [200, 131, 66], [500, 777, 66], 0),
    "8, 1 128": (128, 8, 32, [1301, 0, 835], [1301, 40, 1500], 0),
}


@pytest.mark.parametrize("name", FORMS)
@pytest.mark.parametrize("page,order", [(0, "head"), (0, "key"), (16, "key"), (64, "head")])
@pytest.mark.parametrize("kind,io,causal,window,spoiled", [("f16", "f16", True, 0, False), ("bf16", "bf16", True, 0, True), ("f16", "f32", True, 333, True), ("bf16", "f32", False, 0, False), ("f16", "f16", False, 150, True),
                                                           ("bf16", "bf16", True, 64, False)])
def test_every_form_of_the_packed_attention(gpu, name, page, order, kind, io, causal, window, spoiled):
    """each row tile and split of the waves that a call can get, by its name in the profile, with every kind of mask, infinities in tiles seen whole and in part, strided rows"""
    ctx, ka, torch = gpu
    dim, kv_heads, heads, q_lens, k_lens, max_q = FORMS[name]
    n, ks, rng = len(q_lens), k_lens or q_lens, random.Random(1)
    gen = torch.Generator(device="cuda").manual_seed(2)
    cu, ck = (np.concatenate([[0], np.cumsum(x)]).tolist() for x in (q_lens, ks))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.randn(cu[-1] + 2, heads, dim, generator=gen, device="cuda").mul_(2).to(dt(torch, io))
    out = torch.full((cu[-1] + 2, heads, dim), 7.0, device="cuda").to(dt(torch, io))
    kv = [torch.randn(ck[-1], kv_heads, dim, generator=gen, device="cuda").to(dt(torch, kind)) for _ in range(2)]
    if spoiled:
        for i in range(n):
            for j, d, x in ((ks[i] - 1, 1, math.inf), (ks[i] // 2, 2, -math.inf), (ks[i] // 3, 3, math.nan), (ks[i] // 2 + 1, 4, math.inf), (ks[i] - 2, 4, -math.inf), (0, 5, math.inf)):
                if 0 <= j < ks[i]:
                    kv[1][ck[i] + j, :, d] = x
    args = dict(scale=dim ** -0.5, causal=causal, window=window, max_q=max_q)
    if page:
        held = [-(-x // page) for x in ks]
        table, spread = torch.full((n + 1, max(held)), -1, dtype=torch.int32), rng.sample(range(sum(held) + 3), sum(held))
        seq = rng.sample(range(n + 1), n)
        shape = (sum(held) + 3, kv_heads, page, dim) if order == "head" else (sum(held) + 3, page, kv_heads, dim)
        pools = [torch.full(shape, math.nan, device="cuda").to(dt(torch, kind)) for _ in range(2)]
        pools = pools if order == "head" else [x.transpose(1, 2) for x in pools]
        length, at = torch.zeros(n + 1, dtype=torch.int32), 0
        for i in range(n):
            pages = spread[at : at + held[i]]
            at += held[i]
            table[seq[i], : held[i]] = torch.tensor(pages, dtype=torch.int32)
            length[seq[i]] = ks[i]
            where = torch.arange(ks[i])
            for pool, rows in zip(pools, kv):
                pool[torch.tensor(pages, dtype=torch.long)[where // page].cuda(), :, (where % page).cuda()] = rows[ck[i] : ck[i + 1]]
        zero = lambda m: torch.zeros(m, dtype=torch.int32, device="cuda")  # noqa: E731
        status, dtab, dlen, ref, work = zero(1), table.cuda(), length.cuda(), zero(sum(held) + 3), torch.empty(ka.kv_work_bytes(n + 1, sum(held) + 3), dtype=torch.uint8, device="cuda")
        c = ka.kv_cache(*pools, dtab, dlen, ref, status, work)
        call = ctx.attn_packed_call(q, out, ints(cu), cache=c, seq=ints(seq), **args)
    else:
        wide = [torch.full((ck[-1] + 1, kv_heads, 2 * dim if order == "key" else dim), math.nan, device="cuda").to(dt(torch, kind)) for _ in range(2)]
        for x, rows in zip(wide, kv):
            x[: ck[-1], :, :dim] = rows
        call = ctx.attn_packed_call(q, out, ints(cu), k=wide[0][..., :dim], v=wide[1][..., :dim], cu_k=ints(ck) if k_lens else None, **args)
    torch.cuda.synchronize()
    ctx.prof_reset()
    ctx.prof(True)
    call()
    ctx.sync()
    ran = [r["name"] for r in ctx.prof_report()]
    ctx.prof(False)
    ctx.prof_reset()
    form = f"k_attn_packed<{kind}_ops, {dim}, {str(page > 0).lower()}, {name[:4]}>" if max_q == 0 else f"k_attn_paged<{kind}_ops, {dim}, 1, {0 if page == 16 else 1 if page else 2}, true>"
    assert len(ran) == 1 and form in ran[0], (form, ran)
    assert (out[cu[-1] :] == 7.0).all() and (not page or int(status) == 0)
    for i in range(n):
        Q, L = q_lens[i], ks[i]
        if Q == 0:
            continue
        r = sorted(set(range(min(Q, 6))) | set(range(max(Q - 6, 0), Q)) | set(rng.sample(range(Q), min(Q, 40))))
        j, own = torch.arange(L, device="cuda"), torch.tensor(r, device="cuda")[:, None] + L - Q
        see = j <= own if causal else (j >= 0).expand(len(r), L)
        see = see & (j > own - window) if window else see
        o, tol = expect_rows(torch, q[[cu[i] + x for x in r]], kv[0][ck[i] : ck[i + 1]], kv[1][ck[i] : ck[i + 1]], see, dim ** -0.5, kind, io, io != kind)
        try:
            same(torch, out[[cu[i] + x for x in r]], o.cpu(), tol.cpu())
        except AssertionError as e:
            raise AssertionError(f"sequence {i} of {Q} rows and {L} keys: {e}")


def test_a_decode_loop_captured_into_a_graph_and_replayed(gpu):
    """append, attention, fork and truncate of a step captured once on the context's stream; every replay, with new lists and eager work of the program
    between the replays, equals the same step run eagerly on a second cache"""
    ctx, ka, torch = gpu
    stream = torch.cuda.ExternalStream(ka.lib().mi355x_ctx_stream(ctx.h))
    n, heads = 4, 2
    caches = [Pool(gpu, n_seq=n, n_pages=64, max_pages=16, page=4, heads=heads, dim=64, seed=1) for _ in range(2)]
    for p in caches:
        assert p.append([(s, 5 + 7 * s) for s in range(n)]) == 0
    seq, cu = caches[0].ints(list(range(n))), caches[0].ints(list(range(n + 1)))
    k, v, q = (torch.zeros(n, heads, 64, device="cuda") for _ in range(3))
    src, dst, keep = caches[0].ints([0] * n), caches[0].ints(list(range(n))), caches[0].ints([1000] * n)
    outs, steps = [torch.zeros(n, heads, 64, device="cuda") for _ in caches], []
    for p, out in zip(caches, outs):
        work = torch.empty(max(16, ka.attn_paged_work_bytes(p.c, n, heads)), dtype=torch.uint8, device="cuda")
        steps.append([ctx.kv_append_call(p.c, seq, cu, k, v), ctx.attn_paged_call(p.c, q, out, scale=0.125, work=work), ctx.kv_fork_call(p.c, src, dst), ctx.kv_truncate_call(p.c, seq, keep)])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for call in steps[1]:
            call()
    gen = torch.Generator(device="cuda").manual_seed(8)
    rng = random.Random(8)
    for rep in range(6):
        for x in (k, v, q):
            x.copy_(torch.randn(n, heads, 64, generator=gen, device="cuda"))
        src.copy_(caches[0].ints([rng.randrange(n) for _ in range(n)]))
        keep.copy_(caches[0].ints([rng.choice((1000, 3, 9)) for _ in range(n)]))
        torch.cuda.synchronize()
        for call in steps[0]:
            call()
        ctx.sync()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1])
        for x in ("table", "len", "ref", "status"):
            assert torch.equal(getattr(caches[0], x), getattr(caches[1], x)), (rep, x)
        assert int(caches[0].status) == 0


@pytest.mark.parametrize("kind,dim,kv_heads,heads,page", [("f16", 64, 2, 4, 16), ("bf16", 128, 1, 4, 8)])
def test_serving_streams_from_prompt_to_beams(gpu, kind, dim, kv_heads, heads, page):
    """prompts into the cache and attention over them, a second piece of each over the cache, single tokens with forks between them, a compaction in
    the middle: every result equals attention over the keys that the restatement holds"""
    ctx, ka, torch = gpu
    p = Pool(gpu, n_seq=6, n_pages=120, max_pages=20, page=page, heads=kv_heads, dim=dim, kind=kind)
    scale, gen, rng = 1 / math.sqrt(dim), torch.Generator(device="cuda").manual_seed(3), random.Random(3)

    def queries(rows):
        return torch.randn(rows, heads, dim, generator=gen, device="cuda").to(dt(torch, kind))

    def hold(out, q, i, s, last):
        k, v = (torch.stack([x[w] for x in p.keys[s]]) for w in (0, 1))
        o, tol = expect(torch, q[i].cpu(), k, v, torch.arange(len(k)) <= last, scale, kind, kind, kind, False, True)
        same(torch, out[i], o, tol)

    for piece in ([7, 0, 33], [20, 2, 1]):                           # the prompts in two pieces
        assert p.append(list(enumerate(piece)), kind) == 0
        q, cu = queries(sum(piece)), np.concatenate([[0], np.cumsum(piece)]).tolist()
        out = torch.zeros_like(q)
        p.run(ctx.attn_packed_call(q, out, p.ints(cu), cache=p.c, seq=p.ints([0, 1, 2]), scale=scale))
        for s, x in enumerate(piece):
            for r in range(x):
                hold(out, q, cu[s] + r, s, len(p.keys[s]) - x + r)
    p.fork([(0, 3), (2, 4), (2, 5)])
    for step in range(10):
        live = [0, 2, 3, 4, 5]
        assert p.append([(s, 1) for s in live], kind) == 0
        q = queries(len(live))
        out = torch.zeros_like(q)
        work = torch.empty(max(16, ka.attn_paged_work_bytes(p.c, len(live), heads)), dtype=torch.uint8, device="cuda")
        p.run(ctx.attn_paged_call(p.c, q, out, seq=p.ints(live), scale=scale, work=work))
        p.check(contents=False)
        for i, s in enumerate(live):
            hold(out, q, i, s, len(p.keys[s]) - 1)
        p.fork([(rng.choice((2, 4, 5)), d) for d in (2, 4, 5)])
        if step == 5:
            other = Pool(gpu, n_seq=6, n_pages=90, max_pages=20, page=page, heads=kv_heads, dim=dim, kind=kind, order="key", seed=5)
            p.run(ctx.kv_compact_call(p.c, other.c))
            used = [x for x in range(p.n_pages) if p.count[x]]
            name = {x: i for i, x in enumerate(used)}
            other.rows, other.keys = [[name[x] for x in r] for r in p.rows], p.keys
            other.count = [p.count[x] for x in used] + [0] * (90 - len(used))
            other.content = {(name[a], b): x for (a, b), x in p.content.items() if a in name}
            p = other
            p.check(contents=False)
    p.check(contents=False)


@pytest.mark.parametrize("n,n_seq,width", [(3000, 4000, 13), (8192, 20000, 7), (8192, 8192, 3), (1, 3, 20)])
def test_forks_of_long_lists(gpu, n, n_seq, width):
    """lists whose workgroups need more than 64 KB, or hold fewer columns at a time, against a restatement of tables"""
    ctx, ka, torch = gpu
    gen, rng = torch.Generator().manual_seed(n), random.Random(n)
    n_pages = 500
    lens = torch.randint(0, width * 4 + 1, (n_seq,), generator=gen, dtype=torch.int32)
    column = torch.arange(width)
    table = torch.where(column < (lens[:, None] + 3) // 4, torch.randint(0, n_pages, (n_seq, width), generator=gen), -1).int()
    count = lambda t: torch.bincount(t[t >= 0].long(), minlength=n_pages).int()  # noqa: E731
    k = torch.zeros(n_pages, 1, 4, 64, dtype=torch.float16, device="cuda")
    dtab, dlen, ref, status, work = table.cuda(), lens.cuda(), count(table).cuda(), torch.zeros(1, dtype=torch.int32, device="cuda"), torch.empty(ka.kv_work_bytes(n_seq, n_pages), dtype=torch.uint8, device="cuda")
    c = ka.kv_cache(k, k.clone(), dtab, dlen, ref, status, work)
    dst = rng.sample(range(n_seq), n)
    src = [rng.randrange(-1, n_seq) for _ in range(n)]
    for i in range(0, n, 5):
        dst[i] = -1 if i % 2 else dst[i]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    dsrc, ddst = ints(src), ints(dst)
    torch.cuda.synchronize()
    ctx.kv_fork_call(c, dsrc, ddst)()
    ctx.sync()
    new, new_len = table.clone(), lens.clone()
    for a, b in zip(src, dst):
        if b >= 0:
            new[b], new_len[b] = (table[a], lens[a]) if a >= 0 else (torch.full((width,), -1, dtype=torch.int32), 0)
    assert torch.equal(dtab.cpu(), new) and torch.equal(dlen.cpu(), new_len) and torch.equal(ref.cpu(), count(new)) and int(status) == 0
    if n > 1:                                                        # the last entry once more the first's row: nothing changes
        ddst[0], ddst[-1] = 7, 7
        torch.cuda.synchronize()
        ctx.kv_fork_call(c, dsrc, ddst)()
        ctx.sync()
        assert torch.equal(dtab.cpu(), new) and torch.equal(dlen.cpu(), new_len) and torch.equal(ref.cpu(), count(new)) and int(status) == ka.KV_BAD_ARG


@pytest.mark.parametrize("heads,dim,kind,io,counts", [(64, 128, "bf16", "f32", [3, 1, 700, 20]), (256, 128, "f16", "bf16", [33, 0, 2]), (1, 64, "f16", "f16", [4000, 1, 999, 17]), (5, 64, "bf16", "bf16", [1500, 3000])])
def test_appends_of_wide_rows_and_of_many(gpu, heads, dim, kind, io, counts):
    """rows of more pieces than a workgroup loads at once, and as many narrow rows to a workgroup as it takes"""
    ctx, ka, torch = gpu
    page, n = 16, len(counts)
    held = [-(-x // page) for x in counts]
    p = Pool(gpu, n_seq=n, n_pages=sum(held) + 1, max_pages=max(held), page=page, heads=heads, dim=dim, kind=kind)
    k, v = (torch.randn(sum(counts) + 2, heads, dim, generator=p.gen, device="cuda").to(dt(torch, io)) for _ in range(2))
    cu = np.concatenate([[0], np.cumsum(counts)]).tolist()
    p.run(ctx.kv_append_call(p.c, p.ints(list(range(n))), p.ints(cu), k, v))
    assert int(p.status) == 0 and p.len.tolist() == counts
    table, taken = p.table.cpu(), 0
    for i in range(n):                                               # free pages in ascending order, entry by entry
        assert table[i].tolist() == list(range(taken, taken + held[i])) + [-1] * (max(held) - held[i])
        for pool, rows in ((p.k, k), (p.v, v)):
            got = pool[taken : taken + held[i]].transpose(1, 2).reshape(-1, heads, dim)
            assert torch.equal(got[: counts[i]], rows[cu[i] : cu[i + 1]].to(dt(torch, kind)))
            assert got[counts[i] :].isnan().all()
        taken += held[i]
    assert p.ref.tolist() == [1] * taken + [0] and p.k[taken:].isnan().all()


@pytest.mark.parametrize("kind,dim,order", [("f16", 64, "head"), ("bf16", 128, "key")])
def test_places_beyond_four_gigabytes(gpu, kind, dim, order):
    """pages more than a gigabyte apart, rows of packed prompts too: every byte offset in 64 bits, in each call"""
    ctx, ka, torch = gpu
    page, heads, n_pages, apart = 16, 2, 7, (1 << 30) + 4096       # (elements of 2 bytes: 2 GiB and a bit)
    inner = (page * dim, dim) if order == "head" else (dim, heads * dim)
    whole = [torch.empty(apart * (n_pages - 1) + heads * page * dim, dtype=dt(torch, kind), device="cuda") for _ in range(2)]
    k, v = (x.as_strided((n_pages, heads, page, dim), (apart, *inner, 1)) for x in whole)
    zero = lambda *m: torch.zeros(*m, dtype=torch.int32, device="cuda")  # noqa: E731
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    work = torch.empty(ka.kv_work_bytes(2, n_pages), dtype=torch.uint8, device="cuda")
    table, length, ref, status = zero(2, 5), zero(2), zero(n_pages), zero(1)
    c = ka.kv_cache(k, v, table, length, ref, status, work)
    gen = torch.Generator(device="cuda").manual_seed(1)
    rows = [torch.randn(75, heads, dim, generator=gen, device="cuda").to(dt(torch, kind)) for _ in range(2)]
    q = torch.randn(8, 4, dim, generator=gen, device="cuda").to(dt(torch, kind))

    def run(call):
        torch.cuda.synchronize()
        call()
        ctx.sync()

    def hold(out, i, last, first, keys):
        o, tol = expect(torch, q[i].cpu(), *(x[first : first + keys].cpu() for x in rows), torch.arange(keys) <= last, 0.1, kind, kind, "f32", False, True)
        same(torch, out[i], o, tol)

    run(ctx.kv_reset_call(c))
    run(ctx.kv_append_call(c, ints([1, 0]), ints([0, 5, 75]), *rows))            # sequence 1 in page 0, sequence 0 in pages 1 .. 5
    assert int(status) == 0 and table.tolist() == [[1, 2, 3, 4, 5], [0, -1, -1, -1, -1]]
    small = [torch.zeros(n_pages, heads, page, dim, dtype=dt(torch, kind), device="cuda") for _ in range(2)]
    table2, length2, ref2, work2 = zero(2, 5), zero(2), zero(n_pages), torch.empty_like(work)
    to = ka.kv_cache(*small, table2, length2, ref2, status, work2)
    run(ctx.kv_reset_call(to))
    run(ctx.kv_compact_call(c, to))                                  # from far apart to close together, and back
    for x, y in zip((k, v), small):
        for p, filled in ((0, 5), (1, 16), (3, 16), (5, 6)):
            assert torch.equal(x[p, :, :filled], y[p, :, :filled])
    for which in (c, to):
        out = torch.zeros(2, 4, dim, device="cuda")
        run(ctx.attn_paged_call(which, q[:2], out, scale=0.1))
        hold(out, 0, 69, 5, 70)
        hold(out, 1, 4, 0, 5)
        for max_q in (0, 8):
            out = torch.zeros(8, 4, dim, device="cuda")
            run(ctx.attn_packed_call(q, out, ints([0, 6, 8]), cache=which, scale=0.1, max_q=max_q))
            for i in range(6):
                hold(out, i, 64 + i, 5, 70)
            hold(out, 7, 4, 0, 5)
    del whole, k, v, c, x
    torch.cuda.empty_cache()
    far = [torch.empty(300 * (1 << 24), dtype=dt(torch, kind), device="cuda").as_strided((300, heads, dim), (1 << 24, dim, 1)) for _ in range(2)]     # rows of a prompt 32 MiB apart
    for i, x in enumerate(far):
        x.copy_(torch.cat([rows[i], torch.randn(225, heads, dim, generator=gen, device="cuda").to(dt(torch, kind))]))
    rows = [x.contiguous() for x in far]
    for max_q in (0, 8):
        out = torch.zeros(8, 4, dim, device="cuda")
        run(ctx.attn_packed_call(q[:6], out[:6], ints([0, 6]), k=far[0], v=far[1], cu_k=ints([0, 300]), scale=0.1, max_q=max_q))
        for i in range(6):
            hold(out, i, 294 + i, 0, 300)
    run(ctx.kv_reset_call(to))
    run(ctx.kv_append_call(to, ints([1, 0]), ints([225, 230, 300]), *far))       # the last rows: 7 GiB from the first
    assert int(status) == 0
    assert torch.equal(small[0][1], rows[0][230:246].transpose(0, 1)) and torch.equal(small[1][5, :, :6], rows[1][294:300].transpose(0, 1))
    del far
    torch.cuda.empty_cache()


@pytest.mark.parametrize("page,order", [(1, "head"), (2, "key"), (1024, "head"), (4096, "key")])
@pytest.mark.parametrize("kind,dim", [("f16", 64), ("bf16", 128)])
def test_the_smallest_and_the_largest_pages(gpu, page, order, kind, dim):
    ctx, ka, torch = gpu
    lens = [4500, 0, 1, 700, 1025]
    need = sum(-(-x // page) for x in lens)
    p = Pool(gpu, n_seq=5, n_pages=need + 5, max_pages=-(-4501 // page), page=page, heads=1, dim=dim, kind=kind, order=order)
    assert p.append(list(enumerate(lens)), kind) == 0
    p.fork([(0, 1)])
    assert p.append([(1, 1), (3, 2)], kind) == 0
    p.truncate([(0, 4097)])
    lens = [len(x) for x in p.keys]
    p.check(contents=False)
    q = torch.randn(5 * 6, 4, dim, generator=p.gen, device="cuda").to(dt(torch, kind))
    flat = [[torch.stack([x[w] for x in keys]) for w in (0, 1)] for keys in p.keys]
    out, work = torch.zeros(5, 4, dim, device="cuda"), torch.empty(max(16, ka.attn_paged_work_bytes(p.c, 5, 4)), dtype=torch.uint8, device="cuda")
    p.run(ctx.attn_paged_call(p.c, q[:5], out, scale=0.1, work=work))
    for s in range(5):
        o, tol = expect(torch, q[s].cpu(), *flat[s], torch.ones(lens[s], dtype=torch.bool), 0.1, kind, kind, "f32", False, True)
        same(torch, out[s], o, tol)
    for max_q in (0, 8):
        out = torch.zeros(30, 4, dim, device="cuda")
        p.run(ctx.attn_packed_call(q, out, p.ints([0, 6, 12, 18, 24, 30]), cache=p.c, scale=0.1, max_q=max_q))
        for s in range(5):
            for r in range(6):
                o, tol = expect(torch, q[6 * s + r].cpu(), *flat[s], torch.arange(lens[s]) <= lens[s] - 6 + r, 0.1, kind, kind, "f32", False, True)
                same(torch, out[6 * s + r], o, tol)
    p.check()


def test_prompts_and_a_compaction_captured_into_a_graph_and_replayed(gpu):
    """reset, append, packed attention (the form of eight waves and the one for few rows) and compact in one graph, with new lists and rows between the replays"""
    ctx, ka, torch = gpu
    stream = torch.cuda.ExternalStream(ctx.stream)
    n, heads, kv_heads, dim, rows, keys = 3, 16, 2, 128, 2700, 2700
    ends = [[0, 900, 1800, 2700], [0, 1, 2500, 2700], [0, 0, 2700, 2700], [0, 1300, 1300, 1999]]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    zero = lambda *m: torch.zeros(*m, dtype=torch.int32, device="cuda")  # noqa: E731
    cu, few = ints(ends[0]), ints([0, 4, 8, 12])
    q, k, v = torch.zeros(rows, heads, dim, device="cuda").half(), *(torch.zeros(keys, kv_heads, dim, device="cuda").half() for _ in range(2))
    status, sets = zero(1), []
    for _ in range(2):
        cells = []
        for _ in range(2):
            pool = [torch.zeros(200, kv_heads, 16, dim, device="cuda").half() for _ in range(2)]
            rest = [zero(n, 180), zero(n), zero(200), status, torch.empty(ka.kv_work_bytes(n, 200), dtype=torch.uint8, device="cuda")]
            cells.append((ka.kv_cache(*pool, *rest), pool, rest))
        outs = [torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q[:12])]
        a, b = cells[0][0], cells[1][0]
        seq = ints([2, 0, 1])
        calls = [ctx.kv_reset_call(a), ctx.kv_append_call(a, seq, cu, k, v), ctx.attn_packed_call(q, outs[0], cu, k=k, v=v, scale=0.1, window=500), ctx.kv_reset_call(b), ctx.kv_compact_call(a, b),
                 ctx.attn_packed_call(q, outs[1], cu, cache=b, seq=seq, scale=0.1, window=500), ctx.attn_packed_call(q[:12], outs[2], few, cache=b, seq=seq, scale=0.1, max_q=8)]
        sets.append((calls, cells, outs))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for call in sets[1][0]:
            call()
    gen = torch.Generator(device="cuda").manual_seed(4)
    for rep in range(6):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=gen, device="cuda"))
        cu.copy_(ints(ends[rep % len(ends)]))
        for _, cells, outs in sets:
            for x in outs:
                x.fill_(7.0)
        torch.cuda.synchronize()
        for call in sets[0][0]:
            call()
        ctx.sync()
        graph.replay()
        torch.cuda.synchronize()
        assert int(status) == 0
        for x, y in zip(sets[0][2], sets[1][2]):
            assert torch.equal(x, y), rep
        for (_, pool, rest), (_, pool2, rest2) in zip(sets[0][1], sets[1][1]):
            assert all(torch.equal(x, y) for x, y in zip(pool + rest[:3], pool2 + rest2[:3])), rep


@pytest.mark.parametrize("n", [64, 65, 4097, 20000])
def test_thousands_of_sequences_in_one_call(gpu, n):
    """of 0 to 3 rows: appended, attended to as packed rows (their own and the cache's, few and not) and one token each, where the searches have one, two and three levels"""
    ctx, ka, torch = gpu
    rng, gen, heads, dim, page = random.Random(n), torch.Generator(device="cuda").manual_seed(n), 2, 64, 4
    counts = [rng.choice((0, 1, 2, 3)) for _ in range(n)]
    cu = np.concatenate([[0], np.cumsum(counts)])
    total = int(cu[-1])
    ints = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")  # noqa: E731
    zero = lambda *m: torch.zeros(*m, dtype=torch.int32, device="cuda")  # noqa: E731
    q, k, v = (torch.randn(total, heads, dim, generator=gen, device="cuda").half() for _ in range(3))
    pool = [torch.zeros(n, heads, page, dim, device="cuda").half() for _ in range(2)]
    table, length, ref, status, work = zero(n, 2), zero(n), zero(n), zero(1), torch.empty(ka.kv_work_bytes(n, n), dtype=torch.uint8, device="cuda")
    c = ka.kv_cache(*pool, table, length, ref, status, work)
    # the definition: entry e's rows are cu[e] ..; row r of it sees the entry's rows up to itself, the one token all of them
    starts = torch.tensor(cu[:-1], device="cuda")
    entry = torch.repeat_interleave(torch.arange(n, device="cuda"), torch.tensor(counts, device="cuda"))
    own = torch.arange(total, device="cuda") - starts[entry]

    def define(rows, first, last):
        """rows [R, heads, dim] over the keys first .. last (at most 3) of each; its allowed error as in expect(), with the larger of all bounds"""
        at = (first[:, None] + torch.arange(3, device="cuda")).clamp_max(total - 1)
        see = (torch.arange(3, device="cuda") <= (last - first)[:, None])[:, None]
        x = (rows.double()[:, None] * k[at].double()).sum(3).transpose(1, 2) * 0.1
        w = torch.softmax(torch.where(see, x, -math.inf), 2).nan_to_num(0.0)
        o = (w[..., None] * v[at].double().transpose(1, 2)).sum(2)
        e = 0.1 * float((rows.double().abs()[:, None] * k[at].double().abs()).sum(3).max()) * (dim + 8) * U["f32"]
        return o, (math.expm1(4 * e) + 2 * U["f16"] + 40 * U["f32"]) * float(v.abs().max()) + U["f16"] * o.abs()

    def hold(out, o, tol):
        assert bool(((out.double() - o).abs() <= tol).all())

    def run(call):
        torch.cuda.synchronize()
        call()
        ctx.sync()

    seq = rng.sample(range(n), n)
    dseq, dcu = ints(seq), ints(cu)
    run(ctx.kv_reset_call(c))
    run(ctx.kv_append_call(c, dseq, dcu, k, v))
    assert int(status) == 0
    pages, t = iter(range(n)), table.tolist()
    for e, s in enumerate(seq):
        assert t[s] == ([next(pages), -1] if counts[e] else [-1, -1])
    o, tol = define(q, starts[entry], starts[entry] + own)
    for extra in (dict(k=k, v=v), dict(cache=c, seq=dseq)):
        for max_q in (0, 3):
            out = torch.full_like(q, 7.0)
            run(ctx.attn_packed_call(q, out, dcu, scale=0.1, max_q=max_q, **extra))
            hold(out, o, tol)
    one = torch.randn(n, heads, dim, generator=gen, device="cuda").half()
    out, space = torch.full_like(one, 7.0), torch.empty(max(16, ka.attn_paged_work_bytes(c, n, heads)), dtype=torch.uint8, device="cuda")
    run(ctx.attn_paged_call(c, one, out, seq=dseq, scale=0.1, work=space))
    o, tol = define(one, starts, starts + torch.tensor(counts, device="cuda") - 1)
    hold(out, o, tol)


@pytest.mark.parametrize("n", [4096, 4097])
def test_one_long_sequence_among_thousands_of_short_ones(gpu, n):
    """on both sides of the number of queries from which keys are not split"""
    ctx, ka, torch = gpu
    page, gen, long = 16, torch.Generator(device="cuda").manual_seed(n), 9001
    lens = [i % 3 for i in range(n)]
    lens[n // 2] = long
    held = [-(-x // page) for x in lens]
    k, v = (torch.randn(sum(held), 1, page, 64, generator=gen, device="cuda").half() for _ in range(2))
    table, at = torch.full((n, max(held)), -1, dtype=torch.int32), 0
    for s, h in enumerate(held):
        table[s, :h] = torch.arange(at, at + h)
        at += h
    zero = lambda m: torch.zeros(m, dtype=torch.int32, device="cuda")  # noqa: E731
    status = zero(1)
    c = ka.kv_cache(k, v, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), zero(sum(held)), status, torch.empty(ka.kv_work_bytes(n, sum(held)), dtype=torch.uint8, device="cuda"))
    q = torch.randn(n, 3, 64, generator=gen, device="cuda").half()
    out, need = torch.full_like(q, 7.0), ka.attn_paged_work_bytes(c, n, 3)
    assert (need > 0) == (n <= 4096)
    space = torch.empty(max(16, need), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    ctx.attn_paged_call(c, q, out, scale=0.125, work=space)()
    ctx.sync()
    assert int(status) == 0
    for s in [0, 1, 2, 3, n // 2 - 1, n // 2, n // 2 + 1, n - 3, n - 2, n - 1]:
        flat = [x.cpu()[table[s, : held[s]].long()].transpose(1, 2).reshape(-1, 1, 64)[: lens[s]] for x in (k, v)]
        o, tol = expect(torch, q[s].cpu(), *flat, torch.ones(lens[s], dtype=torch.bool), 0.125, "f16", "f16", "f16", False, True)
        same(torch, out[s], o, tol)


@pytest.mark.parametrize("kind,io", [("f16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("dim,rows,max_q", [(64, 9, 8), (128, 9, 0), (64, 300, 0), (128, 300, 0)])
def test_queries_and_results_inside_larger_arrays(gpu, kind, io, dim, rows, max_q):
    """every third head of a projection's rows, every second row of a result: what lies between is as it was"""
    ctx, ka, torch = gpu
    p = Pool(gpu, n_seq=rows, n_pages=40, max_pages=30, page=16, heads=2, dim=dim, kind=kind)
    assert p.append([(1, 400), (2, 30)], kind) == 0
    wide = torch.randn(2 * rows, 20, dim, generator=p.gen, device="cuda").to(dt(torch, io))
    q = wide[::2, 1:17:3]                                            # 6 heads
    seq = p.ints([1, 2, -1] * (rows // 3))
    for call in (lambda q, o: ctx.attn_paged_call(p.c, q, o, seq=seq, scale=0.1), lambda q, o: ctx.attn_packed_call(q, o, p.ints([0, rows]), cache=p.c, seq=p.ints([1]), scale=0.1, max_q=max_q)):
        plain, big = torch.zeros(rows, 6, dim, device="cuda"), torch.full((2 * rows, 13, dim), 7.0, device="cuda")
        p.run(call(q.contiguous(), plain))
        p.run(call(q, big[1::2, 1::2]))
        assert torch.equal(big[1::2, 1::2], plain) and float(plain.abs().max()) > 0
        assert (big[::2] == 7).all() and (big[:, ::2] == 7).all()
