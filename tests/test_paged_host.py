"""What the calls of the paged cache and its attentions refuse (include/mi355x_kernels.h: mi355x_kv_*, mi355x_attn_paged, mi355x_attn_packed): checked on the
host before anything is launched, so without a device.  The context of a refused call is never touched: a blank block stands for it."""
import ctypes as C

import pytest

from whisper_cpp_amd import kernels_api as ka

BLANK = C.create_string_buffer(65536)
CTX = C.cast(BLANK, C.c_void_p)
MEM = (C.c_char * 4096).from_buffer(bytearray(4096))
AT = (C.addressof(MEM) + 63) // 64 * 64


def cache(**change):
    c = ka.KvCache()
    c.k, c.v, c.type, c.head_dim, c.n_head_kv, c.page_size, c.n_pages, c.n_seq, c.max_pages = AT, AT, ka.F16, 64, 2, 16, 8, 4, 4
    c.nb_key, c.nb_head, c.nb_page = 128, 2048, 4096
    c.table = c.len = c.ref = c.status = c.work = AT
    for name, value in change.items():
        setattr(c, name, value)
    return c


def rows(n=3, heads=2, dim=64, kind=ka.F32, at=AT, nb=None):
    size = 4 if kind == ka.F32 else 2
    return ka.tensor(at, kind, [dim, heads, n], nb or [size, size * dim, size * dim * heads])


def refused(name, *args):
    assert getattr(ka.lib(), name)(CTX, *args) == -1
    assert ka.lib().mi355x_last_error()


BAD_CACHES = [dict(k=None), dict(v=None), dict(table=None), dict(len=None), dict(ref=None), dict(status=None), dict(work=None), dict(type=ka.F32), dict(type=ka.Q8_0), dict(head_dim=80),
              dict(head_dim=0), dict(n_head_kv=0), dict(n_head_kv=513), dict(page_size=0), dict(page_size=24), dict(page_size=8192), dict(n_pages=0), dict(n_seq=0), dict(n_seq=300000),
              dict(max_pages=0), dict(max_pages=1 << 27), dict(nb_key=120), dict(nb_key=64), dict(nb_head=8), dict(nb_page=0), dict(k=AT + 8), dict(table=AT + 2), dict(nb_page=-4096)]


@pytest.mark.parametrize("change", BAD_CACHES, ids=lambda d: "-".join(f"{k}={v}" for k, v in d.items()))
def test_every_call_refuses_a_cache_that_does_not_fit(change):
    c, t = cache(**change), rows()
    d = ka.AttnPagedDesc()
    d.q, d.dst, d.scale = rows(4), rows(4), 1.0
    p = ka.AttnPackedDesc()
    p.q, p.dst, p.cu_q, p.cache, p.n = rows(), rows(), AT, C.pointer(c), 1
    refused("mi355x_kv_reset", C.byref(c))
    refused("mi355x_kv_append", C.byref(c), 1, AT, AT, C.byref(t), C.byref(t))
    refused("mi355x_kv_truncate", C.byref(c), 1, AT, AT)
    refused("mi355x_kv_fork", C.byref(c), 1, AT, AT)
    refused("mi355x_kv_compact", C.byref(c), C.byref(cache(k=AT + 1024, v=AT + 2048)))
    refused("mi355x_kv_compact", C.byref(cache(k=AT + 1024, v=AT + 2048)), C.byref(c))
    refused("mi355x_attn_paged", C.byref(c), C.byref(d))
    refused("mi355x_attn_packed", C.byref(p))


def test_lists_and_rows_that_do_not_fit_are_refused():
    c = cache()
    ok, cases = rows(), [rows(dim=128), rows(heads=3), rows(at=AT + 4), rows(kind=ka.I32), rows(nb=[4, 250, 512]), rows(nb=[8, 512, 1024]), rows(n=4), rows(kind=ka.F16), rows(at=None)]
    for t in cases:
        refused("mi355x_kv_append", C.byref(c), 1, AT, AT, C.byref(ok), C.byref(t))
    refused("mi355x_kv_append", C.byref(c), 1, AT, AT, None, C.byref(ok))
    refused("mi355x_kv_append", C.byref(c), 5, AT, AT, C.byref(ok), C.byref(ok))
    refused("mi355x_kv_append", C.byref(c), -1, AT, AT, C.byref(ok), C.byref(ok))
    refused("mi355x_kv_append", C.byref(c), 1, None, AT, C.byref(ok), C.byref(ok))
    refused("mi355x_kv_append", C.byref(c), 1, AT, AT + 1, C.byref(ok), C.byref(ok))
    refused("mi355x_kv_truncate", C.byref(c), 1, AT, None)
    refused("mi355x_kv_truncate", C.byref(c), -1, AT, AT)
    refused("mi355x_kv_fork", C.byref(c), 1, None, AT)
    refused("mi355x_kv_fork", C.byref(c), 8193, AT, AT)
    other = dict(k=AT + 1024, v=AT + 2048, table=AT + 64, len=AT + 128, ref=AT + 192, work=AT + 256)
    for change in (dict(type=ka.BF16), dict(head_dim=128, nb_key=256), dict(n_head_kv=1), dict(page_size=8), dict(n_seq=5), dict(max_pages=3), dict(k=AT), dict(table=AT), dict(work=AT)):
        refused("mi355x_kv_compact", C.byref(c), C.byref(cache(**{**other, **change})))


def test_attention_of_one_token_refuses_what_it_cannot_do():
    c = cache(max_pages=4096)
    for change in (dict(q=rows(heads=3)), dict(q=rows(dim=128)), dict(dst=rows(4)), dict(dst=rows(kind=ka.Q8_0)), dict(q=rows(5), dst=rows(5)), dict(window=-1), dict(max_len=-1), dict(seq=AT + 2),
                   dict(work=None), dict(work=AT + 4), dict(work_bytes=64)):
        d = ka.AttnPagedDesc()
        d.q, d.dst, d.scale, d.work, d.work_bytes = rows(), rows(), 1.0, AT, 1 << 30
        for name, value in change.items():
            setattr(d, name, value)
        refused("mi355x_attn_paged", C.byref(c), C.byref(d))
    refused("mi355x_attn_paged", C.byref(c), None)
    assert ka.attn_paged_work_bytes(c, 3, 2) > 64                    # 65536 keys: split, so the work area is wanted
    assert ka.attn_paged_work_bytes(c, 3, 2, 100) == 0               # at most 100: not
    big = cache(max_pages=1 << 26)                                   # 2^30 keys: more than 31 of such queries are not split, their costs would not fit 32 bits
    assert ka.attn_paged_work_bytes(big, 31, 2) > 0 and ka.attn_paged_work_bytes(big, 32, 2) == 0
    assert ka.attn_paged_work_bytes(c, 3, 3) == 0 and ka.attn_paged_work_bytes(c, 0, 2) == 0
    assert ka.kv_work_bytes(4, 8) > 0 and ka.kv_work_bytes(0, 8) == 0 and ka.kv_work_bytes(4, -1) == 0


def test_the_work_area_is_for_one_shape_and_the_largest_answer_does_for_all():
    """what the header says of its size: not monotone in the queries; an area that is a byte short of its own shape's is refused"""
    c = cache(n_head_kv=8, max_pages=128, n_seq=256, nb_page=16384)
    need = {n: ka.attn_paged_work_bytes(c, n, 8, 2048) for n in (1, 63, 64, 128)}
    assert need[63] == 268484 > need[1] > 0 and need[64] == need[128] == 0
    sizes = [ka.attn_paged_work_bytes(c, n, 8, 2048) for n in range(1, 129)]
    d = ka.AttnPagedDesc()
    d.scale, d.max_len, d.work = 1.0, 2048, AT
    for n in (1, 2, 62, 63):
        d.q, d.dst, d.work_bytes = rows(n, 8), rows(n, 8), sizes[n - 1] - 1
        refused("mi355x_attn_paged", C.byref(c), C.byref(d))
    assert max(sizes) == sizes[62]


def test_attention_of_packed_rows_refuses_what_it_cannot_do():
    kv = rows(kind=ka.F16)
    for change in (dict(q=rows(heads=3)), dict(q=rows(dim=128)), dict(q=rows(heads=258)), dict(dst=rows(4)), dict(k=rows()), dict(v=rows(kind=ka.BF16)), dict(v=rows(2, kind=ka.F16)), dict(k=rows(dim=80, kind=ka.F16)),
                   dict(v=rows(kind=ka.F16, nb=[2, 128, 512])), dict(cu_q=None), dict(cu_q=AT + 2), dict(cu_k=AT + 2), dict(n=-1), dict(window=-1), dict(max_q=-1), dict(q=rows(at=AT + 8))):
        d = ka.AttnPackedDesc()
        d.q, d.k, d.v, d.dst, d.cu_q, d.n, d.scale = rows(), kv, kv, rows(), AT, 1, 1.0
        for name, value in change.items():
            setattr(d, name, value)
        refused("mi355x_attn_packed", C.byref(d))
    d.cache, d.cu_q, d.n, d.max_q, d.q = C.pointer(cache()), AT, 5, 0, rows()
    refused("mi355x_attn_packed", C.byref(d))                        # more entries than the cache has sequences, and no list of them
    refused("mi355x_attn_packed", None)


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf")])
def test_attention_of_packed_rows_refuses_a_scale_that_is_no_number(scale):
    """(a NaN came out as equal weights)"""
    d = ka.AttnPackedDesc()
    d.q, d.k, d.v, d.dst, d.cu_q, d.n, d.scale = rows(), rows(kind=ka.F16), rows(kind=ka.F16), rows(), AT, 1, scale
    refused("mi355x_attn_packed", C.byref(d))


def test_calls_of_more_threads_than_a_launch_has_are_refused_before_anything_is_launched():
    c = cache()
    refused("mi355x_kv_truncate", C.byref(c), 1 << 24, AT, AT)
    many = rows(n=1 << 24, dim=64, kind=ka.F16)
    refused("mi355x_kv_append", C.byref(c), 1, AT, AT, C.byref(many), C.byref(many))
    refused("mi355x_kv_fork", C.byref(cache(page_size=1, nb_page=2048, max_pages=1 << 28)), 1, AT, AT)
    other = dict(k=AT + 1024, v=AT + 2048, table=AT + 64, len=AT + 128, ref=AT + 192, work=AT + 256)
    refused("mi355x_kv_compact", C.byref(cache(n_pages=1 << 27)), C.byref(cache(n_pages=1 << 27, **other)))
    d = ka.AttnPagedDesc()
    d.scale, d.max_len, d.seq = 1.0, 16, AT
    d.q, d.dst = (rows(n=65535, heads=256) for _ in range(2))
    refused("mi355x_attn_paged", C.byref(cache(max_pages=1)), C.byref(d))
    d.q, d.dst = (rows(n=4096, heads=2048) for _ in range(2))
    refused("mi355x_attn_paged", C.byref(cache(max_pages=1)), C.byref(d))
    p = ka.AttnPackedDesc()
    p.q, p.k, p.v, p.dst, p.cu_q, p.n, p.scale = rows(n=1 << 24, heads=256), rows(n=64, heads=256, kind=ka.F16), rows(n=64, heads=256, kind=ka.F16), rows(n=1 << 24, heads=256), AT, 1, 1.0
    refused("mi355x_attn_packed", C.byref(p))


def test_python_descriptions_refuse_arrays_that_do_not_fit():
    import torch
    k = torch.zeros(8, 2, 16, 64, dtype=torch.float16)
    i = lambda *n: torch.zeros(*n, dtype=torch.int32)  # noqa: E731
    ok = dict(k=k, v=k.clone(), table=i(4, 4), length=i(4), ref=i(8), status=i(1), work=torch.zeros(ka.kv_work_bytes(4, 8), dtype=torch.uint8))
    c = ka.kv_cache(**ok)
    assert (c.n_pages, c.n_head_kv, c.page_size, c.head_dim, c.n_seq, c.max_pages, c.nb_key, c.nb_head, c.nb_page) == (8, 2, 16, 64, 4, 4, 128, 2048, 4096)
    t = ka.kv_cache(**{**ok, "k": k.transpose(1, 2).contiguous().transpose(1, 2), "v": k.transpose(1, 2).contiguous().transpose(1, 2)})
    assert (t.nb_key, t.nb_head) == (256, 128)
    for change in (dict(v=k[:7]), dict(v=k.float()), dict(table=i(4)), dict(table=i(4, 4).long()), dict(length=i(3)), dict(ref=i(7)), dict(work=i(3)), dict(k=k.double(), v=k.double()), dict(table=i(8, 4)[::2])):
        with pytest.raises(ValueError):
            ka.kv_cache(**{**ok, **change})


def test_a_cache_and_its_calls_hold_on_to_their_arrays():
    """a work area made in the call itself, as the documents have it, is not given back while a call can still use it"""
    import gc
    import weakref
    import torch
    ctx = object.__new__(ka.Ctx)
    ctx.h, ctx.device = CTX, 0
    made = []

    class On:
        def __init__(self, t):
            self.t, self.device = t, torch.device("cuda:0")          # (a host array that says it lies on the device: nothing is launched)
            made.append(weakref.ref(self))

        def __getattr__(self, name):
            return getattr(self.t, name)

    i = lambda *n: On(torch.zeros(*n, dtype=torch.int32))  # noqa: E731
    pool = lambda: On(torch.zeros(8, 2, 16, 64, dtype=torch.float16))  # noqa: E731
    c = lambda: ka.kv_cache(pool(), pool(), i(4, 4), i(4), i(8), i(1), On(torch.zeros(ka.kv_work_bytes(4, 8), dtype=torch.uint8)))  # noqa: E731
    row = lambda: On(torch.zeros(3, 2, 64))  # noqa: E731
    calls = [ctx.kv_reset_call(c()), ctx.kv_append_call(c(), i(2), i(3), row(), row()), ctx.kv_truncate_call(c(), i(2), i(2)), ctx.kv_fork_call(c(), i(2), i(2)), ctx.kv_compact_call(c(), c()),
             ctx.attn_paged_call(c(), row(), row(), seq=i(3), work=On(torch.zeros(64, dtype=torch.uint8))), ctx.attn_packed_call(row(), row(), i(3), cache=c(), seq=i(2))]
    gc.collect()
    assert len(made) == 7 * 8 + 16 and all(m() is not None for m in made)
    calls.clear()
    gc.collect()
    assert all(m() is None for m in made)


def test_calls_refuse_arrays_that_are_not_on_the_contexts_device():
    """host memory, or another device's, is no memory for a kernel: refused where the call is made up, before there is anything to launch"""
    import torch
    ctx = object.__new__(ka.Ctx)
    ctx.h, ctx.device = CTX, 0

    class On:
        """a host array that says it lies on a device"""
        def __init__(self, t, device):
            self.t, self.device = t, torch.device(device)

        def __getattr__(self, name):
            return getattr(self.t, name)

    def arrays(device):
        on = lambda t: On(t, device)  # noqa: E731
        i = lambda *n: on(torch.zeros(*n, dtype=torch.int32))  # noqa: E731
        k = torch.zeros(8, 2, 16, 64, dtype=torch.float16)
        a = dict(cache=ka.kv_cache(on(k), on(k.clone()), i(4, 4), i(4), i(8), i(1), on(torch.zeros(ka.kv_work_bytes(4, 8), dtype=torch.uint8))))
        a.update(seq=i(3), cu=i(4), rows=on(torch.zeros(3, 2, 64)), kv=on(torch.zeros(3, 2, 64, dtype=torch.float16)), work=on(torch.zeros(64, dtype=torch.uint8)))
        return a

    calls = {                                                        # of each call, the names of its arrays
        "reset": (lambda a: ctx.kv_reset_call(a["cache"]), "cache"),
        "append": (lambda a: ctx.kv_append_call(a["cache"], a["seq"], a["cu"], a["k"], a["v"]), "cache seq cu k v"),
        "truncate": (lambda a: ctx.kv_truncate_call(a["cache"], a["seq"], a["keep"]), "cache seq keep"),
        "fork": (lambda a: ctx.kv_fork_call(a["cache"], a["src"], a["dst"]), "cache src dst"),
        "compact": (lambda a: ctx.kv_compact_call(a["cache"], a["to"]), "cache to"),
        "paged": (lambda a: ctx.attn_paged_call(a["cache"], a["q"], a["out"], seq=a["seq"], work=a["work"]), "cache q out seq work"),
        "packed": (lambda a: ctx.attn_packed_call(a["q"], a["out"], a["cu"], k=a["kv"], v=a["v16"], cu_k=a["cu_k"]), "q out cu kv v16 cu_k"),
        "packed over a cache": (lambda a: ctx.attn_packed_call(a["q"], a["out"], a["cu"], cache=a["cache"], seq=a["seq"]), "q out cu cache seq"),
    }
    same = dict(k="rows", v="rows", q="rows", out="rows", keep="seq", src="seq", dst="seq", to="cache", v16="kv", cu_k="cu")
    of = lambda a, name: a[same.get(name, name)]  # noqa: E731
    good = arrays("cuda:0")
    for what, (make, names) in calls.items():
        mine = {name: of(good, name) for name in names.split()}
        make(mine)                                                   # (made up, not called)
        for other in ("cpu", "cuda:1"):
            bad = arrays(other)
            for name in names.split():
                with pytest.raises(ValueError, match="context's device"):
                    make({**mine, name: of(bad, name)})
    k = torch.zeros(8, 2, 16, 64, dtype=torch.float16)
    i = lambda *n: torch.zeros(*n, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="one device"):
        ka.kv_cache(k, k.clone(), On(i(4, 4), "cuda:0"), i(4), i(8), i(1), torch.zeros(ka.kv_work_bytes(4, 8), dtype=torch.uint8))


def test_a_call_of_a_closed_context_is_refused():
    """a call keeps the context that it was made up for: after close() that is freed memory"""
    ctx = object.__new__(ka.Ctx)
    ctx.h, ctx.device = CTX, 0
    call = ctx.kv_reset_call(cache())
    reached = []
    call.fn = lambda *args: reached.append(args) or 0
    call()
    assert len(reached) == 1
    ctx.h = None                                                     # what close() leaves
    with pytest.raises(RuntimeError, match="closed"):
        call()
    assert len(reached) == 1
    with pytest.raises(RuntimeError, match="closed"):
        ctx.stream


def test_ctypes_mirrors_of_the_paged_structs(tmp_path):
    import subprocess
    from conftest import ROOT
    probes = {"mi355x_kv_cache": ka.KvCache, "mi355x_attn_paged_desc": ka.AttnPagedDesc, "mi355x_attn_packed_desc": ka.AttnPackedDesc}
    src = ["#include <stdio.h>", "#include <stddef.h>", '#include "mi355x_kernels.h"', "int main(void) {"]
    for s, m in probes.items():
        src.append(f'  printf("{s} %zu", sizeof({s}));')
        src += [f'  printf(" %zu", offsetof({s}, {f[0]}));' for f in m._fields_] + ['  printf("\\n");']
    (tmp_path / "layout.c").write_text("\n".join(src + ["  return 0;", "}"]))
    subprocess.run(["gcc", f"-I{ROOT / 'include'}", str(tmp_path / "layout.c"), "-o", str(tmp_path / "layout")], check=True)
    for line in subprocess.run([str(tmp_path / "layout")], check=True, stdout=subprocess.PIPE, text=True).stdout.strip().splitlines():
        name, size, *offs = line.split()
        assert C.sizeof(probes[name]) == int(size)
        assert [getattr(probes[name], f[0]).offset for f in probes[name]._fields_] == [int(x) for x in offs]


SWEEP = """
import sys
sys.path.insert(0, sys.argv[1])
import __graft_entry__ as graft
graft.load_package()
import ctypes as C
from whisper_cpp_amd import kernels_api as ka
if ka.lib().mi355x_device_count() != 0:
    sys.exit("a device is visible: nothing may be launched")
blank = C.create_string_buffer(65536)
mem = (C.c_char * 4096).from_buffer(bytearray(4096))
at = (C.addressof(mem) + 63) // 64 * 64
seen = set()
for dim in (64, 128):
    for kv_heads in (1, 2):
        for group in range(1, 129):
            for n, rows, keys, max_q in ((1, 200, 200, 0), (1, 1, 1000, 0), (4, 1, 8000, 0), (4, 1, 8000, 1), (1, 4000, 4000, 0), (1, 100, 300, 8), (16, 100000, 100000, 0), (9, 9, 90, 3)):
                for cached in (False, True):
                    H = kv_heads * group
                    d = ka.AttnPackedDesc()
                    d.q, d.dst = (ka.tensor(at, ka.F32, [dim, H, rows], [4, 4 * dim, 4 * dim * H]) for _ in range(2))
                    d.k, d.v = (ka.tensor(at, ka.F16, [dim, kv_heads, keys], [2, 2 * dim, 2 * dim * kv_heads]) for _ in range(2))
                    d.cu_q, d.n, d.scale, d.causal, d.max_q = at, n, 1.0, 1, max_q
                    c = ka.KvCache()
                    c.k, c.v, c.type, c.head_dim, c.n_head_kv, c.page_size, c.n_pages, c.n_seq, c.max_pages = at, at, ka.F16, dim, kv_heads, 16, 8, 16, -(-keys // 16)
                    c.nb_key, c.nb_head, c.nb_page = 2 * dim, 32 * dim, 32 * dim * kv_heads
                    c.table = c.len = c.ref = c.status = c.work = at
                    if cached:
                        d.cache = C.pointer(c)
                    print(dim, H, kv_heads, n, rows, keys, max_q, cached, flush=True)
                    seen.add(ka.lib().mi355x_attn_packed(C.cast(blank, C.c_void_p), C.byref(d)))
print("answers:", *sorted(seen))
"""


def test_every_group_of_heads_finds_a_form_of_the_packed_attention():
    """up to 128 query heads to a K/V head, in every branch of the choice: each call gets as far as its launch, which finds no device (a process of its own, which sees none)"""
    import os
    import subprocess
    import sys
    from conftest import ROOT
    env = {**os.environ, "HIP_VISIBLE_DEVICES": "-1", "ROCR_VISIBLE_DEVICES": "-1"}
    r = subprocess.run([sys.executable, "-c", SWEEP, str(ROOT)], env=env, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, timeout=300)
    lines = r.stdout.strip().splitlines()
    assert r.returncode == 0, (r.returncode, lines[-1:])
    name, *answers = lines[-1].split()
    assert name == "answers:" and answers and all(int(x) > 0 for x in answers), lines[-1]


def test_a_build_compiles_every_kernel_source_when_told_to_and_after_a_change_of_flags(monkeypatch, tmp_path):
    """nothing is run: the commands are"""
    import os
    from whisper_cpp_amd import build
    ran = []
    monkeypatch.setattr(build, "_run", lambda cmd: ran.append([str(x) for x in cmd]) or "")
    monkeypatch.setattr(build, "LIB", tmp_path / "lib")
    monkeypatch.setattr(build, "BUILD", tmp_path / "build")
    compiled = lambda: sorted(os.path.basename(c[c.index("-c") + 1]) for c in ran if "-c" in c)  # noqa: E731
    build.build_kernels()
    assert compiled() == sorted(build.KERNEL_SRCS) and "-shared" in ran[-1]
    now = max(f.stat().st_mtime for f in [build.Path(build.__file__), *(build.CSRC / "kernels").iterdir(), *(build.ROOT / "include").iterdir()]) + 5
    made = [tmp_path / "build" / "kernels" / (s + ".o") for s in build.KERNEL_SRCS] + [tmp_path / "lib" / "libmi355x_kernels.so"]
    for f in made:
        f.write_bytes(b"")
        os.utime(f, (now, now))
    ran.clear()
    build.build_kernels()
    assert ran == []
    build.build_kernels(force=True)
    assert compiled() == sorted(build.KERNEL_SRCS) and "-shared" in ran[-1]
    for f in made[:-1]:
        f.unlink()
    ran.clear()
    build.build_kernels()                                            # the library alone, newer than all sources
    assert ran == []
    build.build_kernels(force=True)
    assert compiled() == sorted(build.KERNEL_SRCS)
    for f in made[:-1]:
        f.write_bytes(b"")
    flags = build.Path(build.__file__).stat().st_mtime
    for f in made:
        os.utime(f, (flags - 1, flags - 1))                          # objects older than the flags
    ran.clear()
    build.build_kernels()
    assert compiled() == sorted(build.KERNEL_SRCS)
