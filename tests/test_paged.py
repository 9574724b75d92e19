"""The paged session cache against plain loops: every array exactly, after each call
and over random runs of calls; refusals; bad indexes; graph replay."""
from __future__ import annotations

import copy
import ctypes as C
import io
import os
import random
import subprocess
import tempfile

import pytest
import torch

from oasis_b200 import _lib, paged
from oracle.paged_oracle import OracleCache
from tests.helpers import ROOT

DEV = "cuda"


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def make(pages=40, page=16, layers=2, heads=3, dim=64, slots=8, width=6, dtype=torch.bfloat16, seed=0):
    c = paged.PagedCache(pages, page, layers, heads, dim, slots, width, dtype=dtype, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(seed)
    c.pool.normal_(generator=g)
    return c, OracleCache(c.pool, c.table, c.lengths, c.refs)


def same(c, o):
    torch.cuda.synchronize()
    assert c.lengths.tolist() == o.lengths
    assert c.refs.tolist() == o.refs
    held = [[p for p in r[: -(-n // o.page)]] for r, n in zip(c.table.tolist(), o.lengths)]
    assert held == [r[: -(-n // o.page)] for r, n in zip(o.table, o.lengths)]
    assert int(c.status.item()) == o.status
    assert torch.equal(c.pool.cpu().view(torch.int16), o.pool.view(torch.int16))


def extend(c, o, seqs, counts, gen, layers=None):
    """Reserve and write on both sides, keys and values as views of packed rows."""
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + max(n, 0))
    start = c.reserve(ints(seqs), ints(cu))
    want = o.reserve(seqs, cu)
    assert start.tolist() == want
    rows = torch.empty(cu[-1] + 2, 2 * c.kv_heads + 1, c.head_dim, dtype=c.dtype, device=DEV).normal_(generator=gen)
    k, v = rows[:, 1 : 1 + c.kv_heads], rows[:, 1 + c.kv_heads :]
    for layer in range(c.layers) if layers is None else layers:
        c.write(layer, k, v, ints(seqs), ints(cu), start)
        o.write(layer, k, v, seqs, cu, want)


# ----------------------------------------------------------------- without a GPU --

def _header_program(body):
    src = f'#include <stdio.h>\n#include "{ROOT}/open-oasis_b200/csrc/pages.cuh"\nusing namespace oasis;\nint main() {{{body}}}'
    with tempfile.TemporaryDirectory() as d:
        f, exe = os.path.join(d, "p.cpp"), os.path.join(d, "p")
        open(f, "w").write(src)
        subprocess.run(["g++", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", f, "-o", exe], check=True)
        return subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()


def test_index_arithmetic_stays_in_bounds():
    """Lengths, table entries and offsets that device memory may hold, good or bad:
    what the kernels make of them stays inside the table, the pool and the lists."""
    out = _header_program(r'''
      const int odd[] = {-2147483647 - 1, -1, 0, 1, 15, 16, 17, 95, 96, 97, 2147483647};
      for (int len : odd) {
        const int e = used_entries(len, 16, 6), t = held_tokens(len, 16, 6);
        if (e < 0 || e > 6 || t < 0 || t > 96 || pages_of(t, 16) != e) printf("entries %d\n", len);
      }
      if (page_ok(-1, 5) || page_ok(5, 5) || !page_ok(4, 5) || !page_ok(0, 5)) printf("page\n");
      const int lists[][5] = {{0, 0, 3, 3, 9}, {5, 4, 3, 2, 1}, {-7, 100, -7, 100, 0}, {0, 0, 0, 0, 0}};
      for (auto& l : lists)
        for (int at : odd)
          for (int n = 1; n <= 5; ++n) {
            const int i = last_not_above(l, n, at);
            if (i < 0 || i >= n) printf("search\n");
          }
      const int s[] = {0, 0, 3, 3, 9};
      if (last_not_above(s, 5, 0) != 1 || last_not_above(s, 5, 2) != 1 || last_not_above(s, 5, 3) != 3 ||
          last_not_above(s, 5, 8) != 3 || last_not_above(s, 5, 99) != 4) printf("which\n");
      PageGeometry g; g.pages = 1 << 20; g.layers = 32; g.kv_heads = 16; g.page_size = 64; g.head_dim = 128;
      const long long end = tile_offset(g, g.pages - 1, 31, 1, 15) + tile_vectors(g);
      if (end != (long long)g.pages * page_vectors(g) || end < (1LL << 31)) printf("offset %lld\n", end);
      printf("done\n");''')
    assert out == ["done"]


def _c_cache(**kw):
    a = dict(pool=16, pages=4, layers=1, kv_heads=1, page_size=16, head_dim=64, dtype=1, table=16, slots=2, width=2,
             lengths=16, refs=16, status=16, workspace=16, workspace_bytes=1 << 20)
    a.update(kw)
    return _lib.OasisPageCache(**a)


@pytest.mark.parametrize("field,value,text", [
    ("pool", 0, b"null"), ("pool", 24, b"16-byte"), ("dtype", 0, b"dtype"), ("pages", 0, b"pages=0"),
    ("page_size", 24, b"page_size=24"), ("page_size", 272, b"page_size"), ("head_dim", 12, b"head_dim=12"),
    ("width", 1 << 30, b"too large"), ("layers", 1 << 25, b"too large"),
])
def test_cache_is_checked(field, value, text):
    lib = _lib.load()
    c = _c_cache(**{field: value})
    for rc in (lib.oasis_pages_free(C.byref(c), 16, 1, None), lib.oasis_pages_fork(C.byref(c), 16, 16, 1, 0, None),
               lib.oasis_pages_reserve(C.byref(c), 16, 16, 1, 16, None), lib.oasis_pages_compact(C.byref(c), None),
               lib.oasis_pages_write(C.byref(c), 0, 16, 16, 64, 64, 64, 64, 16, 16, 16, 1, 1, None)):
        assert rc == -1 and text in lib.oasis_last_error()


def test_calls_are_checked():
    lib = _lib.load()
    c = _c_cache()
    assert lib.oasis_pages_free(C.byref(c), 16, 3, None) == -1 and b"n=3" in lib.oasis_last_error()
    assert lib.oasis_pages_fork(C.byref(c), 16, 0, 1, 0, None) == -1 and b"null" in lib.oasis_last_error()
    assert lib.oasis_pages_reserve(C.byref(c), 16, 16, -1, 16, None) == -1
    for bad in (dict(workspace=0), dict(workspace_bytes=8)):
        d = _c_cache(**bad)
        assert lib.oasis_pages_compact(C.byref(d), None) == -3 and b"workspace" in lib.oasis_last_error()
    write = lambda layer, k, stride: lib.oasis_pages_write(  # noqa: E731
        C.byref(c), layer, k, 16, stride, 64, 64, 64, 16, 16, 16, 1, 1, None)
    assert write(1, 16, 64) == -1 and b"layer=1" in lib.oasis_last_error()
    assert write(0, 18, 64) == -1 and b"16-byte" in lib.oasis_last_error()
    assert write(0, 16, 68) == -1 and b"strides" in lib.oasis_last_error()
    # nothing to do
    assert lib.oasis_pages_free(C.byref(c), None, 0, None) == 0
    assert lib.oasis_pages_workspace_size(0, 4) == 0
    assert lib.oasis_pages_workspace_size(100, 4) > lib.oasis_pages_workspace_size(10, 4) > 0


def test_struct_layout_matches_c():
    with tempfile.TemporaryDirectory() as d:
        lines = [f'printf("%zu\\n", offsetof(OasisPageCache, {f}));' for f, _ in _lib.OasisPageCache._fields_]
        f, exe = os.path.join(d, "l.c"), os.path.join(d, "l")
        open(f, "w").write('#include <stdio.h>\n#include <stddef.h>\n' + f'#include "{ROOT}/include/oasis_b200.h"\n'
                           + "int main(void) {" + "".join(lines) + 'printf("%zu\\n", sizeof(OasisPageCache)); return 0; }')
        subprocess.run(["gcc", "-std=c99", f, "-o", exe], check=True)
        got = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    want = [getattr(_lib.OasisPageCache, f).offset for f, _ in _lib.OasisPageCache._fields_]
    assert got == want + [C.sizeof(_lib.OasisPageCache)]


def test_python_refuses_host_tensors():
    pool = torch.zeros(4, 1, 2, 1, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        paged.PagedCache.from_tensors(pool, torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32),
                                      torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError, match="contiguous"):
        paged.PagedCache.from_tensors(pool.transpose(4, 5), None, None, None)
    with pytest.raises(ValueError, match="bfloat16"):
        paged.PagedCache.from_tensors(pool.float(), None, None, None)


# --------------------------------------------------------------------- on a GPU --

@pytest.mark.gpu
@pytest.mark.parametrize("page,dim,dtype", [(16, 64, torch.bfloat16), (32, 128, torch.float16), (48, 8, torch.bfloat16)])
def test_reserve_write_fork_free_compact(page, dim, dtype):
    c, o = make(page=page, dim=dim, dtype=dtype)
    gen = torch.Generator(device=DEV).manual_seed(1)
    extend(c, o, [0, 3, 5], [page + 3, 2 * page, 1], gen)
    same(c, o)
    extend(c, o, [5, 0], [page - 1, 1], gen)  # fills a page to its end; stays inside one
    same(c, o)
    for src, dst, deep in (([0, 0, 3], [1, 2, 4], False), ([3, 6], [6, 7], True)):  # 6 is empty when the call begins
        c.fork(ints(src), ints(dst), deep=deep)
        o.fork(src, dst, deep)
        same(c, o)
    extend(c, o, [1, 2, 0], [5, 1, 2 * page], gen)  # forks grow apart
    same(c, o)
    for seqs in ([0, 3], [3, 5]):  # 3 is empty by then
        c.free(ints(seqs))
        o.free(seqs)
        same(c, o)
    c.compact()
    o.compact()
    same(c, o)
    c.compact()
    same(c, o)
    c.check()


@pytest.mark.gpu
def test_requests_that_are_refused():
    c, o = make(pages=7, slots=6, width=3)
    gen = torch.Generator(device=DEV).manual_seed(2)
    extend(c, o, [0, 9, 1, 0, -1], [20, 5, 16, 3, 1], gen)  # outside the cache, named twice
    same(c, o)
    assert o.status == 3
    with pytest.raises(_lib.OasisError, match="outside the cache.*named twice"):
        c.check()
    o.status = 0
    extend(c, o, [1, 0, 2], [33, 1, 0], gen)  # 49 tokens do not fit three pages of 16
    same(c, o)
    assert o.status == paged.TOO_LONG
    extend(c, o, [2, 3, 4, 5], [40, 32, 1, 0], gen)  # 4 free pages: 3, then 2 and 1 more do not fit
    same(c, o)
    assert o.status & paged.NO_PAGES and o.lengths[2] == 40 and o.lengths[3] == o.lengths[4] == 0
    for src, dst, deep in (([0, 1, 0], [1, 3, 3], False), ([1, 7], [5, 4], False), ([2, 1], [4, 3], True)):
        c.fork(ints(src), ints(dst), deep=deep)
        o.fork(src, dst, deep)
        same(c, o)
    c.free(ints([2, 2, 6]))
    o.free([2, 2, 6])
    same(c, o)
    bad = c.reserve(ints([2]), ints([4, 1]))  # decreasing offsets
    assert bad.tolist() == [-1]


@pytest.mark.gpu
def test_pages_outside_the_pool_are_skipped():
    c, o = make(pages=8, slots=4, width=4)
    gen = torch.Generator(device=DEV).manual_seed(3)
    extend(c, o, [0, 1], [40, 40], gen)
    before = c.pool.clone()
    c.table[0] = ints([-5, 8, 1 << 30, -1])
    rows = torch.ones(40, c.kv_heads, 64, dtype=torch.bfloat16, device=DEV)
    c.write(0, rows, rows, ints([0]), ints([0, 40]), ints([0]))
    c.fork(ints([0]), ints([2]))
    c.compact()
    c.free(ints([0, 2]))
    torch.cuda.synchronize()
    assert int(c.status.item()) == paged.BAD_PAGE
    assert c.lengths.tolist() == [0, 40, 0, 0]
    kept = c.table[1, :3].long()
    assert torch.equal(c.pool[kept, :, :, :, :8], before[torch.tensor(o.table[1][:3], device=DEV), :, :, :, :8])


@pytest.mark.gpu
@pytest.mark.parametrize("seed,pages,slots", [(0, 30, 9), (1, 200, 17), (2, 17000, 40)])
def test_random_runs(seed, pages, slots):
    """Random calls, refused ones among them; the large pool takes the free-page
    search over more than one round of the planning block."""
    rng = random.Random(seed)
    c, o = make(pages=pages, page=16, layers=1, heads=1, dim=8, slots=slots, width=9, seed=seed)
    if pages > 1000:  # the front of the pool is taken
        c.refs[: pages - 60] = 1
        c.refs[5::1000] = 0
        o.refs = c.refs.tolist()
    gen = torch.Generator(device=DEV).manual_seed(seed)
    for step in range(40):
        pick = lambda: [rng.randrange(-1, slots + 1) for _ in range(rng.randint(1, slots))]  # noqa: E731
        kind = rng.choice(["extend", "extend", "fork", "deep", "free", "compact"])
        if kind == "extend":
            seqs = pick()
            extend(c, o, seqs, [rng.choice([0, 1, 5, 16, 40, 200]) for _ in seqs], gen)
        elif kind == "free":
            seqs = pick()
            c.free(ints(seqs))
            o.free(seqs)
        elif kind == "compact":
            c.compact()
            o.compact()
        else:
            src = pick()
            dst = [rng.randrange(-1, slots + 1) for _ in src]
            c.fork(ints(src), ints(dst), deep=kind == "deep")
            o.fork(src, dst, kind == "deep")
        same(c, o)


@pytest.mark.gpu
@pytest.mark.parametrize("slots", [2500, 9000])
def test_many_requests_at_once(slots):
    """More requests than the planning block has threads; more sequences than it keeps in
    shared memory."""
    c, o = make(pages=4000, page=16, layers=1, heads=1, dim=8, slots=slots, width=3)
    rng = random.Random(5)
    seqs = rng.sample(range(slots), 2499)
    seqs.insert(1300, seqs[7])  # named twice
    rng.shuffle(seqs)
    counts = [rng.choice([0, 1, 16, 17, 48, 49]) for _ in seqs]
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    assert c.reserve(ints(seqs), ints(cu)).tolist() == o.reserve(seqs, cu)
    same(c, o)
    c.free(ints(seqs[:1200]))
    o.free(seqs[:1200])
    c.fork(ints(seqs[1200:2400]), ints(seqs[:1200]))
    o.fork(seqs[1200:2400], seqs[:1200])
    same(c, o)
    c.compact()
    o.compact()
    same(c, o)


@pytest.mark.gpu
def test_graph_replay_and_side_stream():
    """A captured step (free, fork, reserve, write) replayed, then a call on another
    stream behind an event."""
    c, o = make(pages=60, slots=6, width=6)
    gen = torch.Generator(device=DEV).manual_seed(4)
    extend(c, o, [0, 1], [37, 16], gen)
    src, dst, cu = ints([0, 1, 0]), ints([2, 3, 4]), ints([0, 1, 3, 4])
    rows = torch.empty(4, 3, 64, dtype=torch.bfloat16, device=DEV).normal_(generator=gen)

    def step():
        c.free(dst)
        c.fork(src, dst)
        start = c.reserve(dst, cu)
        for layer in range(c.layers):
            c.write(layer, rows, rows, dst, cu, start)
        c.compact()

    def plain():
        o.free([2, 3, 4])
        o.fork([0, 1, 0], [2, 3, 4])
        start = o.reserve([2, 3, 4], [0, 1, 3, 4])
        for layer in range(c.layers):
            o.write(layer, rows, rows, [2, 3, 4], [0, 1, 3, 4], start)
        o.compact()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    plain()
    same(c, o)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    same(c, o)
    for _ in range(3):
        g.replay()
        plain()
    same(c, o)
    ready = torch.cuda.Event()
    ready.record()
    side.wait_event(ready)
    c.free(dst, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    o.free([2, 3, 4])
    same(c, o)


@pytest.mark.gpu
def test_copies_and_stored_caches_are_their_own():
    """A deep copy, or a cache stored and loaded, changes its own tensors and not the first's."""
    c = paged.PagedCache(8, 16, 1, 1, 64, 3, 4, device=DEV)
    seqs, cu = ints([0]), ints([0, 20])
    c.reserve(seqs, cu)
    buffer = io.BytesIO()
    torch.save(c, buffer)
    buffer.seek(0)
    for other in (copy.deepcopy(c), torch.load(buffer, weights_only=False)):
        assert torch.equal(other.table, c.table) and other.table.data_ptr() != c.table.data_ptr()
        other.reserve(seqs, cu)
        assert other.lengths.tolist() == [40, 0, 0] and c.lengths.tolist() == [20, 0, 0]
        assert int(other.refs.sum()) == 3 and int(c.refs.sum()) == 2
    same = copy.copy(c)
    same.reserve(seqs, cu)
    assert c.lengths.tolist() == [40, 0, 0]


@pytest.mark.gpu
def test_python_checks():
    c, _ = make()
    with pytest.raises(ValueError, match="int32"):
        c.free(torch.zeros(2, dtype=torch.int64, device=DEV))
    with pytest.raises(ValueError, match="must be on"):
        c.free(torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="cu must hold 3"):
        c.reserve(ints([0, 1]), ints([0, 1]))
    rows = torch.zeros(3, 3, 64, dtype=torch.bfloat16, device=DEV)
    start = ints([0])
    for k, text in ((rows.half(), "bfloat16"), (rows[:, :2], r"\[rows, 3, 64\]"), (rows[0], "rows"),
                    (torch.zeros(3, 3, 65, dtype=torch.bfloat16, device=DEV)[:, :, 1:], "aligned"),
                    (torch.zeros(3, 64, 3, dtype=torch.bfloat16, device=DEV).transpose(1, 2), "contiguous")):
        with pytest.raises(ValueError, match=text):
            c.write(0, k, k, ints([0]), ints([0, 3]), start)
    with pytest.raises(_lib.OasisError, match="layer=2"):
        c.write(2, rows, rows, ints([0]), ints([0, 3]), start)
    with pytest.raises(_lib.OasisError, match="n=9"):
        c.free(ints(list(range(9))))


@pytest.mark.gpu
@pytest.mark.parametrize("deep", [False, True])
def test_a_fork_of_a_page_outside_the_pool(deep):
    """What the source does not have its fork does not have either: the entry outside the pool
    is the fork's too, no page of the pool stands in its place, and the pages meant for it are
    free. A whole page and the partial last one, which every fork copies."""
    c, o = make(pages=12, slots=4, width=4, layers=1)
    gen = torch.Generator(device=DEV).manual_seed(6)
    extend(c, o, [0], [40], gen)
    pages = c.table[0, :3].tolist()
    c.table[0, 2] = 99
    if deep:
        c.table[0, 0] = -3
    bad = [x for x in c.table[0, :3].tolist()]
    c.fork(ints([0]), ints([1]), deep=deep)
    torch.cuda.synchronize()
    assert int(c.status.item()) == paged.BAD_PAGE
    got = c.table[1, :3].tolist()
    assert c.lengths.tolist() == [40, 40, 0, 0] and got[2] == 99
    refs = [0] * 12
    for p in pages:
        refs[p] = 1
    if deep:
        assert got[0] == -3 and got[1] not in pages
        refs[got[1]] = 1
        assert torch.equal(c.pool[got[1]], c.pool[bad[1]])
    else:
        assert got[:2] == bad[:2]
        refs[bad[0]], refs[bad[1]] = 2, 2
    assert c.refs.tolist() == refs
    q = torch.empty(2, 3, 64, dtype=c.dtype, device=DEV).normal_(generator=gen)
    q[1] = q[0]
    plan = paged.SharedPlan([], [], 40, DEV)
    a = paged.attention_shared(q, c, 0, ints([0, 1]), plan)
    assert torch.equal(a[0], a[1]) and bool(torch.isfinite(a).all())
    c.free(ints([1]))
    left = [0] * 12
    for p in pages:
        left[p] = 1
    assert c.refs.tolist() == left


@pytest.mark.gpu
def test_copies_and_stored_caches_keep_what_was_refused():
    """A copy of a cache, or one stored and loaded, raises what the cache has been refused
    since its last check; a handle on the same tensors shares the word."""
    c = paged.PagedCache(1, 16, 1, 1, 64, 2, 4, device=DEV)
    c.reserve(ints([0]), ints([0, 20]))  # two pages of one
    buffer = io.BytesIO()
    torch.save(c, buffer)
    buffer.seek(0)
    for other in (copy.deepcopy(c), torch.load(buffer, weights_only=False)):
        with pytest.raises(_lib.OasisError, match="no free page"):
            other.check()
        other.check()
    same = copy.copy(c)
    with pytest.raises(_lib.OasisError, match="no free page"):
        same.check()
    c.check()
    fresh = paged.PagedCache.from_tensors(c.pool, c.table, c.lengths, c.refs)
    assert int(fresh.status.item()) == 0
    with pytest.raises(ValueError, match="status must hold 1"):
        paged.PagedCache.from_tensors(c.pool, c.table, c.lengths, c.refs, c.lengths)
