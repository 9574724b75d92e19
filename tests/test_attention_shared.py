"""Attention of single queries over the paged cache, with and without shared prefixes,
against fp64 within the bound of its roundings; then the operators in a run."""
from __future__ import annotations

import copy
import ctypes as C
import math
import os
import random
import subprocess
import sys
import tempfile

import pytest
import torch

from oasis_b200 import _lib, paged
from oracle import paged_oracle as O
from tests.helpers import ROOT

DEV = "cuda"
BF16, FP16 = torch.bfloat16, torch.float16


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def build(groups, page, heads_kv, dim, dtype, seed=0, layers=2):
    """A cache with a scattered table. groups: (prefix pages, [length of each row])."""
    rng = random.Random(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    lists, lengths = [], []
    need = sum(p + sum(-(-max(0, t - p * page) // page) for t in ls) for p, ls in groups)
    order = list(range(need + 3))
    rng.shuffle(order)
    take = lambda n: [order.pop() for _ in range(n)]  # noqa: E731
    for p, ls in groups:
        common = take(p)
        for t in ls:
            lists.append((common + take(-(-max(0, t - p * page) // page)))[: -(-t // page)])
            lengths.append(t)
    n = len(lists)
    slots = list(range(n + 2))
    rng.shuffle(slots)
    seqs = slots[:n]
    width = max(1, max(len(x) for x in lists))
    c = paged.PagedCache(need + 3, page, layers, heads_kv, dim, n + 2, width, dtype=dtype, device=DEV)
    c.pool.normal_(generator=g)
    for s, pages, t in zip(seqs, lists, lengths):
        c.table[s, : len(pages)] = ints(pages)
        c.lengths[s] = t
    plan = paged.SharedPlan([len(ls) for _, ls in groups], [p for p, _ in groups], max(lengths), DEV)
    return c, seqs, plan, g


def queries(n, heads, dim, dtype, gen, scale=2.0):
    return torch.empty(n, heads, dim, dtype=dtype, device=DEV).normal_(generator=gen).mul_(scale)


def check(got, q, c, layer, seqs, scale=None, rows=None):
    table, lengths = c.table.tolist(), c.lengths.tolist()
    want = O.attention_cached(q, c.pool, table, lengths, layer, seqs, scale)
    absolute = c.pool.clone()
    absolute[:, :, 1] = absolute[:, :, 1].abs()
    spread = O.attention_cached(q, absolute, table, lengths, layer, seqs, scale)
    scale_ = q.shape[2] ** -0.5 if scale is None else scale
    finite = torch.nan_to_num(c.pool[:, layer, 0].double(), 0, 0, 0)
    finite = torch.where(finite.abs() > 1e30, 0, finite)  # such a key's probability is 0
    reach = scale_ * float(torch.nan_to_num(q.double()).norm(dim=-1).max() * finite.norm(dim=-1).max())
    bound = O.error_bound(want, spread, reach, max(lengths), q.shape[2], q.dtype)
    off = (got.double() - want).abs()
    rows = slice(None) if rows is None else rows
    assert bool((off <= bound)[rows].all()), float((off / bound)[rows].max())
    return want


# ----------------------------------------------------------------- without a GPU --

def _args(cache=None, **kw):
    c = dict(pool=16, pages=4, layers=1, kv_heads=1, page_size=16, head_dim=64, dtype=1, table=16, slots=2, width=2,
             lengths=16, refs=16, status=16)
    c.update(cache or {})
    keep = _lib.OasisPageCache(**c)
    a = dict(q=16, out=16, q_row_stride=64, q_head_stride=64, out_row_stride=64, out_head_stride=64,
             cache=C.pointer(keep), layer=0, seqs=16, rows=1, heads=1, scale=0.125)
    a.update(kw)
    return _lib.OasisSharedArgs(**a), keep


@pytest.mark.parametrize("cache,kw,text", [
    (dict(dtype=0), {}, b"dtype"), (dict(head_dim=96), {}, b"head_dim=96"), (dict(page_size=8), {}, b"page_size=8"),
    (dict(width=1 << 30), {}, b"too large"), (dict(pool=0), {}, b"null"), (dict(pool=8), {}, b"16-byte"),
    ({}, dict(layer=1), b"layer=1"), ({}, dict(layer=-1), b"layer=-1"), (dict(kv_heads=2), dict(heads=3), b"heads=3"),
    ({}, dict(rows=-1), b"rows=-1"), ({}, dict(groups=-1), b"groups=-1"), ({}, dict(scale=0.0), b"scale"),
    ({}, dict(scale=math.nan), b"scale"), ({}, dict(q=0), b"null"), ({}, dict(out=24), b"16-byte"),
    ({}, dict(q_row_stride=4), b"stride"), ({}, dict(groups=1), b"group arrays"),
    (dict(kv_heads=4), dict(rows=1 << 30, heads=4), b"too many"),
])
def test_arguments_are_checked(cache, kw, text):
    a, _ = _args(cache, **kw)
    lib = _lib.load()
    assert lib.oasis_attention_shared(C.byref(a), None) == -1
    assert text in lib.oasis_last_error()


def test_workspace_is_asked_for():
    lib = _lib.load()
    a, _ = _args(rows=2, groups=1, group_start=16, prefix_pages=16, group_rows_hint=2, prefix_pages_hint=40)
    assert lib.oasis_attention_shared_workspace_size(C.byref(a)) == 0  # each row by itself, in one range
    a, _ = _args(rows=2, groups=1, group_start=16, prefix_pages=16, group_rows_hint=2, prefix_pages_hint=20000)
    size = lib.oasis_attention_shared_workspace_size(C.byref(a))
    assert size > 0
    for ws, n in ((0, size), (16, size - 1)):
        a.workspace, a.workspace_bytes = ws, n
        assert lib.oasis_attention_shared(C.byref(a), None) == -3 and b"workspace" in lib.oasis_last_error()
    a, _ = _args(rows=0)
    assert lib.oasis_attention_shared_workspace_size(C.byref(a)) == 0
    assert lib.oasis_attention_shared(C.byref(a), None) == 0
    assert lib.oasis_attention_shared(None, None) == -1


def test_workspace_of_the_largest_hints():
    """As many groups as rows save nothing: hints of any size ask for ranges of rows that exist."""
    lib, most = _lib.load(), (1 << 31) - 1
    for groups in (1, 2):
        a, _ = _args(rows=2, groups=groups, group_start=16, prefix_pages=16, group_rows_hint=most,
                     prefix_pages_hint=most, own_tokens_hint=most)
        assert 0 <= lib.oasis_attention_shared_workspace_size(C.byref(a)) <= 2 * 128 * (64 * 4 + 8)


def test_struct_layout_matches_c():
    with tempfile.TemporaryDirectory() as d:
        lines = [f'printf("%zu\\n", offsetof(OasisSharedArgs, {f}));' for f, _ in _lib.OasisSharedArgs._fields_]
        f, exe = os.path.join(d, "l.c"), os.path.join(d, "l")
        open(f, "w").write('#include <stdio.h>\n#include <stddef.h>\n' + f'#include "{ROOT}/include/oasis_b200.h"\n'
                           + "int main(void) {" + "".join(lines) + 'printf("%zu\\n", sizeof(OasisSharedArgs)); return 0; }')
        subprocess.run(["gcc", "-std=c99", f, "-o", exe], check=True)
        got = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    want = [getattr(_lib.OasisSharedArgs, f).offset for f, _ in _lib.OasisSharedArgs._fields_]
    assert got == want + [C.sizeof(_lib.OasisSharedArgs)]


def test_plan_is_checked():
    with pytest.raises(ValueError, match="group_rows"):
        paged.SharedPlan([1, 2], [3], 10, "cpu")
    with pytest.raises(ValueError, match="group_rows"):
        paged.SharedPlan([1, -2], [3, 0], 10, "cpu")


# --------------------------------------------------------------------- on a GPU --

# How a call is carried out goes by its sizes: small batches read each row by itself, larger
# ones run one of three kernels for the prefix. These make a small batch take each way.
WAYS = ["as it is", "tensor memory", "mma", "one pass"]


def run(way, q, c, layer, seqs, plan):
    """The call with hints, and with rows of an empty sequence behind the plan's, that
    lead it the given way; the results of the rows in `seqs`."""
    hints, extra = (plan.longest, plan.most_pages), 0
    heads = q.shape[1]
    if way == "tensor memory":
        plan.most_pages = 1 << 16
    elif way != "as it is":
        read = max(1, plan.most_pages) * c.page_size * c.kv_heads * c.head_dim * 4
        extra = 120_000_000 // read + plan.groups + (20_000 // heads if way == "one pass" else 0)
        plan.longest = 1 if way == "one pass" else 1 << 20
    lengths = c.lengths.tolist()
    empty = next(s for s in range(c.sequences) if lengths[s] == 0)
    more = torch.zeros(extra, heads, c.head_dim, dtype=q.dtype, device=DEV)
    got = paged.attention_shared(torch.cat([q, more]), c, layer, ints(list(seqs) + [empty] * extra), plan)
    plan.longest, plan.most_pages = hints
    assert not bool(got[len(seqs) :].any())
    return got[: len(seqs)]


GROUPS = {
    "long prefix": [(33, [600, 540, 528]), (80, [1290, 1281])],
    "long and short": [(40, [645, 100, 0, 700, 639, 641]), (2, [33])],
    "one row": [(0, [1])],
    "lengths": [(0, [1, 15, 16, 17, 0, 64, 65, 200])],
    "prefix": [(2, [33, 40, 32, 64])],
    "no own": [(3, [48, 48])],
    "several": [(1, [20, 17]), (0, [5, 0, 31]), (9, [145, 300, 151]), (2, [32])],
    "shorter than the prefix": [(4, [10, 64, 0, 50, 90])],
    "all short": [(4, [10, 0, 20])],
    "many rows": [(5, [80 + i % 7 for i in range(70)])],
    "long": [(60, [1000, 1900, 961]), (0, [1500, 3])],
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", GROUPS)
@pytest.mark.parametrize("heads,kv,dim,dtype,page", [
    (2, 2, 64, BF16, 16), (6, 2, 128, BF16, 16), (4, 1, 64, FP16, 32), (7, 1, 128, FP16, 48), (40, 2, 64, BF16, 64),
])
def test_groups(name, heads, kv, dim, dtype, page):
    groups = [(-(-p * 16 // page), [t if t < p * 16 else t + (-(-p * 16 // page)) * page - p * 16 for t in ls])
              for p, ls in GROUPS[name]]
    c, seqs, plan, g = build(groups, page, kv, dim, dtype)
    q = queries(len(seqs), heads, dim, dtype, g)
    for way in WAYS:
        check(run(way, q, c, 1, seqs, plan), q, c, 1, seqs)
    alone = paged.SharedPlan([], [], plan.longest, DEV)
    check(paged.attention_shared(q, c, 1, ints(seqs), alone), q, c, 1, seqs)
    c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,dim,dtype,page", [(32, 16, 64, BF16, 16), (20, 20, 128, FP16, 32), (112, 16, 64, FP16, 48)])
@pytest.mark.parametrize("shape", ["forks", "ragged", "alone"])
def test_many_rows_with_few_keys(shape, heads, kv, dim, dtype, page):
    """Enough rows for the one-pass kernel: groups inside, across and larger than a tile,
    short and empty rows, rows in no group."""
    rng = random.Random(7)
    n = 64 * 20 * kv // heads
    if shape == "forks":
        groups = [(1, [page + rng.randint(1, page) for _ in range(16)]) for _ in range(n // 16)]
    elif shape == "ragged":
        groups, left = [], n
        while left > 0:
            r = min(left, rng.choice([1, 2, 5, 150]))
            p = rng.choice([0, 1, 3])
            groups.append((p, [rng.choice([0, 3, p * page, p * page + rng.randint(1, 40)]) for _ in range(r)]))
            left -= r
    else:
        groups = [(0, [rng.randint(0, 50) for _ in range(n)])]
    c, seqs, plan, g = build(groups, page, kv, dim, dtype, layers=1)
    if shape == "ragged":  # the last rows belong to no group
        plan.group_start[-1] -= 1
    q = queries(len(seqs), heads, dim, dtype, g)
    got = paged.attention_shared(q, c, 0, ints(seqs), plan)
    check(got, q, c, 0, seqs)
    assert torch.equal(got, paged.attention_shared(q, c, 0, ints(seqs), plan))
    c.pool[:, :, 1, :, -1] = math.nan  # values behind many rows' last token, seen by others
    got = paged.attention_shared(q, c, 0, ints(seqs), plan)
    want = O.attention_cached(q, c.pool, c.table.tolist(), c.lengths.tolist(), 0, seqs)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and bool(torch.isnan(want).any())
    fine = ~torch.isnan(want).reshape(len(seqs), -1).any(1)
    c.pool[:, :, 1] = torch.nan_to_num(c.pool[:, :, 1])
    check(got, q, c, 0, seqs, rows=fine)
    c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,heads,kv,dim,dtype,page", [
    (300, 2, 2, 64, BF16, 16), (70, 12, 3, 128, BF16, 64), (40, 7, 1, 64, FP16, 48), (140, 2, 1, 128, FP16, 128), (3, 4, 4, 64, BF16, 256),
    (40, 28, 4, 64, FP16, 48), (60, 4, 4, 64, BF16, 256),
])
def test_long_prefixes(rows, heads, kv, dim, dtype, page):
    """The tensor-memory kernel: both tiles, several ranges, pages above and below a block,
    rows of different limits, a page of the prefix that is not in the pool, hints that are
    too small."""
    rng = random.Random(rows)
    first = -(-900 // page)
    groups = [(first, [first * page + rng.choice([-200, 0, 1, 33]) for _ in range(rows - 1)] + [first * page + 5]),
              (-(-300 // page), [-(-300 // page) * page + 2] * 2)]
    c, seqs, plan, g = build(groups, page, kv, dim, dtype)
    q = queries(len(seqs), heads, dim, dtype, g)
    good = paged.attention_shared(q, c, 1, ints(seqs), plan)
    check(good, q, c, 1, seqs)
    assert torch.equal(good, paged.attention_shared(q, c, 1, ints(seqs), plan))
    plan.most_rows, pages = 1, plan.most_pages
    check(paged.attention_shared(q, c, 1, ints(seqs), plan), q, c, 1, seqs)
    plan.most_rows, plan.most_pages = rows, 10 * pages
    check(paged.attention_shared(q, c, 1, ints(seqs), plan), q, c, 1, seqs)
    plan.most_pages = pages
    shared = int(c.table[seqs[0], 1])
    c.pool[shared, 1, 0, 0, 3, :] = math.nan  # a key of the prefix
    got = paged.attention_shared(q, c, 1, ints(seqs), plan)
    want = O.attention_cached(q, c.pool, c.table.tolist(), c.lengths.tolist(), 1, seqs)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and bool(torch.isnan(want).any())
    c.pool[shared, 1, 0, 0, 3, :] = 0
    c.check()
    c.table[torch.tensor(seqs[:rows], device=DEV), 1] = -7  # left out of the sum, for all rows alike
    got = paged.attention_shared(q, c, 1, ints(seqs), plan)
    torch.cuda.synchronize()
    assert int(c.status.item()) == paged.BAD_PAGE
    table, lengths = c.table.tolist(), c.lengths.tolist()
    for b in (0, rows - 1):
        s = seqs[b]
        pages = [p for i, p in enumerate(table[s][: -(-lengths[s] // page)]) if i != 1]
        kv_rows = c.pool[pages, 1].permute(1, 2, 0, 3, 4).reshape(2, kv, -1, dim)[:, :, : lengths[s] - page]
        want = O.attention_rows(q[b : b + 1], kv_rows[0].transpose(0, 1), kv_rows[1].transpose(0, 1))
        assert float((got[b].double() - want[0]).norm() / want.norm()) < 2 * torch.finfo(dtype).eps
    assert _lib.load().oasis_device_error(0) == 0


RANGES = {  # (page, groups, key heads)
    # own keys in one range that joins the ranges of a long prefix; a row that ends inside it
    "one range": (64, lambda r: [(33, [2112 + n for n in (900, 5, 1, 440)] + [1000, 0])], 16),
    # a warp for each item, beside a prefix on part of the SMs
    "one warp": (16, lambda r: [(40, [640 + r.randint(0, 60) for _ in range(300)]), (0, [r.randint(0, 90) for _ in range(9)])], 8),
    # rows of thousands of tokens, ragged, without a common prefix
    "long rows": (128, lambda r: [(0, [5000, 17, 0, 2049, 1024, 1025, 300])], 2),
    # many groups of few rows: their prefixes are too short for tensor memory
    "many groups": (16, lambda r: [(25, [400 + r.randint(0, 30) for _ in range(r.randint(1, 4))]) for _ in range(100)], 8),
    # ranges of own keys behind a prefix in ranges
    "both": (32, lambda r: [(70, [2240 + 20 * n for n in range(60)]), (3, [1900, 96, 97])], 3),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", RANGES)
@pytest.mark.parametrize("per,dim,dtype", [(1, 64, BF16), (4, 128, FP16), (9, 64, FP16)])
def test_ranges(name, per, dim, dtype):
    """Each way that prefixes and own keys are split, with an infinity behind the rows' ends."""
    page, groups, kv = RANGES[name]
    c, seqs, plan, g = build(groups(random.Random(5)), page, kv, dim, dtype, layers=1)
    q = queries(len(seqs), per * kv, dim, dtype, g)
    got = paged.attention_shared(q, c, 0, ints(seqs), plan)
    check(got, q, c, 0, seqs)
    assert torch.equal(got, paged.attention_shared(q, c, 0, ints(seqs), plan))
    table, lengths = c.table.tolist(), c.lengths.tolist()
    for s in seqs:  # a last page that no other row reads ends behind its row's last token
        t = lengths[s]
        if t % page and sum(table[s][t // page] in row for row in table) == 1:
            c.pool[table[s][t // page], 0, :, :, t % page :] = math.inf
    graph, at = torch.cuda.CUDAGraph(), ints(seqs)
    with torch.cuda.graph(graph):
        again = paged.attention_shared(q, c, 0, at, plan)
    for _ in range(3):
        again.zero_()
        graph.replay()
    check(again, q, c, 0, seqs)
    c.check()


@pytest.mark.gpu
def test_hints_only_choose_the_split():
    c, seqs, plan, g = build([(30, [500, 900, 700]), (0, [1200])], 16, 2, 64, BF16)
    q = queries(4, 4, 64, BF16, g)
    most = (1 << 31) - 1
    for longest, rows, pages in ((1, 1, 1), (1 << 20, 1000, 1), (900, 1, 4000), (10, 3, 0), (most, 1, 1)):
        plan.longest, plan.most_rows, plan.most_pages, plan.least_pages = longest, rows, pages, 0
        check(paged.attention_shared(q, c, 0, ints(seqs), plan), q, c, 0, seqs)


@pytest.mark.gpu
@pytest.mark.parametrize("way", WAYS)
def test_rows_outside_the_groups_and_named_twice(way):
    c, seqs, _, g = build([(2, [40, 50, 33])], 16, 1, 64, BF16)
    plan = paged.SharedPlan([2], [2], 64, DEV)
    plan.group_start += 1  # rows 1 and 2
    order = [seqs[2], seqs[0], seqs[1], seqs[0], seqs[2]]
    q = queries(5, 2, 64, BF16, g)
    check(run(way, q, c, 0, order, plan), q, c, 0, order)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("way", WAYS)
def test_what_lies_behind_a_sequence_takes_no_part(way, dim, bad):
    """NaN in pages behind a sequence's last token, and in the prefix behind a shorter
    row; NaN and empty results where the formula has them."""
    groups = [(3, [20, 70, 52, 0, 48]), (0, [7])]
    c, seqs, plan, g = build(groups, 16, 2, dim, BF16)
    lists, lengths = c.table.tolist(), c.lengths.tolist()
    for s in seqs:
        t = lengths[s]
        if t % 16 and t >= 48 or t == 7:
            c.pool[lists[s][t // 16], :, :, :, t % 16:] = bad
    unused = [p for p in range(c.pages) if all(p not in r for r in lists)]
    c.pool[unused] = bad
    q = queries(6, 6, dim, BF16, g)
    got = run(way, q, c, 0, seqs, plan)
    check(got, q, c, 0, seqs)
    c.pool[lists[seqs[1]][2], :, :, :, 5] = bad  # token 37 of the prefix: rows 1, 2 and 4 see it, row 0 does not
    got = run(way, q, c, 0, seqs, plan)
    want = check(got, q, c, 0, seqs, rows=[0, 3, 5])
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and bool(torch.isnan(want[[1, 2, 4]]).any())
    q[1] = math.nan
    got = run(way, q, c, 0, seqs, plan)
    check(got, q, c, 0, seqs, rows=[0, 3, 5])
    assert bool(torch.isnan(got[1]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("way", WAYS)
def test_lowest_scores(way):
    """Keys that score -inf or the lowest value: in the whole prefix, in a row's own part."""
    c, seqs, plan, g = build([(4, [70, 100])], 16, 1, 64, BF16)
    q = queries(2, 2, 64, BF16, g)
    q[:, :, 0] = 1
    c.pool[..., 0] = torch.where(torch.arange(2, device=DEV)[None, None, :, None, None] == 0, 0, c.pool[..., 0])
    common = c.table[seqs[0], :4].long()
    c.pool[common, :, 0, :, :, 0] = -math.inf
    check(run(way, q, c, 0, seqs, plan), q, c, 0, seqs)
    c.pool[common, :, 0, :, :, 0] = torch.finfo(BF16).min
    check(run(way, q, c, 0, seqs, plan), q, c, 0, seqs)
    c.pool[:, :, 0, :, :, 0] = -math.inf
    assert bool(torch.isnan(run(way, q, c, 0, seqs, plan)).all())  # as the formula: 0 / 0


@pytest.mark.gpu
@pytest.mark.parametrize("way", WAYS)
def test_bad_indexes_are_left_out(way):
    c, seqs, plan, g = build([(2, [40, 40]), (0, [64, 20])], 16, 1, 64, BF16)
    q = queries(4, 1, 64, BF16, g)
    good = run(way, q, c, 0, seqs, plan)
    table = c.table.clone()
    c.table[seqs[2], 1] = 1 << 30
    c.table[seqs[3], :2] = ints([-1, c.pages])
    got = run(way, q, c, 0, [seqs[0], 99, seqs[2], seqs[3]], plan)
    torch.cuda.synchronize()
    assert torch.equal(got[0], good[0]) and not bool(got[1].any()) and not bool(got[3].any())
    assert int(c.status.item()) == paged.BAD_SEQUENCE | paged.BAD_PAGE
    c.table.copy_(table)
    pages = c.table[seqs[2], :4].tolist()
    short = O.attention_rows(q[2:3], c.pool[[pages[0], pages[2], pages[3]], 0, 0].transpose(1, 2).reshape(-1, 1, 64),
                             c.pool[[pages[0], pages[2], pages[3]], 0, 1].transpose(1, 2).reshape(-1, 1, 64))
    assert float((got[2].double() - short[0]).norm() / short.norm()) < 2 * 2.0 ** -8


@pytest.mark.gpu
def test_strides_streams_graph():
    c, seqs, plan, g = build([(20, [330, 400]), (0, [100])], 16, 2, 64, BF16)
    rows = torch.empty(3, 8, 64, dtype=BF16, device=DEV).normal_(generator=g)
    q = rows[:, 2:6]  # a view of packed rows
    out = torch.zeros(4, 3, 2, 64, dtype=BF16, device=DEV)[:, :, 0].transpose(0, 1)  # heads outside
    at = ints(seqs)
    paged.attention_shared(q, c, 1, at, plan, out=out)
    check(out, q, c, 1, seqs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    a = paged.attention_shared(q, c, 1, at, plan, stream=side)
    b = paged.attention_shared(q, c, 1, at, plan)  # beside it, each with its own workspace
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, b) and torch.equal(a, out)
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(paged.attention_shared(q, c, 1, at, plan))
        graphs.append(gr)
    side.wait_stream(torch.cuda.current_stream())
    for gr in graphs:
        gr.replay()
    with torch.cuda.stream(side):
        graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], a) and torch.equal(outs[1], a)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A pool of more than 2^32 bytes: pages at its far end."""
    c = paged.PagedCache(4100, 64, 8, 8, 128, 2, 3, device=DEV)  # 8.6 GB
    assert c.pool.numel() > 1 << 32
    pages = [4099, 0, 4098]
    g = torch.Generator(device=DEV).manual_seed(1)
    for p in pages:
        c.pool[p].normal_(generator=g)
    c.table[1] = ints(pages)
    c.lengths[1] = 150
    c.refs[pages] = 1
    q = queries(1, 8, 128, BF16, g)
    small = paged.PagedCache(3, 64, 8, 8, 128, 2, 3, device=DEV)
    small.pool.copy_(c.pool[pages])
    small.table[1] = ints([0, 1, 2])
    small.lengths[1] = 150
    plan = paged.SharedPlan([1], [2], 192, DEV)
    a = paged.attention_shared(q, c, 7, ints([1]), plan)
    b = paged.attention_shared(q, small, 7, ints([1]), plan)
    assert torch.equal(a, b)
    check(b, q, small, 7, [1])
    rows = torch.empty(10, 8, 128, dtype=BF16, device=DEV).normal_(generator=g)
    for x in (c, small):
        start = x.reserve(ints([1]), ints([0, 10]))
        x.write(7, rows, rows, ints([1]), ints([0, 10]), start)
    assert torch.equal(c.pool[4098], small.pool[2])
    c.compact()  # the far pages move to 1 and 2
    assert c.table[1].tolist() == [1 if p == 4098 else 2 if p == 4099 else 0 for p in pages]
    assert torch.equal(c.pool[c.table[1].long()], small.pool)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, FP16)])
def test_a_run_of_them_together(dim, dtype):
    """Two prompts enter, are forked, grow token by token, one branch ends, the pool is
    compacted and the rest goes on: each step's attention against fp64 over the
    tokens that each sequence really holds."""
    rng = random.Random(3)
    heads, kv, page, layers = 6, 2, 16, 2
    c = paged.PagedCache(40, page, layers, kv, dim, 8, 10, dtype=dtype, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(4)
    held = {}  # sequence -> per layer list of (k, v) rows

    def rows(n):
        return torch.empty(layers, n, heads + 2 * kv, dim, dtype=dtype, device=DEV).normal_(generator=g)

    lengths = [70, 37]
    x = rows(sum(lengths))
    cu = [0, 70, 107]
    start = c.reserve(ints([0, 1]), ints(cu))
    for layer in range(layers):
        q, k, v = x[layer, :, :heads], x[layer, :, heads : heads + kv], x[layer, :, heads + kv :]
        got = paged.attention_prompt(q, k, v, ints(cu), 70)
        want, spread = O.attention_prompt(q, k, v, cu), O.attention_prompt(q, k, v.abs(), cu)
        reach = dim ** -0.5 * float(q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max())
        assert bool(((got.double() - want).abs() <= O.error_bound(want, spread, reach, 70, dim, dtype)).all())
        c.write(layer, k, v, ints([0, 1]), ints(cu), start)
    for i, s in enumerate((0, 1)):
        held[s] = x[:, cu[i] : cu[i + 1], heads:].clone()
    c.fork(ints([0, 0, 1]), ints([2, 3, 4]))
    for s, t in ((0, 2), (0, 3), (1, 4)):
        held[t] = held[s].clone()
    order, plan = [0, 2, 3, 1, 4], paged.SharedPlan([3, 2], [70 // page, 37 // page], 100, DEV)
    for step in range(24):
        if step == 9:  # a branch ends
            c.free(ints([2]))
            del held[2]
            order, plan = [0, 3, 1, 4], paged.SharedPlan([2, 2], [70 // page, 37 // page], 100, DEV)
            c.compact()
        if step == 15:  # and its slot takes a copy of another
            c.fork(ints([3]), ints([2]), deep=True)
            held[2] = held[3].clone()
            order, plan = [0, 3, 1, 4, 2], paged.SharedPlan([2, 2], [70 // page, 37 // page], 100, DEV)
        n = len(order)
        x = rows(n)
        one = list(range(n + 1))
        start = c.reserve(ints(order), ints(one))
        for layer in range(layers):
            c.write(layer, x[layer, :, heads : heads + kv], x[layer, :, heads + kv :], ints(order), ints(one), start)
            got = paged.attention_shared(x[layer, :, :heads], c, layer, ints(order), plan)
            for i, s in enumerate(order):
                if layer == 0:
                    held[s] = torch.cat([held[s], x[:, i : i + 1, heads:]], 1)
                k, v = held[s][layer, :, :kv], held[s][layer, :, kv:]
                q = x[layer, i : i + 1, :heads]
                want, spread = O.attention_rows(q, k, v), O.attention_rows(q, k, v.abs())
                reach = dim ** -0.5 * float(q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max())
                bound = O.error_bound(want, spread, reach, k.shape[0], dim, dtype)
                assert bool(((got[i : i + 1].double() - want).abs() <= bound).all()), (step, layer, s)
    c.check()
    assert sorted(c.lengths.tolist()) == sorted(held[s].shape[1] if s in held else 0 for s in range(8))
    c.free(ints(list(range(8))))
    assert not bool(c.refs.any()) and rng


@pytest.mark.gpu
def test_python_checks():
    c, seqs, plan, g = build([(1, [20, 20])], 16, 1, 64, BF16)
    q = queries(2, 1, 64, BF16, g)
    at = ints(seqs)
    call = paged.attention_shared
    for args, text in (((q.half(), c, 0, at, plan), "q must be"), ((q[:1], c, 0, at, plan), "seqs must hold 1"),
                       ((q, c, 0, at.long(), plan), "int32"), ((q[:1], c, 0, at[:1], plan), "plan is for 2"),
                       ((q.cpu(), c, 0, at, plan), "CUDA")):
        with pytest.raises(ValueError, match=text):
            call(*args)
    with pytest.raises(ValueError, match="out has 3"):
        call(q, c, 0, at, plan, out=torch.zeros(3, 1, 64, dtype=BF16, device=DEV))
    with pytest.raises(_lib.OasisError, match="layer=2"):
        call(q, c, 2, at, plan)
    assert call(q[:0], c, 0, at[:0], paged.SharedPlan([], [], 1, DEV)).shape == (0, 1, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, BF16), (64, FP16)])
@pytest.mark.parametrize("way", WAYS)
def test_large_values_that_are_not_seen_change_no_bit(way, dim, dtype):
    """Finite keys and values up to the type's largest behind a sequence's last token and in
    the prefix behind a shorter row: the rows that do not see them keep every bit that they
    have with zeros there."""
    groups = [(15, [250, 100, 0, 17, 241, 242]), (15, [230, 225]), (0, [7])]
    c, seqs, plan, g = build(groups, 16, 2, dim, dtype)
    lists, lengths = c.table.tolist(), c.lengths.tolist()
    places = [(lists[seqs[0]][t // 16], t % 16) for t in range(100, 240)]  # rows 0, 4 and 5 see these
    for b in (0, 4, 5, 6, 8):
        t = lengths[seqs[b]]
        places += [(lists[seqs[b]][t // 16], x) for x in range(t % 16, 16)]
    pages, slots = (torch.tensor(x, device=DEV) for x in zip(*places))
    q = queries(len(seqs), 6, dim, dtype, g)
    blind = [1, 2, 3, 6, 7, 8]
    fill = lambda x: c.pool.__setitem__((pages, slice(None), slice(None), slice(None), slots), x)  # noqa: E731
    fill(0)
    want = run(way, q, c, 0, seqs, plan)
    check(want, q, c, 0, seqs)
    for size in (1e30, 1e36, 3.3e38) if dtype == BF16 else (6e4,):
        fill(size)
        assert torch.equal(run(way, q, c, 0, seqs, plan)[blind], want[blind]), size
    c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("at", [128, 129, 256, 260])
def test_a_score_of_nan_alone_in_a_range(way, dim, at):
    """A shorter row's last token in the prefix is a NaN key at or near the start of a range,
    so that its range may hold no other key that it sees: its result is NaN all the same."""
    c, seqs, plan, g = build([(20, [at + 1, 400, at])], 16, 2, dim, BF16)
    page = c.table[seqs[1]].tolist()[at // 16]
    c.pool[page, 0, 0, :, at % 16, 5] = math.nan
    q = queries(3, 4, dim, BF16, g)
    got = run(way, q, c, 0, seqs, plan)
    assert bool(torch.isnan(got[:2]).all())
    check(got, q, c, 0, seqs, rows=[2])


@pytest.mark.parametrize("hints", [
    dict(group_rows_hint=1 << 30, prefix_pages_hint=15), dict(group_rows_hint=(1 << 31) - 1, prefix_pages_hint=15),
    dict(group_rows_hint=1 << 30, prefix_pages_hint=1000), dict(group_rows_hint=(1 << 31) - 1, prefix_pages_hint=1000),
])
def test_a_group_hint_beyond_the_batch_is_the_batch(hints):
    """A group has no more rows than the batch, whatever the hint: the same workspace, and no
    count that overflows. In a process of its own, which a division by zero would end."""
    code = f'''
import ctypes as C, sys
sys.path.insert(0, {ROOT!r})
import __graft_entry__
__graft_entry__.load_package()
from tests.test_attention_shared import _args
from oasis_b200 import _lib
lib, sizes = _lib.load(), []
for heads in (256, 128, 3):
    for rows in (2000, 1 << 22):
        for hint in ({hints["group_rows_hint"]}, rows):
            a, keep = _args(dict(width=4096), rows=rows, heads=heads, groups=2, group_start=16, prefix_pages=16,
                            group_rows_hint=hint, prefix_pages_hint={hints["prefix_pages_hint"]}, own_tokens_hint=5000)
            sizes.append(lib.oasis_attention_shared_workspace_size(C.byref(a)))
            a.workspace, a.workspace_bytes = 16, 8  # too small: refused before anything is launched
            sizes[-1] = sizes[-1], lib.oasis_attention_shared(C.byref(a), None), lib.oasis_last_error()
print(sizes[0::2] == sizes[1::2], all(x[0] > 8 and x[1] == -3 for x in sizes))
'''
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert run.returncode == 0 and run.stdout.split() == ["True", "True"], (run.returncode, run.stdout, run.stderr[-500:])


@pytest.mark.parametrize("kw,rc,text", [
    (dict(rows=(1 << 31) - 1, heads=1024), -1, b"too many"),
    (dict(rows=1 << 20, heads=1024, groups=1 << 19), -3, b"workspace"),  # mostly empty groups
    (dict(rows=1 << 20, heads=1024, groups=3, group_rows_hint=-5), -3, b"workspace"),
])
def test_batches_of_any_size_are_launched_or_refused(kw, rc, text):
    """The most rows, heads and groups that the arguments hold overflow no count."""
    lib = _lib.load()
    rest = dict(groups=1, group_start=16, prefix_pages=16, group_rows_hint=(1 << 31) - 1, prefix_pages_hint=15,
                own_tokens_hint=5000, workspace=16, workspace_bytes=8)
    a, _ = _args(dict(width=4096), **{**rest, **kw})
    assert lib.oasis_attention_shared(C.byref(a), None) == rc and text in lib.oasis_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("way", WAYS)
def test_the_largest_group_hint(way):
    c, seqs, plan, g = build([(15, [250, 300, 241]), (20, [330, 400])], 16, 2, 64, BF16)
    q = queries(5, 16, 64, BF16, g)
    want = run(way, q, c, 0, seqs, plan)
    check(want, q, c, 0, seqs)
    plan.most_rows = (1 << 31) - 1
    got = run(way, q, c, 0, seqs, plan)
    check(got, q, c, 0, seqs)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("way", WAYS)
def test_values_whose_sum_overflows(way, dim):
    """Values near the type's largest: their weighted mean is finite, their sum is not."""
    c, seqs, plan, g = build([(15, [250, 100, 0, 17, 241]), (0, [7, 1])], 16, 2, dim, BF16)
    c.pool[:, :, 1].uniform_(1e38, 3e38, generator=g)
    c.pool[:, :, 1, :, :, 1::2] *= -1
    q = queries(len(seqs), 4, dim, BF16, g)
    check(run(way, q, c, 0, seqs, plan), q, c, 0, seqs)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("way", WAYS)
def test_values_of_keys_that_weigh_nothing(way, dim):
    """Keys that a row sees and that score thousands below its others: whatever finite value
    they have, none of it is in the result."""
    c, seqs, plan, g = build([(15, [250, 300, 0, 17, 241]), (0, [40])], 16, 2, dim, BF16)
    q = queries(len(seqs), 4, dim, BF16, g)
    q[:, :, 0] = 1
    c.pool[:, :, 0, :, :, 0] = 0
    c.pool[:, :, 0, :, 1::3, 0] = -3e4
    c.pool[:, :, 1, :, 1::3] = 3e38
    check(run(way, q, c, 0, seqs, plan), q, c, 0, seqs)


@pytest.mark.gpu
@pytest.mark.parametrize("name,pages,longest", [
    ("alone", 0, 400), ("alone in ranges", 0, 1 << 14), ("tensor memory", 1 << 16, 300), ("tensor memory in ranges", 1 << 11, 1 << 16),
    ("mma", 15, 300), ("mma in ranges", 15, 1 << 14),
])
def test_steps_without_a_pause(name, pages, longest):
    """Decoding steps queued one behind the other, kernels of a step starting while the last
    one ends, leave the bits of the same steps with a wait between all calls."""
    rows, kv, steps = 40, 16, 60
    g = torch.Generator(device=DEV).manual_seed(8)
    c = paged.PagedCache(400, 16, 1, kv, 64, rows, 24, device=DEV)
    new = torch.empty(250, 2 * kv, 64, dtype=BF16, device=DEV).normal_(generator=g)
    start = c.reserve(ints([0]), ints([0, 250]))
    c.write(0, new[:, :kv], new[:, kv:], ints([0]), ints([0, 250]), start)
    c.fork(ints([0] * (rows - 1)), ints(list(range(1, rows))))
    seqs, one = ints(list(range(rows))), ints(list(range(rows + 1)))
    plan = paged.SharedPlan([rows], [15], longest, DEV)
    plan.most_pages = pages
    qkv = torch.empty(steps, rows, 3 * kv, 64, dtype=BF16, device=DEV).normal_(generator=g)

    def go(cache, wait):
        outs = []
        for x in qkv:
            at = cache.reserve(seqs, one)
            wait()
            cache.write(0, x[:, kv : 2 * kv], x[:, 2 * kv :], seqs, one, at)
            wait()
            outs.append(paged.attention_shared(x[:, :kv], cache, 0, seqs, plan))
            wait()
        return torch.stack(outs)

    other = copy.deepcopy(c)
    torch.cuda.synchronize()
    quick = go(c, lambda: None)
    slow = go(other, torch.cuda.synchronize)
    assert torch.equal(quick, slow)
    check(quick[-1], qkv[-1, :, :kv], c, 0, list(range(rows)))
    c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 48)])
@pytest.mark.parametrize("way", WAYS)
def test_a_sum_that_overflows_beside_pages_outside_the_pool(way, dim, page):
    """Rows that are worked out again leave out what lies outside the pool, and one that has
    nothing in it gives zeros."""
    c, seqs, plan, g = build([(2, [5 * page + 3, 3 * page]), (0, [4 * page, page + 1, 70])], page, 2, dim, BF16)
    c.pool[:, :, 1].uniform_(1e38, 3e38, generator=g)
    q = queries(len(seqs), 4, dim, BF16, g)
    c.table[seqs[0], 3] = -1
    c.table[seqs[2], 0], c.table[seqs[2], 2] = 1 << 30, c.pages
    c.table[seqs[3], :2] = ints([-1, -1])
    got = run(way, q, c, 0, seqs, plan)
    torch.cuda.synchronize()
    assert int(c.status.item()) == paged.BAD_PAGE
    table, lengths = c.table.tolist(), c.lengths.tolist()
    for b, s in enumerate(seqs):
        held = [(p, x) for t in range(lengths[s]) for p, x in [(table[s][t // page], t % page)] if 0 <= p < c.pages]
        if not held:
            assert b == 3 and not bool(got[b].any())
            continue
        pages, slots = (torch.tensor(x, device=DEV) for x in zip(*held))
        kv = c.pool[pages, 0, :, :, slots]  # [tokens, 2, heads, dim]
        want = O.attention_rows(q[b : b + 1], kv[:, 0], kv[:, 1])
        reach = dim ** -0.5 * float(q.double().norm(dim=-1).max() * kv[:, 0].double().norm(dim=-1).max())
        bound = O.error_bound(want, want, reach, len(held), dim, BF16)
        assert bool(((got[b : b + 1].double() - want).abs() <= bound).all()), b


@pytest.mark.gpu
@pytest.mark.parametrize("dim,dtype", [(64, FP16), (128, FP16), (64, BF16)])
@pytest.mark.parametrize("nats", [10, 14, 15.5])
@pytest.mark.parametrize("way", WAYS)
def test_one_key_outweighs_the_others(way, nats, dim, dtype):
    """A first token that takes nearly all of the weight and has a value of zero: what the
    others, `nats` below it, add is as exact as a probability's one rounding (the bound as for
    packed prompts)."""
    c, seqs, plan, g = build([(15, [250, 300, 1100, 241]), (0, [900, 70])], 16, 1, dim, dtype)
    c.pool.zero_()
    c.pool[:, :, 0, :, :, 0] = -nats * dim ** 0.5
    c.pool[:, :, 0, :, :, 1] = torch.empty(c.pool.shape[:2] + c.pool.shape[3:5], device=DEV).uniform_(-2, 2, generator=g)
    c.pool[:, :, 1] = 1
    for s in seqs:
        c.pool[int(c.table[s, 0]), :, :, :, 0] = 0
    q = torch.zeros(len(seqs), 2, dim, dtype=dtype, device=DEV)
    q[:, :, :2] = 1
    got = run(way, q, c, 0, seqs, plan)
    want = O.attention_cached(q, c.pool, c.table.tolist(), c.lengths.tolist(), 0, seqs)
    reach = dim ** -0.5 * float(q.double().norm(dim=-1).max() * c.pool[:, 0, 0].double().norm(dim=-1).max())
    allowed = 2.0 ** -24 * (1 + 2 * 1100) if dtype == FP16 else 2.0 ** -120
    bound = O.error_bound(want, want, reach, 1100, dim, dtype) - allowed + 2.0 ** (-25 if dtype == FP16 else -120)
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 48, 256])
@pytest.mark.parametrize("tokens", [150, 700])
@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, FP16)])
@pytest.mark.parametrize("way", WAYS)
def test_what_lies_behind_the_sequences_changes_no_bit(way, dim, dtype, tokens, page):
    """NaN and infinities behind the last token of a group's rows, also where all of them end
    inside the named prefix, leave every bit that zeros there leave: no row is worked out
    another way because of them."""
    n = -(-tokens // page)
    groups = [(n, [n * page - 7, n * page - 100, 0]), (n, [n * page + 5, n * page + 21]), (1, [9]), (0, [40, 3])]
    c, seqs, plan, g = build(groups, page, 2, dim, dtype, layers=1)
    q = queries(len(seqs), 6, dim, dtype, g)
    lists, lengths = c.table.tolist(), c.lengths.tolist()
    places = []
    for b in (0, 3, 4, 5, 6, 7):
        t = lengths[seqs[b]]
        places += [(lists[seqs[b]][t // page], x) for x in range(t % page, page)]
    pages, slots = (torch.tensor(x, device=DEV) for x in zip(*places))
    c.pool[pages, :, :, :, slots] = 0
    want = run(way, q, c, 0, seqs, plan)
    check(want, q, c, 0, seqs)
    for bad in (math.nan, math.inf, -math.inf):
        c.pool[pages, :, :, :, slots] = bad
        assert torch.equal(run(way, q, c, 0, seqs, plan), want)
    c.check()
