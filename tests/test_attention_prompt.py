"""Packed causal attention with grouped heads against fp64, element by element within
the bound of its roundings."""
from __future__ import annotations

import ctypes as C
import math
import os
import random
import subprocess
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


def starts(lengths, at=0):
    cu = [at]
    for n in lengths:
        cu.append(cu[-1] + n)
    return cu


def inputs(lengths, heads, kv, dim, dtype, seed=0, extra=0, scale=2.0):
    """q, k, v as views of packed rows, `extra` rows behind the last sequence."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    rows = torch.empty(sum(lengths) + extra, heads + 2 * kv, dim, dtype=dtype, device=DEV).normal_(generator=g)
    rows[:, :heads] *= scale
    return rows[:, :heads], rows[:, heads : heads + kv], rows[:, heads + kv :]


def check(got, q, k, v, cu, scale=None):
    scale_ = q.shape[2] ** -0.5 if scale is None else scale
    want, spread = O.attention_prompt(q, k, v, cu, scale), O.attention_prompt(q, k, v.abs(), cu, scale)
    for a, b in zip(cu, cu[1:]):
        if a == b:
            continue
        reach = scale_ * float(q[a:b].double().norm(dim=-1).max() * k[a:b].double().norm(dim=-1).max())
        bound = O.error_bound(want[a:b], spread[a:b], reach, b - a, q.shape[2], q.dtype)
        off = (got[a:b].double() - want[a:b]).abs()
        assert bool((off <= bound).all()), (a, b, float((off / bound).max()))


# ----------------------------------------------------------------- without a GPU --

def _args(**kw):
    a = dict(q=16, k=16, v=16, out=16, q_row_stride=64, q_head_stride=64, k_row_stride=64, k_head_stride=64,
             v_row_stride=64, v_head_stride=64, out_row_stride=64, out_head_stride=64, rows=4, cu=16, n=1, longest=4,
             heads=1, kv_heads=1, head_dim=64, dtype=1, scale=0.125)
    a.update(kw)
    return _lib.OasisPromptArgs(**a)


@pytest.mark.parametrize("field,value,text", [
    ("rows", -1, b"rows=-1"), ("n", -1, b"n=-1"), ("dtype", 0, b"dtype=0"), ("head_dim", 96, b"head_dim=96"),
    ("kv_heads", 0, b"kv_heads=0"), ("kv_heads", 2, b"kv_heads=2"), ("heads", 2048, b"heads=2048"),
    ("scale", 0.0, b"scale"), ("scale", math.nan, b"scale"), ("scale", -1.0, b"scale"), ("scale", math.inf, b"scale"),
    ("q", 0, b"null"), ("cu", 0, b"null"), ("out", 8, b"16-byte"), ("k", 24, b"16-byte"), ("k_row_stride", 68, b"stride"),
    ("out_head_stride", 0, b"stride"), ("v_head_stride", -64, b"stride"),
])
def test_arguments_are_checked(field, value, text):
    a = _args(**{field: value})
    lib = _lib.load()
    assert lib.oasis_attention_prompt(C.byref(a), None) == -1
    assert text in lib.oasis_last_error()


def test_nothing_to_do_and_too_much():
    lib = _lib.load()
    assert lib.oasis_attention_prompt(None, None) == -1
    assert lib.oasis_attention_prompt(C.byref(_args(rows=0, q=0)), None) == 0
    assert lib.oasis_attention_prompt(C.byref(_args(n=0, cu=0)), None) == 0
    assert lib.oasis_attention_prompt(C.byref(_args(rows=(1 << 31) - 1, heads=1024)), None) == -1
    assert b"too many" in lib.oasis_last_error()


def test_struct_layout_matches_c():
    with tempfile.TemporaryDirectory() as d:
        lines = [f'printf("%zu\\n", offsetof(OasisPromptArgs, {f}));' for f, _ in _lib.OasisPromptArgs._fields_]
        f, exe = os.path.join(d, "l.c"), os.path.join(d, "l")
        open(f, "w").write('#include <stdio.h>\n#include <stddef.h>\n' + f'#include "{ROOT}/include/oasis_b200.h"\n'
                           + "int main(void) {" + "".join(lines) + 'printf("%zu\\n", sizeof(OasisPromptArgs)); return 0; }')
        subprocess.run(["gcc", "-std=c99", f, "-o", exe], check=True)
        got = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    want = [getattr(_lib.OasisPromptArgs, f).offset for f, _ in _lib.OasisPromptArgs._fields_]
    assert got == want + [C.sizeof(_lib.OasisPromptArgs)]


# --------------------------------------------------------------------- on a GPU --

LENGTHS = [
    [1], [2, 1, 1], [17], [64, 64], [63, 1, 65], [128], [129], [127, 128, 1, 256], [255, 257], [300, 0, 5, 0, 0, 40],
    [3] * 50 + [1, 9, 2, 8, 31, 32, 33], [700], [144, 288, 1, 432],
]


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda v: f"{len(v)}x{sum(v)}")
@pytest.mark.parametrize("heads,kv,dim,dtype", [(2, 2, 64, BF16), (6, 2, 128, BF16), (4, 1, 64, FP16), (3, 3, 128, FP16)])
@pytest.mark.parametrize("hint", ["short", "long"])
def test_lengths_heads_types(lengths, heads, kv, dim, dtype, hint):
    q, k, v = inputs(lengths, heads, kv, dim, dtype, extra=3)
    cu = starts(lengths)
    out = torch.full((q.shape[0], heads, dim), 7.0, dtype=dtype, device=DEV)
    got = paged.attention_prompt(q, k, v, ints(cu), 1 if hint == "short" else 1 << 20, out=out)
    assert got is out
    check(got, q, k, v, cu)
    assert bool((got[cu[-1]:] == 7).all()), "rows behind the last sequence are left"


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,heads,kv,dim,dtype", [
    ([4608, 144, 1440], 2, 2, 64, BF16), ([3001, 2000], 4, 2, 128, BF16), ([2500], 3, 1, 128, FP16), ([2048, 2049], 8, 1, 64, FP16),
])
def test_long(lengths, heads, kv, dim, dtype):
    q, k, v = inputs(lengths, heads, kv, dim, dtype, seed=3)
    cu = starts(lengths)
    check(paged.attention_prompt(q, k, v, ints(cu), max(lengths)), q, k, v, cu)


@pytest.mark.gpu
@pytest.mark.parametrize("hint", [1, 1 << 20])
@pytest.mark.parametrize("scale,size", [(None, 30.0), (1.0, 4.0), (0.001, 1.0)])
def test_peaked_and_flat_scores(scale, size, hint):
    """Scores far apart (the running maximum moves by more than the exponent's range)
    and all alike."""
    lengths = [400, 77]
    q, k, v = inputs(lengths, 2, 1, 64, BF16, seed=5, scale=size)
    k[:400] *= torch.linspace(0.1, 3, 400, device=DEV)[:, None, None]  # later keys outweigh earlier ones
    cu = starts(lengths)
    check(paged.attention_prompt(q, k, v, ints(cu), hint, scale=scale), q, k, v, cu, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("hint", [1, 1 << 20])
def test_strides(hint):
    """Heads outside rows, gaps between rows, an output that is a view."""
    lengths = [150, 33, 200]
    cu, n = starts(lengths), sum(lengths)
    g = torch.Generator(device=DEV).manual_seed(6)
    make = lambda *s: torch.empty(*s, dtype=BF16, device=DEV).normal_(generator=g)  # noqa: E731
    q = make(4, n, 64).transpose(0, 1)
    k = make(n, 5, 72)[:, 1:3, :64]
    v = make(n, 2, 2, 64)[:, 1]
    out = torch.zeros(n, 6, 128, dtype=BF16, device=DEV)
    paged.attention_prompt(q, k, v, ints(cu), hint, out=out[:, 1:5, 64:])
    check(out[:, 1:5, 64:], q, k, v, cu)
    rest = out.clone()
    rest[:, 1:5, 64:] = 0
    assert not bool(rest.any())


@pytest.mark.gpu
@pytest.mark.parametrize("hint", [1, 1 << 20])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dim", [64, 128])
def test_what_is_not_seen_takes_no_part(hint, bad, dim):
    """NaN and infinities in keys and values that a row does not see: later rows of its
    sequence, its neighbours' rows, rows behind the last sequence."""
    lengths = [90, 200, 61]
    q, k, v = inputs(lengths, 2, 1, dim, BF16, seed=7, extra=40)
    cu = starts(lengths)
    for r in (60, 89, 90 + 130, 290 + 50, 351, 380):
        k[r], v[r] = bad, bad
    q[351:] = bad
    out = torch.zeros(q.shape, dtype=BF16, device=DEV)
    paged.attention_prompt(q, k, v, ints(cu), hint, out=out)
    want, spread = O.attention_prompt(q, k, v, cu), O.attention_prompt(q, k, torch.nan_to_num(v, 0, 0, 0).abs(), cu)
    for a, first in zip(cu, (60, 89 + 131, 340)):
        fine = slice(a, first)
        reach = dim ** -0.5 * float(q[fine].double().norm(dim=-1).max() * k[fine].double().norm(dim=-1).max())
        bound = O.error_bound(want[fine], spread[fine], reach, 200, dim, BF16)
        assert bool(((out[fine].double() - want[fine]).abs() <= bound).all())
    for a, b in zip(cu, cu[1:]):  # rows that see them: not finite where the formula is not
        assert torch.equal(torch.isnan(out[a:b]), torch.isnan(want[a:b]))
        assert torch.equal(torch.isinf(out[a:b]), torch.isinf(want[a:b]))


@pytest.mark.gpu
@pytest.mark.parametrize("hint", [1, 1 << 20])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_score_that_is_not_finite_reaches_the_result(hint, dtype, bad):
    """One key of NaN, or one that scores +inf, at each place of a block in turn, its value
    finite: every row that sees it is NaN, no other is."""
    n = 130
    q, k, v = inputs([n], 1, 1, 64, dtype, seed=13)
    q[:, :, 0] = 1
    for at in list(range(0, n, 7)) + [126, 127, 128, 129]:
        kk = k.clone()
        kk[at, 0, 0] = bad
        got = paged.attention_prompt(q, kk, v, ints([0, n]), hint)
        seen = torch.isnan(got).reshape(n, -1)
        assert bool(seen[at:].all()) and not bool(seen[:at].any()), at


@pytest.mark.gpu
@pytest.mark.parametrize("hint", [1, 1 << 20])
def test_keys_at_the_lowest_value(hint):
    """Scores of -inf and of the type's lowest value before, between and after others."""
    lengths = [260]
    q, k, v = inputs(lengths, 1, 1, 64, BF16, seed=8)
    q[:, :, 0] = 1
    k[:, :, 0] = 0
    k[:130, :, 0] = -math.inf  # nothing that counts in the first tile's keys
    k[200, :, 0] = torch.finfo(BF16).min
    cu = starts(lengths)
    got = paged.attention_prompt(q, k, v, ints(cu), hint)
    want = O.attention_prompt(q, k, v, cu)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and bool(torch.isnan(want[:130]).all())
    spread = O.attention_prompt(q, k, v.abs(), cu)
    reach = 64 ** -0.5 * float(q.double().norm(dim=-1).max() * k[201:].double().norm(dim=-1).max())
    bound = O.error_bound(want[130:], spread[130:], reach, 260, 64, BF16)
    assert bool(((got[130:].double() - want[130:]).abs() <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("hint", [1, 1 << 20])
def test_rows_of_no_sequence(hint):
    """Offsets that begin behind row 0, and offsets that pass the rows."""
    q, k, v = inputs([300], 2, 2, 64, BF16, seed=9)
    out = torch.full((300, 2, 64), 7.0, dtype=BF16, device=DEV)
    paged.attention_prompt(q, k, v, ints([40, 100, 220]), hint, out=out)
    check(out, q, k, v, [40, 100, 220])
    assert bool((out[:40] == 7).all()) and bool((out[220:] == 7).all())
    out.fill_(7)
    paged.attention_prompt(q, k, v, ints([0, 10, 900]), hint, out=out)
    check(out, q, k, v, [0, 10, 300])
    out.fill_(7)
    paged.attention_prompt(q, k, v, ints([0, 0, 0]), hint, out=out)
    assert bool((out == 7).all())


@pytest.mark.gpu
def test_same_results_again_and_in_a_graph():
    """The same bits on each call, beside another stream's call and from a graph whose
    inputs change between replays."""
    lengths = [500, 3, 260]
    cu = ints(starts(lengths))
    q, k, v = (t.contiguous() for t in inputs(lengths, 4, 2, 64, BF16, seed=10))
    for hint in (1, 500):
        a = paged.attention_prompt(q, k, v, cu, hint)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        b = paged.attention_prompt(q, k, v, cu, hint, stream=side)
        c = paged.attention_prompt(q, k, v, cu, hint)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(a, b) and torch.equal(a, c)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            d = paged.attention_prompt(q, k, v, cu, hint)
        g.replay()
        assert torch.equal(a, d)
        old = v.clone()
        v.mul_(2)  # exact in bf16: the result doubles
        g.replay()
        assert torch.equal(2 * a, d)
        v.copy_(old)


@pytest.mark.gpu
def test_memory_of_a_side_stream_is_its_own():
    """A result on a side stream does not land in memory that the current stream has given
    back but still reads, and is not given to that side stream again while the current
    one reads it."""
    q, k, v = inputs([100], 16, 16, 64, BF16, seed=16)
    cu, side, zero = ints([0, 100]), torch.cuda.Stream(), torch.zeros(100, 16, 64, dtype=BF16, device=DEV)
    want = paged.attention_prompt(q, k, v, cu, 100)
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        old = torch.full_like(want, 3.0)
        torch.cuda._sleep(20_000_000)  # the current stream is busy for some milliseconds
        kept = old.clone()
        del old
        out = paged.attention_prompt(q, k, v, cu, 100, stream=side)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda._sleep(20_000_000)
        again = out.clone()
        del out
        paged.attention_prompt(q, k, zero, cu, 100, stream=side)
        torch.cuda.synchronize()
        assert bool((kept == 3).all()) and torch.equal(again, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_beside_matrix_products(dim):
    """Products that use tensor memory before and behind the attention, without a pause:
    each starts while the one before it still runs."""
    lengths, heads = [150, 90, 16], 8
    q, k, v = inputs(lengths, heads, 4, dim, BF16, seed=15)
    cu, rows, width = ints(starts(lengths)), sum(lengths), heads * dim
    w = (torch.randn(1024, width, device=DEV) * 0.05).to(BF16)
    big = torch.randn(4096, width, device=DEV).to(BF16)
    y, z = torch.empty(rows, 1024, device=DEV), torch.empty(4096, 1024, device=DEV)
    ws = torch.empty(64 << 20, dtype=torch.uint8, device=DEV)
    stream = torch.cuda.current_stream().cuda_stream

    def product(a, out, block_n):
        args = _lib.OasisGemmArgs()
        args.a, args.lda, args.w = a.data_ptr(), width, w.data_ptr()
        args.m, args.n, args.k, args.mode = a.shape[0], 1024, width, 0
        args.out, args.ldo, args.rows_per_frame, args.rope_div, args.rope_mod = out.data_ptr(), 1024, 1, 1, 1
        args.block_n, args.splits, args.workspace, args.workspace_bytes = block_n, 1, ws.data_ptr(), ws.numel()
        _lib.call("oasis_gemm", C.byref(args), stream)

    for block_n in (32, 64, 256):
        for _ in range(20):
            product(big, z, block_n)
            out = paged.attention_prompt(q, k, v, cu, 1 << 20)
            product(out, y, block_n)
        check(out, q, k, v, starts(lengths))
        want = out.reshape(rows, width).double() @ w.double().T
        assert float((y.double() - want).norm() / want.norm()) < 1e-5
    assert _lib.load().oasis_device_error(0) == 0


@pytest.mark.gpu
def test_against_the_temporal_attention():
    """One length for all sequences and 16 heads of 64: what oasis_attention_temporal computes."""
    B, T, P = 3, 8, 144
    g = torch.Generator(device=DEV).manual_seed(11)
    qkv = torch.empty(B * T * P, 48, 64, dtype=BF16, device=DEV).normal_(generator=g)
    want = torch.empty(B * T * P, 16, 64, dtype=BF16, device=DEV)
    _lib.call("oasis_attention_temporal", qkv.data_ptr(), want.data_ptr(), B, T, 16, torch.cuda.current_stream().cuda_stream)
    rows = qkv.view(B, T, P, 48, 64).transpose(1, 2).reshape(-1, 48, 64)
    got = paged.attention_prompt(rows[:, :16], rows[:, 16:32], rows[:, 32:], ints(starts([T] * (B * P))), T)
    want = want.view(B, T, P, 16, 64).transpose(1, 2).reshape(-1, 16, 64)
    assert float((got.double() - want.double()).norm() / want.double().norm()) < 2 * 2.0 ** -8  # half a step each, twice


@pytest.mark.gpu
def test_random_batches():
    rng = random.Random(12)
    for seed in range(12):
        kv = rng.choice([1, 2, 3])
        heads, dim, dtype = kv * rng.choice([1, 2, 3, 7, 8]), rng.choice([64, 128]), rng.choice([BF16, FP16])
        lengths = [int(math.exp(rng.uniform(0, 6.2))) - 1 for _ in range(rng.randint(1, 9))] + [1]
        q, k, v = inputs(lengths, heads, kv, dim, dtype, seed=seed)
        cu = starts(lengths)
        check(paged.attention_prompt(q, k, v, ints(cu), rng.choice([1, max(lengths), 1 << 30])), q, k, v, cu)


@pytest.mark.gpu
def test_python_checks():
    q, k, v = inputs([10], 4, 2, 64, BF16)
    cu = ints([0, 10])
    call = paged.attention_prompt
    for args, text in (((q.float(), k, v, cu), "bfloat16"), ((q, k.half(), v, cu), "k must be"),
                       ((q, k[:5], v, cu), "rows"), ((q, k, v[:, :1], cu), "v must be"), ((q, k, v, cu.long()), "int32"),
                       ((q[:, :, :32], k, v, cu), "k must be"), ((q.cpu(), k, v, cu), "CUDA"),
                       ((q, k, v.cpu(), cu), "v must be on")):
        with pytest.raises(ValueError, match=text):
            call(*args, 10)
    with pytest.raises(ValueError, match="out"):
        call(q, k, v, cu, 10, out=torch.zeros(9, 4, 64, dtype=BF16, device=DEV))
    with pytest.raises(_lib.OasisError, match="kv_heads=2"):
        call(q[:, :3], k, v, cu, 10)
    assert call(q[:0], k[:0], v[:0], ints([0]), 0).shape == (0, 4, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("hint", [1, 1 << 20])
@pytest.mark.parametrize("heads,kv,dim,dtype", [(2, 1, 64, BF16), (2, 1, 128, BF16), (3, 1, 64, BF16), (2, 1, 64, FP16)])
def test_large_values_that_are_not_seen_change_no_bit(hint, heads, kv, dim, dtype):
    """Finite keys and values up to the type's largest in later rows of a sequence, in its
    neighbours and behind the last sequence: the rows that do not see them keep every bit
    that they have with zeros there."""
    lengths = [200, 130, 61]
    q, k, v = inputs(lengths, heads, kv, dim, dtype, seed=17, extra=130)
    hidden = torch.zeros(q.shape[0], dtype=torch.bool, device=DEV)
    for a, b in ((150, 200), (300, 330), (391, 521)):
        hidden[a:b] = True
    cu = ints(starts(lengths))
    k[hidden], v[hidden] = 0, 0
    want = paged.attention_prompt(q, k, v, cu, hint)
    assert bool(torch.isfinite(want[:391]).all())
    for size in (1e30, 1e36, 3.3e38) if dtype == BF16 else (6e4,):
        k[hidden], v[hidden] = size, size
        v[hidden] *= torch.where(torch.arange(dim, device=DEV) % 2 == 0, 1, -1).to(dtype)
        got = paged.attention_prompt(q, k, v, cu, hint)
        assert torch.equal(got[~hidden], want[~hidden]), size


def test_what_a_block_covers():
    """The tiles of a block, over many offsets: each row's keys lie in its tile's key blocks,
    and a tile's queries are fetched exactly where a product waits for them, so that no copy
    is left on its way when a block without a second (or a first) tile ends."""
    src = f'#include <stdio.h>\n#include <stdlib.h>\n#include "{ROOT}/open-oasis_b200/csrc/prompt_unit.cuh"\n' + r'''
    using namespace oasis;
    int main() {
      srand(1);
      int one_tile[2] = {0, 0};
      for (int run = 0; run < 4000; ++run) {
        int cu[9], n = 1 + rand() % 8;
        cu[0] = run % 3 ? 0 : rand() % 400;
        for (int i = 0; i < n; ++i) cu[i + 1] = cu[i] + (rand() % 4 ? rand() % (run % 2 ? 40 : 300) : 0);
        const int rows = 1 + rand() % (cu[n] + 300), end = rows < cu[n] ? rows : cu[n];
        for (int pair = 0; pair < 2; ++pair) {
          const int tile_rows = pair ? kPromptTile : 2 * kPromptTile;
          for (int rt = 0; rt < (rows + tile_rows - 1) / tile_rows; ++rt) {
            const PromptUnit u = prompt_unit(cu, n, pair, end, 0, rt);
            int blocks = 0;
            for (int t = 0; t < 2; ++t) {
              bool waited = false;  // as the warp that issues the products walks the blocks
              for (int j = 0; j < u.blocks; ++j)
                if (j >= u.first[t] && j < u.last[t]) waited = true;
              if (waited != u.has(t)) printf("waits %d %d\n", run, t);
              if (u.last[t] > blocks) blocks = u.last[t];
              if (u.blocks > 0 && !u.has(t)) ++one_tile[t];
              for (int r = u.r0[t]; r < u.r0[t] + kPromptTile && r < end; ++r) {
                if (r < cu[0]) continue;
                const int a = cu[last_not_above(cu, n, r)];
                if (a < u.begin + u.first[t] * kPromptTile || r >= u.begin + u.last[t] * kPromptTile)
                  printf("keys %d %d\n", run, r);
              }
            }
            if (blocks != u.blocks || u.blocks < 0) printf("blocks %d\n", run);
          }
        }
      }
      printf(one_tile[0] > 0 && one_tile[1] > 0 ? "done\n" : "no block of one tile\n");
      return 0;
    }'''
    with tempfile.TemporaryDirectory() as d:
        f, exe = os.path.join(d, "u.cpp"), os.path.join(d, "u")
        open(f, "w").write(src)
        subprocess.run(["g++", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", f, "-o", exe], check=True)
        assert subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split("\n")[:-1] == ["done"]


def test_queries_are_fetched_only_for_tiles_that_wait():
    """In the kernel: each copy into a tile's Q stands behind that tile's `has`."""
    text = open(f"{ROOT}/open-oasis_b200/csrc/attention_prompt_tc.cu").read()
    loads = [line for line in text.splitlines() if "&tmQ, &q_full" in line]
    assert len(loads) == 2 and all(f"if (u.has({t})) load(" in line for t, line in enumerate(loads))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("begin,lengths,extra", [(0, [300], 0), (0, [513], 200), (140, [300], 0), (400, [20, 250], 90)])
def test_blocks_of_one_tile(dim, begin, lengths, extra):
    """Heads that do not pair: blocks whose second tile, or whose first, has no row."""
    cu = starts(lengths, begin)
    q, k, v = inputs([cu[-1]], 3, 1, dim, BF16, seed=20, extra=extra)
    out = torch.full(q.shape, 7.0, dtype=BF16, device=DEV)
    for _ in range(3):
        paged.attention_prompt(q, k, v, ints(cu), 1 << 20, out=out)
    check(out, q, k, v, cu)
    assert bool((out[:begin] == 7).all()) and bool((out[cu[-1] :] == 7).all())
    assert _lib.load().oasis_device_error(0) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("hint", [1, 1 << 20])
@pytest.mark.parametrize("dim", [64, 128])
def test_values_whose_sum_overflows(hint, dim):
    """Values near the type's largest: their weighted mean is finite, their sum is not."""
    lengths = [140, 3, 60]
    q, k, v = inputs(lengths, 2, 1, dim, BF16, seed=18)
    v.uniform_(1e38, 3e38, generator=torch.Generator(device=DEV).manual_seed(19))
    v[:, :, 1::2] *= -1
    cu = starts(lengths)
    check(paged.attention_prompt(q, k, v, ints(cu), hint), q, k, v, cu)


@pytest.mark.gpu
@pytest.mark.parametrize("hint", [1, 1 << 20])
@pytest.mark.parametrize("dim", [64, 128])
def test_values_of_keys_that_weigh_nothing(hint, dim):
    """Keys that a row sees and that score thousands below its others: whatever finite value
    they have, none of it is in the result."""
    q, k, v = inputs([300], 2, 1, dim, BF16, seed=21)
    q[:, :, 0] = 1
    k[:, :, 0] = 0
    low = torch.arange(300, device=DEV) % 3 == 1
    k[low, :, 0], v[low] = -3e4, 3e38
    got = paged.attention_prompt(q, k, v, ints([0, 300]), hint)
    check(got, q, k, v, [0, 300])


@pytest.mark.gpu
@pytest.mark.parametrize("hint", [1, 1 << 20])
@pytest.mark.parametrize("heads,kv,dim,dtype", [(2, 1, 64, BF16), (3, 3, 64, FP16), (2, 1, 128, FP16), (3, 1, 128, BF16)])
@pytest.mark.parametrize("lengths,extra", [([70], 1), ([140, 3, 90], 100), ([300], 15), ([129, 255], 300), ([64, 64, 128], 64)])
def test_what_lies_behind_the_last_sequence_changes_no_bit(lengths, extra, heads, kv, dim, dtype, hint):
    """NaN and infinities in padding rows leave every bit that zeros there leave: no row is
    worked out another way because of them (which took hundreds of times as long)."""
    q, k, v = inputs(lengths, heads, kv, dim, dtype, seed=22, extra=extra)
    cu, n = ints(starts(lengths)), sum(lengths)
    q[n:], k[n:], v[n:] = 0, 0, 0
    want = paged.attention_prompt(q, k, v, cu, hint)
    check(want, q, k, v, starts(lengths))
    for bad in (math.nan, math.inf, -math.inf):
        q[n:], k[n:], v[n:] = bad, bad, bad
        out = torch.full_like(want, 7.0)
        paged.attention_prompt(q, k, v, cu, hint, out=out)
        assert torch.equal(out[:n], want[:n]) and bool((out[n:] == 7).all())


@pytest.mark.gpu
def test_a_batch_of_nan_is_not_worked_out_key_by_key():
    """A diverged model's NaN cost a few times a clean call (4 as measured, 1000 where each row
    went through all of its keys one by one)."""
    q, k, v = (t.contiguous() for t in inputs([2000, 2000], 16, 16, 64, BF16, seed=23))
    cu = ints([0, 2000, 4000])

    def took():
        paged.attention_prompt(q, k, v, cu, 2000)
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(3):
            out = paged.attention_prompt(q, k, v, cu, 2000)
        b.record()
        b.synchronize()
        return a.elapsed_time(b), out

    clean, _ = took()
    for t in (q, k, v):
        t[:] = math.nan
    dirty, out = took()
    assert bool(torch.isnan(out).all()) and dirty < 40 * clean, (clean, dirty)


@pytest.mark.gpu
@pytest.mark.parametrize("hint", [1, 1 << 20])
@pytest.mark.parametrize("dim,dtype", [(64, FP16), (128, FP16), (64, BF16)])
@pytest.mark.parametrize("nats", [10, 14, 15.5])
def test_one_key_outweighs_the_others(nats, dim, dtype, hint):
    """A first key that takes nearly all of the weight and has a value of zero: what the others,
    `nats` below it, add is as exact as a probability's one rounding. The bound is the usual
    one without its allowance for probabilities that underflow; half a subnormal step for
    results among the type's subnormal numbers."""
    n = 3000
    g = torch.Generator(device=DEV).manual_seed(24)
    q, k, v = (torch.zeros(n, 1, dim, dtype=dtype, device=DEV) for _ in range(3))
    q[:, :, :2] = 1
    k[1:, 0, 0] = -nats * dim ** 0.5
    k[1:, 0, 1] = torch.empty(n - 1, device=DEV).uniform_(-2, 2, generator=g).to(dtype)
    v[1:] = 1
    got = paged.attention_prompt(q, k, v, ints([0, n]), hint)
    want = O.attention_prompt(q, k, v, [0, n])
    reach = dim ** -0.5 * float(q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max())
    allowed = 2.0 ** -24 * (1 + 2 * n) if dtype == FP16 else 2.0 ** -120
    bound = O.error_bound(want, want, reach, n, dim, dtype) - allowed + 2.0 ** (-25 if dtype == FP16 else -120)
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())
