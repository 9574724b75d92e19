"""Measured cases of the paged-cache operators: attention over packed prompts,
attention of single queries over a paged cache whose sequences share a prefix, and
the management of the cache's pages.

`run` computes a case with elementary torch operations in 32 bits (`own` false) or
through the framework's entry points (`own` true), on the same state.

Sizes: 16 heads x 64, 144 patches per frame, windows of 8 and up to 32 frames and 64
sessions are this model's; grouped heads, head dim 128 and the longer lengths are
generic.
"""
from __future__ import annotations

import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
PATCHES = 144


def _device() -> str:
    return "cuda" if torch.cuda.is_available() else "cpu"


# --------------------------------------------------------------------- cases --

def listed():
    return [
        # one new session with a few tokens: the smallest call, all latency
        dict(name="prompt: one short sequence", op="prompt", type="fp16", heads=16, kv_heads=16, dim=64, sequences=1,
             repeat=1, step=1, longest=17, mix=1),
        # temporal attention of a batch of 64 sessions that hold 1 to 8 frames each:
        # one sequence per (session, patch), thousands of sequences of a few tokens
        dict(name="prompt: frames per patch", op="prompt", type="bf16", heads=16, kv_heads=16, dim=64, sequences=64,
             repeat=PATCHES, step=1, longest=8, mix=2),
        # whole contexts of 1 to 32 frames of 144 tokens, eight sessions packed
        dict(name="prompt: sessions of frames", op="prompt", type="bf16", heads=16, kv_heads=16, dim=64, sequences=8,
             repeat=1, step=PATCHES, longest=32 * PATCHES, mix=3),
        # long ragged prompts with grouped heads of 128
        dict(name="prompt: grouped heads", op="prompt", type="bf16", heads=32, kv_heads=8, dim=128, sequences=4, repeat=1,
             step=1, longest=6001, mix=4),
        # three forks of one frame, one token each: latency
        dict(name="shared: three forks", op="shared", type="bf16", heads=16, kv_heads=16, dim=64, groups=1, rows=3,
             page=16, prefix=144, own=40, mix=5),
        # the generated frame of 64 sessions forked from a 16-frame prompt: a group per
        # patch, one query per (patch, session)
        dict(name="shared: forks per patch", op="shared", type="bf16", heads=16, kv_heads=16, dim=64, groups=PATCHES,
             rows=64, page=16, prefix=16, own=16, mix=6),
        # 64 sequences behind one long prompt, grouped heads
        dict(name="shared: long prefix", op="shared", type="bf16", heads=32, kv_heads=8, dim=128, groups=1, rows=64,
             page=64, prefix=8192, own=1024, mix=7),
        # groups of different sizes and prefixes, one without a prefix, an empty
        # sequence, an odd number of heads per key head
        dict(name="shared: ragged groups", op="shared", type="fp16", heads=28, kv_heads=4, dim=128, groups=5, rows=12,
             page=32, prefix=2999, own=700, mix=8),
        # two small sessions end and two others take their places
        dict(name="pages: admit", op="admit", type="bf16", layers=2, heads=16, dim=64, page=16, sequences=2, longest=40,
             mix=9),
        # 60 branches are dropped and forked anew from four sessions
        dict(name="pages: fork", op="fork", type="bf16", deep=False, layers=16, heads=16, dim=64, page=16, sequences=4,
             copies=60, longest=500, mix=10),
        # full copies of six sessions
        dict(name="pages: copy", op="fork", type="bf16", deep=True, layers=8, heads=8, dim=128, page=32, sequences=6,
             copies=6, longest=1500, mix=11),
        # sessions end and the pool is compacted before others arrive, twice
        dict(name="pages: roll", op="roll", type="bf16", layers=4, heads=16, dim=64, page=64, sequences=24, longest=640,
             mix=12),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5)))))))


def draw(rng):
    mix = rng.randrange(1 << 20)
    kind = rng.choice(["prompt", "prompt", "prompt", "shared", "shared", "shared", "admit", "fork", "roll"])
    typ, dim = rng.choice(["bf16", "fp16"]), rng.choice([64, 128])
    kv = rng.choice([1, 2, 3, 4, 8, 16])
    heads = kv * rng.choice([g for g in (1, 2, 3, 4, 7, 8) if kv * g <= 32])
    if kind == "prompt":
        form = rng.choice(["few", "many", "frames"])
        if form == "many":  # many sequences of a few tokens
            return dict(op="prompt", type=typ, heads=16, kv_heads=16, dim=64, sequences=_log(rng, 1, 32), repeat=PATCHES,
                        step=1, longest=_log(rng, 1, 16), mix=mix)
        if form == "frames":
            return dict(op="prompt", type=typ, heads=16, kv_heads=16, dim=64, sequences=_log(rng, 1, 8), repeat=1,
                        step=PATCHES, longest=PATCHES * rng.randint(1, 24), mix=mix)
        longest = _log(rng, 1, 6001)
        most = max(1, min(64, (1 << 31) // (heads * longest * longest)))
        return dict(op="prompt", type=typ, heads=heads, kv_heads=kv, dim=dim, sequences=_log(rng, 1, most), repeat=1,
                    step=1, longest=longest, mix=mix)
    if kind == "shared":
        rows = _log(rng, 1, 64)
        prefix, more = _log(rng, 1, 8192), _log(rng, 1, 1024)
        most = max(1, min(PATCHES, (1 << 28) // (rows * (prefix + more) * kv * dim)))
        return dict(op="shared", type=typ, heads=heads, kv_heads=kv, dim=dim, groups=_log(rng, 1, most), rows=rows,
                    page=rng.choice([16, 32, 64]), prefix=prefix, own=more, mix=mix)
    page, layers = rng.choice([16, 32, 64]), rng.choice([1, 2, 4, 8])
    longest, n = _log(rng, 1, 640), _log(rng, 1, 16)
    case = dict(op=kind, type=typ, layers=layers, heads=kv, dim=dim, page=page, sequences=n, longest=longest, mix=mix)
    if kind == "fork":
        case.update(deep=rng.random() < 0.5, copies=_log(rng, 1, 16))
    return case


def _lengths(case, n):
    """Lengths of n sequences: one the longest, the others spread over the logarithm of the range."""
    rng = random.Random(case["mix"])
    step = case.get("step", 1)
    most = case["longest"] // step
    got = [step * most] + [step * _log(rng, 1, most) for _ in range(n - 1)]
    rng.shuffle(got)
    return got


def _groups(case):
    """Rows, whole prefix pages and row lengths of each group of a shared case."""
    rng = random.Random(case["mix"])
    G, rows, page = case["groups"], case["rows"], case["page"]
    even = G >= PATCHES or G == 1
    sizes = [rows] + [rows if even else _log(rng, 1, rows) for _ in range(G - 1)]
    pages = [-(-case["prefix"] // page)] + [-(-(case["prefix"] if even else _log(rng, 1, case["prefix"])) // page)
                                            for _ in range(G - 1)]
    lengths = [[p * page + _log(rng, 1, case["own"]) for _ in range(r)] for r, p in zip(sizes, pages)]
    lengths[0][0] = pages[0] * page + case["own"]
    if not even:
        pages[-1] = 0
        lengths[-1] = [_log(rng, 1, case["own"]) for _ in lengths[-1]]
        lengths[-1][-1] = 0
    return sizes, pages, lengths


def work(case):
    if case["op"] == "prompt":
        lengths = [t for t in _lengths(case, case["sequences"]) for _ in range(case["repeat"])]
        H, K, D = case["heads"], case["kv_heads"], case["dim"]
        return dict(bytes=sum(lengths) * (2 * H + 2 * K) * D * 2, flops=4 * H * D * sum(t * (t + 1) // 2 for t in lengths))
    if case["op"] == "shared":
        sizes, pages, lengths = _groups(case)
        H, K, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
        keys = sum(p * page + sum(max(0, t - p * page) for t in ls) for p, ls in zip(pages, lengths))
        return dict(bytes=keys * 2 * K * D * 2 + sum(sizes) * 2 * H * D * 2 + sum(sum(-(-t // page) for t in ls) for ls in lengths) * 4,
                    flops=4 * H * D * sum(sum(ls) for ls in lengths))
    token = case["layers"] * 2 * case["heads"] * case["dim"] * 2
    page, n = case["page"], case["sequences"]
    lengths = _lengths(case, n)
    if case["op"] == "fork":
        took = [lengths[i % n] for i in range(case["copies"])]
        rows = sum(t if case["deep"] else t % page for t in took)
        return dict(bytes=rows * token * 2 + sum(-(-t // page) for t in took) * 4 * 4, flops=0)
    if case["op"] == "admit":
        return dict(bytes=2 * sum(lengths) * token + sum(-(-t // page) for t in lengths) * 4 * 4, flops=0)
    held = sum(-(-t // page) for t in lengths)
    return dict(bytes=2 * (2 * held * page * token + 2 * sum(lengths) * token), flops=0)


# -------------------------------------------------------------------- inputs --

def _starts(lengths, dev):
    at = [0]
    for t in lengths:
        at.append(at[-1] + t)
    return torch.tensor(at, dtype=torch.int32, device=dev)


def _fill(shape, typ, dev, gen, scale=1.0):
    t = torch.empty(shape, dtype=TYPES[typ], device=dev)
    t.normal_(generator=gen)
    return t if scale == 1.0 else t.mul_(scale)


def _hand_out(lengths, page, order):
    """Page lists of sequences, taken from `order`, and what is left of it."""
    lists = []
    for t in lengths:
        need = -(-t // page)
        lists.append(order[:need])
        order = order[need:]
    return lists, order


def prepare(case, seed):
    dev = _device()
    gen = torch.Generator(device=dev).manual_seed(seed)
    typ = case["type"]
    D = case["dim"]
    if case["op"] == "prompt":
        H, K = case["heads"], case["kv_heads"]
        lengths = [t for t in _lengths(case, case["sequences"]) for _ in range(case["repeat"])]
        # the packed rows that a projection of q, k and v leaves
        qkv = _fill((sum(lengths), (H + 2 * K) * D), typ, dev, gen)
        qkv[:, : H * D] *= 2
        rows = qkv.view(-1, H + 2 * K, D)
        return dict(case=case, q=rows[:, :H], k=rows[:, H : H + K], v=rows[:, H + K :], cu=_starts(lengths, dev),
                    longest=max(lengths))
    rng = random.Random(seed)
    if case["op"] == "shared":
        H, K, page = case["heads"], case["kv_heads"], case["page"]
        sizes, pages, lengths = _groups(case)
        flat = [t for ls in lengths for t in ls]
        private = [max(0, t - p * page) for p, ls in zip(pages, lengths) for t in ls]
        total = sum(pages) + sum(-(-t // page) for t in private)
        order = list(range(total + 5))
        rng.shuffle(order)
        common, order = _hand_out([p * page for p in pages], page, order)
        mine, order = _hand_out(private, page, order)
        rows, at = [], 0
        for g, r in enumerate(sizes):
            rows += [(common[g] + mine[at + i]) if flat[at + i] else [] for i in range(r)]
            at += r
        width = max(len(r) for r in rows) + 1
        table = torch.tensor([r + [-1] * (width - len(r)) for r in rows], dtype=torch.int32, device=dev)
        refs = torch.zeros(total + 5, dtype=torch.int32, device=dev)
        refs.index_add_(0, table[table >= 0].long(), torch.ones_like(table[table >= 0]))
        pool = _fill((total + 5, 2, 2, K, page, D), typ, dev, gen)
        return dict(case=case, q=_fill((len(flat), H, D), typ, dev, gen, 2.0), pool=pool, table=table,
                    lengths=torch.tensor(flat, dtype=torch.int32, device=dev), refs=refs, layer=1, sizes=sizes, pages=pages,
                    seqs=torch.arange(len(flat), dtype=torch.int32, device=dev), longest=max(flat))
    # a pool with sessions in scattered pages and free slots
    K, page, L, n = case["heads"], case["page"], case["layers"], case["sequences"]
    lengths = _lengths(case, n)
    if case["op"] == "fork":
        slots, room = n + case["copies"], [lengths[i % n] for i in range(case["copies"])]
        live = lengths
    elif case["op"] == "admit":
        slots, room, live = n + 2, [], lengths + [page + 3, page]
    else:
        slots, room, live = 3 * n, [], lengths + lengths + lengths
    total = sum(-(-t // page) for t in live + room) + len(live) + 3
    order = list(range(total))
    rng.shuffle(order)
    lists, _ = _hand_out(live, page, order)
    width = -(-case["longest"] // page) + 2
    table = torch.full((slots, width), -1, dtype=torch.int32)
    for i, pages in enumerate(lists):
        table[i, : len(pages)] = torch.tensor(pages, dtype=torch.int32)
    refs = torch.zeros(total, dtype=torch.int32)
    refs[table[table >= 0].long()] = 1
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    state = dict(case=case, pool=_fill((total, L, 2, K, page, D), typ, dev, gen), table=table.to(dev), refs=refs.to(dev),
                 lengths=ints(live + [0] * (slots - len(live))))
    if case["op"] == "fork":
        state.update(src=ints([i % n for i in range(case["copies"])]), dst=ints(list(range(n, slots))))
    else:
        rows = _fill((L, sum(lengths), 2 * K * D), typ, dev, gen).view(L, -1, 2 * K, D)
        state.update(cu=_starts(lengths, dev), k=rows[:, :, :K], v=rows[:, :, K:],
                     cohorts=[ints(list(range(n)))] if case["op"] == "admit" else
                     [ints(list(range(n))), ints(list(range(2 * n, 3 * n)))])
    return state


# --------------------------------------------------------------- plain forms --

def _plain_prompt(s):
    """softmax(q k^T / sqrt(D)) v over j <= i, on sequences padded to the longest."""
    q, k, v, cu, T = s["q"], s["k"], s["v"], s["cu"].long(), s["longest"]
    H, K, D = q.shape[1], k.shape[1], q.shape[2]
    n = cu.numel() - 1
    at = torch.arange(T, device=q.device)
    row = cu[:-1, None] + at
    inside = row < cu[1:, None]
    row = row.clamp_(max=q.shape[0] - 1)
    qp = q[row].float().permute(0, 2, 1, 3).reshape(n, K, (H // K) * T, D)
    kp = k[row].float().permute(0, 2, 3, 1)
    vp = v[row].float().permute(0, 2, 1, 3)
    x = torch.matmul(qp, kp).view(n, K, H // K, T, T)
    x.mul_(1 / math.sqrt(D)).masked_fill_(at > at[:, None], -math.inf)
    x.sub_(x.amax(-1, keepdim=True)).exp_()
    total = x.sum(-1, keepdim=True)
    y = torch.matmul(x.view(n, K, -1, T), vp).view(n, K, H // K, T, D).div_(total)
    return y.permute(0, 3, 1, 2, 4).reshape(n, T, H, D)[inside].to(q.dtype)


def _plain_shared(s):
    """softmax(q k^T / sqrt(D)) v over the first length tokens of each row's pages; zero for an empty row."""
    q, layer, page = s["q"], s["layer"], s["case"]["page"]
    pool, table, length = s["pool"], s["table"][s["seqs"].long()].long(), s["lengths"][s["seqs"].long()]
    B, H, D = q.shape
    K = pool.shape[3]
    at = torch.arange(s["longest"], device=q.device)
    where = table[:, at // page].clamp_(min=0)
    slot = (at % page).expand(B, -1)
    k = pool[:, layer, 0].transpose(1, 2)[where, slot].float()
    v = pool[:, layer, 1].transpose(1, 2)[where, slot].float()
    x = torch.matmul(q.float().view(B, K, H // K, D), k.permute(0, 2, 3, 1)).mul_(1 / math.sqrt(D))
    hidden = (at >= length[:, None])[:, None, None]
    x.masked_fill_(hidden, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True)).masked_fill_(hidden, 0)
    y = torch.matmul(x, v.transpose(1, 2)) / x.sum(-1, keepdim=True).clamp_min(1e-30)
    return y.view(B, H, D).to(q.dtype)


def _plain_free(s, seqs):
    at = seqs.long()
    pages = s["table"][at]
    pages = pages[pages >= 0].long()
    s["refs"].index_add_(0, pages, torch.full_like(pages, -1, dtype=torch.int32))
    s["table"][at] = -1
    s["lengths"][at] = 0


def _free_pages(s):
    return torch.argsort((s["refs"] > 0).int(), stable=True)


def _plain_fork(s, src, dst, deep):
    page, table = s["case"]["page"], s["table"]
    a, b = src.long(), dst.long()
    length = s["lengths"][a].long()
    last = (length + page - 1) // page
    first = torch.zeros_like(length) if deep else length // page
    need = last - first
    base = torch.cumsum(need, 0) - need
    col = torch.arange(table.shape[1], device=table.device)
    mine = (col >= first[:, None]) & (col < last[:, None])
    free = _free_pages(s)
    new = free[(base[:, None] + col - first[:, None]).clamp_(0, free.numel() - 1)]
    old = table[a].long()
    got = torch.where(mine, new, torch.where(col < last[:, None], old, -1))
    table[b] = got.int()
    s["lengths"][b] = length.int()
    used = got[got >= 0]
    s["refs"].index_add_(0, used, torch.ones_like(used, dtype=torch.int32))
    fill = (length[:, None] - col * page).clamp_(max=page)[mine]
    keep = torch.arange(page, device=table.device) < fill[:, None]
    keep = keep[:, None, None, None, :, None]
    s["pool"][new[mine]] = torch.where(keep, s["pool"][old[mine]], s["pool"][new[mine]])


def _plain_reserve(s, seqs, cu):
    page, table, at = s["case"]["page"], s["table"], seqs.long()
    begin = s["lengths"][at].long()
    end = begin + (cu[1:] - cu[:-1]).long()
    first, last = (begin + page - 1) // page, (end + page - 1) // page
    need = last - first
    base = torch.cumsum(need, 0) - need
    col = torch.arange(table.shape[1], device=table.device)
    mine = (col >= first[:, None]) & (col < last[:, None])
    free = _free_pages(s)
    new = free[(base[:, None] + col - first[:, None]).clamp_(0, free.numel() - 1)]
    table[at] = torch.where(mine, new, table[at].long()).int()
    s["refs"][new[mine]] = 1
    s["lengths"][at] = end.int()
    return begin.int()


def _plain_write(s, layer, k, v, seqs, cu, start):
    page = s["case"]["page"]
    row = torch.arange(k.shape[0], device=k.device)
    which = torch.searchsorted(cu[1:].long(), row, right=True)
    at = start.long()[which] + row - cu.long()[which]
    where = s["table"][seqs.long()[which], at // page].long()
    s["pool"][where, layer, 0, :, at % page] = k
    s["pool"][where, layer, 1, :, at % page] = v


def _plain_compact(s):
    held = s["refs"] > 0
    count = held.sum()
    index = torch.arange(held.numel(), device=held.device)
    source, target = index[held & (index >= count)], index[~held & (index < count)]
    s["pool"][target] = s["pool"][source]
    to = index.clone()
    to[source] = target
    s["refs"][target] = s["refs"][source]
    s["refs"][source] = 0
    s["table"].copy_(torch.where(s["table"] >= 0, to[s["table"].clamp(min=0).long()].int(), s["table"]))


# ----------------------------------------------------------------------- run --

class _Plain:
    """The page operations on a state's tensors."""

    def __init__(self, s):
        self.s = s

    def free(self, seqs):
        _plain_free(self.s, seqs)

    def fork(self, src, dst, deep=False):
        _plain_fork(self.s, src, dst, deep)

    def reserve(self, seqs, cu):
        return _plain_reserve(self.s, seqs, cu)

    def write(self, layer, k, v, seqs, cu, start):
        _plain_write(self.s, layer, k, v, seqs, cu, start)

    def compact(self):
        _plain_compact(self.s)


def _paged():
    import __graft_entry__

    __graft_entry__.load_package()
    from oasis_b200 import paged

    return paged


def _cache(s):
    """The cache handle that a program keeps beside its tensors."""
    if "cache" not in s:
        s["cache"] = _paged().PagedCache.from_tensors(s["pool"], s["table"], s["lengths"], s["refs"])
    return s["cache"]


def run(s):
    op = s["case"]["op"]
    if op == "prompt":
        if own:
            return _paged().attention_prompt(s["q"], s["k"], s["v"], s["cu"], s["longest"])
        return _plain_prompt(s)
    if op == "shared":
        if own:
            if "plan" not in s:
                s["plan"] = _paged().SharedPlan(s["sizes"], s["pages"], s["longest"], s["q"].device)
            return _paged().attention_shared(s["q"], _cache(s), s["layer"], s["seqs"], s["plan"])
        return _plain_shared(s)
    cache = _cache(s) if own else _Plain(s)
    if op == "fork":
        cache.free(s["dst"])
        cache.fork(s["src"], s["dst"], deep=s["case"]["deep"])
    else:
        for seqs in s["cohorts"]:
            cache.free(seqs)
            if op == "roll":
                cache.compact()
            start = cache.reserve(seqs, s["cu"])
            for layer in range(s["case"]["layers"]):
                cache.write(layer, s["k"][layer], s["v"][layer], seqs, s["cu"], start)
    return dict(pool=s["pool"], table=s["table"], lengths=s["lengths"], refs=s["refs"])


# --------------------------------------------------------------------- exact --

def exact(case, seed):
    if case["op"] not in ("prompt", "shared"):
        return None  # bytes that are moved and whole numbers
    s = prepare(case, seed)
    H, K, D = case["heads"], case["kv_heads"], case["dim"]
    q = s["q"].double()
    out = torch.zeros_like(q)
    if case["op"] == "prompt":
        k, v, cu = s["k"].double(), s["v"].double(), s["cu"].tolist()
        by_length = {}
        for a, b in zip(cu, cu[1:]):
            by_length.setdefault(b - a, []).append(a)
        for t, begins in by_length.items():
            rows = torch.tensor(begins, device=q.device)[:, None] + torch.arange(t, device=q.device)
            seen = torch.ones(t, t, dtype=torch.bool, device=q.device).tril()
            for h in range(H):
                e = torch.einsum("nid,njd->nij", q[rows, h], k[rows, h // (H // K)]) * D ** -0.5
                p = torch.softmax(torch.where(seen, e, torch.tensor(-math.inf, dtype=e.dtype, device=e.device)), -1)
                out[rows, h] = torch.einsum("nij,njd->nid", p, v[rows, h // (H // K)])
        return out
    page, layer = case["page"], s["layer"]
    lengths, table = s["lengths"].tolist(), s["table"].tolist()
    for b, t in enumerate(lengths):
        if t:
            pages = torch.tensor(table[b][: -(-t // page)], device=q.device)
            kv = s["pool"][pages, layer].double().permute(1, 2, 0, 3, 4).reshape(2, K, -1, D)[:, :, :t]
            e = torch.einsum("kgd,ktd->kgt", q[b].view(K, H // K, D), kv[0]) / D ** 0.5
            out[b] = torch.einsum("kgt,ktd->kgd", torch.softmax(e, -1), kv[1]).reshape(H, D)
    return out
