"""CPU restatement of the paged session cache and of the attention over it: plain
loops over sequences, whole numbers in Python, attention in fp64. The tests compare
the kernels with it."""
from __future__ import annotations

import math

import torch

BAD_SEQUENCE, IN_USE, NO_PAGES, TOO_LONG, BAD_PAGE = 1, 2, 4, 8, 16


class OracleCache:
    """The same arrays as PagedCache, on the CPU, changed request by request."""

    def __init__(self, pool, table, lengths, refs):
        self.pool, self.table = pool.cpu().clone(), table.cpu().tolist()
        self.lengths, self.refs = lengths.cpu().tolist(), refs.cpu().tolist()
        self.page = pool.shape[4]
        self.slots, self.width = len(self.table), table.shape[1]
        self.status = 0

    def _pages(self, tokens):
        return -(-tokens // self.page)

    def _lowest_free(self):
        return [p for p, r in enumerate(self.refs) if r == 0]

    def _targets(self, seqs):
        """Whether request i is the first valid one that names its target."""
        seen, ok = set(), []
        for s in seqs:
            if not 0 <= s < self.slots:
                self.status |= BAD_SEQUENCE
                ok.append(False)
            elif s in seen:
                self.status |= IN_USE
                ok.append(False)
            else:
                seen.add(s)
                ok.append(True)
        return ok

    def reserve(self, seqs, cu):
        free, used, full, start = self._lowest_free(), 0, False, []
        for i, (s, ok) in enumerate(zip(seqs, self._targets(seqs))):
            more = cu[i + 1] - cu[i]
            if not ok:
                start.append(-1)
                continue
            begin = self.lengths[s]
            if more < 0:
                self.status |= BAD_SEQUENCE
                start.append(-1)
            elif begin + more > self.width * self.page:
                self.status |= TOO_LONG
                start.append(-1)
            else:
                need = self._pages(begin + more) - self._pages(begin)
                if need and (full or used + need > len(free)):
                    full = True
                    self.status |= NO_PAGES
                    start.append(-1)
                    continue
                for k in range(need):
                    self.table[s][self._pages(begin) + k] = free[used + k]
                    self.refs[free[used + k]] = 1
                used += need
                self.lengths[s] = begin + more
                start.append(begin)
        return start

    def write(self, layer, k, v, seqs, cu, start):
        for i, s in enumerate(seqs):
            if start[i] < 0:
                continue
            for r in range(cu[i], min(cu[i + 1], k.shape[0])):
                at = start[i] + r - cu[i]
                if at >= self.lengths[s]:
                    continue
                page = self.table[s][at // self.page]
                self.pool[page, layer, 0, :, at % self.page] = k[r].cpu()
                self.pool[page, layer, 1, :, at % self.page] = v[r].cpu()

    def fork(self, src, dst, deep=False):
        lengths, tables = list(self.lengths), [list(r) for r in self.table]
        free, used, full = self._lowest_free(), 0, False
        for i, ok in enumerate(self._targets(dst)):
            if not ok:
                continue
            s, t = src[i], dst[i]
            if not 0 <= s < self.slots:
                self.status |= BAD_SEQUENCE
                continue
            if lengths[t]:
                self.status |= IN_USE
                continue
            L = lengths[s]
            whole = 0 if deep else L // self.page
            need = self._pages(L) - whole
            if need and (full or used + need > len(free)):
                full = True
                self.status |= NO_PAGES
                continue
            for c in range(self._pages(L)):
                page = tables[s][c]
                if c < whole:
                    self.refs[page] += 1
                else:
                    new = free[used]
                    used += 1
                    self.refs[new] = 1
                    fill = min(self.page, L - c * self.page)
                    self.pool[new, :, :, :, :fill] = self.pool[page, :, :, :, :fill]
                    page = new
                self.table[t][c] = page
            self.lengths[t] = L

    def free(self, seqs):
        for s in seqs:
            if not 0 <= s < self.slots:
                self.status |= BAD_SEQUENCE
                continue
            for c in range(self._pages(self.lengths[s])):
                self.refs[self.table[s][c]] -= 1
                self.table[s][c] = -1
            self.lengths[s] = 0

    def compact(self):
        live = [p for p, r in enumerate(self.refs) if r]
        source = [p for p in live if p >= len(live)]
        target = [p for p in range(len(live)) if self.refs[p] == 0]
        name = dict(zip(source, target))
        for s, t in name.items():
            self.pool[t] = self.pool[s]
            self.refs[t], self.refs[s] = self.refs[s], 0
        for s in range(self.slots):
            for c in range(self._pages(self.lengths[s])):
                self.table[s][c] = name.get(self.table[s][c], self.table[s][c])


def attention_rows(q, k, v, scale=None):
    """One sequence's queries [t, H, D] over all its keys [n, K, D]; query i sees keys
    j <= n - t + i. fp64; a query that sees nothing gives zero. Keys that are not seen
    take no part, whatever they hold."""
    t, H, D = q.shape
    n, K = k.shape[0], k.shape[1]
    scale = 1 / math.sqrt(D) if scale is None else scale
    q, k, v = q.double(), k.double(), v.double()
    out = torch.zeros(t, H, D, dtype=torch.float64, device=q.device)
    if n >= t > 0 and bool(torch.isfinite(k).all()) and bool(torch.isfinite(v).all()):
        hidden = torch.arange(n, device=q.device) > torch.arange(n - t, n, device=q.device)[:, None]
        for h in range(H):
            x = (q[:, h] @ k[:, h // (H // K)].T * scale).masked_fill_(hidden, -math.inf)
            out[:, h] = torch.softmax(x, -1) @ v[:, h // (H // K)]
        return out
    for i in range(t):
        seen = n - t + i + 1
        if seen <= 0:
            continue
        x = torch.einsum("kgd,jkd->kgj", q[i].view(K, H // K, D), k[:seen]) * scale
        out[i] = torch.einsum("kgj,jkd->kgd", torch.softmax(x, -1), v[:seen]).reshape(H, D)
    return out


def attention_prompt(q, k, v, cu, scale=None):
    """Causal attention within each packed sequence; rows from cu[-1] on are not written (NaN here)."""
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device=q.device)
    for a, b in zip(cu, cu[1:]):
        out[a:b] = attention_rows(q[a:b], k[a:b], v[a:b], scale)
    return out


def attention_cached(q, pool, table, lengths, layer, seqs, scale=None):
    """One query per row b over the tokens of sequence seqs[b]."""
    page, out = pool.shape[4], []
    for b, s in enumerate(seqs):
        n = lengths[s]
        pages = torch.tensor(table[s][: -(-n // page)], dtype=torch.long, device=pool.device)
        kv = pool[pages, layer].permute(1, 2, 0, 3, 4).reshape(2, pool.shape[3], -1, pool.shape[5])[:, :, :n]
        out.append(attention_rows(q[b : b + 1], kv[0].transpose(0, 1), kv[1].transpose(0, 1), scale))
    return torch.cat(out)


def error_bound(want, spread, reach, keys, D, dtype):
    """How far a kernel with 16-bit probabilities, 32-bit scores, sums and maxima may be
    from `want` in 64 bits, element by element. `spread`: the attention over |v|;
    `reach`: a bound of scale * sum_d |q_d k_d|; `keys`: the most keys of a row.
    With u half a step of the type: each probability rounded once (u), the result once
    (u); a score's sum of D products and its scaling (D + 4 roundings of 2^-24 of
    `reach`), the maximum subtracted in the base-2 exponent (4 more), a probability
    that is exp(score) moved by as much, in the sum and in the total (twice); the
    exponential's own error twice (2^-21 from the special-function unit, 2^-13.7 for bf16
    and 2^-18.4 for fp16 where a polynomial takes its place: the measured maxima of the
    two polynomials over their interval); the sums over keys (keys 2^-24 twice). `tiny`: what
    underflows (probabilities below 2^-25 of the largest in fp16, results below the
    smallest step)."""
    u = torch.finfo(dtype).eps / 2
    drift = 2 * ((D + 8) * reach * 1.4427 + 2 * keys) * 2.0 ** -24 + 2 * 2.0 ** (-18.4 if dtype == torch.float16 else -13.7)
    tiny = 2.0 ** -24 if dtype == torch.float16 else 2.0 ** -120
    rel = (1 + u) * (1 + drift) * (1 + u) - 1
    return (rel * spread + u * want.abs()) * 1.0001 + tiny * (1 + keys * (dtype == torch.float16) * 2)
