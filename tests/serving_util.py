"""Plain 64-bit references and builders of the serving operators' tests."""

import math

import torch


def build_pool(lens, page, hkv, d, dtype, gen, *, spare=3, fill=None):
    """Random pages [P, Hkv, page, D] (k and v), a scattered table and the lengths, on the CPU."""
    held = [(n + page - 1) // page for n in lens]
    n_pages = sum(held) + spare
    ids = torch.randperm(n_pages, generator=gen).tolist()
    table = torch.full((len(lens), max(1, max(held))), -1, dtype=torch.int32)
    for s, n in enumerate(held):
        for j in range(n):
            table[s, j] = ids.pop()
    k = torch.randn(n_pages, hkv, page, d, generator=gen).to(dtype)
    v = torch.randn(n_pages, hkv, page, d, generator=gen).to(dtype)
    if fill is not None:  # what no sequence owns
        own = torch.zeros(n_pages, page, dtype=torch.bool)
        for s, n in enumerate(lens):
            for j in range(n):
                own[table[s, j // page], j % page] = True
        for t in (k, v):
            f = t.float()
            f[~own[:, None, :].expand(-1, hkv, -1)] = fill
            t.copy_(f.to(dtype))
    return k, v, table, torch.tensor(lens, dtype=torch.int32)


def gather(pages, table_row, n, g):
    """The first n rows of head g of a sequence, 64-bit [n, D]."""
    page = pages.shape[2]
    ids = table_row[: (n + page - 1) // page].long()
    if pages.element_size() == 1:  # 8-bit types are indexed as bytes
        rows = pages.view(torch.uint8)[ids, g].view(pages.dtype)
    else:
        rows = pages[ids, g]
    return rows.float().double().reshape(-1, pages.shape[3])[:n]


def attend64(q, k, v, table, lens, scale, mask=None, ks=None, vs=None, seqs=None):
    """(out, lse) in 64 bits; mask [B or 1, L] covers the first L keys, hidden keys count as absent."""
    b, h, d = q.shape
    hkv = k.shape[1]
    out = torch.zeros(b, h, d, dtype=torch.float64)
    lse = torch.full((b, h), -math.inf, dtype=torch.float64)
    for i in range(b):
        s = i if seqs is None else int(seqs[i])
        n = int(lens[s])
        if n == 0:
            continue
        keep = torch.ones(n, dtype=torch.bool)
        add = torch.zeros(n, dtype=torch.float64)
        if mask is not None:
            m = mask[min(i, mask.shape[0] - 1), :n]
            if m.dtype == torch.bool:
                keep[: len(m)] = m
            else:
                keep[: len(m)] = m != -math.inf
                add[: len(m)] = m.double()
        if not keep.any():
            continue
        for hh in range(h):
            g = hh // (h // hkv)
            kk, vv = gather(k, table[s], n, g)[keep], gather(v, table[s], n, g)[keep]
            if ks is not None:
                kk = kk * ks[g].double()
            if vs is not None:
                vv = vv * vs[g].double()
            x = kk @ q[i, hh].double() * scale + add[keep]
            lse[i, hh] = torch.logsumexp(x, 0)
            out[i, hh] = torch.softmax(x, 0) @ vv
    return out, lse


class PoolModel:
    """The page operations as their documentation puts them, one sequence after the other."""

    def __init__(self, table, lens, refs, data, page):
        self.table, self.lens, self.refs = table.clone(), lens.clone(), refs.clone()
        self.data, self.page = data.clone(), page

    def held(self, s):
        return -(-int(self.lens[s]) // self.page)

    def _release(self, s):
        for j in range(self.held(s)):
            self.refs[self.table[s, j]] -= 1
            self.table[s, j] = -1
        self.lens[s] = 0

    def _free_ids(self):
        return [p for p in range(len(self.refs)) if self.refs[p] <= 0]

    def free(self, seqs):
        for s in seqs:
            if 0 <= s < len(self.lens):
                self._release(s)

    def _pairs(self, src, dst):
        n = len(self.lens)
        for i, (s, d) in enumerate(zip(src, dst)):
            ok = 0 <= s < n and 0 <= d < n and d not in src and d not in dst[:i]
            yield i, s, d, ok

    def fork(self, src, dst):
        for _, s, d, ok in self._pairs(src, dst):
            if not ok:
                continue
            self._release(d)
            for j in range(self.held(s)):
                self.table[d, j] = self.table[s, j]
                self.refs[self.table[s, j]] += 1
            self.lens[d] = self.lens[s]

    def copy(self, src, dst):
        granted = [0] * len(src)
        pairs = [(i, s, d) for i, s, d, ok in self._pairs(src, dst) if ok]
        for _, _, d in pairs:
            self._release(d)
        free, at = self._free_ids(), 0
        for i, s, d in pairs:
            need = self.held(s)
            at += need
            if need and at > len(free):
                continue
            for j in range(need):
                p = free[at - need + j]
                self.table[d, j] = p
                self.refs[p] = 1
                self.data[:, p] = self.data[:, self.table[s, j]]
            self.lens[d] = self.lens[s]
            granted[i] = int(self.lens[s])
        return granted

    def reserve(self, seqs, new):
        granted, plans = [0] * len(seqs), {}
        most = self.table.shape[1] * self.page
        sharers = {}
        for i, (s, a) in enumerate(zip(seqs, new)):
            if not 0 <= s < len(self.lens) or s in seqs[:i] or a < 0 or int(self.lens[s]) + a > most:
                continue
            n = int(self.lens[s])
            tail = int(self.table[s, n // self.page]) if a > 0 and n % self.page else None
            if tail is not None and self.refs[tail] > 1:
                sharers.setdefault(tail, []).append(i)
            else:
                tail = None
            plans[i] = [s, a, tail, -(-(n + a) // self.page) - self.held(s)]
        keeps = {who[-1] for t, who in sharers.items() if len(who) == int(self.refs[t])}
        free, at, served = self._free_ids(), 0, {}
        for i, (s, a, tail, need) in sorted(plans.items()):
            need += tail is not None and i not in keeps
            at += need
            if need == 0 or at <= len(free):
                served[i] = free[at - need:at]
        for i in list(served):
            tail = plans[i][2]
            if i in keeps and any(j not in served for j in sharers[tail]):
                del served[i]
        for i, ids in served.items():
            s, a, tail, need = plans[i]
            held = self.held(s)
            if tail is not None and i not in keeps:
                p = ids[0]
                ids = ids[1:]
                self.data[:, p] = self.data[:, tail]
                self.refs[tail] -= 1
                self.refs[p] = 1
                self.table[s, int(self.lens[s]) // self.page] = p
            for j, p in enumerate(ids):
                self.table[s, held + j] = p
                self.refs[p] = 1
            self.lens[s] += a
            granted[i] = a
        return granted

    def compact(self):
        live = int((self.refs > 0).sum())
        holes = [p for p in range(live) if self.refs[p] <= 0]
        high = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        to = dict(zip(high, holes))
        for a, b in to.items():
            self.data[:, b] = self.data[:, a]
            self.refs[b], self.refs[a] = int(self.refs[a]), 0
        for s in range(len(self.lens)):
            for j in range(self.held(s)):
                p = int(self.table[s, j])
                self.table[s, j] = to.get(p, p)
        return live
