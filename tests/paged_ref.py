"""64-bit definitions of the dense paged-cache operators and the tolerances their outputs are held to."""

import math

import torch

D = 128


class Cache:
    """Pages in either vLLM layout with a permuted block table, and the rows they hold as [B][H, n, 128] views."""

    def __init__(self, lens, H, dtype, block=16, layout="rows", seed=0, device="cuda", spare=4, room=None):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.H, self.block, self.layout, self.dtype = list(lens), H, block, layout, dtype
        B = len(lens)
        room = max(max(lens), 1) + 16 if room is None else room
        self.per = -(-room // block)
        blocks = B * self.per + spare
        shape = (2, blocks, block, H, D) if layout == "rows" else (blocks, H, block, 2 * D)
        self.kv = torch.randn(shape, generator=g).to(dtype).to(device)
        self.table = torch.randperm(blocks, generator=g)[: B * self.per].view(B, self.per).to(torch.int32).to(device)
        self.seq_lens = torch.tensor(self.lens, dtype=torch.int32, device=device)
        self.cap = self.per * block

    def views(self):
        """keys, values [blocks, block, H, 128]"""
        if self.layout == "rows":
            return self.kv[0], self.kv[1]
        return self.kv[..., :D].transpose(1, 2), self.kv[..., D:].transpose(1, 2)

    def rows(self, r, h, n):
        i = torch.arange(n, device=self.kv.device)
        blk = self.table[r].long()[i // self.block]
        k, v = self.views()
        return k[blk, i % self.block, h], v[blk, i % self.block, h]

    def put(self, r, h, slot, k, v):
        ks, vs = self.views()
        blk = int(self.table[r, slot // self.block])
        ks[blk, slot % self.block, h], vs[blk, slot % self.block, h] = k, v


def visible(pos, p, first, window, sinks):
    ok = (pos >= first) & (pos <= p)
    if window:
        ok &= (p - pos < window) | (pos - first < sinks)
    return ok


def attend(cache, q, scale=None, softcap=0.0, slopes=None, window=0, sinks=0, first=None, key_pos=None, query_pos=None):
    """(out, lse, weights, tolerance of out, bound on a score's error) in 64 bits; weights [B][H] -> [n] sums over rows.

    Tolerance of an output element, from the arithmetic the operator documents: products of the inputs are exact in
    fp32 and summed there (128 terms, each addition off by at most 2^-24 of the sum of magnitudes; 2^-23 allows for
    truncating adders), so a score is off by at most ds = 2^-23 (130 scale sum|q k| + 8 |s| + 4); numerator and
    denominator each move by ds relatively, the exponential adds 2^-22, the n additions 2^-24 each, a p rounded to the
    16-bit type half a step, and so does the output."""
    B, T, Hq, _ = q.shape
    H = cache.H
    G = Hq // H
    scale = 1 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64, device=q.device)
    lse = torch.full((B, T, Hq), -math.inf, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    dsm = torch.zeros_like(lse)
    half = torch.finfo(q.dtype).eps / 2
    weights = [[None] * H for _ in range(B)]
    for r, n in enumerate(cache.lens):
        n = max(n, 0)
        for h in range(H):
            k, v = (x.double() for x in cache.rows(r, h, n))
            pos = torch.arange(n, device=q.device) if key_pos is None else key_pos[r, h, :n].long()
            f = max(int(first[r]), 0) if first is not None else 0
            weights[r][h] = torch.zeros(n, dtype=torch.float64, device=q.device)
            for t in range(T):
                p = (n - 1 if query_pos is None else int(query_pos[r])) - (T - 1 - t)
                at = visible(pos, p, f, window, sinks).nonzero().view(-1)
                if at.numel() == 0:
                    continue
                qq = q[r, t, h * G : (h + 1) * G].double()
                s = scale * (qq @ k[at].T)
                mag = abs(scale) * (qq.abs() @ k[at].abs().T)
                if softcap:
                    s = softcap * torch.tanh(s / softcap)
                bias = torch.zeros_like(s)
                if slopes is not None:
                    bias = slopes[h * G : (h + 1) * G].double().view(G, 1) * (p - pos[at]).double()
                s = s - bias
                # the log2 units the kernels work in multiply a score's rounding by 1.45: counted in the 8 |s|
                ds = (2.0**-23 * (130 * mag + 8 * (s.abs() + bias.abs()) + 4)).amax(1)
                z = torch.logsumexp(s, 1)
                w = torch.exp(s - z.view(G, 1))
                rows = slice(h * G, (h + 1) * G)
                out[r, t, rows], lse[r, t, rows] = w @ v[at], z
                wv = w @ v[at].abs()
                rel = 2 * ds.view(G, 1) + 2.0**-22 * 2 + 2.0**-24 * (at.numel() + 300)
                if q.dtype != torch.float32:
                    rel = rel + half
                tol[r, t, rows] = half * out[r, t, rows].abs() + rel * wv + 1e-30
                if q.dtype == torch.float16:
                    tol[r, t, rows] += 2.0**-24  # half a step of its smallest numbers
                dsm[r, t, rows] = ds
                weights[r][h][at] += w.sum(0)
    return out, lse, weights, tol, dsm


def evict(mass, pos, n, budget, sinks, recent, last):
    """Former slot of each of the first min(n, budget) slots after an eviction, by sorting (lists of plain numbers)."""
    if n <= budget:
        return list(range(n))

    def key(i):
        x = float(mass[i])
        if int(pos[i]) < sinks or int(pos[i]) > last - recent:
            return math.inf
        return -math.inf if math.isnan(x) else x

    kept = sorted(sorted(range(n), key=lambda i: (-key(i), i))[:budget])
    stay = {i for i in kept if i < budget}
    late = iter([i for i in kept if i >= budget])
    return [i if i in stay else next(late) for i in range(budget)]
