"""Rounds of drafted trees over paged caches for the tests, and their definitions in 64 bits, row by row."""
import math

import numpy as np
import torch

PAGE = 64


class Round:
    """Requests with committed tokens `lengths` and trees `parents` (None: a chain of `counts[s]` rows); pages in random order."""

    def __init__(self, lengths, counts, device="cpu", seed=0, trees=True, pad=0, slots=None, spare=2, width=None):
        self.rs = np.random.RandomState(seed)
        self.lengths, self.counts, self.device = list(lengths), list(counts), device
        S = len(self.lengths)
        self.slots = list(slots) if slots is not None else None
        n_slots = max(self.slots) + 1 if self.slots else S
        self.parents = [[-1 if j == 0 else int(self.rs.randint(-1 if self.rs.rand() < 0.1 else max(0, j - 6), j)) for j in range(n)] if trees
                        else [j - 1 for j in range(n)] for n in self.counts]
        self.trees = trees
        self.starts = [0, *np.cumsum(self.counts).tolist()]
        self.R = self.starts[-1] + pad
        need = [-(-(a + b) // PAGE) for a, b in zip(self.lengths, self.counts)]
        self.n_pages = sum(need) + spare
        order = self.rs.permutation(self.n_pages)
        self.table = np.full((n_slots, width or max(need + [1])), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[self.slot(s), :n] = order[at: at + n]
            at += n
        self.anc = []
        for p in self.parents:
            m = np.eye(len(p), dtype=bool)
            for j, a in enumerate(p):
                if a >= 0:
                    m[j] |= m[a]
            self.anc.append(m)

    def slot(self, s):
        return self.slots[s] if self.slots else s

    def i32(self, x):
        return torch.tensor(np.asarray(x), dtype=torch.int32, device=self.device).contiguous()

    def rows(self, s):
        t = np.arange(self.lengths[s] + self.counts[s])
        return self.table[self.slot(s), t // PAGE].astype(np.int64) * PAGE + t % PAGE

    def flat_parents(self):
        out = np.full(self.R, -1, np.int32)
        for s, p in enumerate(self.parents):
            out[self.starts[s]: self.starts[s + 1]] = p
        return out

    def inputs(self):
        """Arguments of `slot_maps`."""
        d = {"lengths": self.i32(self.lengths), "counts": self.i32(self.counts), "tables": self.i32(self.table), "rows": self.R}
        if self.slots:
            d["slots"] = self.i32(self.slots)
        if self.trees:
            d.update(parents=self.i32(self.flat_parents()), nodes=max(self.counts + [1]))
        return d

    def randn(self, *shape, dtype=torch.float32):
        g = torch.Generator().manual_seed(int(self.rs.randint(1 << 30)))
        return torch.randn(*shape, generator=g).to(dtype).to(self.device)


def want_maps(r):
    """starts, slot, index, pos, cache_row, ancestors [R, nodes] (bool)."""
    slot, index, pos, row = (np.full(r.R, -1, np.int64) for _ in range(4))
    nodes = max(r.counts + [1])
    anc = np.zeros((r.R, nodes), bool)
    for s, (L, n) in enumerate(zip(r.lengths, r.counts)):
        sl = slice(r.starts[s], r.starts[s] + n)
        slot[sl], index[sl], row[sl] = r.slot(s), np.arange(n), r.rows(s)[L:]
        pos[sl] = L + r.anc[s].sum(1) - 1
        anc[sl, :n] = r.anc[s]
    return np.array(r.starts), slot, index, pos, row, anc


def want_attention(r, q, k, v, scale, softcap=0.0, bias=None, slopes=None, sink=None, window=0, chunk=0, gate=None, out_scale=1.0, rounded=0.0):
    """(outputs, error bound) in 64 bits.  The bound counts, in fp32 half steps u = 2^-24: a score's products and sums in any order ((D + 8) u of
    their magnitudes, times two for a score and its row's maximum against one another), an exponential and a weight's scale (16 u), the sum of
    n weighted values (n u); `rounded`: half step of the weights' type; and half a step of the outputs' type."""
    H, D, G, V = q.shape[1], q.shape[2], k.shape[2], v.shape[3]
    dev, u = q.device, 2.0 ** -24
    out, tol = (torch.zeros(q.shape[0], H, V, dtype=torch.float64, device=dev) for _ in range(2))
    kf, vf = k.reshape(-1, G, D), v.reshape(-1, G, V)
    for s, (L, n) in enumerate(zip(r.lengths, r.counts)):
        if n == 0:
            continue
        r0, t = r.starts[s], torch.arange(L + n, device=dev)
        tree = torch.tensor(r.anc[s], device=dev)
        pos = L + tree.sum(1) - 1
        at = torch.cat((t[:L], pos))
        dist = pos.unsqueeze(1) - at
        seen = torch.cat((torch.ones(n, L, dtype=torch.bool, device=dev), tree), 1)
        if chunk:
            seen &= at >= (pos // chunk * chunk).unsqueeze(1)
        if window:
            seen &= dist < window
        rows = torch.tensor(r.rows(s), device=dev)
        for h in range(H):
            g = h // (H // G)
            kk, vv, qq = kf[rows, g].double(), vf[rows, g].double(), q[r0: r0 + n, h].double()
            x, e = qq @ kk.T * scale, (qq.abs() @ kk.abs().T) * abs(scale) * (D + 8) * u
            if softcap:
                x = softcap * torch.tanh(x / softcap)
                e = e + softcap * 8 * u
            if bias is not None:
                x = x + bias[h].double()[dist.clamp(0, bias.shape[1] - 1)]
            if slopes is not None:
                x = x - slopes[h].double() * dist
                e = e + (slopes[h].double() * dist).abs() * 4 * u
            x = x.masked_fill(~seen, -math.inf)
            usual = x.abs() < 1e30
            e = 2 * e.masked_fill(~seen, 0).amax(1) + 4 * u * x.masked_fill(~usual, 0).abs().amax(1)
            top = x.amax(1)
            if sink is not None:
                top = torch.maximum(top, sink[h].double())
            ref = top.masked_fill(top == -math.inf, 0).unsqueeze(1)
            p = torch.exp(x - ref)
            z = p.sum(1) + (torch.exp(sink[h].double() - ref[:, 0]) if sink is not None else 0)
            p = p / z.masked_fill(z == 0, 1).unsqueeze(1)
            f = out_scale * (torch.sigmoid(gate[r0: r0 + n, h].double()) if gate is not None else torch.ones(n, dtype=torch.float64, device=dev))
            out[r0: r0 + n, h] = p @ vv * f.unsqueeze(1)
            tol[r0: r0 + n, h] = (p @ vv.abs()) * (f.abs() * (e + (16 + seen.sum(1)) * u + rounded)).unsqueeze(1)
    return out.cpu(), tol.cpu()


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, want, tol, dtype):
    """Every value within its bound and half a step of its type."""
    err = (got.double().cpu() - want).abs()
    lim = tol + half_step(dtype) * (want.abs() + tol) + 1e-30
    worst = (err / lim).max() if err.numel() else torch.tensor(0.0)
    assert bool((err <= lim).all()), f"{float(worst):.3f} of the bound"
    return float(worst)


def want_conv(r, x, w, tail):
    """y [R, C] and its magnitude (sum of the products' absolute values)."""
    taps = w.shape[0]
    x, w, tail = x.double().cpu(), w.double().cpu(), tail.double().cpu()
    y, mag = torch.zeros_like(x), torch.zeros_like(x)
    for s, p in enumerate(r.parents):
        for j in range(len(p)):
            line, at = [], j
            while at >= 0:
                line.append(x[r.starts[s] + at])
                at = p[at]
            line = (line + list(tail[r.slot(s)].flip(0)))[:taps]
            for t, u in enumerate(line):
                y[r.starts[s] + j] += w[taps - 1 - t] * u
                mag[r.starts[s] + j] += (w[taps - 1 - t] * u).abs()
    return y, mag


def path_of(r, s, j):
    """Path from the root to node j."""
    line = []
    while j >= 0:
        line.append(j)
        j = r.parents[s][j]
    return line[::-1]
