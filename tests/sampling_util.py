"""Rows of logits and settings for the sampling tests, and the operators' definitions in 64 bits, row by row."""
import math

import numpy as np
import torch

from spark_engine_b200 import ops
from spark_engine_b200.spec.sampling import uniform_ref

F32 = np.float32


class Rows:
    """R rows of V logits and everything that is drawn by; `kind`: peaked, flat, equal (many ties), holes (-inf, NaN), one (a single token)."""

    def __init__(self, R, V, kind="peaked", dtype=torch.float32, seed=0, device="cpu", pad=0):
        self.rs, self.R, self.V, self.device = np.random.RandomState(seed), R, V, device
        z = self.rs.randn(R, V)
        if kind == "peaked":
            z *= 1.8
            z[np.arange(R)[:, None], self.rs.randint(0, V, (R, 40))] = 6 + 9 * self.rs.rand(R, 40) ** 2
        elif kind == "equal":
            z = np.round(z)
        elif kind == "same":
            z[:] = 1.25
        elif kind == "holes":
            z[self.rs.rand(R, V) < 0.7] = -np.inf
            z[self.rs.rand(R, V) < 0.1] = np.nan
        elif kind == "one":
            at = self.rs.randint(0, V, R)
            z[:] = -np.inf
            z[np.arange(R), at] = self.rs.randn(R)
        wide = torch.full((R, V + pad), 77.0, dtype=dtype)
        wide[:, :V] = torch.tensor(z.astype(F32)).to(dtype)
        self.logits = wide.to(device)[:, :V]                 # rows `pad` apart
        self.z = self.logits.float().cpu().numpy()
        self.seeds, self.positions = self.rs.randint(0, 1 << 40, R), self.rs.randint(0, 1 << 20, R)

    def t(self, x, dtype):
        return torch.tensor(np.asarray(x), dtype=dtype, device=self.device).contiguous()

    def draw(self, temps, top_k=None, top_p=None, min_p=None, adjust=None):
        f, i = torch.float32, torch.int32
        full = lambda x: np.broadcast_to(np.asarray(x), (self.R,))
        opt = lambda x, d: None if x is None else self.t(full(x), d)
        got = ops.sample_tokens(self.logits, self.t(full(temps), f), self.t(self.seeds, torch.int64), self.t(self.positions, torch.int64), top_k=opt(top_k, i),
                                top_p=opt(top_p, f), min_p=opt(min_p, f), adjust=adjust)
        return got.cpu().numpy()

    def want(self, temps, top_k=None, top_p=None, min_p=None, z=None):
        full = lambda x, none: np.broadcast_to(np.asarray(none if x is None else x), (self.R,))
        k, p, m, t = full(top_k, 0), full(top_p, 1.0), full(min_p, 0.0), full(temps, 0)
        z = self.z if z is None else z
        return np.array([want_token(z[r], t[r], int(self.seeds[r]), int(self.positions[r]), int(k[r]), p[r], m[r]) for r in range(self.R)], np.int32)


def order(z):
    """Ids of a row in its order, without what is no token."""
    ids = np.arange(z.shape[0])
    ids = ids[~np.isnan(z) & (z > -np.inf)]
    return ids[np.lexsort((ids, -z[ids].astype(np.float64)))]


def want_kept(z, temp, k, p, m):
    """Ids that a row keeps, in its order (at least one)."""
    ids = order(z)
    if k > 0:
        ids = ids[:k]
    d = (z[ids].astype(np.float64) - float(z[ids[0]])) / float(F32(temp))
    if m > 0:
        n = max(1, int((d >= math.log(float(F32(m)))).sum()))
        ids, d = ids[:n], d[:n]
    if p < 1:
        w = np.exp(d)
        before = np.concatenate(([0.0], np.cumsum(w)[:-1]))
        ids = ids[: max(1, int((before < float(F32(p)) * w.sum()).sum()))]
    return ids


def want_token(z, temp, seed, position, k, p, m):
    ids = order(z)
    if not len(ids):
        return -1
    with np.errstate(over="ignore"):
        if not temp > 0 or not abs(F32(z[ids[0]]) / F32(temp)) < 2.0 ** 30:      # (beside which noise is nothing)
            return int(ids[0])
    kept = want_kept(z, temp, k, p, m)
    u = uniform_ref(seed, position, z.shape[0]).numpy()[kept]
    with np.errstate(over="ignore"):
        score = z[kept].astype(F32) / F32(temp) + (-np.log(-np.log(u))).astype(F32)
    return int(kept[score == score.max()].min())


def want_logprobs(z, t, top):
    """(log-probability, rank, ids, log-probabilities) of a row."""
    ids = order(z)
    lp = np.full(z.shape[0], -np.inf)
    if len(ids):
        with np.errstate(invalid="ignore"):
            d = np.where(z[ids] == z[ids[0]], 0.0, z[ids].astype(np.float64) - float(z[ids[0]]))
        lp[ids] = d - math.log(np.exp(d).sum())
    there = 0 <= t < z.shape[0]
    rank = 0
    if there:
        real = np.nan_to_num(z.astype(np.float64), nan=-np.inf, posinf=np.inf, neginf=-np.inf)
        rank = 1 + int(((real > real[t]) | ((real == real[t]) & (np.arange(z.shape[0]) < t))).sum())
    first = list(ids[:top]) + [-1] * max(0, top - len(ids))
    return lp[t] if there else -np.inf, rank, first, [lp[i] if i >= 0 else -np.inf for i in first]


def near(got, want):
    """fp32 log-probabilities: the sum of exponentials is off by at most 2^-21 of itself (their own error, that of their arguments times the
    argument, fp32 partial sums of a few terms), the differences and the result by half a step each."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    fine = np.isfinite(want)
    assert np.array_equal(fine, np.isfinite(got)) and np.array_equal(got[~fine], want[~fine])
    err, tol = np.abs(got[fine] - want[fine]), 2.0 ** -21 + 2.0 ** -22 * np.abs(want[fine])
    assert (err <= tol).all(), (err / tol).max()


class Table:
    """Adjustments of R rows, k rows of a request each, and what they make of logits in 64 bits."""

    def __init__(self, rows: Rows, per=1, drafts=0, biases=0, allowed=None, prompt=50, answer=30, dup=False):
        rs, R, V = rows.rs, rows.R, rows.V
        self.r, S = rows, -(-R // per)
        self.counts = np.zeros((S, V), np.int64)
        for s in range(S):
            self.counts[s, rs.randint(0, V, prompt)] |= 1
            np.add.at(self.counts[s], rs.randint(0, V, answer), 2)
        self.slots = np.arange(R) // per
        self.slots[rs.rand(R) < 0.1] = -1
        self.drafted = rs.randint(0, V, (R, drafts)) if drafts else None
        if drafts:
            self.drafted[rs.rand(R, drafts) < 0.3] = -1
            self.drafted[rs.rand(R) < 0.3, -1] = self.drafted[0, 0]      # (some twice)
        self.rep, self.pres, self.freq = (F32(x) for x in (0.8 + rs.rand(R), rs.rand(R), 0.5 * rs.rand(R)))
        self.bias_ids = self.bias = None
        if biases:
            self.bias_ids = np.stack([rs.choice(V, biases, replace=dup or biases > V) for _ in range(R)])
            self.bias_ids[rs.rand(R, biases) < 0.2] = -1
            self.bias = F32(rs.randn(R, biases) * 3)
        self.bits = None
        if allowed is not None:
            self.bits = rs.rand(R, V) < allowed
            if R > 2:
                self.bits[1] = False

    def adjust(self):
        r = self.r
        words = None
        if self.bits is not None:
            n = -(-r.V // 32)
            b = np.zeros((r.R, n * 32), np.uint64)
            b[:, : r.V] = self.bits
            words = (b.reshape(r.R, n, 32) << np.arange(32, dtype=np.uint64)).sum(2).astype(np.uint32).view(np.int32)
        i, f = torch.int32, torch.float32
        opt = lambda x, d: None if x is None else r.t(x, d)
        return ops.Adjust(counts=r.t(self.counts, i), slots=r.t(self.slots, i), drafted=opt(self.drafted, i), repetition=r.t(self.rep, f), presence=r.t(self.pres, f),
                          frequency=r.t(self.freq, f), bias_ids=opt(self.bias_ids, i), bias=opt(self.bias, f), allowed=opt(words, i))

    def want(self):
        """(adjusted logits in 64 bits, how far fp32 may be off: half a step of every intermediate result)."""
        z = self.r.z.astype(np.float64)
        tol = np.zeros_like(z)
        half = lambda x: np.abs(np.where(np.isfinite(x), x, 0)) * 2.0 ** -24
        for r in range(self.r.R):
            if self.slots[r] >= 0:
                c = self.counts[self.slots[r]] >> 1
                prompt = self.counts[self.slots[r]] & 1
                if self.drafted is not None:
                    c = c + np.bincount(self.drafted[r][self.drafted[r] >= 0], minlength=self.r.V)
                rep = np.where((c > 0) | (prompt > 0), float(self.rep[r]), 1.0)
                z[r] = np.where(z[r] > 0, z[r] / rep, z[r] * rep)
                tol[r] += half(z[r]) + half(float(self.freq[r]) * c)
                z[r] = z[r] - float(self.freq[r]) * c
                tol[r] += half(z[r])
                z[r] = z[r] - float(self.pres[r]) * (c > 0)
                tol[r] += half(z[r])
            if self.bias is not None:
                for i, b in zip(self.bias_ids[r], self.bias[r]):
                    if i >= 0:
                        z[r, i] += float(b)
                        tol[r, i] += half(z[r, i])
            if self.bits is not None:
                z[r][~self.bits[r]] = -np.inf
        return z, tol * (1 + 2.0 ** -20)
