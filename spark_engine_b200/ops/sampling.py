"""From a round's logits to its tokens: counts of what a request has said, penalties, biases and allowed tokens, draws with top-k, top-p and min-p,
log-probabilities (`csrc/kernels/token_counts.cu`, `sample_rows.cu`).

A row's tokens are ordered by descending logit, the lower id first where logits are equal; NaN and -inf are no tokens.  Draws are Gumbel-max with
noise that (seed, position, id) determine (`spec/sampling.py`): a row's token depends on its logits and settings only, and without filters it is the one
that `gumbel_perturb` and `argmax` draw.

Settings and state live on the device, the calls neither wait for it nor read from it, and a captured call may be replayed with others.  A slot outside
the counts sets the device status word and the row goes without any penalties, drafted tokens' too (or its tokens are not counted); for tensors on the host
it is a ValueError.  Ids outside the vocabulary are left out."""
from __future__ import annotations

import ctypes
import importlib.util
import math
import os
import sysconfig
from typing import NamedTuple, Optional

import torch

from . import cuda_ops, use_kernels

_ENTRIES = ("spark_count_tokens", "spark_adjust_rows", "spark_sample_rows", "spark_logprob_rows")
_mod = None
_bound = None
_known = set()                                     # devices that the bindings know


def _native():
    """The bindings (`csrc/bindings/sampling_ops.cpp`): checks of arguments, outputs, launches."""
    global _mod
    if _mod is None:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "_lib", "_sampling" + sysconfig.get_config_var("EXT_SUFFIX"))
        if not os.path.exists(path):
            from ..build import build_sampling
            path = build_sampling()
        spec = importlib.util.spec_from_file_location("_sampling", path)
        _mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(_mod)
    return _mod


def _kernels(t: torch.Tensor) -> bool:
    """Whether the kernels run on this tensor; the bindings then know them and its device."""
    if not use_kernels(t):
        return False
    index = t.get_device()
    if index not in _known:
        _bind(index)
    return True


def _same_layout(mod, dll):
    """The bindings fill structures that the kernels read: both have to come from one header."""
    if not hasattr(dll, "spark_sampling_layout"):
        raise RuntimeError(f"{dll._name} has no sampling kernels: run `python -m spark_engine_b200.build`")
    dll.spark_sampling_layout.restype = ctypes.c_uint
    if dll.spark_sampling_layout() != mod.layout():
        raise RuntimeError(f"{dll._name} and {mod.__file__} were built from different sources: run `python -m spark_engine_b200.build`")


def _bind(index: int):
    global _bound
    mod, cu = _native(), cuda_ops()
    if _bound is None:
        dll = cu.lib()
        _same_layout(mod, dll._dll)
        for name in _ENTRIES:
            mod.bind_entry(name, ctypes.cast(getattr(dll._dll, name), ctypes.c_void_p).value)
        _bound = dll
    mod.bind_device(index, cu.status_word(torch.device("cuda", index)).data_ptr(), torch.cuda.get_device_properties(index).multi_processor_count)
    _known.add(index)


def _count():
    """Counts the kernels that the last call launched (none where there is nothing to do)."""
    cuda_ops().add_launches(_mod.take_launched())


class Adjust(NamedTuple):
    """What a row's logits go through before a token is drawn; tensors on the logits' device, None: none of the kind."""
    counts: Optional[torch.Tensor] = None          # int32 [slots, V]: 2 * times generated + (1 if in the prompt), see `count_tokens`
    slots: Optional[torch.Tensor] = None           # int32 [R]: a row's row of counts (None: its number; negative: the row has no penalties)
    drafted: Optional[torch.Tensor] = None         # int32 [R, n]: tokens on the way to the row that count as generated on top, negative: none
    repetition: Optional[torch.Tensor] = None      # fp32 [R]
    presence: Optional[torch.Tensor] = None        # fp32 [R]
    frequency: Optional[torch.Tensor] = None       # fp32 [R]
    bias_ids: Optional[torch.Tensor] = None        # int32 [R, n]: ids whose logits get the biases (each of an id's), negative: none
    bias: Optional[torch.Tensor] = None            # fp32 [R, n]
    allowed: Optional[torch.Tensor] = None         # int32 [R, (V + 31) / 32]: bit c % 32 of word c / 32 says whether column c may be drawn


# ----------------------------------------------------------------------------- counts
def count_tokens(counts, tokens, n, slots=None, prompt: bool = False, reset: bool = False):
    """Count the first n[s] of tokens[s] ([S, P] int32) in row slots[s] (None: s; negative: nowhere) of counts int32 [slots, V], in place: tokens of
    the answer add 2 each, tokens of the `prompt` set the lowest bit.  `reset`: the rows are zeroed first, as for a new request; its slots are different."""
    run = _kernels(counts)
    _native().count_tokens(counts, tokens, n, slots, prompt, reset, run)
    if run:
        _count()
        return
    for s, k in enumerate(n.tolist()):
        slot = s if slots is None else int(slots[s])
        if slot < 0:
            continue
        if slot >= counts.shape[0]:
            raise ValueError("a slot outside the counts")
        if reset:
            counts[slot] = 0
        ids = tokens[s, : max(k, 0)].long()
        ids = ids[(ids >= 0) & (ids < counts.shape[1])]
        if prompt:
            counts[slot, ids] |= 1
        else:
            counts[slot] += 2 * torch.bincount(ids, minlength=counts.shape[1]).to(torch.int32)


# ----------------------------------------------------------------------------- adjustments
def adjust_logits(logits, adjust: Adjust, offset: int = 0, out=None) -> torch.Tensor:
    """fp32 logits [R, V] after a row's adjustments: of tokens that were generated (or drafted) or are in the prompt, z / repetition where z > 0, else
    z * repetition; minus frequency times the times generated, minus presence if generated; plus the biases of the id; -inf where not allowed.  Logits fp32,
    bf16 or fp16, of ids offset .. offset + V (counts and allowed words are of these columns, ids in the lists are the vocabulary's).  Into `out` if
    given, which may be the logits."""
    run = _kernels(logits)
    y = _native().adjust_logits(logits, adjust, offset, out, run)
    if run:
        _count()
        return y
    return y.copy_(_plain_adjust(logits, adjust, offset))


def _plain_adjust(logits, a, offset: int = 0):
    z = logits.float().clone()
    R, V = z.shape
    for r in range(R):
        slot = r if a.slots is None else int(a.slots[r])
        count = torch.zeros(V, dtype=torch.int32, device=z.device)
        if slot >= 0:
            if a.counts is not None:
                if slot >= a.counts.shape[0]:
                    raise ValueError("a slot outside the counts")
                count = a.counts[slot]
            times, seen = count >> 1, count > 0
            if a.drafted is not None:
                ids = a.drafted[r].long() - offset
                more = torch.bincount(ids[(a.drafted[r] >= 0) & (ids >= 0) & (ids < V)], minlength=V).to(torch.int32)
                times, seen = times + more, seen | (more > 0)
            if a.repetition is not None:
                z[r] = torch.where(seen, torch.where(z[r] > 0, z[r] / a.repetition[r], z[r] * a.repetition[r]), z[r])
            if a.frequency is not None:
                z[r] -= a.frequency[r] * times
            if a.presence is not None:
                z[r] -= torch.where(times > 0, a.presence[r], torch.zeros_like(a.presence[r]))
        if a.bias is not None:
            for i, b in zip(a.bias_ids[r].tolist(), a.bias[r]):
                if i >= 0 and 0 <= i - offset < V:
                    z[r, i - offset] += b
        if a.allowed is not None:
            at = torch.arange(V, device=z.device)
            z[r].masked_fill_((a.allowed[r][at // 32] >> (at % 32)) & 1 == 0, -math.inf)
    return z


# ----------------------------------------------------------------------------- tokens
def sample_tokens(logits, temps, seeds, positions, top_k=None, top_p=None, min_p=None, adjust: Optional[Adjust] = None) -> torch.Tensor:
    """One token per row of logits [R, V] (fp32, bf16, fp16; after `adjust` if given): int32 [R], -1 where a row has none.  temps, top_p, min_p fp32 [R],
    top_k int32 [R], seeds and positions int64 [R].  Kept are the first top_k tokens of the row's order (<= 0: all); of these the ones at least min_p
    times as probable as the first (<= 0: all); of these the shortest run of the order that has top_p of their probability (>= 1: all; one at least).
    Drawn is the arg-max over kept of fp32(logit / temperature) + fp32(g), g = -log(-log u), u from (seed, position, id); rows of temperature <= 0, and
    rows whose best logit / temperature is 2^30 or more in size, beside which noise is nothing, take the first of the order.

    Weights are fp32 (to about 2^-20 of themselves), their sums whole numbers of 2^-40: only where the probability up to a token comes that close to top_p
    can the last one kept be its neighbour, and it is the same one in every batch and wherever the row lies.  An `adjust` takes a workspace of R * V fp32 from torch's allocator, which a captured call keeps."""
    run = _kernels(logits)
    t = _native().sample_tokens(logits, temps, seeds, positions, top_k, top_p, min_p, adjust, run)
    if run:
        _count()
        return t
    z = _plain_adjust(logits, adjust) if adjust is not None else logits.float()
    rows = [_plain_sample(z[r], *(x[r].item() if x is not None else None for x in (temps, seeds, positions, top_k, top_p, min_p))) for r in range(z.shape[0])]
    return t.copy_(torch.tensor(rows, dtype=torch.int32))


def _plain_sample(z, temp, seed, position, k, p, m) -> int:
    from ..spec.sampling import gumbel_noise_ref
    z = torch.where(torch.isnan(z), torch.full_like(z, -math.inf), z)
    z, ids = torch.sort(z, descending=True, stable=True)
    if z[0] == -math.inf:
        return -1
    temp = torch.tensor(temp, dtype=torch.float32, device=z.device)
    if not temp > 0 or not torch.abs(z[0] / temp) < 2.0 ** 30:
        return int(ids[0])
    d = (z.double() - z[0].double()) / temp.double()
    n = int((z > -math.inf).sum())
    if k is not None and k > 0:
        n = min(n, k)
    if m is not None and m > 0:
        n = max(1, min(n, int((d >= math.log(m)).sum())))
    if p is not None and p < 1:
        w = torch.exp(d[:n])
        upto = torch.cumsum(w, 0)
        n = max(1, int((upto - w < p * upto[-1]).sum()))
    score = z[:n] / temp + gumbel_noise_ref(seed, position, z.shape[0], z.device)[ids[:n]]
    return int(ids[:n][score == score.max()].min())


# ----------------------------------------------------------------------------- log-probabilities
class Logprobs(NamedTuple):
    logprob: torch.Tensor                          # fp32 [R]: of the given tokens
    rank: torch.Tensor                             # int32 [R]: their places in the row's order, from 1
    ids: torch.Tensor                              # int32 [R, top]: the first of the order, -1 where a row has fewer
    logprobs: torch.Tensor                         # fp32 [R, top]


def token_logprobs(logits, tokens, top: int = 0) -> Logprobs:
    """log softmax(logits) of tokens int32 [R] and of the `top` (256 at most) most probable ones of every row, for logits [R, V] (fp32, bf16, fp16).  What is
    not in the vocabulary has -inf and rank 0; tokens that are none (-inf, NaN) have -inf.

    Exponentials are fp32, their sums 64 bits beyond 32 of them, differences 64 bits: results are off by about a step of fp32 (2^-21 of the sum at most, and half a
    step).  They are the same in every batch; where rows begin elsewhere between two 16-byte boundaries the last bit may be another."""
    run = _kernels(logits)
    out = Logprobs(*_native().token_logprobs(logits, tokens, top, run))
    if run:
        _count()
        return out
    z = logits.float()
    z = torch.where(torch.isnan(z), torch.full_like(z, -math.inf), z)
    for r in range(z.shape[0]):
        v, ids = torch.sort(z[r], descending=True, stable=True)
        d = torch.where(v == v[0], torch.zeros_like(v), v - v[0]).double()       # (infinite logits: a limit)
        lp = torch.where(v == -math.inf, d.new_tensor(-math.inf), d - torch.log(torch.exp(d).sum()))
        t = int(tokens[r])
        there = 0 <= t < z.shape[1]
        at = int((ids == t).nonzero()) if there else -1
        out.logprob[r], out.rank[r] = (lp[at] if there else -math.inf), at + 1
        n = min(top, int((v > -math.inf).sum()))
        out.ids[r], out.logprobs[r] = -1, -math.inf
        out.ids[r, :n], out.logprobs[r, :n] = ids[:n].to(torch.int32), lp[:n].float()
    return out
