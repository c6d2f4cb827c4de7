"""Verification of drafted trees over paged caches: block tables and row maps made from request lengths on the device, the short
convolution along a node's path, attention of the nodes, the commit of accepted paths (`csrc/kernels/tree_rows.cu`, `tree_attn.cu`).

A round's rows are the requests' rows one after another: request s brings counts[s] rows, row j of it is written to the cache at the
request's token lengths[s] + j.  In a tree, parents[row] is the parent's index within the request (-1: hangs off the committed tokens),
below the row's own; a row's position is lengths[s] plus its depth, and it sees the committed tokens, its ancestors and itself.  Without
parents the rows are chains.  Lengths, counts, parents, tables and paths live on the device: a captured round may be replayed with others.
The maps refer to lengths, tables, slots and parents, which have to stay as they are until the round is committed; requests of one round
have different slots, and pages that only one of them writes to.

`block_tables` is for callers that keep their free pages on the device as well; the engine's own pages are leased by the host's pool
(`cache/kv.py`), whose tables `slot_maps` and the others read as they are.

The calls neither wait for the device nor read from it.  What they can only find out there sets the device status word: what would be
written to a missing page or read from one is left out, a row whose parent is not in front of it hangs off the committed tokens, and
`commit_paths` skips a request whose path does not ascend or whose pages are missing.  The plain forms, for tensors on the host, leave missing
pages out as well, and raise for such parents and commits before anything has changed."""
from __future__ import annotations

import ctypes
import importlib.util
import math
import os
import sysconfig
from typing import Sequence, Tuple

import torch

from . import cuda_ops, use_kernels

PAGE = 64
_ENTRIES = ("spark_block_tables", "spark_slot_maps", "spark_path_conv", "spark_commit_paths", "spark_tree_attn")
_mod = None
_bound = None
_known = set()                                     # devices that the bindings know


def _native():
    """The bindings (`csrc/bindings/tree_ops.cpp`): checks of arguments, outputs, launches."""
    global _mod
    if _mod is None:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "_lib", "_tree" + sysconfig.get_config_var("EXT_SUFFIX"))
        if not os.path.exists(path):
            from ..build import build_tree
            path = build_tree()
        spec = importlib.util.spec_from_file_location("_tree", path)
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
    if not hasattr(dll, "spark_tree_layout"):
        raise RuntimeError(f"{dll._name} has no tree kernels: run `python -m spark_engine_b200.build`")
    dll.spark_tree_layout.restype = ctypes.c_uint
    if dll.spark_tree_layout() != mod.layout():
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


def _need(ok: bool, what: str):
    if not ok:
        raise ValueError(what)


def __getattr__(name):
    if name == "RowMaps":
        return _native().RowMaps
    raise AttributeError(name)


# ----------------------------------------------------------------------------- block tables
def block_tables(lengths, tables, held, free, n_free) -> torch.Tensor:
    """Let the requests' pages follow their lengths, in place.  lengths [S] int32: tokens request s needs room for (negative: it is left
    as it is); tables [S, pages] int32: its pages in position order, -1 behind the held[s] it has; free int32: stack of free pages, of which
    n_free[0] lie on it, with room for every page of the pool.  Pages go back first (the last request's last page first), then requests
    take theirs in order, each from the top, so that giving back what was just taken restores the stack; a request whose pages are not all
    there gets none, nor does one behind it that needs any.  Returns the tokens [S] int32 that each request now has room for."""
    run = _kernels(tables)
    room = _native().block_tables(lengths, tables, held, free, n_free, run)
    if run:
        _count()
        return room
    return _plain_tables(lengths, tables, held, free, n_free)


def _plain_tables(lengths, tables, held, free, n_free):
    stack, have = free[: int(n_free)].tolist(), held.tolist()
    need = [h if n < 0 else min(-(-n // PAGE), tables.shape[1]) for n, h in zip(lengths.tolist(), have)]
    for s in reversed(range(len(have))):
        for p in reversed(range(need[s], have[s])):
            stack.append(int(tables[s, p]))
            tables[s, p] = -1
        have[s] = min(have[s], need[s])
    asked, top, took = 0, len(stack), 0
    for s, n in enumerate(need):
        asked += n - have[s]
        if asked <= top:
            for p in range(have[s], n):
                took += 1
                tables[s, p] = stack[top - took]
            have[s] = n
    free[:top] = torch.tensor(stack, dtype=torch.int32)
    n_free.fill_(top - took)
    held.copy_(torch.tensor(have, dtype=torch.int32))
    return held * PAGE


# ----------------------------------------------------------------------------- row maps
def slot_maps(lengths, counts, tables, rows: int, slots=None, parents=None, nodes: int = 0) -> "RowMaps":
    """Maps of a round's rows.  lengths, counts [S] int32: committed tokens and new rows of the requests; tables [slots, pages] int32;
    rows: rows of the round's tensors (at least the sum of the counts; the ones behind it belong to nobody); slots [S] int32: the requests'
    rows of the tables (None: their numbers); parents [rows] int32 and nodes, at least the largest count: trees."""
    run = _kernels(tables)
    m = _native().slot_maps(lengths, counts, tables, rows, slots, parents, nodes, run)
    if run:
        _count()
        return m
    return _plain_maps(m)


def _plain_maps(m):
    counts = [max(c, 0) for c in m.counts.tolist()]
    _need(sum(counts) <= m.rows, "more rows than the round's tensors have")
    for t in (m.slot, m.index, m.pos, m.cache_row):
        t.fill_(-1)
    if m.anc is not None:
        m.anc.zero_()
    r, starts = 0, [0]
    slots = m.slots.tolist() if m.slots is not None else range(len(counts))
    for slot, L, n in zip(slots, m.lengths.tolist(), counts):
        L = max(L, 0)
        par = m.parents[r: r + n].tolist() if m.parents is not None else [j - 1 for j in range(n)]
        _need(all(-1 <= p < j for j, p in enumerate(par)) and (m.parents is None or n <= m.nodes), "a tree's nodes must follow their parents")
        depth, anc = [], []
        for j, p in enumerate(par):
            depth.append(depth[p] + 1 if p >= 0 else 0)
            anc.append((anc[p] if p >= 0 else 0) | 1 << j) if m.anc is not None else None
            tok = L + j
            page = int(m.tables[slot, tok // PAGE]) if 0 <= slot < m.tables.shape[0] and tok // PAGE < m.tables.shape[1] else -1
            m.cache_row[r + j] = page * PAGE + tok % PAGE if page >= 0 else -1
            if m.anc is not None:
                w = [(anc[j] >> 32 * i) & 0xffffffff for i in range(m.anc.shape[1])]
                m.anc[r + j] = torch.tensor([x - (1 << 32) if x >> 31 else x for x in w], dtype=torch.int32)
        m.slot[r: r + n], m.index[r: r + n] = slot, torch.arange(n, dtype=torch.int32)
        m.pos[r: r + n] = L + torch.tensor(depth, dtype=torch.int32)
        r += n
        starts.append(r)
    m.starts.copy_(torch.tensor(starts, dtype=torch.int32))
    return m


def _cache_rows(maps, slot: int, tokens, pages: int) -> torch.Tensor:
    """Cache rows of a request's tokens; -1 where its table leads nowhere in a cache of `pages` pages."""
    tables = maps.tables
    t = torch.as_tensor(tokens, dtype=torch.long, device=tables.device)
    if not 0 <= slot < tables.shape[0]:
        return torch.full_like(t, -1)
    page = tables[slot, (t // PAGE).clamp_max(tables.shape[1] - 1)].long()
    there = (t // PAGE < tables.shape[1]) & (page >= 0) & (page < pages)
    return torch.where(there, page * PAGE + t % PAGE, -1)


# ----------------------------------------------------------------------------- convolution along paths
def path_conv(x, w, tail, maps: "RowMaps", nq: int, k, v) -> torch.Tensor:
    """y_j = sum_t w[t] u_t over the row itself (t = taps - 1), its ancestors, then the request's past `tail` [slots, taps - 1, C] (newest
    last).  x [R, C], w fp32 [taps, C].  The first nq channels of y are returned [R, nq]; the others, the row's keys and values, go to its
    row of the caches k, v [pages, 64, ...].  `tail` is left as it is: `commit_paths` advances it.  Rows behind the last request give rows of
    zeros."""
    run = _kernels(x)
    q = _native().path_conv(x, w, tail, maps, nq, k, v, run)
    if run:
        _count()
        return q
    return _plain_conv(x, w, tail, maps, nq, k, v)


def _flat(t, width):
    """(pages, tokens) view of a cache whose pages may be apart."""
    return t.as_strided((t.shape[0], PAGE, width), (t.stride(0), t.stride(1), 1))


def _plain_conv(x, w, tail, maps, nq, k, v):
    taps, nk = w.shape[0], int(math.prod(k.shape[2:]))
    y = torch.zeros_like(x, dtype=torch.float32)
    kf, vf = _flat(k, nk), _flat(v, x.shape[1] - nq - nk)
    for r in range(x.shape[0]):
        slot, j, row = int(maps.slot[r]), int(maps.index[r]), int(maps.cache_row[r])
        if not 0 <= slot < tail.shape[0]:
            continue
        at, back = j, 0
        for t in reversed(range(taps)):
            if at >= 0:
                u = x[r - j + at]
                at = int(maps.parents[r - j + at]) if maps.parents is not None else at - 1
            else:
                back += 1
                u = tail[slot, taps - 1 - back]
            y[r] += w[t] * u.float()
        if 0 <= row < k.shape[0] * PAGE:
            kf[row // PAGE, row % PAGE] = y[r, nq: nq + nk].to(k.dtype)
            vf[row // PAGE, row % PAGE] = y[r, nq + nk:].to(v.dtype)
    return y[:, :nq].to(x.dtype)


# ----------------------------------------------------------------------------- attention
def tree_attention(q, k, v, maps: "RowMaps", scale: float, softcap: float = 0.0, bias=None, slopes=None, sink=None, window: int = 0, chunk: int = 0,
                   gate=None, out_scale: float = 1.0, out=None) -> torch.Tensor:
    """Attention of a round's rows over the paged caches, which hold the rows' own keys and values already: q [R, H, D], k [pages, 64, G, D],
    v [pages, 64, G, V], query head h on key / value head h // (H / G); bf16, or fp32 throughout.  Scores scale * q.k are soft-capped
    (softcap * tanh(s / softcap)), get bias[h, min(distance, n - 1)] (fp32 [H, n]) or lose slopes[h] * distance; rows see the tokens of their
    own aligned `chunk` of positions or of the `window` positions that end at theirs.  sink fp32 [H] enters the denominators, gate [R, H]
    (logits, in q's type) and out_scale scale the outputs.  Into `out` [R, H, V] if given (rows behind the last request are left as they
    were), else a new tensor (they are zero).  A row that sees nothing is zero; what a row does not see has no effect on it, whatever it holds.

    Scores, statistics and sums are fp32.  bf16 heads of up to 256 run on the tensor cores, where a weight enters the product as two bf16 terms
    (2^-17 of it is lost; infinite values that a row sees may give NaN for infinity); what fp32 and wider heads run on keeps weights in fp32.  A call takes a workspace from torch's allocator (39 MB for
    values of 128 in bf16, however small the round), which a captured call keeps."""
    run = _kernels(q)
    o = _native().tree_attention(q, k, v, maps, scale, softcap, bias, slopes, sink, window, chunk, gate, out_scale, out, run)
    if run:
        _count()
        return o
    return _plain_attention(q, k, v, maps, scale, softcap, bias, slopes, sink, window, chunk, gate, out_scale, o, out is None)


def _plain_attention(q, k, v, maps, scale, softcap, bias, slopes, sink, window, chunk, gate, out_scale, out, fresh):
    (R, H, D), G, V = q.shape, k.shape[2], v.shape[3]
    if fresh:
        out.zero_()
    kf, vf = _flat(k, G * D), _flat(v, G * V)
    starts, lengths = maps.starts.tolist(), maps.lengths.tolist()
    slots = maps.slots.tolist() if maps.slots is not None else range(len(lengths))
    for s, (slot, L) in enumerate(zip(slots, lengths)):
        r0, n = starts[s], starts[s + 1] - starts[s]
        if n == 0:
            continue
        L = min(max(L, 0), maps.tables.shape[1] * PAGE)          # (what lies behind the table's last page is not there)
        t = torch.arange(L + n, device=q.device)
        row = _cache_rows(maps, slot, t, k.shape[0])
        page = row.clamp_min(0) // PAGE
        kk, vv = kf[page, t % PAGE].float().view(-1, G, D), vf[page, t % PAGE].float().view(-1, G, V)
        pos, j = maps.pos[r0: r0 + n].long(), torch.arange(n, device=q.device)
        at = torch.cat((t[:L], pos))
        if maps.anc is not None:
            tree = (maps.anc[r0: r0 + n][:, j // 32] >> (j % 32)) & 1 == 1
        else:
            tree = j.unsqueeze(1) >= j
        dist = pos.unsqueeze(1) - at
        seen = torch.cat((torch.ones(n, L, dtype=torch.bool, device=q.device), tree), 1) & (row >= 0)
        if window:
            seen &= dist < window
        if chunk:
            seen &= pos.unsqueeze(1) // chunk == at // chunk
        x = torch.einsum("tgrd,sgd->grts", q[r0: r0 + n].float().view(n, G, H // G, D), kk).reshape(H, n, -1) * scale
        if softcap:
            x = softcap * torch.tanh(x / softcap)
        if bias is not None:
            x = x + bias[:, dist.clamp(0, bias.shape[1] - 1)]
        if slopes is not None:
            x = x - slopes.view(H, 1, 1) * dist
        x = x.masked_fill(~seen, -math.inf)
        m = x.amax(-1, keepdim=True)
        m = torch.maximum(m, sink.view(H, 1, 1)) if sink is not None else m
        m = torch.where(m == -math.inf, torch.zeros_like(m), m)
        p = torch.exp(x - m)
        z = p.sum(-1, keepdim=True) + (torch.exp(sink.view(H, 1, 1) - m) if sink is not None else 0)
        p = torch.where(z == 0, torch.zeros_like(p), p / z).view(G, H // G, n, -1)
        y = torch.einsum("grts,sgd->tgrd", p, vv).reshape(n, H, V)
        odd = ~torch.isfinite(vv).all(-1).all(-1)                # what a row does not see stays out of it
        if bool(odd.any()):
            for i in range(n):
                y[i] = torch.einsum("grs,sgd->grd", p[:, :, i, seen[i]], vv[seen[i]]).reshape(H, V)
        if gate is not None:
            y = y * torch.sigmoid(gate[r0: r0 + n].float()).unsqueeze(-1)
        out[r0: r0 + n] = (y * out_scale).to(out.dtype)
    return out


# ----------------------------------------------------------------------------- commit
def commit_paths(maps: "RowMaps", path, n_path, caches: Sequence[torch.Tensor], tails: Sequence[Tuple[torch.Tensor, torch.Tensor]] = ()):
    """Keep the accepted rows of every request: path [S, P] int32, its first n_path[s] entries the accepted rows' indices in ascending order
    (0: nothing happens to the request).  In every cache [pages, 64, ...] row path[i] of the request moves to its token length + i, and each
    tail [slots, kept, C] of `tails` = [(x [R, C], tail), ...] becomes the last `kept` of (tail, accepted rows of x).  A request whose path
    does not ascend, or whose accepted rows are not in pages that all caches of the call have, stays as it is in every cache and tail.  No
    two of the caches and tails may share memory."""
    run = _kernels(maps.tables)
    _native().commit_paths(maps, path, n_path, caches, tails, run)
    if run:
        _count()
    else:
        _plain_commit(maps, path, n_path, caches, tails)


def _plain_commit(maps, path, n_path, caches, tails):
    slots = maps.slots.tolist() if maps.slots is not None else range(maps.lengths.shape[0])
    pages = min((c.shape[0] for c in caches), default=None)
    todo = []
    for s, (slot, L, n) in enumerate(zip(slots, maps.lengths.tolist(), n_path.tolist())):
        rows = path[s, : max(n, 0)].tolist()
        count = int(maps.starts[s + 1] - maps.starts[s])
        _need(all(0 <= a < count for a in rows) and all(a < b for a, b in zip(rows, rows[1:])), "an accepted path must ascend within its request")
        if not rows:
            continue
        _need(0 <= slot < maps.tables.shape[0], "a request without a row of the tables")
        src = dst = None
        if pages is not None:
            src, dst = (_cache_rows(maps, slot, [max(L, 0) + j for j in at], pages).tolist() for at in (rows, range(len(rows))))
            _need(min(src + dst) >= 0, "an accepted row without a page")
        todo.append((slot, int(maps.starts[s]), rows, src, dst))
    for slot, r0, rows, src, dst in todo:            # (nothing has moved until all of them are known to be good)
        for c in caches:
            flat = _flat(c, int(math.prod(c.shape[2:])))
            for a, b in zip(src, dst):
                if a != b:
                    flat[b // PAGE, b % PAGE] = flat[a // PAGE, a % PAGE]
        for x, t in tails:
            t[slot] = torch.cat((t[slot], x[r0 + torch.tensor(rows, device=x.device)]))[len(rows):]
