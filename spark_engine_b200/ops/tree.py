"""Verification of drafted trees over paged caches: block tables and row maps made from request lengths on the device, the short
convolution along a node's path, attention of the nodes, the commit of accepted paths (`csrc/kernels/tree_rows.cu`, `tree_attn.cu`).

A round's rows are the requests' rows one after another: request s brings counts[s] rows, row j of it is written to the cache at the
request's token lengths[s] + j.  In a tree, parents[row] is the parent's index within the request (-1: hangs off the committed tokens),
below the row's own; a row's position is lengths[s] plus its depth, and it sees the committed tokens, its ancestors and itself.  Without
parents the rows are chains.  Lengths, counts, parents, tables and paths live on the device: a captured round may be replayed with others.

The calls neither wait for the device nor read from it.  What they can only find out there (a missing page, a parent behind its child, a
path that does not ascend) skips the row, or the request in `commit_paths`, and sets the device status word."""
from __future__ import annotations

import contextlib
import ctypes as C
import math
from typing import List, Optional, Sequence, Tuple

import torch

PAGE = 64
MAX_ROWS = 1 << 22           # of a round
MAX_NODES = 1024             # of a request's tree
MAX_PATH = 1024
MAX_HEAD = 512               # channels of a head

_i, _p, _l, _f = C.c_int, C.c_void_p, C.c_longlong, C.c_float


def _struct(*groups):
    return [(n, t) for t, names in groups for n in names.split()]


class _BlockTables(C.Structure):
    _fields_ = _struct((_p, "lengths tables held free n_free room status"), (_i, "S ld cap"))


class _SlotMaps(C.Structure):
    _fields_ = _struct((_p, "lengths counts tables slots parents starts slot index pos anc cache_row status"), (_i, "S R ld n_slots nodes words"))


class _PathConv(C.Structure):
    _fields_ = _struct((_p, "x w tail q k v slot index parents cache_row status"), (_l, "k_page k_tok v_page v_tok cache_rows"),
                       (_i, "ldx R C taps nq nk n_slots"))


class _CommitJob(C.Structure):
    _fields_ = _struct((_p, "base x"), (_l, "page tok"), (_i, "bytes extent kept pad"))


_JOBS = 64


class _CommitPaths(C.Structure):
    _fields_ = [("job", _CommitJob * _JOBS)] + _struct((_p, "path n_path starts lengths slots tables status"), (_i, "S P ld n_slots"))


class _TreeAttn(C.Structure):
    _fields_ = _struct((_p, "q k v out starts lengths slots pos pages anc bias slopes sink gate part_o part_ml split status"),
                       (_l, "k_page k_tok v_page v_tok"),
                       (_i, "S R words page_ld n_slots n_pages H G D V ldq hq ldo ho ldg bias_n window chunk bm sms ctas min_tiles zero_rest"),
                       (_f, "scale cap out_scale"))


_SIGS = {"spark_block_tables": [_p, _p], "spark_slot_maps": [_p, _p], "spark_path_conv": [_p, _i, _p], "spark_commit_paths": [_p, _i, _i, _p],
         "spark_tree_attn": [_p, _i, _i, _p]}
_bound = None


def _cu():
    """The bindings with this module's entry points declared."""
    global _bound
    from . import cuda as cu
    dll = cu.lib()
    if _bound is not dll:
        for name, sig in _SIGS.items():
            fn = getattr(dll._dll, name)
            fn.argtypes, fn.restype = sig, _i
        cu._KERNELS_PER_CALL["spark_tree_attn"] = 2
        _bound = dll
    return cu


def _call(name: str, dev, *args):
    """Launch on the tensors' device, on its current stream."""
    cu = _cu()
    here = contextlib.nullcontext() if dev.index is None or dev.index == torch.cuda.current_device() else torch.cuda.device(dev)
    with here:
        cu.check(getattr(cu.lib(), name)(*args, torch.cuda.current_stream(dev).cuda_stream), name)


def _use(t) -> bool:
    from . import use_kernels
    return use_kernels(t)


def _need(ok: bool, what: str):
    if not ok:
        raise ValueError(what)


def _ints(name: str, t, shape, dev):
    _need(torch.is_tensor(t) and t.dtype == torch.int32 and t.device == dev and t.is_contiguous() and t.dim() == len(shape)
          and all(a == b for a, b in zip(t.shape, shape) if b is not None),
          f"{name} must be a contiguous int32 tensor {tuple('any' if s is None else s for s in shape)} on {dev}")


# ----------------------------------------------------------------------------- block tables
def block_tables(lengths, tables, held, free, n_free) -> torch.Tensor:
    """Let the requests' pages follow their lengths, in place.  lengths [S] int32: tokens request s needs room for (negative: it is left
    as it is); tables [S, pages] int32: its pages in position order, -1 behind the held[s] it has; free int32: stack of free pages, of which
    n_free[0] lie on it, with room for every page of the pool.  Pages go back first (the last request's last page first), then requests
    take theirs in order, each from the top, so that giving back what was just taken restores the stack; a request whose pages are not all
    there gets none, nor does one behind it that needs any.  Returns the tokens [S] int32 that each request now has room for."""
    dev = tables.device
    _need(tables.dim() == 2 and tables.shape[1] > 0, "tables must be [requests, pages]")
    S, ld = tables.shape
    _ints("tables", tables, (None, None), dev)
    _ints("lengths", lengths, (S,), dev)
    _ints("held", held, (S,), dev)
    _ints("free", free, (None,), dev)
    _ints("n_free", n_free, (1,), dev)
    _need(tables.numel() <= 1 << 24, "tables of more than 2^24 entries")
    if not _use(tables):
        return _plain_tables(lengths, tables, held, free, n_free)
    room = torch.empty(S, dtype=torch.int32, device=dev)
    cu = _cu()
    a = _BlockTables(cu.P(lengths), cu.P(tables), cu.P(held), cu.P(free), cu.P(n_free), cu.P(room), cu.P(cu.status_word(dev)), S, ld, free.shape[0])
    _call("spark_block_tables", dev, C.byref(a))
    return room


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
class RowMaps:
    """Where a round's rows belong (int32 unless said otherwise; -1 for rows behind the last request): slot [R] row of the tables, index
    [R] within the request, pos [R], cache_row [R] int64 (page * 64 + token; -1 too where the table has no page), starts [S + 1] first row
    of every request, anc [R, words] ancestors-or-self as bits over the request's rows (trees; else None)."""

    def __init__(self, starts, slot, index, pos, cache_row, anc, lengths, counts, tables, slots, parents, nodes):
        self.starts, self.slot, self.index, self.pos, self.cache_row, self.anc = starts, slot, index, pos, cache_row, anc
        self.lengths, self.counts, self.tables, self.slots, self.parents, self.nodes = lengths, counts, tables, slots, parents, nodes

    @property
    def rows(self) -> int:
        return self.slot.shape[0]


def slot_maps(lengths, counts, tables, rows: int, slots=None, parents=None, nodes: int = 0) -> RowMaps:
    """Maps of a round's rows.  lengths, counts [S] int32: committed tokens and new rows of the requests; tables [slots, pages] int32;
    rows: rows of the round's tensors (at least the sum of the counts; the ones behind it belong to nobody); slots [S] int32: the requests'
    rows of the tables (None: their numbers); parents [rows] int32 and nodes, at least the largest count: trees."""
    dev = tables.device
    _need(tables.dim() == 2 and tables.shape[1] > 0, "tables must be [slots, pages]")
    _ints("tables", tables, (None, None), dev)
    _ints("lengths", lengths, (None,), dev)
    S = lengths.shape[0]
    _ints("counts", counts, (S,), dev)
    if slots is not None:
        _ints("slots", slots, (S,), dev)
    else:
        _need(S <= tables.shape[0], "more requests than rows of the tables")
    if parents is not None:
        _ints("parents", parents, (rows,), dev)
        _need(0 < nodes <= MAX_NODES, f"a request's tree has 1 to {MAX_NODES} nodes (`nodes`)")
    else:
        _need(nodes == 0, "`nodes` belongs to `parents`")
    _need(0 <= rows <= MAX_ROWS and S <= 8192, f"at most {MAX_ROWS} rows of 8192 requests")
    words = -(-nodes // 32)
    new = lambda *s, dt=torch.int32: torch.empty(*s, dtype=dt, device=dev)
    m = RowMaps(new(S + 1), new(rows), new(rows), new(rows), new(rows, dt=torch.int64), new(rows, words) if words else None, lengths, counts, tables,
                slots, parents, nodes)
    if not _use(tables):
        return _plain_maps(m)
    if S == 0:
        for t in (m.slot, m.index, m.pos, m.cache_row):
            t.fill_(-1)
        m.starts.zero_()
        return m
    cu = _cu()
    a = _SlotMaps(cu.P(lengths), cu.P(counts), cu.P(tables), cu.P(slots), cu.P(parents), cu.P(m.starts), cu.P(m.slot), cu.P(m.index), cu.P(m.pos),
                  cu.P(m.anc), cu.P(m.cache_row), cu.P(cu.status_word(dev)), S, rows, tables.shape[1], tables.shape[0], nodes, words)
    _call("spark_slot_maps", dev, C.byref(a))
    return m


def _plain_maps(m: RowMaps) -> RowMaps:
    counts = [max(c, 0) for c in m.counts.tolist()]
    _need(sum(counts) <= m.rows, "more rows than the round's tensors have")
    for t in (m.slot, m.index, m.pos, m.cache_row):
        t.fill_(-1)
    if m.anc is not None:
        m.anc.zero_()
    r, starts = 0, [0]
    slots = m.slots.tolist() if m.slots is not None else range(len(counts))
    for slot, L, n in zip(slots, m.lengths.tolist(), counts):
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


# ----------------------------------------------------------------------------- caches
def _cache(name: str, t, dtype, dev, width: Optional[int] = None) -> Tuple[int, int]:
    """Strides (elements) of the pages and of the tokens of a cache [pages, 64, ...] whose tokens are contiguous."""
    inner = int(math.prod(t.shape[2:])) if torch.is_tensor(t) and t.dim() >= 3 else 0
    _need(inner > 0 and t.shape[1] == PAGE and t.dtype == dtype and t.device == dev, f"{name} must be a {dtype} cache [pages, {PAGE}, heads, channels] on {dev}")
    want, st = 1, list(t.stride())
    for n, s in zip(reversed(t.shape[2:]), reversed(st[2:])):
        _need(n == 1 or s == want, f"{name}: a token's channels must be contiguous")
        want *= n
    e = 16 // t.element_size()
    _need(t.data_ptr() % 16 == 0 and st[0] % e == 0 and st[1] % e == 0 and inner % e == 0 and st[1] >= inner, f"{name}: tokens must start on 16 bytes")
    _need(width is None or inner == width, f"{name} holds {inner} channels of a token, not {width}")
    _need(t.shape[0] <= 1 << 24, f"{name} has more than 2^24 pages")
    return st[0], st[1]


def _rows16(t):
    """Rows that start on 16 bytes (a copy where they do not)."""
    e = 16 // t.element_size()
    ok = t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s % e == 0 for s in t.stride()[:-1])
    return t if ok else t.contiguous()


# ----------------------------------------------------------------------------- convolution along paths
def path_conv(x, w, tail, maps: RowMaps, nq: int, k, v) -> torch.Tensor:
    """y_j = sum_t w[t] u_t over the row itself (t = taps - 1), its ancestors, then the request's past `tail` [slots, taps - 1, C] (newest
    last).  x [R, C], w fp32 [taps, C].  The first nq channels of y are returned [R, nq]; the others, the row's keys and values, go to its
    row of the caches k, v [pages, 64, ...].  `tail` is left as it is: `commit_paths` advances it.  Rows behind the last request give rows of
    zeros."""
    dev, taps = x.device, w.shape[0]
    _need(x.dim() == 2 and x.dtype in (torch.bfloat16, torch.float32), "rows must be bf16 or fp32 [rows, channels]")
    R, Cn = x.shape
    _need(R == maps.rows, "the maps are another round's")
    _need(w.shape == (taps, Cn) and w.dtype == torch.float32 and w.device == dev and w.is_contiguous() and taps > 0, "w must be fp32 [taps, channels]")
    _need(tail.dim() == 3 and tail.shape[1:] == (taps - 1, Cn) and tail.dtype == x.dtype and tail.device == dev and tail.is_contiguous(),
          "tail must be [slots, taps - 1, channels] in the rows' type")
    _need(tail.shape[0] == maps.tables.shape[0], "tail and tables must have the same slots")
    kp, kt = _cache("k", k, x.dtype, dev)
    nk = int(math.prod(k.shape[2:]))
    vp, vt = _cache("v", v, x.dtype, dev, Cn - nq - nk)
    _need(k.shape[0] == v.shape[0], "k and v must have the same pages")
    _need(nq >= 0 and nq % 8 == 0 and nk % 8 == 0 and Cn % 8 == 0, "channels must be multiples of 8")
    if not _use(x):
        return _plain_conv(x, w, tail, maps, nq, k, v)
    q = torch.empty(R, nq, dtype=x.dtype, device=dev)
    if R == 0:
        return q
    x = _rows16(x)
    if x.stride(0) % 8:
        x = x.contiguous()
    cu = _cu()
    a = _PathConv(cu.P(x), cu.P(w), cu.P(tail), cu.P(q), cu.P(k), cu.P(v), cu.P(maps.slot), cu.P(maps.index), cu.P(maps.parents), cu.P(maps.cache_row),
                  cu.P(cu.status_word(dev)), kp, kt, vp, vt, k.shape[0] * PAGE, x.stride(0), R, Cn, taps, nq, nk, tail.shape[0])
    _call("spark_path_conv", dev, C.byref(a), int(x.dtype == torch.float32))
    return q


def _flat(t, width):
    """(pages, tokens) view of a cache whose pages may be apart."""
    return t.as_strided((t.shape[0], PAGE, width), (t.stride(0), t.stride(1), 1))


def _plain_conv(x, w, tail, maps, nq, k, v):
    taps, nk = w.shape[0], int(math.prod(k.shape[2:]))
    y = torch.zeros_like(x, dtype=torch.float32)
    kf, vf = _flat(k, nk), _flat(v, x.shape[1] - nq - nk)
    for r in range(x.shape[0]):
        slot, j, row = int(maps.slot[r]), int(maps.index[r]), int(maps.cache_row[r])
        if slot < 0:
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
        if row >= 0:
            kf[row // PAGE, row % PAGE] = y[r, nq: nq + nk].to(k.dtype)
            vf[row // PAGE, row % PAGE] = y[r, nq + nk:].to(v.dtype)
    return y[:, :nq].to(x.dtype)


# ----------------------------------------------------------------------------- attention
def tree_attention(q, k, v, maps: RowMaps, scale: float, softcap: float = 0.0, bias=None, slopes=None, sink=None, window: int = 0, chunk: int = 0,
                   gate=None, out_scale: float = 1.0, out=None) -> torch.Tensor:
    """Attention of a round's rows over the paged caches, which hold the rows' own keys and values already: q [R, H, D], k [pages, 64, G, D],
    v [pages, 64, G, V], query head h on key / value head h // (H / G); bf16, or fp32 throughout.  Scores scale * q.k are soft-capped
    (softcap * tanh(s / softcap)), get bias[h, min(distance, n - 1)] (fp32 [H, n]) or lose slopes[h] * distance; rows see the tokens of their
    own aligned `chunk` of positions or of the `window` positions that end at theirs.  sink fp32 [H] enters the denominators, gate [R, H]
    (logits, in q's type) and out_scale scale the outputs.  Into `out` [R, H, V] if given (rows behind the last request are left as they
    were), else a new tensor (they are zero).  A row that sees nothing is zero; what a row does not see has no effect on it, whatever it holds."""
    dev, dt = q.device, q.dtype
    _need(q.dim() == 3 and dt in (torch.bfloat16, torch.float32), "queries must be bf16 or fp32 [rows, heads, channels]")
    R, H, D = q.shape
    kp, kt = _cache("k", k, dt, dev)
    vp, vt = _cache("v", v, dt, dev)
    _need(k.dim() == 4 and v.dim() == 4 and k.shape[:3] == v.shape[:3] and k.shape[3] == D, "caches must be [pages, 64, heads, channels], keys as wide as queries")
    G, V = k.shape[2], v.shape[3]
    _need(G > 0 and H % G == 0, "query heads must be a multiple of the key / value heads")
    _need(D % 8 == 0 and V % 8 == 0 and D <= MAX_HEAD and V <= MAX_HEAD, f"head widths must be multiples of 8 up to {MAX_HEAD}")
    _need(R == maps.rows and maps.tables.device == dev, "the maps are another round's")
    _need(window >= 0 and chunk >= 0 and not (window and chunk), "either a window or a chunk")
    _need(softcap >= 0 and math.isfinite(softcap) and math.isfinite(scale), "scale and soft cap must be finite, the cap not negative")
    for name, t, shape in (("bias", bias, (H, None)), ("slopes", slopes, (H,)), ("sink", sink, (H,))):
        _need(t is None or (t.dtype == torch.float32 and t.device == dev and t.is_contiguous() and t.dim() == len(shape) and t.shape[0] == H and t.numel() > 0),
              f"{name} must be a contiguous fp32 tensor of {H} heads on {dev}")
    _need(gate is None or (gate.shape == (R, H) and gate.dtype == dt and gate.device == dev and gate.stride(1) == 1), "gate must be [rows, heads] in the queries' type")
    fresh = out is None
    if fresh:
        out = torch.empty(R, H, V, dtype=dt, device=dev)
    else:
        e = 16 // out.element_size()
        _need(out.shape == (R, H, V) and out.dtype == dt and out.device == dev and out.stride(2) == 1 and out.data_ptr() % 16 == 0
              and out.stride(0) % e == 0 and out.stride(1) % e == 0, "out must be [rows, heads, value channels] in the queries' type, heads on 16 bytes")
    if R == 0 or H == 0:
        return out
    if maps.lengths.shape[0] == 0:
        return out.zero_() if fresh else out
    if not _use(q):
        return _plain_attention(q, k, v, maps, scale, softcap, bias, slopes, sink, window, chunk, gate, out_scale, out, fresh)
    q = _rows16(q)
    cu = _cu()
    sms = torch.cuda.get_device_properties(dev).multi_processor_count
    # tensor cores: one tile of 128 (node, head) rows per CTA and two CTAs per SM, or two tiles that share the keys (trees of more rows)
    tc = dt == torch.bfloat16 and max(D, V) <= 256
    if tc:
        bm = 256 if max(D, V) <= 128 and min(maps.nodes or R, R) * (H // G) > 128 else 128
        ctas = sms if bm == 256 or max(D, V) > 128 else 2 * sms
    else:
        bm, ctas = 32, 3 * sms
    part_o = torch.empty(ctas * 2 * bm * V, dtype=torch.float32, device=dev)
    part_ml = torch.empty(ctas * 2 * bm * 2, dtype=torch.float32, device=dev)
    split = torch.empty(ctas * 4, dtype=torch.int32, device=dev)
    P = cu.P
    a = _TreeAttn(P(q), P(k), P(v), P(out), P(maps.starts), P(maps.lengths), P(maps.slots), P(maps.pos), P(maps.tables), P(maps.anc), P(bias), P(slopes),
                  P(sink), P(gate), P(part_o), P(part_ml), P(split), P(cu.status_word(dev)), kp, kt, vp, vt, maps.lengths.shape[0], R,
                  maps.anc.shape[1] if maps.anc is not None else 0, maps.tables.shape[1], maps.tables.shape[0], k.shape[0], H, G, D, V, q.stride(0),
                  q.stride(1), out.stride(0), out.stride(1), gate.stride(0) if gate is not None else 0, bias.shape[1] if bias is not None else 0, window,
                  chunk, bm, sms, ctas, 1, int(fresh), scale, softcap, out_scale)
    _call("spark_tree_attn", dev, C.byref(a), int(dt == torch.float32), int(tc))
    return out


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
        t = torch.arange(L + n, device=q.device)
        page = maps.tables[slot, t // PAGE].long()
        kk, vv = kf[page.clamp_min(0), t % PAGE].float().view(-1, G, D), vf[page.clamp_min(0), t % PAGE].float().view(-1, G, V)
        pos, j = maps.pos[r0: r0 + n].long(), torch.arange(n, device=q.device)
        at = torch.cat((t[:L], pos))
        if maps.anc is not None:
            tree = (maps.anc[r0: r0 + n][:, j // 32] >> (j % 32)) & 1 == 1
        else:
            tree = j.unsqueeze(1) >= j
        dist = pos.unsqueeze(1) - at
        seen = torch.cat((torch.ones(n, L, dtype=torch.bool, device=q.device), tree), 1) & (page >= 0)
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
def commit_paths(maps: RowMaps, path, n_path, caches: Sequence[torch.Tensor], tails: Sequence[Tuple[torch.Tensor, torch.Tensor]] = ()):
    """Keep the accepted rows of every request: path [S, P] int32, its first n_path[s] entries the accepted rows' indices in ascending order
    (0: nothing happens to the request).  In every cache [pages, 64, ...] row path[i] of the request moves to its token length + i, and each
    tail [slots, kept, C] of `tails` = [(x [R, C], tail), ...] becomes the last `kept` of (tail, accepted rows of x)."""
    dev, S = maps.tables.device, maps.lengths.shape[0]
    _ints("path", path, (S, None), dev)
    _ints("n_path", n_path, (S,), dev)
    P = path.shape[1]
    _need(P <= MAX_PATH, f"paths of at most {MAX_PATH} rows")
    jobs: List[tuple] = []
    for i, c in enumerate(caches):
        _need(torch.is_tensor(c) and c.dtype in (torch.bfloat16, torch.float32), "caches must be bf16 or fp32")
        cp, ct = _cache(f"cache {i}", c, c.dtype, dev)
        e = c.element_size()
        jobs.append((c.data_ptr(), None, cp * e, ct * e, int(math.prod(c.shape[2:])) * e, c.shape[0], 0, 0))
    for x, t in tails:
        _need(t.dim() == 3 and t.is_contiguous() and t.shape[0] == maps.tables.shape[0] and t.device == dev, "tails must be contiguous [slots, kept, channels]")
        _need(x.dim() == 2 and x.shape == (maps.rows, t.shape[2]) and x.dtype == t.dtype and x.device == dev and x.stride(1) == 1,
              "the rows behind a tail must be [rows, channels] in its type")
        e = t.element_size()
        _need(t.shape[2] * e % 16 == 0 and x.stride(0) * e % 16 == 0 and x.data_ptr() % 16 == 0 and t.data_ptr() % 16 == 0, "rows and tails must start on 16 bytes")
        jobs.append((t.data_ptr(), x.data_ptr(), x.stride(0) * e, t.shape[2] * e, t.shape[2] * e, t.shape[0], t.shape[1], 0))
    jobs = [j for j in jobs if j[0]]                     # (tensors without elements have no address)
    _need(len({j[0] for j in jobs}) == len(jobs), "a cache or tail is given twice")
    if not jobs or S == 0 or P == 0 or maps.rows == 0:
        return
    if not _use(maps.tables):
        return _plain_commit(maps, path, n_path, caches, tails)
    cu = _cu()
    ptr = cu.P
    for at in range(0, len(jobs), _JOBS):
        part = jobs[at: at + _JOBS]
        a = _CommitPaths((_CommitJob * _JOBS)(*[_CommitJob(*j) for j in part]), ptr(path), ptr(n_path), ptr(maps.starts), ptr(maps.lengths), ptr(maps.slots),
                         ptr(maps.tables), ptr(cu.status_word(dev)), S, P, maps.tables.shape[1], maps.tables.shape[0])
        _call("spark_commit_paths", dev, C.byref(a), len(part), max(j[4] for j in part))


def _plain_commit(maps, path, n_path, caches, tails):
    slots = maps.slots.tolist() if maps.slots is not None else range(maps.lengths.shape[0])
    for s, (slot, L, n) in enumerate(zip(slots, maps.lengths.tolist(), n_path.tolist())):
        rows = path[s, : max(n, 0)].tolist()
        count = int(maps.starts[s + 1] - maps.starts[s])
        _need(all(0 <= a < count for a in rows) and all(a < b for a, b in zip(rows, rows[1:])), "an accepted path must ascend within its request")
        at = lambda j: (int(maps.tables[slot, (L + j) // PAGE]), (L + j) % PAGE)
        for c in caches:
            flat = _flat(c, int(math.prod(c.shape[2:])))
            for i, j in enumerate(rows):
                if i != j:
                    flat[at(i)] = flat[at(j)]
        for x, t in tails:
            if rows:
                t[slot] = torch.cat((t[slot], x[int(maps.starts[s]) + torch.tensor(rows, device=x.device)]))[len(rows):]
