"""Drafted trees over a paged cache: the operators of one verification round, each in its plain form and as the framework's call.

  maps    room for the round's rows in the requests' block tables, the rows' maps (positions, cache rows, ancestors), and the room
          given back: what a round does before its layers run and after its drafts were turned down
  conv    the short convolution in front of the cache along every node's path: queries out, keys and values into their pages
  attn    attention of the trees' nodes over committed tokens and their own ancestors
  commit  the accepted path's cache rows of all layers moved together, the convolutions' tails advanced along it

Caches are pages of 64 tokens in no particular order.  A case's lengths and node counts are spread evenly (lengths: over their
logarithm) from its lowest to its highest, so that its work does not depend on the seed; which request has which does.
"""
import math

import numpy as np
import torch

own = False
PAGE = 64


def listed():
    return [
        # four streams with sixteen drafts each: the smallest call, launches and latency count
        {"name": "maps-round-4", "op": "maps", "requests": 4, "length_min": 300, "length_max": 5000, "rows_min": 16, "rows_max": 16, "tree": True, "pad": 0},
        # prompts of many requests admitted together: the maps of some 300 thousand rows
        {"name": "maps-prompts-256", "op": "maps", "requests": 256, "length_min": 1, "length_max": 32000, "rows_min": 1, "rows_max": 2300,
         "tree": False, "pad": 77},
        # two streams, trees of 25 nodes, four taps
        {"name": "conv-2x25", "op": "conv", "requests": 2, "rows_min": 25, "rows_max": 25, "length_min": 200, "length_max": 900, "H": 16, "G": 2,
         "D": 128, "V": 128, "taps": 4, "dtype": "bf16"},
        # many streams with large trees
        {"name": "conv-96x64", "op": "conv", "requests": 96, "rows_min": 40, "rows_max": 64, "length_min": 1, "length_max": 900, "H": 32, "G": 8,
         "D": 128, "V": 128, "taps": 4, "dtype": "bf16"},
        # one interactive stream, a small tree
        {"name": "attn-1x8-900", "op": "attn", "requests": 1, "rows_min": 8, "rows_max": 8, "length_min": 900, "length_max": 900, "H": 16, "G": 4,
         "D": 128, "V": 128, "dtype": "bf16"},
        # four streams behind long prompts, wide heads
        {"name": "attn-4x16-16k", "op": "attn", "requests": 4, "rows_min": 16, "rows_max": 16, "length_min": 16001, "length_max": 16001, "H": 16,
         "G": 2, "D": 256, "V": 256, "dtype": "bf16"},
        # streams of very different lengths; soft cap, distance bias and sink, as the chunked models have them
        {"name": "attn-16x25-ragged", "op": "attn", "requests": 16, "rows_min": 9, "rows_max": 25, "length_min": 60, "length_max": 30000, "H": 16,
         "G": 4, "D": 128, "V": 128, "dtype": "bf16", "cap": 50.0, "bias": 1025, "chunk": 2048, "sink": True},
        # window attention with slopes and gates far into a context
        {"name": "attn-8x32-window", "op": "attn", "requests": 8, "rows_min": 32, "rows_max": 32, "length_min": 20000, "length_max": 33000, "H": 16,
         "G": 4, "D": 128, "V": 128, "dtype": "bf16", "window": 1024, "slopes": True, "gate": True},
        # a full batch with large trees: the largest call, products count as much as bytes
        {"name": "attn-64x64-4k", "op": "attn", "requests": 64, "rows_min": 64, "rows_max": 64, "length_min": 4000, "length_max": 4100, "H": 32,
         "G": 8, "D": 128, "V": 128, "dtype": "bf16"},
        # the 32-bit mode, odd head sizes
        {"name": "attn-3x11-f32", "op": "attn", "requests": 3, "rows_min": 5, "rows_max": 11, "length_min": 700, "length_max": 2100, "H": 6, "G": 2,
         "D": 80, "V": 48, "dtype": "f32"},
        # four streams, twelve layers
        {"name": "commit-4x12", "op": "commit", "requests": 4, "rows_min": 25, "rows_max": 25, "path_min": 3, "path_max": 6, "length_min": 200,
         "length_max": 900, "layers": 12, "G": 4, "D": 128, "V": 128, "taps": 4, "C": 2048, "dtype": "bf16"},
        # a full batch, long accepted paths
        {"name": "commit-64x24", "op": "commit", "requests": 64, "rows_min": 64, "rows_max": 64, "path_min": 3, "path_max": 17, "length_min": 1,
         "length_max": 900, "layers": 24, "G": 8, "D": 128, "V": 128, "taps": 4, "C": 4096, "dtype": "bf16"},
    ]


# --------------------------------------------------------------------------------------------------- drawn cases
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _span(rng, key, lo, hi):
    a, b = sorted((_log(rng, lo, hi), _log(rng, lo, hi)))
    return {key + "_min": a, key + "_max": b}


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6.5e12, w["flops"] / 1.6e15)


def draw(rng):
    op = rng.choice(["maps", "conv", "attn", "attn", "attn", "commit"])
    most = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        case = _drawn(rng, op)
        if _cost(case) <= most and (case.get("dtype") != "f32" or op != "attn" or work(case)["flops"] <= 6e10):
            return case


def _drawn(rng, op):
    if op == "maps":
        tree = rng.random() < 0.5
        return {"op": op, "requests": _log(rng, 1, 256), **_span(rng, "length", 1, 32000), **_span(rng, "rows", 1, 64 if tree else 2300), "tree": tree,
                "pad": rng.choice([0, 0, 1, 100])}
    G, rep = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 8, 12])
    D = rng.choice([32, 64, 80, 96, 128, 128, 192, 256])
    case = {"op": op, "requests": _log(rng, 1, 96), **_span(rng, "rows", 1, 64), "G": G, "D": D, "V": D if rng.random() < 0.7 else rng.choice([32, 64, 128]),
            "dtype": "bf16" if rng.random() < 0.8 else "f32"}
    if op == "commit":
        a, b = sorted((rng.randint(3, 17), rng.randint(3, 17)))
        case.update(_span(rng, "length", 1, 900), **_span(rng, "rows", 8, 64), path_min=a, path_max=b, layers=rng.randint(1, 24), taps=rng.randint(2, 4),
                    C=16 * rng.randint(1, 256))
        return case
    case["H"] = G * rep
    if op == "conv":
        case.update(_span(rng, "length", 1, 900), taps=rng.randint(1, 5))
        return case
    case.update(_span(rng, "length", 1, 40000))
    if rng.random() < 0.3:
        case["cap"] = rng.choice([20.0, 50.0])
    if rng.random() < 0.3:
        case["bias"] = rng.choice([33, 257, 1025])
    elif rng.random() < 0.3:
        case["slopes"] = True
    if rng.random() < 0.4:
        case[rng.choice(["window", "chunk"])] = rng.choice([100, 1024, 2048])
    for k in ("sink", "gate"):
        if rng.random() < 0.3:
            case[k] = True
    case["pad"] = rng.choice([0, 0, 3])
    return case


# --------------------------------------------------------------------------------------------------- sizes of a case
def _spread(lo, hi, n, log=False):
    if n == 1:
        return [hi]
    if log:
        return [int(round(math.exp(math.log(lo) + (math.log(hi) - math.log(lo)) * i / (n - 1)))) for i in range(n)]
    return [int(round(lo + (hi - lo) * i / (n - 1))) for i in range(n)]


def _sizes(case):
    """(committed length, new rows) per request, before they are shuffled."""
    n = case["requests"]
    lengths = _spread(case["length_min"], case["length_max"], n, log=True)
    counts = _spread(case["rows_min"], case["rows_max"], n)
    return lengths, counts[::2] + counts[1::2][::-1]           # not in step with the lengths


def _path_sizes(case):
    """Accepted rows per request."""
    _, counts = _sizes(case)
    p = _spread(case["path_min"], case["path_max"], case["requests"])
    return [min(a, (c + 1) // 2) for a, c in zip(p, counts)]


def _first(case, p):
    if case.get("chunk"):
        return p // case["chunk"] * case["chunk"]
    return max(p - case["window"] + 1, 0) if case.get("window") else 0


def work(case):
    lengths, counts = _sizes(case)
    R, e = sum(counts), 2 if case.get("dtype") == "bf16" else 4
    if case["op"] == "maps":
        pages = sum(-(-(a + b) // PAGE) - -(-a // PAGE) for a, b in zip(lengths, counts))
        words = -(-max(counts) // 32) if case["tree"] else 0
        # both lengths, counts and held pages of a request; slot, index, request, position, cache row (and parent, ancestors) of a row;
        # every entry of the tables taken, read and given back
        return {"bytes": 40 * len(lengths) + R * (24 + (4 + 4 * words if case["tree"] else 0)) + pages * 20, "flops": 0}
    if case["op"] == "conv":
        C = case["H"] * case["D"] + case["G"] * (case["D"] + case["V"])
        tails = len(lengths) * (case["taps"] - 1) * C * e
        return {"bytes": 2 * R * C * e + tails + 4 * case["taps"] * C, "flops": 2 * R * C * case["taps"]}
    if case["op"] == "commit":
        moved = sum(_path_sizes(case)) - sum(max(1, p // 2) for p in _path_sizes(case))
        rows = 2 * moved * case["G"] * (case["D"] + case["V"])
        return {"bytes": case["layers"] * e * (rows + 2 * len(lengths) * (case["taps"] - 1) * case["C"]), "flops": 0}
    H, G, D, V = case["H"], case["G"], case["D"], case["V"]
    seen = [a + b - _first(case, a) for a, b in zip(lengths, counts)]
    keys = sum(b * (a - _first(case, a) + math.log2(b) + 1) for a, b in zip(lengths, counts))
    return {"bytes": e * (sum(seen) * G * (D + V) + R * H * (D + V)), "flops": 2 * (D + V) * H * keys}


# --------------------------------------------------------------------------------------------------- inputs
def _tree(rs, n):
    """Parents of n nodes in the order they were drafted: the last sampled token, then nodes that hang off one of the few before them."""
    return [-1] + [int(rs.randint(max(0, j - 6), j)) for j in range(1, n)]


def _path_tree(rs, n, length):
    """(parents, path): the accepted path starts on the greedy spine, which was drafted first, and leaves it for a later branch."""
    m = max(1, length // 2)
    rest = sorted(rs.choice(np.arange(max(length, m), n), size=length - m, replace=False).tolist()) if length > m else []
    path = list(range(m)) + rest
    parents = [-1] + [int(rs.randint(max(0, j - 6), j)) for j in range(1, n)]
    for a, b in zip(path, path[1:]):
        parents[b] = a
    return parents, path


def _tables(rs, lengths, spare):
    """(table [requests, pages], free pages): the pool's pages in random order."""
    need = [-(-n // PAGE) for n in lengths]
    width, order = max(need), rs.permutation(sum(need) + spare)
    table, at = np.full((len(lengths), width), -1, np.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = order[at: at + n]
        at += n
    return table, order[at:].astype(np.int32)


def _i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def _ancestors(parents):
    """[n, n]: node j sees node i."""
    m = np.eye(len(parents), dtype=bool)
    for j, p in enumerate(parents):
        if p >= 0:
            m[j] |= m[p]
    return m


def _requests(case, seed):
    """Sizes, trees and tables of a seed, on the host."""
    rs = np.random.RandomState(seed % (1 << 31))
    lengths, counts = _sizes(case)
    order = rs.permutation(len(lengths))
    lengths, counts = [lengths[i] for i in order], [counts[i] for i in order]
    h = {"lengths": lengths, "counts": counts, "R": sum(counts) + case.get("pad", 0), "starts": np.concatenate(([0], np.cumsum(counts))).astype(np.int64)}
    if case["op"] == "commit":
        sizes = _path_sizes(case)
        both = [_path_tree(rs, n, sizes[order[i]]) for i, n in enumerate(counts)]
        h["parents"], h["path"] = [p for p, _ in both], [p for _, p in both]
    elif case["op"] != "maps" or case["tree"]:
        h["parents"] = [_tree(rs, n) for n in counts]
    if case["op"] == "maps":
        grown = [a + b for a, b in zip(lengths, counts)]
        held = [-(-n // PAGE) for n in lengths]
        table, free = _tables(rs, grown, 37)
        taken = [-(-n // PAGE) for n in grown]
        # a round starts with the committed tokens' pages; the others lie on the stack
        back = [table[i, j] for i in range(len(held)) for j in range(held[i], taken[i])]
        for i, n in enumerate(held):
            table[i, n:] = -1
        stack = np.concatenate((free, np.array(back, np.int32)[rs.permutation(len(back))])).astype(np.int32)
        h.update(table=table, held=held, stack=stack, n_pages=sum(taken) + 37)
    else:
        h["table"], spare = _tables(rs, [a + b for a, b in zip(lengths, counts)], 3)
        h["n_pages"] = int((h["table"] >= 0).sum()) + len(spare)
    return h


def _flat_parents(h):
    out = np.full(h["R"], -1, np.int32)
    out[: h["starts"][-1]] = np.concatenate([np.array(p, np.int32) for p in h["parents"]])
    return out


def _slot_rows(h):
    """Per request: cache rows of its positions."""
    tokens = [np.arange(a + b) for a, b in zip(h["lengths"], h["counts"])]
    return [h["table"][i, t // PAGE].astype(np.int64) * PAGE + t % PAGE for i, t in enumerate(tokens)]


def _inputs(case, seed):
    h = _requests(case, seed)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = torch.bfloat16 if case.get("dtype") == "bf16" else torch.float32
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g, dtype=torch.float32)
    s = {"case": case, "R": h["R"], "lengths": _i32(h["lengths"]), "counts": _i32(h["counts"]), "tables": _i32(h["table"]), "host": h}
    if "parents" in h:
        s["parents"], s["nodes"] = _i32(_flat_parents(h)), max(h["counts"])
    if case["op"] == "maps":
        s.update(held=_i32(h["held"]), free=torch.cat((_i32(h["stack"]), _i32(np.full(h["n_pages"] - len(h["stack"]), -1)))), n_free=_i32([len(h["stack"])]),
                 grown=_i32([a + b for a, b in zip(h["lengths"], h["counts"])]))
        return s
    R, n = h["R"], h["n_pages"]
    pool = lambda width: torch.cat([rnd(min(1024, n - i), PAGE, *width).to(dt) for i in range(0, n, 1024)])
    if case["op"] == "commit":
        layers = range(case["layers"])
        s["k"], s["v"] = (torch.stack([pool((case["G"], w)) for _ in layers]) for w in (case["D"], case["V"]))
        s["tail"] = torch.stack([rnd(len(h["lengths"]), case["taps"] - 1, case["C"]).to(dt) for _ in layers])
        s["caches"] = [*s["k"], *s["v"]]
        s["tails"] = [(rnd(R, case["C"]).to(dt), t) for t in s["tail"]]
        width = max(len(p) for p in h["path"])
        s["path"], s["n_path"] = _i32([p + [0] * (width - len(p)) for p in h["path"]]), _i32([len(p) for p in h["path"]])
    else:
        H, G, D, V = case["H"], case["G"], case["D"], case["V"]
        s["k"], s["v"] = pool((G, D)), pool((G, V))
        s["x"] = rnd(R, H * D + G * (D + V)).to(dt)             # projected rows
        if case["op"] == "conv":
            s["w"] = rnd(case["taps"], s["x"].shape[1]) * case["taps"] ** -0.5
            s["tail"] = rnd(len(h["lengths"]), case["taps"] - 1, s["x"].shape[1]).to(dt)
        else:
            s["q"] = s["x"][:, : H * D].unflatten(1, (H, D))
            s["scale"] = D ** -0.5
            s["opt"] = {"softcap": case.get("cap", 0.0), "window": case.get("window", 0), "chunk": case.get("chunk", 0),
                        "bias": rnd(H, case["bias"]) * 0.5 if case.get("bias") else None,
                        "slopes": torch.tensor([2.0 ** (-8 * (i + 1) / H) for i in range(H)], device="cuda") if case.get("slopes") else None,
                        "sink": rnd(H) if case.get("sink") else None, "gate": rnd(R, H).to(dt) if case.get("gate") else None}
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    h = s["host"]
    if case["op"] == "maps":
        return s
    if own:
        from spark_engine_b200 import ops
        s["maps"] = ops.slot_maps(s["lengths"], s["counts"], s["tables"], s["R"], parents=s["parents"], nodes=s["nodes"])
    else:                                                       # the same plan for the plain forms
        s["cache_rows"] = [torch.tensor(x, device="cuda") for x in _slot_rows(h)]
        s["anc"] = [torch.tensor(_ancestors(p), device="cuda") for p in h["parents"]]
        s["depth"] = [a.sum(1) - 1 for a in s["anc"]]
        if case["op"] == "conv":
            s["taps_at"] = _taps_at(case, h)
    return s


def _taps_at(case, h):
    """[R, taps]: row of every tap; negative: -1 - i for entry taps - 2 - i of the tail (the newest is -1)."""
    out = np.zeros((h["R"], case["taps"]), np.int64)
    for s, p in enumerate(h["parents"]):
        for j in range(len(p)):
            at, back = j, 0
            for t in range(case["taps"] - 1, -1, -1):
                if at >= 0:
                    out[h["starts"][s] + j, t] = h["starts"][s] + at
                    at = p[at]
                else:
                    back += 1
                    out[h["starts"][s] + j, t] = -back
    return torch.tensor(out, device="cuda")


# --------------------------------------------------------------------------------------------------- one pass
def run(state):
    return {"maps": _maps, "conv": _conv, "attn": _attn, "commit": _commit}[state["case"]["op"]](state)


def _maps(s):
    """Room for the round's rows, their maps, and the room given back."""
    if own:
        from spark_engine_b200 import ops
        room = ops.block_tables(s["grown"], s["tables"], s["held"], s["free"], s["n_free"])
        m = ops.slot_maps(s["lengths"], s["counts"], s["tables"], s["R"], parents=s.get("parents"), nodes=s.get("nodes", 0))
        left = ops.block_tables(s["lengths"], s["tables"], s["held"], s["free"], s["n_free"])
        out = {"room": room, "left": left, "starts": m.starts, "slot": m.slot, "index": m.index, "pos": m.pos, "cache_row": m.cache_row}
        if m.anc is not None:
            out["anc"] = m.anc
    else:
        room = _plain_tables(s, s["grown"])
        out = _plain_maps(s)
        out.update(room=room, left=_plain_tables(s, s["lengths"]))
    out.update(tables=s["tables"], held=s["held"], n_free=s["n_free"], free=s["free"])
    return out


def _plain_tables(s, lengths):
    t, held, free, n_free = s["tables"], s["held"], s["free"], s["n_free"]
    at = torch.arange(t.shape[1], device=t.device).unsqueeze(0)
    need = (lengths + PAGE - 1) // PAGE
    given = torch.clamp(held - need, min=0)
    total = given.sum()
    before = torch.cumsum(given, 0) - given
    gone = (at >= need.unsqueeze(1)) & (at < held.unsqueeze(1))
    to = n_free.long() + total - 1 - (before.unsqueeze(1) + at - need.unsqueeze(1))
    pool = torch.cat((free, free[:1]))
    pool.index_put_((torch.where(gone, to, torch.full_like(to, free.shape[0])),), t)
    free.copy_(pool[:-1])
    held2 = torch.minimum(held, need)
    top = n_free + total
    take = need - held2
    ends = torch.cumsum(take, 0)
    take = torch.where(ends <= top, take, torch.zeros_like(take))
    new = (at >= held2.unsqueeze(1)) & (at < (held2 + take).unsqueeze(1))
    src = top - 1 - ((ends - (need - held2)).unsqueeze(1) + at - held2.unsqueeze(1))
    t.copy_(torch.where(new, free[torch.clamp(src, 0, free.shape[0] - 1)], torch.where(gone, torch.full_like(t, -1), t)))
    held.copy_(held2 + take)
    n_free.copy_(top - take.sum())
    return (held * PAGE).to(torch.int32)


def _plain_maps(s):
    R, S, W = s["R"], s["lengths"].shape[0], s["tables"].shape[1]
    ends = torch.cumsum(s["counts"], 0)
    starts = torch.cat((torch.zeros_like(ends[:1]), ends))
    r = torch.arange(R, device=ends.device)
    req = torch.clamp(torch.searchsorted(ends, r, right=True), max=S - 1)
    there = r < ends[-1]
    j = r - starts[req]
    none = torch.full_like(j, -1)
    tok = s["lengths"][req] + j
    page = s["tables"][req, torch.clamp(tok // PAGE, max=W - 1)].long()
    out = {"starts": starts.to(torch.int32), "slot": torch.where(there, req, none).to(torch.int32), "index": torch.where(there, j, none).to(torch.int32),
           "cache_row": torch.where(there, page * PAGE + tok % PAGE, none)}
    depth = j
    if "parents" in s:
        words = (s["nodes"] + 31) // 32
        anc = torch.zeros(R, words, dtype=torch.int64, device=r.device)
        word = torch.arange(words, device=r.device).unsqueeze(0)
        at, depth = torch.where(there, j, none), none
        for _ in range(s["nodes"]):                              # every node walks up to its root
            on = at >= 0
            bit = torch.ones_like(at) << torch.clamp(at, min=0) % 32
            anc += torch.where(on.unsqueeze(1) & (torch.clamp(at, min=0).unsqueeze(1) // 32 == word), bit.unsqueeze(1), 0)
            depth = depth + on
            at = torch.where(on, s["parents"][torch.clamp(starts[req] + at, 0, R - 1)].long(), none)
        out["anc"] = anc.to(torch.int32)
    out["pos"] = torch.where(there, s["lengths"][req] + depth, none).to(torch.int32)
    return out


def _conv(s):
    c = s["case"]
    nq, G = c["H"] * c["D"], c["G"]
    if own:
        from spark_engine_b200 import ops
        q = ops.path_conv(s["x"], s["w"], s["tail"], s["maps"], nq, s["k"], s["v"])
        return {"q": q, "k": s["k"], "v": s["v"]}
    h, x, taps = s["host"], s["x"].float(), c["taps"]
    req = torch.repeat_interleave(torch.arange(len(h["counts"]), device=x.device), s["counts"], output_size=x.shape[0])
    y = torch.zeros_like(x)
    for t in range(taps):
        at = s["taps_at"][:, t]
        u = x[torch.clamp(at, min=0)]
        if taps > 1:
            u = torch.where((at >= 0).unsqueeze(1), u, s["tail"].float()[req, torch.clamp(taps - 1 + at, 0, taps - 2)])
        y += s["w"][t] * u
    y = y.to(s["x"].dtype)
    rows = torch.cat([a[n:] for a, n in zip(s["cache_rows"], h["lengths"])])
    s["k"].view(-1, G * c["D"])[rows] = y[:, nq: nq + G * c["D"]]
    s["v"].view(-1, G * c["V"])[rows] = y[:, nq + G * c["D"]:]
    return {"q": y[:, :nq].contiguous(), "k": s["k"], "v": s["v"]}


def _attn(s):
    if own:
        from spark_engine_b200 import ops
        return ops.tree_attention(s["q"], s["k"], s["v"], s["maps"], s["scale"], **s["opt"])
    c, o, h = s["case"], s["opt"], s["host"]
    H, G, D, V = c["H"], c["G"], c["D"], c["V"]
    out = torch.zeros(s["R"], H, V, device="cuda", dtype=s["q"].dtype)
    kc, vc = s["k"].view(-1, G, D), s["v"].view(-1, G, V)
    for i, (L, n) in enumerate(zip(h["lengths"], h["counts"])):
        first = _first(c, L)
        r0, rows = int(h["starts"][i]), s["cache_rows"][i][first:]
        k, v = kc[rows].float(), vc[rows].float()
        q = s["q"][r0: r0 + n].float().view(n, G, H // G, D)
        x = (q.permute(1, 2, 0, 3).reshape(G, -1, D) @ k.permute(1, 2, 0)).view(H, n, -1) * s["scale"]
        if o["softcap"]:
            x = o["softcap"] * torch.tanh(x / o["softcap"])
        at = torch.cat((torch.arange(first, L, device=x.device), L + s["depth"][i]))
        pos = (L + s["depth"][i]).unsqueeze(1)
        dist = pos - at
        seen = torch.cat((torch.ones(n, L - first, dtype=torch.bool, device=x.device), s["anc"][i]), 1)
        if o["chunk"]:
            seen = seen & (pos // o["chunk"] == at // o["chunk"])
        if o["window"]:
            seen = seen & (dist < o["window"])
        if o["bias"] is not None:
            x = x + o["bias"][:, torch.clamp(dist, 0, c["bias"] - 1)]
        if o["slopes"] is not None:
            x = x - o["slopes"].view(H, 1, 1) * dist
        x = torch.where(seen, x, torch.full_like(x, -math.inf))
        m = x.amax(-1, keepdim=True)
        if o["sink"] is not None:
            m = torch.maximum(m, o["sink"].view(H, 1, 1))
        p = torch.exp(x - m)
        z = p.sum(-1, keepdim=True)
        if o["sink"] is not None:
            z = z + torch.exp(o["sink"].view(H, 1, 1) - m)
        y = ((p / z).view(G, -1, p.shape[-1]) @ v.permute(1, 0, 2)).view(H, n, V).transpose(0, 1)
        if o["gate"] is not None:
            y = y / (1 + torch.exp(-o["gate"][r0: r0 + n].float())).unsqueeze(-1)
        out[r0: r0 + n] = y.to(out.dtype)
    return out


def _commit(s):
    if own:
        from spark_engine_b200 import ops
        ops.commit_paths(s["maps"], s["path"], s["n_path"], s["caches"], s["tails"])
    else:
        src = torch.cat([a[n + s["path"][i, : len(p)].long()] for i, (a, n, p) in enumerate(zip(s["cache_rows"], s["host"]["lengths"], s["host"]["path"]))])
        dst = torch.cat([a[n: n + len(p)] for a, n, p in zip(s["cache_rows"], s["host"]["lengths"], s["host"]["path"])])
        for c in s["caches"]:
            flat = c.view(-1, c.shape[2] * c.shape[3])
            flat[dst] = flat[src]
        kept = s["case"]["taps"] - 1
        at = s["n_path"].long().unsqueeze(1) - kept + torch.arange(kept, device=dst.device)        # negative: entry kept + at of the tail
        starts = (torch.cumsum(s["counts"], 0) - s["counts"]).unsqueeze(1)
        rows = starts + torch.gather(s["path"].long(), 1, torch.clamp(at, 0, s["path"].shape[1] - 1))
        req = torch.arange(at.shape[0], device=dst.device).unsqueeze(1)
        for x, tail in s["tails"]:
            tail.copy_(torch.where((at >= 0).unsqueeze(2), x[rows], tail[req, torch.clamp(kept + at, 0, kept - 1)]))
    return {"k": s["k"], "v": s["v"], "tail": s["tail"]}


# --------------------------------------------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    h = s["host"]
    if case["op"] == "maps":
        return _exact_maps(case, s, h)
    if case["op"] == "commit":
        return _exact_commit(s, h)
    return _exact_conv(case, s, h) if case["op"] == "conv" else _exact_attn(case, s, h)


def _exact_maps(case, s, h):
    S, R = len(h["lengths"]), h["R"]
    out = {k: np.full(R, -1, np.int64) for k in ("slot", "index", "pos", "cache_row")}
    stack, grown = list(h["stack"]), []
    for i in range(S):                                           # the pool holds enough for every request
        pages = list(h["table"][i, : h["held"][i]])
        while len(pages) * PAGE < h["lengths"][i] + h["counts"][i]:
            pages.append(stack.pop())
        grown.append(np.array(pages, np.int64))
    words = (max(h["counts"]) + 31) // 32
    anc = np.zeros((R, words), np.uint32)
    for i, (L, n) in enumerate(zip(h["lengths"], h["counts"])):
        r0 = int(h["starts"][i])
        sl, j = slice(r0, r0 + n), np.arange(n)
        out["slot"][sl], out["index"][sl] = i, j
        out["cache_row"][sl] = grown[i][(L + j) // PAGE] * PAGE + (L + j) % PAGE
        if case["tree"]:
            m = _ancestors(h["parents"][i])
            out["pos"][sl] = L + m.sum(1) - 1
            for a, b in zip(*np.nonzero(m)):
                anc[r0 + a, b // 32] |= np.uint32(1 << (b % 32))
        else:
            out["pos"][sl] = L + j
    res = {k: torch.tensor(v, dtype=torch.int64 if k == "cache_row" else torch.int32, device="cuda") for k, v in out.items()}
    if case["tree"]:
        res["anc"] = torch.tensor(anc.view(np.int32), device="cuda")
    room = lambda n: _i32([-(-x // PAGE) * PAGE for x in n])
    res.update(starts=_i32(h["starts"]), room=room([a + b for a, b in zip(h["lengths"], h["counts"])]), left=room(h["lengths"]), tables=_i32(h["table"]),
               held=_i32(h["held"]), n_free=_i32([len(h["stack"])]), free=s["free"])
    return res


def _exact_conv(case, s, h):
    taps, nq, G, D, V = case["taps"], case["H"] * case["D"], case["G"], case["D"], case["V"]
    x, w, tail = s["x"].double(), s["w"].double(), s["tail"].double()
    y = torch.zeros_like(x)
    k, v = s["k"].double().view(-1, G * D), s["v"].double().view(-1, G * V)
    rows = _slot_rows(h)
    for i, (L, n) in enumerate(zip(h["lengths"], h["counts"])):
        r0 = int(h["starts"][i])
        past = torch.cat((tail[i], x[r0: r0 + n]))              # row j of the tree is row taps - 1 + j
        up = np.array([taps - 2 if p < 0 else taps - 1 + p for p in h["parents"][i]])
        before = np.concatenate((np.arange(taps - 1) - 1, up)).clip(0)
        at = np.arange(n) + taps - 1
        for t in range(taps - 1, -1, -1):
            y[r0: r0 + n] += w[t] * past[torch.tensor(at, device="cuda")]
            at = before[at]
        dst = torch.tensor(rows[i][L:], device="cuda")
        k[dst], v[dst] = y[r0: r0 + n, nq: nq + G * D], y[r0: r0 + n, nq + G * D:]
    return {"q": y[:, :nq], "k": k.view(s["k"].shape), "v": v.view(s["v"].shape)}


def _exact_attn(case, s, h):
    H, G, D, V, o = case["H"], case["G"], case["D"], case["V"], s["opt"]
    out = torch.zeros(s["R"], H, V, dtype=torch.float64, device="cuda")
    rows = _slot_rows(h)
    for i, (L, n) in enumerate(zip(h["lengths"], h["counts"])):
        r0, lo = int(h["starts"][i]), _first(case, L)
        idx = torch.tensor(rows[i][lo:], device="cuda")
        tree = _ancestors(h["parents"][i])
        pos = L + tree.sum(1) - 1
        at = np.concatenate((np.arange(lo, L), pos))
        dist = pos[:, None] - at[None]
        seen = np.concatenate((np.ones((n, L - lo), bool), tree), 1)
        if o["window"]:
            seen &= dist < o["window"]
        if o["chunk"]:
            seen &= (pos // o["chunk"])[:, None] == (at // o["chunk"])[None]
        seen, dist = torch.tensor(seen, device="cuda"), torch.tensor(dist, device="cuda")
        for g in range(G):
            k, v = s["k"].view(-1, G, D)[idx, g].double(), s["v"].view(-1, G, V)[idx, g].double()
            for a in range(g * H // G, (g + 1) * H // G):
                x = s["q"][r0: r0 + n, a].double() @ k.T * s["scale"]
                if o["softcap"]:
                    x = torch.tanh(x / o["softcap"]) * o["softcap"]
                if o["bias"] is not None:
                    x = x + o["bias"][a].double()[dist.clamp(0, case["bias"] - 1)]
                if o["slopes"] is not None:
                    x = x - dist * o["slopes"][a].double()
                x = x.masked_fill(~seen, -math.inf)
                if o["sink"] is not None:                        # a key without a value
                    x = torch.cat((x, o["sink"][a].double().expand(n, 1)), 1)
                y = torch.softmax(x, 1)[:, : k.shape[0]] @ v
                if o["gate"] is not None:
                    y = y * torch.sigmoid(o["gate"][r0: r0 + n, a].double()).unsqueeze(1)
                out[r0: r0 + n, a] = y
    return out


def _exact_commit(s, h):
    rows = _slot_rows(h)
    caches, tails = [c.clone() for c in s["caches"]], [t.clone() for _, t in s["tails"]]
    src = np.concatenate([rows[i][L + np.array(p)] for i, (L, p) in enumerate(zip(h["lengths"], h["path"]))])
    dst = np.concatenate([rows[i][L: L + len(p)] for i, (L, p) in enumerate(zip(h["lengths"], h["path"]))])
    src, dst = torch.tensor(src, device="cuda"), torch.tensor(dst, device="cuda")
    for c, old in zip(caches, s["caches"]):
        c.view(-1, c.shape[2], c.shape[3])[dst] = old.view(-1, c.shape[2], c.shape[3])[src]
    for t, (x, old) in zip(tails, s["tails"]):
        for i, p in enumerate(h["path"]):
            seen = [old[i, e] for e in range(old.shape[1])] + [x[int(h["starts"][i]) + j] for j in p]
            t[i] = torch.stack(seen[-old.shape[1]:])
    n = len(tails)
    return {"k": torch.stack(caches[:n]).double(), "v": torch.stack(caches[n:]).double(), "tail": torch.stack(tails).double()}
