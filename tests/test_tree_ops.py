"""Block tables, row maps, path convolutions, attention of drafted trees and commits of accepted paths: the plain forms (CPU) against
definitions in 64 bits, and what the calls refuse."""
import numpy as np
import pytest
import torch
import tree_util as U

from spark_engine_b200 import ops


def _tables_state(pages, held, width, stack, device="cpu"):
    t = np.full((len(held), width), -1, np.int32)
    for i, n in enumerate(held):
        t[i, :n] = [pages.pop() for _ in range(n)]
    cap = sum(held) + len(stack)
    i32 = lambda x: torch.tensor(np.asarray(x, dtype=np.int32), device=device)
    return i32(t), i32(held), torch.cat((i32(stack), i32([-1] * (cap - len(stack))))), i32([len(stack)])


def walk_tables(device):
    """Requests grow, shrink and run out of pages; every step against a model with lists."""
    rs = np.random.RandomState(3)
    for S, width in ((1, 4), (5, 9), (33, 40), (1500, 6)):
        total = S * width // 2 + 3
        tables, held, free, n_free = _tables_state([], [0] * S, width, rs.permutation(total).tolist(), device)
        free = torch.cat((free, torch.full((3,), -7, dtype=torch.int32, device=device)))
        lists, stack = [[] for _ in range(S)], free[: int(n_free)].tolist()
        for _ in range(6):
            want = rs.randint(-1, width * 64 + 1, S)
            need = [len(x) if n < 0 else -(-int(n) // 64) for x, n in zip(lists, want)]
            for i in reversed(range(S)):
                while len(lists[i]) > need[i]:
                    stack.append(lists[i].pop())
            left, asked = len(stack), 0
            for i in range(S):
                asked += max(0, need[i] - len(lists[i]))
                if asked <= left:
                    while len(lists[i]) < need[i]:
                        lists[i].append(stack.pop())
            room = ops.block_tables(torch.tensor(want, dtype=torch.int32, device=device), tables, held, free, n_free)
            assert room.tolist() == [64 * len(x) for x in lists] and held.tolist() == [len(x) for x in lists]
            assert int(n_free) == len(stack) and free[: len(stack)].tolist() == stack and free[-3:].tolist() == [-7] * 3
            assert [[p for p in row if p >= 0] for row in tables.tolist()] == lists
            assert all(row[len(x):] == [-1] * (width - len(x)) for row, x in zip(tables.tolist(), lists))


def test_block_tables_follow_lengths():
    walk_tables("cpu")


def test_giving_back_restores_the_stack():
    tables, held, free, n_free = _tables_state(list(range(100, 110)), [2, 0, 3], 8, [5, 9, 2, 7, 1, 0, 3])
    before = [t.clone() for t in (tables, held, free, n_free)]
    ops.block_tables(torch.tensor([300, 64, 200], dtype=torch.int32), tables, held, free, n_free)
    assert held.tolist() == [5, 1, 4]
    ops.block_tables(torch.tensor([128, 0, 150], dtype=torch.int32), tables, held, free, n_free)
    assert all(torch.equal(a, b) for a, b in zip(before, (tables, held, free, n_free)))


ROUNDS = {
    "one row, no past": dict(lengths=[0], counts=[1]),
    "a tree over a page's end": dict(lengths=[61], counts=[9]),
    "ragged, an empty request": dict(lengths=[130, 0, 64, 1], counts=[5, 7, 0, 64], pad=3),
    "more than 64 nodes": dict(lengths=[20, 7], counts=[100, 33]),
    "chains": dict(lengths=[5, 200], counts=[70, 3], trees=False, pad=1),
    "slots out of order": dict(lengths=[33, 190], counts=[4, 6], slots=[3, 1]),
}


def check_maps(r):
    m = ops.slot_maps(**r.inputs())
    starts, slot, index, pos, row, anc = U.want_maps(r)
    for got, want in ((m.starts, starts), (m.slot, slot), (m.index, index), (m.pos, pos), (m.cache_row, row)):
        assert got.tolist() == want.tolist()
    assert m.cache_row.dtype == torch.int64
    if r.trees:
        bits = np.unpackbits(m.anc.cpu().numpy().view(np.uint8).reshape(r.R, -1), axis=1, bitorder="little").astype(bool)
        assert np.array_equal(bits[:, : anc.shape[1]], anc) and not bits[:, anc.shape[1]:].any()
    else:
        assert m.anc is None
    return m


@pytest.mark.parametrize("name", list(ROUNDS))
def test_row_maps(name):
    check_maps(U.Round(**ROUNDS[name]))


def check_conv(r, nq, nk, nv, taps, dtype, page_gap=0):
    dev, C = r.device, nq + nk + nv
    x, w, tail = r.randn(r.R, C, dtype=dtype), r.randn(taps, C) * taps ** -0.5, r.randn(r.table.shape[0], taps - 1, C, dtype=dtype)
    k, v = (r.randn(r.n_pages, 64, 1 + page_gap, n, dtype=dtype)[:, :, :1] for n in (nk, nv))
    before = k.clone(), v.clone(), tail.clone()
    q = ops.path_conv(x, w, tail, ops.slot_maps(**r.inputs()), nq, k, v)
    y, mag = U.want_conv(r, x, w, tail)
    tol = mag * (taps + 1) * 2.0 ** -24
    n = r.starts[-1]
    U.close(q[:n], y[:n, :nq], tol[:n, :nq], dtype)
    rows = torch.tensor(np.concatenate([r.rows(s)[L:] for s, L in enumerate(r.lengths)]), dtype=torch.long)
    for t, old, a in ((k, before[0], nq), (v, before[1], nq + nk)):
        flat, old = t.reshape(r.n_pages * 64, -1).cpu(), old.reshape(r.n_pages * 64, -1).cpu()
        U.close(flat[rows], y[:n, a: a + flat.shape[1]], tol[:n, a: a + flat.shape[1]], dtype)
        rest = torch.ones(len(flat), dtype=torch.bool)
        rest[rows] = False
        assert torch.equal(flat[rest], old[rest])
    assert torch.equal(tail, before[2])


@pytest.mark.parametrize("taps", [1, 2, 4, 7])
@pytest.mark.parametrize("name", list(ROUNDS))
def test_path_convolution(name, taps):
    check_conv(U.Round(**ROUNDS[name]), 24, 16, 8, taps, torch.float32)


FEATURES = {
    "plain": {},
    "soft cap, bias, sink": dict(softcap=2.0, bias=9, sink=True),
    "window, slopes, gate": dict(window=30, slopes=True, gate=True, out_scale=0.7),
    "chunk of 16": dict(chunk=16, bias=40),
    "window of one": dict(window=1, sink=True),
    "bias with masks of the lowest value": dict(bias=50, masked=True),
}


def check_attention(r, H, G, D, V, dtype, f, rounded=0.0, strided=False, layout="plain"):
    dev = r.device
    q = r.randn(r.R, H, D + 8, dtype=dtype)[:, :, :D] if strided else r.randn(r.R, H, D, dtype=dtype)
    if layout == "interleaved":                      # keys and values of a token side by side
        both = r.randn(r.n_pages, 64, G * (D + V), dtype=dtype)
        k, v = both[:, :, : G * D].unflatten(2, (G, D)), both[:, :, G * D:].unflatten(2, (G, V))
    else:
        k, v = r.randn(r.n_pages, 64, G, D, dtype=dtype), r.randn(r.n_pages, 64, G, V, dtype=dtype)
    opt = {n: f[n] for n in ("softcap", "window", "chunk", "out_scale") if n in f}
    if "bias" in f:
        opt["bias"] = r.randn(H, f["bias"])
        if f.get("masked"):
            opt["bias"][:, 3::4] = torch.finfo(torch.float32).min
            opt["bias"][0, 5::4] = -float("inf")
            opt["bias"][1] = torch.finfo(torch.float32).min
    if f.get("slopes"):
        opt["slopes"] = torch.tensor([2.0 ** (-8 * (h + 1) / H) for h in range(H)], device=dev)
    if f.get("sink"):
        opt["sink"] = r.randn(H)
    if f.get("gate"):
        opt["gate"] = r.randn(r.R, H, dtype=dtype)
    m = ops.slot_maps(**r.inputs())
    got = ops.tree_attention(q, k, v, m, D ** -0.5, **opt)
    want, tol = U.want_attention(r, q, k, v, D ** -0.5, rounded=rounded, **opt)
    U.close(got, want, tol, dtype)
    assert not got[r.starts[-1]:].any()
    # into a buffer of the caller's: rows behind the last request are left alone
    wide = torch.full((r.R, H, V + 16), 3.0, dtype=dtype, device=dev)
    assert ops.tree_attention(q, k, v, m, D ** -0.5, out=wide[:, :, :V], **opt).data_ptr() == wide.data_ptr()
    assert torch.equal(wide[: r.starts[-1], :, :V], got[: r.starts[-1]]) and bool((wide[r.starts[-1]:] == 3).all() and (wide[:, :, V:] == 3).all())


@pytest.mark.parametrize("name", list(ROUNDS))
def test_attention_of_rounds(name):
    check_attention(U.Round(**ROUNDS[name]), 4, 2, 16, 24, torch.float32, {})


@pytest.mark.parametrize("name", list(FEATURES))
def test_attention_features(name):
    check_attention(U.Round([70, 3], [9, 12], pad=2), 4, 2, 16, 8, torch.float32, FEATURES[name])


def check_hidden(device, dtype, H=4, G=2, D=64, V=64):
    """What a row does not see may hold anything: siblings, tokens outside the window, tokens behind the last one, free pages."""
    for kind in ("siblings", "window", "behind"):
        r = U.Round([200, 30], [12, 5], device=device, seed=7)
        q, k, v = r.randn(r.R, H, D, dtype=dtype), r.randn(r.n_pages, 64, G, D, dtype=dtype), r.randn(r.n_pages, 64, G, V, dtype=dtype)
        m = ops.slot_maps(**r.inputs())
        opt = dict(window=50) if kind == "window" else {}
        want = ops.tree_attention(q, k, v, m, 0.1, **opt)
        spoiled, odd = set(), []
        if kind == "siblings":
            odd, spoiled = [r.rows(0)[200 + 4]], {j for j in range(12) if r.anc[0][j, 4]}
            assert 0 < len(spoiled) < 12
        elif kind == "window":
            odd = r.rows(0)[:150].tolist()
        else:
            used = set(r.rows(0).tolist()) | set(r.rows(1).tolist())
            odd = [t for t in range(r.n_pages * 64) if t not in used]
        for n, x in enumerate((float("nan"), float("inf"), -float("inf"))):
            for t in odd[n::3] if len(odd) > 2 else odd:
                k.view(-1, G, D)[t], v.view(-1, G, V)[t, :, n::3] = x, x
            got = ops.tree_attention(q, k, v, m, 0.1, **opt)
            for row in range(r.R):
                if row in spoiled:
                    assert not torch.isfinite(got[row]).all()
                else:
                    assert torch.equal(got[row], want[row]), (kind, x, row)


def test_hidden_tokens_have_no_effect():
    check_hidden("cpu", torch.float32, D=16, V=16)


def check_commit(r, dtype, widths, taps, C):
    dev, S = r.device, len(r.counts)
    caches = [r.randn(r.n_pages, 64, 2, n, dtype=dtype) for n in widths]
    tails = [(r.randn(r.R, C, dtype=dtype), r.randn(r.table.shape[0], taps - 1, C, dtype=dtype)) for _ in range(3)] if taps else []
    paths = [U.path_of(r, s, int(r.rs.randint(n))) if n and s != 1 else [] for s, n in enumerate(r.counts)]
    width = max(len(p) for p in paths) + 1
    want_c, want_t = [c.clone() for c in caches], [t.clone() for _, t in tails]
    for s, p in enumerate(paths):
        at = r.rows(s)[r.lengths[s]:]
        for c, old in zip(want_c, caches):
            for i, j in enumerate(p):
                c.view(-1, c.shape[2] * c.shape[3])[at[i]] = old.view(-1, c.shape[2] * c.shape[3])[at[j]]
        for t, (x, old) in zip(want_t, tails):
            line = list(old[r.slot(s)]) + [x[r.starts[s] + j] for j in p]
            if taps > 1:
                t[r.slot(s)] = torch.stack(line[len(line) - (taps - 1):])
    ops.commit_paths(ops.slot_maps(**r.inputs()), r.i32([p + [99] * (width - len(p)) for p in paths]), r.i32([len(p) for p in paths]), caches, tails)
    assert all(torch.equal(a, b) for a, b in zip(caches, want_c)) and all(torch.equal(t, b) for (_, t), b in zip(tails, want_t))


@pytest.mark.parametrize("taps", [0, 1, 4, 9])
@pytest.mark.parametrize("name", list(ROUNDS))
def test_commit_of_paths(name, taps):
    check_commit(U.Round(**ROUNDS[name], seed=5), torch.float32, (8, 12, 4), taps, 24)


# ----------------------------------------------------------------------------- refusals
def _args(**over):
    r = U.Round([70], [5])
    d = dict(q=r.randn(5, 4, 16), k=r.randn(r.n_pages, 64, 2, 16), v=r.randn(r.n_pages, 64, 2, 8), maps=ops.slot_maps(**r.inputs()), scale=0.25)
    d.update({k: f(d) for k, f in over.items()})
    return d


@pytest.mark.parametrize("over", [
    dict(q=lambda d: d["q"].half()), dict(q=lambda d: d["q"][:4]), dict(q=lambda d: d["q"][:, :3]), dict(q=lambda d: d["q"][:, :, :8]),
    dict(k=lambda d: d["k"].bfloat16()), dict(k=lambda d: d["k"][:, :32]), dict(k=lambda d: d["k"][:, :, :1]), dict(v=lambda d: d["v"][:1]),
    dict(v=lambda d: d["v"].transpose(2, 3).contiguous().transpose(2, 3)), dict(window=lambda d: -1), dict(chunk=lambda d: 4, window=lambda d: 4),
    dict(softcap=lambda d: float("nan")), dict(scale=lambda d: float("inf")), dict(bias=lambda d: torch.zeros(4, 0)), dict(bias=lambda d: torch.zeros(3, 5)),
    dict(sink=lambda d: torch.zeros(4).bfloat16()), dict(slopes=lambda d: torch.zeros(8)[::2]), dict(gate=lambda d: torch.zeros(5, 3)),
    dict(out=lambda d: torch.zeros(5, 4, 16)), dict(out=lambda d: torch.zeros(5, 8, 4).transpose(1, 2)),
    dict(q=lambda d: torch.zeros(5, 4, 520), k=lambda d: torch.zeros(d["k"].shape[0], 64, 2, 520)),
    dict(q=lambda d: torch.zeros(5, 4, 12), k=lambda d: torch.zeros(d["k"].shape[0], 64, 2, 12)),
])
def test_attention_refuses(over):
    with pytest.raises(ValueError):
        ops.tree_attention(**_args(**over))


@pytest.mark.parametrize("over", [
    dict(out=lambda d: torch.zeros(5, 1, 8).expand(5, 4, 8)), dict(out=lambda d: torch.zeros(1, 4, 8).expand(5, 4, 8)),
    dict(k=lambda d: d["k"][:1].expand_as(d["k"])), dict(v=lambda d: d["v"][:1].expand_as(d["v"])),
])
def test_attention_refuses_memory_that_overlaps(over):
    with pytest.raises(ValueError):
        ops.tree_attention(**_args(**over))


def check_sink_of_nothing(device, dtype):
    """A sink may be -inf: a row that sees nothing is still zero."""
    r = U.Round([0, 70], [3, 2], device=device)
    q, k, v = r.randn(r.R, 4, 64, dtype=dtype), r.randn(r.n_pages, 64, 2, 64, dtype=dtype), r.randn(r.n_pages, 64, 2, 64, dtype=dtype)
    m = ops.slot_maps(**r.inputs())
    want = ops.tree_attention(q, k, v, m, 0.1)
    m.anc[1].zero_()
    got = ops.tree_attention(q, k, v, m, 0.1, sink=torch.full((4,), -float("inf"), device=device))
    assert not got[1].any() and torch.equal(got[[0, 2, 3, 4]], want[[0, 2, 3, 4]])


def test_sink_of_nothing():
    check_sink_of_nothing("cpu", torch.float32)


def test_maps_and_tables_refuse():
    r = U.Round([70, 9], [5, 6])
    good = r.inputs()
    ops.slot_maps(**good)
    for k, x in (("lengths", good["lengths"].long()), ("counts", good["counts"][:1]), ("tables", good["tables"][0]), ("parents", good["parents"][:3]),
                 ("nodes", 0), ("nodes", 5000), ("slots", good["counts"][:1]), ("rows", 10), ("rows", 1 << 23), ("tables", good["tables"][:1])):
        with pytest.raises(ValueError):
            ops.slot_maps(**{**good, k: x})
    with pytest.raises(ValueError):
        ops.slot_maps(**{k: x for k, x in good.items() if k != "parents"})
    with pytest.raises(ValueError):                  # a parent behind its child
        ops.slot_maps(**{**good, "parents": torch.full((11,), 3, dtype=torch.int32)})
    i = lambda *x: torch.tensor(x, dtype=torch.int32)
    for args in ((i(1), i(1, 2).view(1, 2), i(0, 0), i(3), i(1)), (i(1).long(), i(1, 2).view(1, 2), i(0), i(3), i(1)), (i(1), i(1, 2), i(0), i(3), i(1)),
                 (i(1), i(1, 2).view(1, 2), i(0), i(3), i(1, 1))):
        with pytest.raises(ValueError):
            ops.block_tables(*args)


def test_convolution_and_commit_refuse():
    r = U.Round([70], [5])
    m = ops.slot_maps(**r.inputs())
    good = dict(x=r.randn(5, 48), w=r.randn(4, 48), tail=r.randn(1, 3, 48), maps=m, nq=24, k=r.randn(r.n_pages, 64, 2, 8), v=r.randn(r.n_pages, 64, 1, 8))
    ops.path_conv(**good)
    for k, x in (("x", good["x"][:4]), ("x", good["x"].half()), ("w", good["w"][:, :40]), ("w", good["w"].bfloat16()), ("tail", good["tail"][:, :2]),
                 ("tail", good["tail"].expand(2, 3, 48)), ("nq", 16), ("k", good["k"].bfloat16()), ("k", good["k"][:, :, :, :4]), ("v", good["v"][:1])):
        with pytest.raises(ValueError):
            ops.path_conv(**{**good, k: x})
    path, n = torch.tensor([[0, 2]], dtype=torch.int32), torch.tensor([2], dtype=torch.int32)
    k, t = good["k"], (good["x"], good["tail"])
    ops.commit_paths(m, path, n, [k], [t])
    for args in ((path.long(), n, [k], []), (path, n[:0], [k], []), (path, n, [k, k], []), (path, n, [k.half()], []), (path, n, [k], [(good["x"][:4], good["tail"])]),
                 (path, n, [k[:, :, :, :4].expand(-1, -1, -1, 4)[:, :, :, :3]], []), (path.flip(1), n, [k], []), (path + 4, n, [k], [])):
        with pytest.raises(ValueError):
            ops.commit_paths(m, *args)


# ----------------------------------------------------------------------------- rows that start anywhere
ANYWHERE = {                                         # of a buffer: rows that kernels cannot read 16 bytes at a time as they are
    "contiguous, one element in": lambda b: b[1: 1 + 3 * 32].view(3, 32),
    "contiguous, three elements in": lambda b: b[3: 3 + 3 * 32].view(3, 32),
    "rows of an odd pitch": lambda b: b[: 4 * 37].view(4, 37)[:3, :32],
    "one row of an odd pitch": lambda b: b[: 4 * 37].view(4, 37)[:1, :32],
    "one row of an odd pitch, in the middle": lambda b: b[: 4 * 37].view(4, 37)[2:3, 3: 35],
    "columns": lambda b: b[: 32 * 8].view(32, 8).t(),
    "one value for all channels": lambda b: b[:3].view(3, 1).expand(3, 32),
}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", list(ANYWHERE))
def test_rows_that_start_anywhere_are_made_readable(name, dtype):
    """What the launches take: 16-byte starts, whatever a contiguous tensor's offset or a single row's stride."""
    from spark_engine_b200.ops import tree
    x = ANYWHERE[name](torch.arange(600, dtype=torch.float32).remainder(251).to(dtype))
    y = tree._native().pieces(x, 8)
    assert torch.equal(x, y) and y.data_ptr() % 16 == 0 and y.stride(1) == 1 and (y.shape[0] == 1 or y.stride(0) % 8 == 0)
    heads = x.unflatten(1, (4, x.shape[1] // 4))
    if x.shape[1] // 4 % 8 == 0:
        y = tree._native().pieces(heads, 8)
        assert torch.equal(heads, y) and y.data_ptr() % 16 == 0 and y.stride(2) == 1 and all(y.shape[i] == 1 or y.stride(i) % 8 == 0 for i in range(2))
    good = torch.zeros(3, 40, dtype=dtype)[:, :32]
    assert tree._native().pieces(good, 8).data_ptr() == good.data_ptr()


# ----------------------------------------------------------------------------- tables that lead nowhere
def _spoiled(bad):
    """A request that crosses into a page that is not there, one beside it that is whole."""
    r = U.Round([60, 90], [9, 6], spare=1)
    r.table[0, 1] = r.n_pages if bad == "past the cache" else -1
    d = r.inputs()
    if bad == "past the table":
        r.table[0, 1] = 0
        d["tables"] = r.i32(r.table)
        d["lengths"] = r.i32([126, 90])
    if bad == "no row of the tables":
        d["slots"] = r.i32([7, 1])
    return r, ops.slot_maps(**d)


@pytest.mark.parametrize("bad", ["missing", "past the cache", "past the table", "no row of the tables"])
def test_commit_without_a_page_changes_nothing(bad):
    r, m = _spoiled(bad)
    caches, tail = [r.randn(r.n_pages, 64, 2, 8), r.randn(r.n_pages, 64, 1, 12)], (r.randn(r.R, 24), r.randn(2, 3, 24))
    before = [c.clone() for c in caches] + [tail[1].clone()]
    path = r.i32([[0, 1, 2, 5, 6, 8], [0, 2, 3, 9, 9, 9]])
    with pytest.raises(ValueError):
        ops.commit_paths(m, path, r.i32([6, 3]), caches, [tail])
    assert all(torch.equal(a, b) for a, b in zip(before, caches + [tail[1]]))
    ops.commit_paths(m, path, r.i32([0, 3]), caches, [tail])          # the other request alone
    assert torch.equal(tail[1][0], before[2][0]) and torch.equal(tail[1][1], tail[0][[9, 11, 12]])


@pytest.mark.parametrize("bad", ["missing", "past the cache", "past the table"])
def test_rows_without_a_page_are_left_out(bad):
    """Attention does not see what is not there, and the convolution writes nothing: no other page is read or written in its place."""
    r, m = _spoiled(bad)
    q, k, v = r.randn(r.R, 4, 16), r.randn(r.n_pages, 64, 2, 16), r.randn(r.n_pages, 64, 2, 8)
    got = ops.tree_attention(q, k, v, m, 0.25)
    good = U.Round([60, 90], [9, 6], spare=1)
    there = ops.slot_maps(**good.inputs())
    want = ops.tree_attention(q, k, v, there, 0.25)
    assert torch.isfinite(got).all() and torch.equal(got[9:], want[9:])
    if bad != "past the table":                      # tokens 0 .. 63 alone: nodes 0 .. 3 are in the first page
        anc = there.anc.clone()
        there.anc[:9] &= 15
        assert torch.allclose(got[:9], ops.tree_attention(q, k, v, there, 0.25)[:9], rtol=1e-5, atol=1e-6)
        there.anc.copy_(anc)
    w, tail, x = r.randn(3, 40), r.randn(2, 2, 40), r.randn(r.R, 40)
    k, v = r.randn(r.n_pages, 64, 2, 8), r.randn(r.n_pages, 64, 1, 8)
    k0, k1 = k.clone(), k.clone()
    out = ops.path_conv(x, w, tail, m, 16, k, v)
    assert torch.equal(out, ops.path_conv(x, w, tail, there, 16, k1, v.clone()))
    used = set(good.rows(1)[90:].tolist()) | (set(r.rows(0)[60:64].tolist()) if bad != "past the table" else set(r.table[0, 1] * 64 + np.arange(62, 64)))
    changed = set(torch.nonzero((k != k0).flatten(2).any(2).flatten()).flatten().tolist())
    assert changed == {int(t) for t in used}


def test_negative_lengths_are_zero():
    r = U.Round([0, 70], [3, 4])
    d = r.inputs()
    want = ops.slot_maps(**d)
    got = ops.slot_maps(**{**d, "lengths": r.i32([-1, 70])})
    assert torch.equal(got.pos, want.pos) and torch.equal(got.cache_row, want.cache_row)
    q, k, v = r.randn(r.R, 4, 16), r.randn(r.n_pages, 64, 2, 16), r.randn(r.n_pages, 64, 2, 8)
    assert torch.equal(ops.tree_attention(q, k, v, got, 0.25), ops.tree_attention(q, k, v, want, 0.25))


# ----------------------------------------------------------------------------- the two native parts
def test_kernels_of_other_sources_are_refused():
    """The bindings and the kernels share argument structures: what was built from another header is not launched."""
    import ctypes

    from spark_engine_b200 import build
    from spark_engine_b200.ops import cuda, tree
    mod = tree._native()
    flag, = build._tree_layout()
    assert f"={mod.layout()}u" in flag and mod.layout() != 0
    assert mod.__file__.endswith(build.sysconfig.get_config_var("EXT_SUFFIX"))

    class Fn:
        def __init__(self, value):
            self.value = value

        def __call__(self):
            return self.value

    class Lib:
        _name = "libother.so"

    dll = Lib()
    with pytest.raises(RuntimeError, match="no tree kernels"):
        tree._same_layout(mod, dll)
    dll.spark_tree_layout = Fn(mod.layout() ^ 1)
    with pytest.raises(RuntimeError, match="different sources"):
        tree._same_layout(mod, dll)
    dll.spark_tree_layout = Fn(mod.layout())
    tree._same_layout(mod, dll)
    try:
        real = ctypes.CDLL(cuda.LIB_PATH)
    except OSError:
        return
    tree._same_layout(mod, real)


def test_a_model_with_trees_builds_both_parts(monkeypatch):
    """`kernel_library` keeps the bindings in step with the kernels, and a changed argument header makes the complete library stale."""
    from spark_engine_b200 import build
    called, seen = [], []
    monkeypatch.setattr(build, "build_runtime", lambda: called.append("runtime"))
    monkeypatch.setattr(build, "build_tree", lambda: called.append("tree"))
    monkeypatch.setattr(build, "build_kernels", lambda **kw: called.append(kw.get("family", "all")))
    monkeypatch.setattr(build, "_newer", lambda srcs, out: seen.extend(srcs) or True)
    build.kernel_library("debisun")
    assert called == ["runtime", "tree", "debisun"] and any(s.endswith("tree_args.h") for s in seen)
    called.clear()
    build.kernel_library("vabunex")
    assert called == ["runtime", "vabunex"]
    called.clear()
    build.kernel_library("another family")
    assert called == ["runtime", "tree", "all"]


# ----------------------------------------------------------------------------- memory that overlaps itself
def test_pieces_that_share_memory_are_known():
    from spark_engine_b200.ops import tree
    rs = np.random.RandomState(0)
    for _ in range(3000):
        n0, n1, w = int(rs.randint(1, 7)), int(rs.randint(1, 7)), int(rs.randint(1, 5))
        s0, s1 = int(rs.randint(0, 30)), int(rs.randint(0, 30))
        at = [a * s0 + b * s1 + c for a in range(n0) for b in range(n1) for c in range(w)]
        assert tree._native().apart(n0, s0, n1, s1, w) == (len(set(at)) == len(at)), (n0, s0, n1, s1, w)


def test_outputs_and_caches_that_overlap_themselves_are_refused():
    d = _args()
    ops.tree_attention(**d)
    heads_on_rows = torch.zeros(200).as_strided((5, 4, 8), (8, 8, 1))           # head 1 of a row is head 0 of the next
    with pytest.raises(ValueError):
        ops.tree_attention(**d, out=heads_on_rows)
    heads_first = torch.zeros(4, 5, 8).transpose(0, 1)                          # (rows within heads do not overlap)
    assert torch.equal(ops.tree_attention(**d, out=heads_first), ops.tree_attention(**d))
    pages = d["k"].shape[0]
    sliding = torch.randn(pages * 64 * 32).as_strided((pages, 64, 2, 16), (32, 32, 16, 1))        # a page's token 1 is the next page's token 0
    with pytest.raises(ValueError):
        ops.tree_attention(**{**d, "k": sliding})
    with pytest.raises(ValueError):
        ops.commit_paths(d["maps"], torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32), [sliding])
    tokens_first = torch.randn(64, pages, 2, 16).transpose(0, 1)
    ops.tree_attention(**{**d, "k": tokens_first})


def check_rest_of_convolution(device, dtype):
    """Rows that are nobody's, behind the last request or of one without a row of the tables, are zeros whatever weights and rows hold."""
    for lengths, counts, pad, slots in (([70, 3], [5, 9], 7, None), ([0], [1], 80, None), ([5, 9, 2], [3, 70, 2], 1, [0, 9, 1])):
        r = U.Round(lengths, counts, device=device, pad=pad)
        d = r.inputs()
        if slots:
            d["slots"] = r.i32(slots)
        m = ops.slot_maps(**d)
        w, x, tail = r.randn(3, 40), r.randn(r.R, 40, dtype=dtype), r.randn(len(lengths), 2, 40, dtype=dtype)
        k, v = r.randn(r.n_pages, 64, 2, 8, dtype=dtype), r.randn(r.n_pages, 64, 1, 8, dtype=dtype)
        want = ops.path_conv(x, w, tail, m, 16, k.clone(), v.clone())
        w[0, 3], w[1, 5], w[2, 7] = float("inf"), float("nan"), -float("inf")
        dead = torch.ones(r.R, dtype=torch.bool)
        for s in range(len(lengths)):
            if slots is None or slots[s] < r.table.shape[0]:
                dead[r.starts[s]: r.starts[s + 1]] = False
        x[dead.to(device)] = float("nan")
        got = ops.path_conv(x, w, tail, m, 16, k, v)
        assert not got[dead.to(device)].any() and bool(got[~dead.to(device)][:, [3, 5, 7]].isfinite().logical_not().all())
        fine = [c for c in range(16) if c not in (3, 5, 7)]
        assert torch.equal(got[:, fine], want[:, fine])


def test_rest_of_convolution():
    check_rest_of_convolution("cpu", torch.float32)


def test_tiles_go_by_a_requests_rows():
    """Not by those of all requests: chains of one row are no tree of many."""
    from spark_engine_b200.ops import tree
    tile = tree._native().tile_rows
    assert tile(64, 64, 0, 4) == 128 and tile(64 * 32, 64, 0, 4) == 128 and tile(64 * 33, 64, 0, 4) == 256 and tile(500, 1, 0, 4) == 256
    assert tile(64 * 32, 64, 32, 4) == 128 and tile(64 * 33, 64, 33, 4) == 256 and tile(9, 1, 64, 8) == 128 and tile(563, 64, 0, 4) == 128
