"""Drafted trees over paged caches on a B200: block tables, row maps, path convolutions, attention and commits against definitions in 64
bits; captured rounds, other streams, caches beyond 32-bit offsets, tables and paths that lead nowhere."""
import numpy as np
import pytest
import test_tree_ops as T
import torch
import tree_util as U

from spark_engine_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32
DTYPES = [F32, BF16]
WEIGHTS = {F32: 0.0, BF16: U.half_step(BF16)}          # of a weight: one or two bf16 terms enter the product


@pytest.fixture(autouse=True)
def status_stays_clear():
    cu = ops.cuda_ops()
    cu.clear_status(DEV)
    yield
    torch.cuda.synchronize()
    got = cu.read_status(DEV)
    cu.clear_status(DEV)
    assert got[0] == 0, got


def expect_status():
    torch.cuda.synchronize()
    cu = ops.cuda_ops()
    assert cu.read_status(DEV)[0] != 0
    cu.clear_status(DEV)


def test_block_tables_follow_lengths():
    T.walk_tables(DEV)


@pytest.mark.parametrize("name", list(T.ROUNDS))
def test_row_maps(name):
    T.check_maps(U.Round(**T.ROUNDS[name], device=DEV))


@pytest.mark.parametrize("trees", [False, True])
def test_row_maps_of_many_requests(trees):
    rs = np.random.RandomState(1)
    T.check_maps(U.Round(rs.randint(0, 5000, 700), rs.randint(0, 70, 700), device=DEV, trees=trees, pad=301))


def test_rows_without_pages_are_marked():
    r = U.Round([100, 40], [60, 5], device=DEV)
    r.table[0, 2] = -1
    d = r.inputs()
    m = ops.slot_maps(**d)
    expect_status()
    assert (m.cache_row[:28] >= 0).all() and (m.cache_row[28:60] == -1).all() and (m.cache_row[60:] >= 0).all()
    d["parents"][7] = 9                              # behind its child: hangs off the committed tokens
    m = ops.slot_maps(**d)
    expect_status()
    assert int(m.pos[7]) == 100 and m.anc[7].tolist() == [1 << 7, 0]
    d = U.Round([10, 40], [6, 5], device=DEV).inputs()
    m = ops.slot_maps(**{**d, "rows": 8, "parents": d["parents"][:8].contiguous()})       # more rows than the round's tensors
    expect_status()
    assert m.starts.tolist() == [0, 6, 8]
    m = ops.slot_maps(**{**d, "nodes": 3})
    expect_status()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("taps", [1, 2, 3, 4, 7])
@pytest.mark.parametrize("name", list(T.ROUNDS))
def test_path_convolution(name, taps, dtype):
    T.check_conv(U.Round(**T.ROUNDS[name], device=DEV), 24, 16, 8, taps, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_path_convolution_of_wide_rows(dtype):
    T.check_conv(U.Round([50, 0, 131], [33, 64, 7], device=DEV, pad=5), 2048, 264, 520, 4, dtype, page_gap=1)


SIZES = {
    "one row, no past": (dict(lengths=[0], counts=[1]), 4, 4, 64, 64),
    "heads of 128": (dict(lengths=[130, 0, 64, 1], counts=[5, 7, 0, 64], pad=3), 8, 2, 128, 128),
    "heads of 256": (dict(lengths=[300, 63], counts=[16, 3]), 16, 2, 256, 256),
    "odd heads": (dict(lengths=[700, 1], counts=[11, 2], pad=1), 6, 2, 80, 48),
    "narrow values": (dict(lengths=[90], counts=[21]), 5, 1, 192, 32),
    "wide values": (dict(lengths=[90], counts=[5]), 2, 1, 64, 200),
    "narrow heads": (dict(lengths=[190, 3], counts=[33, 8]), 12, 4, 8, 16),
    "40 query heads per key head": (dict(lengths=[129], counts=[13]), 40, 1, 16, 8),
    "more pairs than a tile": (dict(lengths=[500, 20], counts=[90, 40]), 16, 2, 64, 64),
    "200 nodes": (dict(lengths=[65], counts=[200]), 2, 2, 128, 64),
    "very wide heads": (dict(lengths=[77], counts=[9]), 3, 1, 320, 272),
    "chains": (dict(lengths=[5, 200], counts=[70, 3], trees=False, pad=1), 8, 4, 64, 128),
    "slots out of order": (dict(lengths=[33, 190], counts=[4, 6], slots=[3, 1]), 4, 2, 64, 64),
    "a long past": (dict(lengths=[20000, 5], counts=[3, 9]), 8, 2, 64, 64),
    "300 requests": (dict(lengths=list(range(300)), counts=[1 + i % 4 for i in range(300)], pad=2), 2, 1, 32, 32),
}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", list(SIZES))
def test_attention_of_sizes(name, dtype):
    r, *heads = SIZES[name]
    T.check_attention(U.Round(**r, device=DEV), *heads, dtype, {}, rounded=WEIGHTS[dtype])


@pytest.mark.parametrize("nodes", [1, 4, 10, 17, 45])     # of 3 query heads: tiles of 8, 16, 32 and 64 rows, and two of them
@pytest.mark.parametrize("D,V", [(64, 48), (136, 128), (40, 256), (264, 512), (512, 64)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_of_tiles(D, V, nodes, dtype):
    T.check_attention(U.Round([150, 64], [nodes, 2], device=DEV), 6, 2, D, V, dtype, {}, rounded=WEIGHTS[dtype])


@pytest.mark.parametrize("D,f", [(64, {}), (64, dict(window=300)), (128, dict(softcap=3.0)), (128, dict(slopes=True, chunk=256)), (64, dict(bias=40))])
def test_large_trees_again_and_again(D, f):
    """Two tiles of a request's rows share its keys and run apart, through pages (ends of windows, trees over a page's end) that not every
    row sees whole."""
    rs = np.random.RandomState(5)
    r = U.Round(rs.randint(900, 1100, 40), rs.randint(33, 65, 40), device=DEV)
    T.check_attention(r, 16, 4, D, D, BF16, f, rounded=WEIGHTS[BF16])
    q, k, v, m = r.randn(r.R, 16, D, dtype=BF16), r.randn(r.n_pages, 64, 4, D, dtype=BF16), r.randn(r.n_pages, 64, 4, D, dtype=BF16), ops.slot_maps(**r.inputs())
    opt = {n: x for n, x in f.items() if n in ("softcap", "window", "chunk")}
    if "bias" in f:
        opt["bias"] = r.randn(16, f["bias"])
    if "slopes" in f:
        opt["slopes"] = torch.linspace(0.01, 0.5, 16, device=DEV)
    first = ops.tree_attention(q, k, v, m, D ** -0.5, **opt)
    for _ in range(40):
        assert torch.equal(ops.tree_attention(q, k, v, m, D ** -0.5, **opt), first)


@pytest.mark.parametrize("sharp", [1.0, 40.0])
@pytest.mark.parametrize("window", [0, 333])
@pytest.mark.parametrize("rep", [4, 32])
@pytest.mark.parametrize("dtype", DTYPES)
def test_steep_slopes(dtype, rep, window, sharp):
    """Slopes that outweigh the scores within a page and others that do not, towards the nearest token and away from it, with and without sinks."""
    r = U.Round([700, 1500, 3], [9, 7, 2], device=DEV)
    q, k, v = r.randn(r.R, 2 * rep, 64, dtype=dtype) * sharp, r.randn(r.n_pages, 64, 2, 64, dtype=dtype), r.randn(r.n_pages, 64, 2, 64, dtype=dtype)
    slopes = torch.tensor([[3.0, 0.7, 0.3, -0.2, 0.05, -1.5, 0.0, 0.01][h % 8] for h in range(2 * rep)], device=DEV)
    m = ops.slot_maps(**r.inputs())
    for sink in (None, torch.linspace(-90, 30, 2 * rep, device=DEV)):
        got = ops.tree_attention(q, k, v, m, 0.125, slopes=slopes, sink=sink, window=window)
        U.close(got, *U.want_attention(r, q, k, v, 0.125, slopes=slopes, sink=sink, window=window, rounded=WEIGHTS[dtype]), dtype)


@pytest.mark.parametrize("layout", ["plain", "interleaved"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", list(T.FEATURES))
def test_attention_features(name, dtype, layout):
    r = U.Round([70, 3, 400], [9, 12, 70], device=DEV, pad=2)
    T.check_attention(r, 4, 2, 64, 128, dtype, T.FEATURES[name], rounded=WEIGHTS[dtype], strided=True, layout=layout)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 256, 24])
def test_hidden_tokens_have_no_effect(D, dtype):
    T.check_hidden(DEV, dtype, D=D, V=D)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_see_nothing_are_zero(dtype):
    r = U.Round([0, 70], [6, 4], device=DEV)
    q, k, v = r.randn(r.R, 4, 64, dtype=dtype), r.randn(r.n_pages, 64, 2, 64, dtype=dtype), r.randn(r.n_pages, 64, 2, 64, dtype=dtype)
    m = ops.slot_maps(**r.inputs())
    m.anc[2].zero_()                                 # neither itself nor an ancestor, and there is no past
    got = ops.tree_attention(q, k, v, m, 0.1)
    assert not got[2].any() and got[[0, 1, 3, 4, 5]].abs().amax((1, 2)).min() > 0
    low = torch.full((4, 2000), -float("inf"), device=DEV)
    assert not ops.tree_attention(q, k, v, m, 0.1, bias=low).any()
    assert not ops.tree_attention(q, k, v, m, 0.1, bias=low, sink=torch.zeros(4, device=DEV)).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("length", [70, 9000])         # one CTA to a request's keys, and many
def test_what_is_not_a_number_shows(length, dtype):
    r = U.Round([length, length], [9, 9], device=DEV)
    q, k, v = r.randn(r.R, 4, 64, dtype=dtype), r.randn(r.n_pages, 64, 2, 64, dtype=dtype), r.randn(r.n_pages, 64, 2, 64, dtype=dtype)
    maps = ops.slot_maps(**r.inputs())
    clean = ops.tree_attention(q, k, v, maps, 0.125)
    q[3, 1] = float("nan")                             # every score of the row
    got = ops.tree_attention(q, k, v, maps, 0.125)
    assert got[3, 1].isnan().all()
    got[3, 1] = clean[3, 1]
    # rows beside it may be held against another reference: 2^-17 of a weight and half a step of the output on either side
    assert ((got - clean).abs().float() <= 2 * U.half_step(dtype) * clean.abs().float() + 2.0 ** -16 * v.abs().max().float()).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_missing_pages_are_not_read(dtype):
    r = U.Round([300], [5], device=DEV)
    q, k, v = r.randn(r.R, 4, 64, dtype=dtype), r.randn(r.n_pages, 64, 2, 64, dtype=dtype), r.randn(r.n_pages, 64, 2, 64, dtype=dtype)
    m = ops.slot_maps(**r.inputs())
    want = ops.tree_attention(q, k, v, m, 0.1, window=70)
    for bad in (-1, r.n_pages, 1 << 30):
        m.tables[0, 1] = bad
        assert torch.equal(ops.tree_attention(q, k, v, m, 0.1, window=70), want)          # outside the window
        assert torch.isfinite(ops.tree_attention(q, k, v, m, 0.1)).all()
        expect_status()


@pytest.mark.parametrize("dtype", DTYPES)
def test_sink_of_nothing(dtype):
    T.check_sink_of_nothing(DEV, dtype)


@pytest.mark.parametrize("length", [200, 1 << 20, (1 << 31) - 1])
@pytest.mark.parametrize("dtype", DTYPES)
def test_lengths_beyond_the_table(dtype, length):
    r = U.Round([150, 90], [6, 4], device=DEV)
    q, k, v = r.randn(r.R, 4, 64, dtype=dtype), r.randn(r.n_pages, 64, 2, 64, dtype=dtype), r.randn(r.n_pages, 64, 2, 64, dtype=dtype)
    want = ops.tree_attention(q, k, v, ops.slot_maps(**r.inputs()), 0.1)
    d = r.inputs()
    d["lengths"] = torch.tensor([length, 90], dtype=torch.int32, device=DEV)          # the table has three pages
    m = ops.slot_maps(**d)
    expect_status()
    got = ops.tree_attention(q, k, v, m, 0.1)
    expect_status()
    assert torch.isfinite(got).all() and torch.equal(got[6:], want[6:])


@pytest.mark.parametrize("dtype", DTYPES)
def test_caches_beyond_32_bit_offsets(dtype):
    """The last pages of a cache of more than 2^31 elements (and bytes)."""
    r = U.Round([200], [9], device=DEV)
    G, D = 8, 128
    pages = (1 << 31) // (64 * G * D) + 8
    k, v = torch.zeros(pages, 64, G, D, dtype=dtype, device=DEV), torch.zeros(pages, 64, G, 8, dtype=dtype, device=DEV)
    off = pages - r.n_pages
    r.table[r.table >= 0] += off
    kn, vn = r.randn(r.n_pages, 64, G, D, dtype=dtype), r.randn(r.n_pages, 64, G, 8, dtype=dtype)
    k[off:], v[off:] = kn, vn
    q, m = r.randn(r.R, G, D, dtype=dtype), ops.slot_maps(**r.inputs())
    got = ops.tree_attention(q, k, v, m, 0.1)
    r.table[r.table >= 0] -= off
    want, tol = U.want_attention(r, q, kn, vn, 0.1, rounded=WEIGHTS[dtype])
    U.close(got, want, tol, dtype)
    C = G * (2 * D + 8)
    x, w, tail = r.randn(r.R, C, dtype=dtype), r.randn(2, C), r.randn(1, 1, C, dtype=dtype)
    ops.path_conv(x, w, tail, m, G * D, k, v)
    y, mag = U.want_conv(r, x, w, tail)
    rows = torch.tensor(r.rows(0)[200:], device=DEV) + off * 64
    U.close(k.view(-1, G * D)[rows], y[:, G * D: 2 * G * D], mag[:, G * D: 2 * G * D] * 2.0 ** -22, dtype)
    path = U.path_of(r, 0, 8)
    src = k.view(-1, G * D)[rows[path]].clone()
    ops.commit_paths(m, r.i32([path]), r.i32([len(path)]), [k])
    assert torch.equal(k.view(-1, G * D)[rows[: len(path)]], src)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("taps", [0, 1, 2, 4, 9])
@pytest.mark.parametrize("name", list(T.ROUNDS))
def test_commit_of_paths(name, taps, dtype):
    T.check_commit(U.Round(**T.ROUNDS[name], device=DEV, seed=5), dtype, (8, 12, 4, 520), taps, 1032)


def test_commit_of_many_layers():
    T.check_commit(U.Round([30, 200, 7], [9, 64, 20], device=DEV, seed=6), BF16, (64,) * 150, 4, 64)


def test_paths_that_lead_nowhere_move_nothing():
    r = U.Round([70, 9], [5, 6], device=DEV)
    m, k = ops.slot_maps(**r.inputs()), r.randn(r.n_pages, 64, 2, 8)
    before = k.clone()
    for bad in ([0, 2, 2, 3], [1, 0, 2, 3], [0, 1, 2, 5], [0, -1, 2, 3], [0, 1, 2, 1 << 30]):
        ops.commit_paths(m, r.i32([bad, [0, 0, 0, 0]]), r.i32([4, 0]), [k])
        expect_status()
        assert torch.equal(k, before)


def _round_of(r, dtype, seed):
    """A whole round: room, maps, convolution, attention, commit, room given back.  Returns (call, outputs' owner)."""
    H, G, D = 8, 2, 64
    C = (H + 2 * G) * D
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s, dt=dtype: torch.randn(*s, generator=g).to(dt).to(DEV)
    d = r.inputs()
    held = [-(-n // 64) for n in r.lengths]
    taken = [int((row >= 0).sum()) for row in r.table]
    back = [int(r.table[s, p]) for s in reversed(range(len(held))) for p in reversed(range(held[s], taken[s]))]
    for s, n in enumerate(held):
        d["tables"][s, n:] = -1
    st = {"x": rnd(r.R, C), "w": rnd(4, C, dt=F32) * 0.5, "tail": rnd(len(held), 3, C), "k": rnd(r.n_pages, 64, G, D), "v": rnd(r.n_pages, 64, G, D),
          "held": r.i32(held), "free": r.i32(back + [-1] * (r.n_pages - len(back))), "n_free": r.i32([len(back)]), "grown": r.i32(np.add(r.lengths, r.counts)),
          "path": r.i32([(U.path_of(r, s, n - 1) + [0] * 64)[:64] if n else [0] * 64 for s, n in enumerate(r.counts)]),
          "n_path": r.i32([len(U.path_of(r, s, n - 1)) if n else 0 for s, n in enumerate(r.counts)]), "d": d}

    def call():
        ops.block_tables(st["grown"], d["tables"], st["held"], st["free"], st["n_free"])
        m = ops.slot_maps(**d)
        q = ops.path_conv(st["x"], st["w"], st["tail"], m, H * D, st["k"], st["v"])
        o = ops.tree_attention(q.view(r.R, H, D), st["k"], st["v"], m, D ** -0.5, softcap=20.0, sink=torch.zeros(H, device=DEV))
        ops.commit_paths(m, st["path"], st["n_path"], [st["k"], st["v"]], [(st["x"], st["tail"])])
        ops.block_tables(d["lengths"] + st["n_path"], d["tables"], st["held"], st["free"], st["n_free"])
        return o
    return call, st


def _want_round(r, st0):
    """The same from the definitions."""
    H, G, D = 8, 2, 64
    y, mag = U.want_conv(r, st0["x"], st0["w"], st0["tail"])
    dt = st0["x"].dtype
    y = y.to(dt)
    k, v = st0["k"].clone(), st0["v"].clone()
    for s, L in enumerate(r.lengths):
        rows = torch.tensor(r.rows(s)[L:], device=DEV)
        sl = slice(r.starts[s], r.starts[s + 1])
        k.view(-1, G * D)[rows], v.view(-1, G * D)[rows] = y[sl, H * D: (H + G) * D].to(DEV), y[sl, (H + G) * D:].to(DEV)
    return U.want_attention(r, y[:, : H * D].to(DEV).view(r.R, H, D), k, v, D ** -0.5, softcap=20.0, sink=torch.zeros(H, device=DEV), rounded=WEIGHTS[dt])


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_round_captured_and_replayed_on_another_one(dtype):
    """A captured round gives, on other lengths, trees, pages and rows of the same capacity, what the eager round gives, bit for bit."""
    rounds = [U.Round(L, n, device=DEV, seed=i, pad=40 - sum(n), width=8, spare=30 - sum(-(-(a + b) // 64) for a, b in zip(L, n)))
              for i, (L, n) in enumerate((([70, 200, 3], [9, 12, 4]), ([63, 0, 330], [1, 20, 19]), ([5, 5, 5], [0, 3, 1])))]
    for r in rounds:
        assert r.R == 40 and r.n_pages == 30
    calls = [_round_of(r, dtype, i) for i, r in enumerate(rounds)]
    for c, st in calls:
        st["d"]["nodes"] = 20
    before = [{k: (t.clone() if torch.is_tensor(t) else {a: b.clone() if torch.is_tensor(b) else b for a, b in t.items()}) for k, t in st.items()} for _, st in calls]

    def reset(st, old):
        for k, t in st.items():
            if torch.is_tensor(t):
                t.copy_(old[k])
            else:
                for a, b in t.items():
                    if torch.is_tensor(b):
                        b.copy_(old[k][a])
    eager = []
    for (c, st), old, r in zip(calls, before, rounds):
        o = c().clone()
        eager.append((o, {k: st[k].clone() for k in ("k", "v", "tail", "held", "n_free")}, st["d"]["tables"].clone()))
        want, tol = _want_round(r, old)
        # queries and keys that were rounded at a border may differ by a step: compared loosely here, closely where inputs are given
        assert (o.double().cpu() - want).abs().max() < (1e-4 if dtype == F32 else 0.06)
        reset(st, old)
    call, st = calls[0]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for old, (o, state, tables) in list(zip(before, eager)) * 2:
        reset(st, old)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, o) and torch.equal(st["d"]["tables"], tables)
        assert all(torch.equal(st[k], t) for k, t in state.items())


def test_two_calls_at_once():
    """Calls on two streams and two captured graphs replayed together share no workspace."""
    rs = [U.Round([3000, 500], [20, 9], device=DEV, seed=i) for i in range(2)]
    args = []
    for r in rs:
        q, k, v = r.randn(r.R, 8, 128, dtype=BF16), r.randn(r.n_pages, 64, 2, 128, dtype=BF16), r.randn(r.n_pages, 64, 2, 128, dtype=BF16)
        args.append((q, k, v, ops.slot_maps(**r.inputs()), 0.09))
    want = [ops.tree_attention(*a) for a in args]
    streams = [torch.cuda.Stream() for _ in args]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for s, a in zip(streams, args):
            with torch.cuda.stream(s):
                got.append(ops.tree_attention(*a))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for a in args:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.tree_attention(*a))
        graphs.append(g)
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_results_do_not_depend_on_the_other_requests():
    """The same request alone and in a batch: within the bounds; run to run: bit for bit."""
    r = U.Round([900, 64, 2000, 1], [12, 5, 30, 7], device=DEV)
    q, k, v = r.randn(r.R, 8, 64, dtype=BF16), r.randn(r.n_pages, 64, 2, 64, dtype=BF16), r.randn(r.n_pages, 64, 2, 64, dtype=BF16)
    m = ops.slot_maps(**r.inputs())
    got = ops.tree_attention(q, k, v, m, 0.125)
    for _ in range(3):
        assert torch.equal(ops.tree_attention(q, k, v, m, 0.125), got)


def test_unaligned_queries_are_taken():
    r = U.Round([70], [5], device=DEV)
    k, v, m = r.randn(r.n_pages, 64, 1, 64, dtype=BF16), r.randn(r.n_pages, 64, 1, 64, dtype=BF16), ops.slot_maps(**r.inputs())
    wide = r.randn(r.R, 2 * 64 + 3, dtype=BF16)
    q = wide[:, 1: 129].unflatten(1, (2, 64))
    assert torch.equal(ops.tree_attention(q, k, v, m, 0.1), ops.tree_attention(q.contiguous(), k, v, m, 0.1))


def test_empty_calls():
    r = U.Round([70, 3], [0, 0], device=DEV, trees=False)
    m = ops.slot_maps(**r.inputs())
    k = r.randn(r.n_pages, 64, 1, 64)
    assert ops.tree_attention(torch.empty(0, 2, 64, device=DEV), k, k.clone(), m, 0.1).shape == (0, 2, 64)
    ops.commit_paths(m, torch.zeros(2, 3, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV), [k])
    r = U.Round([70, 3], [0, 0], device=DEV, pad=4)
    m = ops.slot_maps(**r.inputs())
    assert m.slot.tolist() == [-1] * 4
    assert not ops.tree_attention(torch.ones(4, 2, 64, device=DEV), k, k.clone(), m, 0.1).any()


def _anywhere(x, how):
    """The rows x [R, C] again, where kernels cannot read them 16 bytes at a time."""
    R, C = x.shape
    if how == "contiguous, one element in":
        b = x.new_zeros(R * C + 1)
        y = b[1:].view(R, C)
    else:                                            # one row, or rows, of an odd pitch
        b = x.new_zeros(R + 1, C + 5)
        y = b[:R, :C]
    y.copy_(x)
    return y


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 2, 9])
@pytest.mark.parametrize("how", ["contiguous, one element in", "an odd pitch"])
def test_rows_that_start_anywhere(how, rows, dtype):
    r = U.Round([70], [rows], device=DEV)
    H, G, D, taps = 4, 2, 64, 3
    C = (H + 2 * G) * D
    m, k, v = ops.slot_maps(**r.inputs()), r.randn(r.n_pages, 64, G, D, dtype=dtype), r.randn(r.n_pages, 64, G, D, dtype=dtype)
    x, w, tail = r.randn(rows, C, dtype=dtype), r.randn(taps, C), r.randn(1, taps - 1, C, dtype=dtype)
    k2, v2 = k.clone(), v.clone()
    want = ops.path_conv(x, w, tail, m, H * D, k, v)
    got = ops.path_conv(_anywhere(x, how), w, tail, m, H * D, k2, v2)
    assert torch.equal(got, want) and torch.equal(k, k2) and torch.equal(v, v2)
    q = r.randn(rows, H * D, dtype=dtype)
    want = ops.tree_attention(q.view(rows, H, D), k, v, m, 0.1)
    assert torch.equal(ops.tree_attention(_anywhere(q, how).unflatten(1, (H, D)), k, v, m, 0.1), want)
    one = q[:1].expand(rows, -1)                     # one row for all
    assert torch.equal(ops.tree_attention(one.unflatten(1, (H, D)), k, v, m, 0.1), ops.tree_attention(one.contiguous().view(rows, H, D), k, v, m, 0.1))


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_row_and_one_head_have_any_stride(dtype):
    """Strides of dimensions with one entry mean nothing: outputs, gates and rows behind a tail."""
    r = U.Round([70], [1], device=DEV)
    m, k, v = ops.slot_maps(**r.inputs()), r.randn(r.n_pages, 64, 1, 64, dtype=dtype), r.randn(r.n_pages, 64, 1, 64, dtype=dtype)
    q, gate = r.randn(1, 1, 64, dtype=dtype), r.randn(1, 1, dtype=dtype)
    want = ops.tree_attention(q, k, v, m, 0.1, gate=gate)
    out = torch.zeros(200, dtype=dtype, device=DEV).as_strided((1, 1, 64), (67, 5, 1))
    got = ops.tree_attention(q, k, v, m, 0.1, gate=torch.zeros(9, dtype=dtype, device=DEV).as_strided((1, 1), (3, 7)).copy_(gate), out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(got, want)
    x, tail = r.randn(1, 64, dtype=dtype), r.randn(1, 2, 64, dtype=dtype)
    last = tail[0, 1].clone()
    ops.commit_paths(m, r.i32([[0]]), r.i32([1]), [k], [(torch.cat((x, x), 1).as_strided((1, 64), (67, 1)), tail)])
    assert torch.equal(tail[0], torch.stack((last, x[0])))


@pytest.mark.parametrize("length", [200, 1 << 20, (1 << 31) - 1024, (1 << 31) - 2, (1 << 31) - 1])
def test_commit_of_lengths_beyond_the_table(length):
    """Token numbers are formed in 64 bits: the request is skipped, the one beside it is not."""
    r = U.Round([150, 90], [6, 4], device=DEV)
    good, k = ops.slot_maps(**r.inputs()), r.randn(r.n_pages, 64, 2, 8)
    want = k.clone()
    ops.commit_paths(good, r.i32([[0, 0, 0], [0, 2, 3]]), r.i32([0, 3]), [want])
    d = r.inputs()
    d["lengths"] = torch.tensor([length, 90], dtype=torch.int32, device=DEV)          # the table has three pages
    m = ops.slot_maps(**d)
    expect_status()
    ops.commit_paths(m, r.i32([[0, 2, 5], [0, 2, 3]]), r.i32([3, 3]), [k])
    expect_status()
    assert torch.equal(k, want)


@pytest.mark.parametrize("layers", [1, 70])            # one launch, and two
def test_a_request_is_committed_everywhere_or_nowhere(layers):
    """A missing page, or one that only some of the caches have: neither caches nor tails of the request change, those of the others do."""
    for bad in (-1, "past the smallest cache", 1 << 30):
        r = U.Round([60, 90, 126], [9, 6, 4], device=DEV, spare=4)
        m = ops.slot_maps(**r.inputs())
        caches = [r.randn(r.n_pages, 64, 2, 8) for _ in range(layers)] + [r.randn(r.n_pages, 64, 1, 16, dtype=BF16)]
        tails = [(r.randn(r.R, 32), r.randn(3, 2, 32)) for _ in range(layers)]
        path, n_path = r.i32([[0, 2, 4, 6, 8], [0, 2, 3, 3, 3], [0, 1, 3, 3, 3]]), r.i32([5, 3, 3])
        want_c, want_t = [c.clone() for c in caches], [t.clone() for _, t in tails]
        ops.commit_paths(m, path, r.i32([0, 3, 3]), want_c, [(x, t) for (x, _), t in zip(tails, want_t)])
        if bad == "past the smallest cache":
            most = r.table[1:].max() + 1
            keep = max(most, r.table[0, 0] + 1)
            if r.table[0, 1] < keep:                   # (the request's second page lies behind all others)
                m.tables[0, 1] = int(keep)
            caches.append(r.randn(int(keep), 64, 2, 8))
            want_c.append(caches[-1].clone())
            ops.commit_paths(m, path, r.i32([0, 3, 3]), want_c[-1:])
        else:
            m.tables[0, 1] = bad
        ops.commit_paths(m, path, n_path, caches, tails)
        expect_status()
        assert all(torch.equal(a, b) for a, b in zip(caches, want_c)) and all(torch.equal(t, b) for (_, t), b in zip(tails, want_t))
    m.tables[0, 1] = -1                              # without caches nothing depends on pages
    x, t = tails[0]
    ops.commit_paths(m, path, r.i32([5, 0, 0]), [], [(x, t)])
    assert torch.equal(t[0], x[[6, 8]]) and torch.equal(t[1:], want_t[0][1:])


OPTIONS = {
    "soft cap": dict(softcap=2.0), "soft cap and bias": dict(softcap=30.0, bias=100), "bias": dict(bias=100), "slopes": dict(slopes=True),
    "soft cap, slopes, sink": dict(softcap=5.0, slopes=True, sink=True),
}


@pytest.mark.parametrize("name", list(OPTIONS))
@pytest.mark.parametrize("near", [0.01, 3.0])          # scores far below the cap's bend, and past it
@pytest.mark.parametrize("length", [70, 9000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_what_is_not_a_number_shows_with_options(dtype, length, near, name):
    """NaN in a query, in a visible key and in an option's table: the rows that it reaches are NaN, the others are as the definition has them."""
    f = OPTIONS[name]
    r = U.Round([length, length], [9, 9], device=DEV)
    q, k, v = r.randn(r.R, 4, 64, dtype=dtype) * near, r.randn(r.n_pages, 64, 2, 64, dtype=dtype), r.randn(r.n_pages, 64, 2, 64, dtype=dtype)
    opt = {"softcap": f["softcap"]} if "softcap" in f else {}
    if "bias" in f:
        opt["bias"] = r.randn(4, f["bias"])
    if "slopes" in f:
        opt["slopes"] = torch.linspace(0.001, 0.02, 4, device=DEV)
    if "sink" in f:
        opt["sink"] = r.randn(4)
    m = ops.slot_maps(**r.inputs())
    want, tol = U.want_attention(r, q, k, v, 0.125, rounded=WEIGHTS[dtype], **opt)

    def check(rows, heads, q=q, k=k, opt=opt):
        got = ops.tree_attention(q, k, v, m, 0.125, **opt)
        hit = torch.zeros(r.R, 4, dtype=torch.bool)
        hit[torch.tensor(rows)[:, None], torch.tensor(heads)] = True
        assert torch.equal(got.isnan().all(-1).cpu(), hit) and torch.equal(got.isnan().any(-1).cpu(), hit)
        U.close(got.cpu()[~hit], want[~hit], tol[~hit], dtype)

    spoiled = q.clone()
    spoiled[3, 1] = float("nan")
    check([3], [1], q=spoiled)
    for at, rows in ((5, list(range(9))), (length - 1, list(range(9))), (length + 4, [j for j in range(9) if r.anc[0][j, 4]])):
        spoiled = k.clone()
        spoiled.view(-1, 2, 64)[r.rows(0)[at], 1, 7] = float("nan")
        check(rows, [2, 3], k=spoiled)
    for n in ("bias", "slopes", "sink"):
        if n in opt:
            spoiled = opt[n].clone()
            spoiled[2] = float("nan")
            check(list(range(r.R)), [2], opt={**opt, n: spoiled})


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinite_scores_are_capped(dtype):
    """Products past the largest number are scores of plus and minus the cap (held to 8 half steps of fp32, a weight to 16, the sums to one a token)."""
    r = U.Round([300], [9], device=DEV)
    q, k, v = r.randn(r.R, 4, 64, dtype=dtype), r.randn(r.n_pages, 64, 2, 64, dtype=dtype), r.randn(r.n_pages, 64, 2, 64, dtype=dtype)
    q[:, :, 5], k[:, :, :, 5] = 3e38, 3e38 * torch.sign(k[:, :, :, 5].float()).to(dtype)
    got = ops.tree_attention(q, k, v, ops.slot_maps(**r.inputs()), 1.0, softcap=3.0)
    rows, seen = torch.tensor(r.rows(0), device=DEV), torch.ones(9, 309, dtype=torch.bool, device=DEV)
    seen[:, 300:] = torch.tensor(r.anc[0], device=DEV)
    want = torch.zeros(9, 4, 64, dtype=torch.float64, device=DEV)
    tol = torch.zeros_like(want)
    for h in range(4):
        x = torch.where(seen, 3.0 * torch.sign(k.view(-1, 2, 64)[rows, h // 2, 5].double()), -torch.inf)
        p, vv = torch.softmax(x, 1), v.view(-1, 2, 64)[rows, h // 2].double()
        want[:, h], tol[:, h] = p @ vv, p @ vv.abs() * ((2 * 3 * 8 + 16 + 309) * 2.0 ** -24 + WEIGHTS[dtype])
    U.close(got, want.cpu(), tol.cpu(), dtype)


@pytest.mark.parametrize("G,rep,D,V,nodes", [(2, 4, 64, 64, 7), (2, 4, 128, 128, 50), (1, 8, 64, 128, 60), (2, 2, 256, 256, 9), (1, 16, 96, 48, 33)])
@pytest.mark.parametrize("f", [{}, dict(softcap=4.0)])
def test_weights_keep_two_terms(G, rep, D, V, nodes, f):
    """Scores near 0 and values of either sign: outputs that cancel show what the weights lose, which may be 2^-17 of each for any size of tree."""
    r = U.Round([90, 40], [nodes, 3], device=DEV, seed=4)
    q, k = r.randn(r.R, G * rep, D, dtype=BF16) * 0.05, r.randn(r.n_pages, 64, G, D, dtype=BF16)
    v = torch.sign(r.randn(r.n_pages, 64, G, V)).to(BF16)
    got = ops.tree_attention(q, k, v, ops.slot_maps(**r.inputs()), D ** -0.5, **f)
    U.close(got, *U.want_attention(r, q, k, v, D ** -0.5, rounded=2.0 ** -17, **f), BF16)


@pytest.mark.parametrize("dtype", DTYPES)
def test_caches_and_outputs_in_any_order(dtype):
    """Pages inside tokens, heads outside rows: what does not overlap is taken."""
    r = U.Round([300, 63], [16, 3], device=DEV)
    q, k, v, m = r.randn(r.R, 4, 64, dtype=dtype), r.randn(r.n_pages, 64, 2, 64, dtype=dtype), r.randn(r.n_pages, 64, 2, 64, dtype=dtype), ops.slot_maps(**r.inputs())
    want = ops.tree_attention(q, k, v, m, 0.125)
    turned = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.zeros(4, r.R, 64, dtype=dtype, device=DEV).transpose(0, 1)
    assert torch.equal(ops.tree_attention(turned(q), turned(k), turned(v), m, 0.125, out=out), want) and torch.equal(out, want)
    path, n = r.i32([[0, 3, 9], [0, 2, 2]]), r.i32([3, 2])
    other = turned(k)
    ops.commit_paths(m, path, n, [k])
    ops.commit_paths(m, path, n, [other])
    assert torch.equal(k, other)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rest_of_convolution(dtype):
    T.check_rest_of_convolution(DEV, dtype)
    expect_status()                                  # (a request without a row of the tables)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [0, 40])
def test_visible_infinities_show_in_every_page(window, dtype):
    """A visible token counts even where its weight is 0: an infinite value of it makes NaN, in pages that all rows see whole and in others."""
    r = U.Round([200], [9], device=DEV, seed=7)
    q, v = r.randn(r.R, 4, 64, dtype=dtype), r.randn(r.n_pages, 64, 2, 64, dtype=dtype)
    k, m, bias = r.randn(r.n_pages, 64, 2, 64, dtype=dtype), ops.slot_maps(**r.inputs()), r.randn(4, 300)
    for at in (10, 100, 150, 195, 204):              # pages seen whole, the edge of the window, the tree's own page
        low = bias.clone()
        dist = m.pos.long() - (at if at < 200 else int(m.pos[at - 200]))
        low[:, dist.clamp(0, 299)] = -float("inf")
        bad = v.clone()
        bad.view(-1, 2, 64)[r.rows(0)[at], :, 3] = float("inf")
        got = ops.tree_attention(q, k, bad, m, 0.125, bias=low, window=window)
        seen = torch.tensor(r.anc[0][:, at - 200]) if at >= 200 else torch.ones(9, dtype=torch.bool)
        if window:
            seen &= (dist < window).cpu()
        assert torch.equal(got[:, :, 3].isnan().all(1).cpu(), seen) and torch.equal(got[:, :, 3].isnan().any(1).cpu(), seen)
        assert torch.isfinite(got[:, :, [2, 4, 63]]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("low", [-200.0, -float("inf")])
def test_visible_infinities_show_in_every_part(low, dtype):
    """The same of a request whose pages many CTAs share: a part that weighs nothing beside the others."""
    r = U.Round([9000], [5], device=DEV)
    q, k, v = r.randn(r.R, 4, 64, dtype=dtype), r.randn(r.n_pages, 64, 2, 64, dtype=dtype), r.randn(r.n_pages, 64, 2, 64, dtype=dtype)
    m, bias = ops.slot_maps(**r.inputs()), torch.zeros(4, 9100, device=DEV)
    bias[:, 4000:6000] = low
    assert torch.isfinite(ops.tree_attention(q, k, v, m, 0.125, bias=bias)).all()
    v.view(-1, 2, 64)[r.rows(0)[4100], 1, 3] = float("inf")
    got = ops.tree_attention(q, k, v, m, 0.125, bias=bias).isfinite().cpu()
    want = torch.ones_like(got)
    want[:, 2:, 3] = False
    assert torch.equal(got, want)


def test_launches_are_counted_where_there_are_any():
    cu = ops.cuda_ops()
    r, none = U.Round([70, 9], [5, 6], device=DEV), U.Round([70, 3], [0, 0], device=DEV, trees=False)
    k, v = r.randn(r.n_pages, 64, 1, 64), r.randn(r.n_pages, 64, 1, 64)
    m, empty = ops.slot_maps(**r.inputs()), ops.slot_maps(**none.inputs())
    i32 = r.i32

    def counted(call):
        cu.reset_launch_count()
        call()
        return cu.launch_count()
    x, w, tail = r.randn(r.R, 256), r.randn(2, 256), r.randn(2, 1, 256)
    assert counted(lambda: ops.slot_maps(**r.inputs())) == 1
    assert counted(lambda: ops.path_conv(x, w, tail, m, 128, k, v)) == 1
    assert counted(lambda: ops.path_conv(x[:0], w, tail, empty, 128, k, v)) == 0
    assert counted(lambda: ops.tree_attention(r.randn(r.R, 2, 64), k, v, m, 0.1)) == 2
    assert counted(lambda: ops.tree_attention(x[:0, :128].view(0, 2, 64), k, v, empty, 0.1)) == 0
    assert counted(lambda: ops.commit_paths(m, i32([[0], [0]]), i32([1, 1]), [k, v])) == 1
    assert counted(lambda: ops.commit_paths(m, i32([[0], [0]]), i32([1, 1]), [r.randn(r.n_pages, 64, 1, 8) for _ in range(130)])) == 2
    assert counted(lambda: ops.commit_paths(m, i32([[0], [0]]), i32([1, 1]), [])) == 0
    nobody = torch.zeros(0, dtype=torch.int32, device=DEV)
    assert counted(lambda: ops.block_tables(nobody, torch.zeros(0, 3, dtype=torch.int32, device=DEV), nobody, nobody, i32([0]))) == 0


@pytest.mark.parametrize("counts", [[1] * 40, [1] * 39 + [150], [4, 200], [70]])
def test_chains_of_any_lengths(counts):
    r = U.Round(np.random.RandomState(2).randint(0, 700, len(counts)), counts, device=DEV, trees=False, pad=2)
    T.check_attention(r, 16, 4, 64, 64, BF16, {}, rounded=WEIGHTS[BF16])
    T.check_attention(r, 16, 4, 128, 64, BF16, dict(softcap=3.0, window=100), rounded=WEIGHTS[BF16])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [(8, 2), (16, 1)])
def test_requests_alone_and_in_a_batch(heads, dtype):
    """A request's outputs beside others, whose lengths move where its pages are divided, and by itself: both within the bounds of the definition."""
    r = U.Round([900, 64, 2000, 1, 300], [12, 5, 30, 7, 9], device=DEV)
    H, G = heads
    q, k, v = r.randn(r.R, H, 64, dtype=dtype), r.randn(r.n_pages, 64, G, 64, dtype=dtype), r.randn(r.n_pages, 64, G, 64, dtype=dtype)
    opt = dict(softcap=9.0, sink=r.randn(H))
    want, tol = U.want_attention(r, q, k, v, 0.125, rounded=2.0 ** -17 if dtype == BF16 else 0.0, **opt)
    d = r.inputs()
    U.close(ops.tree_attention(q, k, v, ops.slot_maps(**d), 0.125, **opt), want, tol, dtype)
    for s in range(5):
        sl = slice(r.starts[s], r.starts[s + 1])
        m = ops.slot_maps(d["lengths"][s: s + 1].clone(), d["counts"][s: s + 1].clone(), d["tables"], r.counts[s], slots=r.i32([s]),
                          parents=d["parents"][sl].clone(), nodes=r.counts[s])
        U.close(ops.tree_attention(q[sl], k, v, m, 0.125, **opt), want[sl], tol[sl], dtype)
