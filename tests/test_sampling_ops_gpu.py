"""The kernels between a round's logits and its tokens against the definitions in 64 bits."""
import numpy as np
import pytest
import torch

from spark_engine_b200 import ops
from tests.sampling_util import Rows, Table, near, want_logprobs, want_token

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
FILTERS = [dict(), dict(top_k=1), dict(top_k=5), dict(top_k=300), dict(top_p=0.0), dict(top_p=0.3), dict(top_p=0.95), dict(top_p=0.9999999), dict(min_p=0.05),
           dict(min_p=1.0), dict(min_p=2.0), dict(top_k=40, top_p=0.9, min_p=0.02), dict(top_k=10**6, top_p=1.0, min_p=0.0), dict(top_k=3000, top_p=0.9)]


def _sound():
    from spark_engine_b200.ops import cuda
    torch.cuda.synchronize()
    assert cuda.read_status(torch.device("cuda"))[0] == 0


# ----------------------------------------------------------------------------- draws
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("kind", ["peaked", "flat", "equal", "same", "holes", "one"])
@pytest.mark.parametrize("V", [1, 2, 31, 1000, 4099, 50257])
def test_draws_follow_the_definition(V, kind, dtype):
    rows = Rows(4 if V > 5000 else 9, V, kind, TYPES[dtype], seed=V, device="cuda")
    for i, s in enumerate(FILTERS):
        T = (0.8, 1.7, 0.3)[i % 3]
        assert np.array_equal(rows.draw(T, **s), rows.want(T, **s)), (s, T)
    assert np.array_equal(rows.draw(0.0), rows.want(0.0))
    _sound()


@pytest.mark.parametrize("R, V, kind", [(1, 151936, "peaked"), (1, 151936, "flat"), (3, 151936, "equal"), (40, 129280, "peaked"), (160, 20011, "flat"),
                                        (2, 786432, "flat"), (2, 300001, "peaked"), (700, 3000, "peaked"), (5, 65537, "same")])
def test_rows_of_every_size(R, V, kind):
    """Each row with settings of its own, rows a few elements apart."""
    rows = Rows(R, V, kind, seed=R, device="cuda", pad=3)
    r = rows.rs
    s = dict(top_k=r.choice([0, 0, 1, 20, 50, 1000, 20000], R), top_p=r.choice([1.0, 0.5, 0.9, 0.95, 0.999], R), min_p=r.choice([0.0, 0.0, 0.1, 1e-4], R))
    T = r.choice([0.0, 0.5, 1.0, 1.6], R)
    assert np.array_equal(rows.draw(T, **s), rows.want(T, **s))
    _sound()


def test_a_row_draws_the_same_in_every_batch():
    rows = Rows(200, 50001, "flat", seed=4, device="cuda")
    s = dict(top_k=2000, top_p=0.8)
    every = rows.draw(1.2, **s)
    for r in (0, 17, 199):
        one = ops.sample_tokens(rows.logits[r: r + 1], *(rows.t([x], d) for x, d in ((1.2, torch.float32), (rows.seeds[r], torch.int64), (rows.positions[r], torch.int64))),
                                top_k=rows.t([2000], torch.int32), top_p=rows.t([0.8], torch.float32))
        assert int(one) == every[r]
    few = Rows(200, 50001, "flat", seed=4, device="cuda")
    few.logits, few.seeds, few.positions, few.R = rows.logits[:5], rows.seeds[:5], rows.positions[:5], 5
    assert np.array_equal(few.draw(1.2, **s), every[:5])


def test_without_filters_it_is_the_token_of_perturbed_logits():
    rows = Rows(33, 30011, "flat", seed=6, device="cuda")
    x = ops.gumbel_perturb(rows.logits, [0.9] * 33, rows.seeds.tolist(), rows.positions.tolist(), 0, 30011)
    assert np.array_equal(rows.draw(0.9), ops.argmax(x).cpu().numpy())


@pytest.mark.parametrize("T", [1e-40, 1e-30, 1e-8, 1e-7, 1e-6, 1e-5, 1e6, float("inf")])
def test_extreme_temperatures(T):
    for kind in ("flat", "equal"):
        rows = Rows(6, 3001, kind, seed=8, device="cuda")
        for s in (dict(), dict(top_k=30), dict(top_p=0.7), dict(min_p=0.5)):
            assert np.array_equal(rows.draw(T, **s), rows.want(T, **s)), s


def test_large_logits_and_infinities():
    rows = Rows(6, 2000, "flat", seed=9, device="cuda")
    big = rows.z.copy()
    big[0] *= 1e6
    big[1] *= 1e37
    big[2, 5] = big[2, 900] = np.inf
    big[3] -= 1e5
    big[4, :] = -np.inf
    big[5, :] = np.nan
    rows.logits, rows.z = rows.t(big, torch.float32), big.astype(np.float32)
    for s in (dict(), dict(top_k=30), dict(top_p=0.7), dict(min_p=0.5)):
        assert np.array_equal(rows.draw(1.0, **s), rows.want(1.0, **s)), s


@pytest.mark.parametrize("R, V, per, drafts, biases, allowed", [(8, 151936, 4, 3, 8, None), (1, 4099, 1, 0, 0, 0.01), (300, 4099, 3, 2, 30, 0.5), (5, 1001, 5, 64, 700, 0.9),
                                                              (2, 33, 1, 1, 40, None), (64, 20000, 1, 0, 300, 0.001)])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_adjusted_draws_are_draws_from_adjusted_logits(R, V, per, drafts, biases, allowed, dtype):
    rows = Rows(R, V, "peaked", TYPES[dtype], seed=V, device="cuda")
    table = Table(rows, per, drafts, biases, allowed, dup=V < 2000)
    a = table.adjust()
    z = ops.adjust_logits(rows.logits, a)
    want, tol = table.want()
    got = z.double().cpu().numpy()
    fine = np.isfinite(want)
    assert np.array_equal(np.isfinite(got), fine) and (np.abs(got[fine] - want[fine]) <= tol[fine]).all()
    host = lambda x: None if x is None else x.cpu()
    names = ("counts", "slots", "drafted", "repetition", "presence", "frequency", "bias_ids", "bias", "allowed")
    plain = ops.adjust_logits(rows.logits.cpu(), ops.Adjust(**{k: host(getattr(a, k)) for k in names}))
    assert torch.equal(plain, z.cpu())                                   # the same roundings, in the same order
    for s in (dict(), dict(top_k=20, top_p=0.9)):
        assert np.array_equal(rows.draw(0.8, adjust=a, **s), rows.want(0.8, z=got.astype(np.float32), **s))
    assert np.array_equal(rows.draw(0.0, adjust=a), rows.want(0.0, z=got.astype(np.float32)))
    if dtype == "f32":
        x = rows.logits.clone()
        assert ops.adjust_logits(x, a, out=x) is x and torch.equal(x, z)
        wide = torch.zeros(R, V + 5, device="cuda")
        ops.adjust_logits(rows.logits, a, out=wide[:, 2: V + 2])
        assert torch.equal(wide[:, 2: V + 2], z) and not wide[:, :2].any() and not wide[:, V + 2:].any()
    _sound()


def test_slices_of_a_vocabulary_are_adjusted_alike():
    rows = Rows(6, 9000, seed=2, device="cuda")
    a = Table(rows, drafts=2, biases=20).adjust()
    whole = ops.adjust_logits(rows.logits, a)
    for o, n in ((0, 4001), (4001, 4999)):
        part = ops.Adjust(counts=a.counts[:, o: o + n], slots=a.slots, drafted=a.drafted, repetition=a.repetition, presence=a.presence, frequency=a.frequency,
                          bias_ids=a.bias_ids, bias=a.bias)
        assert torch.equal(ops.adjust_logits(rows.logits[:, o: o + n], part, offset=o), whole[:, o: o + n])


def test_slots_outside_the_counts_are_reported():
    from spark_engine_b200.ops import cuda
    rows = Rows(2, 100, device="cuda")
    try:
        a = ops.Adjust(counts=torch.full((2, 100), 2, dtype=torch.int32, device="cuda"), slots=rows.t([5, -1], torch.int32), frequency=rows.t([1.0, 1.0], torch.float32))
        assert torch.equal(ops.adjust_logits(rows.logits, a), rows.logits)
        assert cuda.read_status(torch.device("cuda"))[0] != 0
        cuda.clear_status(torch.device("cuda"))
        c = torch.zeros(2, 100, dtype=torch.int32, device="cuda")
        for reset in (False, True):
            ops.count_tokens(c, rows.t([[1], [2]], torch.int32), rows.t([1, 1], torch.int32), slots=rows.t([2, -1], torch.int32), reset=reset)
            assert not c.any() and cuda.read_status(torch.device("cuda"))[0] != 0
            cuda.clear_status(torch.device("cuda"))
    finally:
        cuda.clear_status(torch.device("cuda"))


# ----------------------------------------------------------------------------- log-probabilities
@pytest.mark.parametrize("R, V", [(1, 1), (3, 2), (5, 33), (600, 1000), (7, 50257), (1, 151936), (200, 30001), (2, 786432)])
@pytest.mark.parametrize("kind", ["peaked", "flat", "equal", "same", "holes", "one"])
@pytest.mark.parametrize("top", [0, 1, 2, 20, 256])
def test_logprobs_follow_the_definition(R, V, kind, top):
    rows = Rows(R, V, kind, list(TYPES.values())[(R + top) % 3], seed=R, device="cuda", pad=R % 4)
    t = np.where(rows.rs.rand(R) < 0.5, rows.rs.randint(-1, V + 1, R), np.nan_to_num(rows.z, nan=-1e30).argmax(1))
    got = ops.token_logprobs(rows.logits, rows.t(t, torch.int32), top)
    got = [x.cpu().numpy() for x in got]
    for r in range(0, R, 1 + R // 20):
        lp, rank, ids, lps = want_logprobs(rows.z[r], int(t[r]), top)
        assert got[1][r] == rank and got[2][r].tolist() == [int(i) for i in ids]
        near(got[0][r: r + 1], [lp])
        near(got[3][r], lps)
    _sound()


def test_logprobs_of_infinite_logits():
    z = torch.zeros(3, 5000, device="cuda")
    z[0, 7] = z[0, 4000] = float("inf")
    z[1] = float("-inf")
    z[2, :10] = float("nan")
    r = ops.token_logprobs(z, torch.tensor([4000, 3, 2], dtype=torch.int32, device="cuda"), 3)
    assert r.ids.tolist() == [[7, 4000, 0], [-1, -1, -1], [10, 11, 12]] and r.rank.tolist() == [2, 4, 4993]
    near(r.logprob.cpu(), [np.log(0.5), -np.inf, -np.inf])
    near(r.logprobs[0].cpu(), [np.log(0.5), np.log(0.5), -np.inf])


# ----------------------------------------------------------------------------- counts
@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("S, V, P", [(1, 1, 1), (3, 1000, 5000), (16, 151936, 4), (9, 50001, 3000), (300, 77, 60)])
@pytest.mark.parametrize("reset", [False, True])
def test_counts_follow_the_tokens(S, V, P, prompt, reset):
    rs = np.random.RandomState(S)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    slots = rs.permutation(S + 3)[:S]
    slots[rs.rand(S) < 0.2] = -1
    n = rs.randint(-1, P + 3, S)
    tokens = rs.randint(-2, V + 2, (S, P + 5))
    tokens[:, : P // 2] = np.minimum(tokens[:, : P // 2], 3)             # (often the same)
    was = rs.randint(0, 9, (S + 3, V + 2))
    wide = i32(was)
    counts = wide[:, 1: V + 1]
    ops.count_tokens(counts, i32(tokens)[:, :P], i32(n), slots=i32(slots), prompt=prompt, reset=reset)
    want = was.copy()
    for s in range(S):
        if slots[s] < 0:
            continue
        row = want[slots[s], 1: V + 1]
        if reset:
            row[:] = 0
        ids = tokens[s, : min(max(n[s], 0), P)]
        ids = ids[(ids >= 0) & (ids < V)]
        if prompt:
            row[ids] |= 1
        else:
            np.add.at(row, ids, 2)
    assert np.array_equal(wide.cpu().numpy(), want)
    _sound()


# ----------------------------------------------------------------------------- together, on streams, in graphs
def _round(rows, counts, slots, settings, n, tokens):
    """What a round does behind its head: draw with penalties, score, count."""
    a = ops.Adjust(counts=counts, slots=slots, frequency=settings["f"], presence=settings["f"], repetition=settings["r"])
    t = ops.sample_tokens(rows.logits, settings["t"], settings["s"], settings["p"], top_k=settings["k"], top_p=settings["q"], adjust=a)
    lp = ops.token_logprobs(rows.logits, t, 4)
    tokens.copy_(t.view(-1, 1))
    ops.count_tokens(counts, tokens, n, slots=slots)
    settings["p"].add_(1)
    return t, lp


def _settings(rows):
    R = rows.R
    f, i = torch.float32, torch.int32
    return {"f": rows.t(np.full(R, 0.5), f), "r": rows.t(np.full(R, 1.2), f), "t": rows.t(np.full(R, 0.9), f), "s": rows.t(rows.seeds, torch.int64),
            "p": rows.t(rows.positions, torch.int64), "k": rows.t(np.full(R, 50), i), "q": rows.t(np.full(R, 0.9), f)}


def _host_round(rows, counts, settings):
    """The same by the definitions; advances counts and positions."""
    z = rows.z.copy()
    for r in range(rows.R):
        c, seen = counts[r] >> 1, counts[r] > 0
        rep = np.float32(1.2)
        z[r] = np.where(seen, np.where(z[r] > 0, z[r] / rep, z[r] * rep), z[r])
        z[r] = z[r] - np.float32(0.5) * c.astype(np.float32)
        z[r] = z[r] - np.float32(0.5) * (c > 0).astype(np.float32)
    got = rows.want(0.9, top_k=50, top_p=0.9, z=z)
    counts[np.arange(rows.R), got] += 2
    rows.positions = rows.positions + 1
    return got


@pytest.mark.parametrize("captured", [False, True])
def test_rounds_follow_the_definitions(captured):
    """Five rounds of a small vocabulary, where penalties matter; on a stream of their own, captured and replayed with states that move on."""
    rows = Rows(12, 60, "flat", seed=11, device="cuda")
    st = _settings(rows)
    counts = torch.zeros(12, 60, dtype=torch.int32, device="cuda")
    slots = rows.t(np.arange(12), torch.int32)
    n, tokens = rows.t(np.ones(12), torch.int32), torch.zeros(12, 1, dtype=torch.int32, device="cuda")
    ops.count_tokens(counts, rows.t(np.arange(12 * 4).reshape(12, 4), torch.int32), rows.t(np.full(12, 4), torch.int32), prompt=True, reset=True)
    host = counts.cpu().numpy().astype(np.int64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        if captured:
            keep = [x.clone() for x in (counts, st["p"])]
            _round(rows, counts, slots, st, n, tokens)
            counts.copy_(keep[0])
            st["p"].copy_(keep[1])
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                t, lp = _round(rows, counts, slots, st, n, tokens)
        for _ in range(5):
            if captured:
                g.replay()
            else:
                t, lp = _round(rows, counts, slots, st, n, tokens)
            side.synchronize()
            want = _host_round(rows, host, st)
            assert np.array_equal(t.cpu().numpy(), want)
            assert np.array_equal(counts.cpu().numpy(), host)
            for r in range(12):
                near(lp.logprob[r: r + 1].cpu(), [want_logprobs(rows.z[r], int(want[r]), 0)[0]])
    _sound()


def test_two_graphs_and_two_streams_at_once():
    a, b = Rows(30, 40001, seed=1, device="cuda"), Rows(2, 151936, "flat", seed=2, device="cuda")
    s = dict(top_k=40, top_p=0.9)
    want = [a.draw(0.8, **s), b.draw(1.3, top_p=0.95)]
    streams = [torch.cuda.Stream() for _ in range(2)]

    sa, pa = a.t(a.seeds, torch.int64), a.t(a.positions, torch.int64)
    ka, qa = a.t(np.full(30, 40), torch.int32), a.t(np.full(30, 0.9), torch.float32)
    ta = a.t(np.full(30, 0.8), torch.float32)
    sb, pb, tb, qb = b.t(b.seeds, torch.int64), b.t(b.positions, torch.int64), b.t([1.3, 1.3], torch.float32), b.t([0.95, 0.95], torch.float32)
    calls = [lambda: ops.sample_tokens(a.logits, ta, sa, pa, top_k=ka, top_p=qa), lambda: ops.sample_tokens(b.logits, tb, sb, pb, top_p=qb)]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for call, st in zip(calls, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(call())
        graphs.append(g)
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert all(np.array_equal(o.cpu().numpy(), w) for o, w in zip(outs, want))


def test_strided_and_transposed_logits():
    x = torch.randn(700, 6, device="cuda").t()                           # columns apart: copied
    want = x.contiguous()
    t = torch.arange(6, dtype=torch.int32, device="cuda")
    for a, b in zip(ops.token_logprobs(x, t, 3), ops.token_logprobs(want, t, 3)):
        assert torch.equal(a, b)
    one = torch.randn(1, 500, device="cuda").expand(40, 500)             # the same row again and again
    r = ops.token_logprobs(one, torch.arange(40, dtype=torch.int32, device="cuda"), 1)
    assert len(set(r.ids[:, 0].tolist())) == 1 and len(set(r.rank.tolist())) == 40


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("V", [700, 9000, 60000])
def test_masks_of_the_lowest_value(V, dtype):
    """Most of a row (whole stretches of it) masked by the type's lowest finite value, which is a token, if an improbable one."""
    rows = Rows(6, V, "flat", TYPES[dtype], seed=V, device="cuda")
    low = torch.finfo(TYPES[dtype]).min
    x = rows.logits.clone()
    x[:, V // 100: -5] = low
    x[1] = low
    x[2, 1:] = low
    rows.logits, rows.z = x, x.float().cpu().numpy()
    for s in (dict(), dict(top_k=30), dict(top_p=0.7), dict(min_p=0.05), dict(top_k=V - 1, top_p=0.9), dict(top_p=0.999, min_p=0.001)):
        assert np.array_equal(rows.draw(0.8, **s), rows.want(0.8, **s)), s
    t = rows.rs.randint(0, V, 6)
    got = [y.cpu().numpy() for y in ops.token_logprobs(rows.logits, rows.t(t, torch.int32), 5)]
    for r in range(6):
        lp, rank, ids, lps = want_logprobs(rows.z[r], int(t[r]), 5)
        assert got[1][r] == rank and got[2][r].tolist() == [int(i) for i in ids]
        near(np.maximum(got[0][r: r + 1], -3e38), np.maximum([lp], -3e38))
        near(np.maximum(got[3][r], -3e38), np.maximum(lps, -3e38))
    _sound()


# ----------------------------------------------------------------------------- ways through the kernels that sizes above do not take
@pytest.mark.parametrize("R, V", [(300, 170001), (300, 400003), (200, 700001)])
def test_many_long_rows(R, V):
    """More rows than leave several CTAs for each, of more logits than groups of eight are kept for.  (One row under many settings.)"""
    rows = Rows(1, V, "peaked", seed=V, device="cuda", pad=1)
    one = rows.z[0]
    rs = rows.rs
    rows.R, rows.logits, rows.z = R, rows.logits.expand(R, V), np.broadcast_to(one, (R, V))
    rows.seeds, rows.positions = rs.randint(0, 1 << 40, R), rs.randint(0, 1 << 20, R)
    s = dict(top_k=rs.choice([0, 0, 30, 1500, 30000], R), top_p=rs.choice([1.0, 0.6, 0.97], R), min_p=rs.choice([0.0, 0.02], R))
    T = rs.choice([0.0, 0.8, 1.5], R)
    got = rows.draw(T, **s)
    t = rs.randint(0, V, R)
    lp = [x.cpu().numpy() for x in ops.token_logprobs(rows.logits, rows.t(t, torch.int32), 20)]
    for r in range(0, R, 17):
        assert got[r] == want_token(one, T[r], int(rows.seeds[r]), int(rows.positions[r]), int(s["top_k"][r]), s["top_p"][r], s["min_p"][r])
        a, rank, ids, b = want_logprobs(one, int(t[r]), 20)
        assert lp[1][r] == rank and lp[2][r].tolist() == [int(i) for i in ids]
        near(lp[0][r: r + 1], [a])
        near(lp[3][r], b)
    _sound()


@pytest.mark.parametrize("at", [0.0, 0.4, 0.97])
def test_likely_tokens_side_by_side(at):
    """All that is kept lies in one CTA's part of the row: more than its share of the leader's inbox."""
    V = 151936
    rows = Rows(2, V, "flat", seed=3, device="cuda")
    z = rows.z.copy()
    first = int(at * V)
    z[:, first: first + 1700] += 12
    rows.logits, rows.z = rows.t(z, torch.float32), z
    for s in (dict(top_k=1200), dict(top_k=1600, top_p=0.9), dict(top_p=0.95), dict(min_p=1e-3), dict(top_k=200)):
        assert np.array_equal(rows.draw(0.9, **s), rows.want(0.9, **s)), s
    got = ops.token_logprobs(rows.logits, rows.t([first, 5], torch.int32), 256)
    for r in range(2):
        assert got.ids[r].tolist() == [int(i) for i in want_logprobs(z[r], 0, 256)[2]]
    _sound()


def test_scores_next_to_one_another():
    """Thousands of draws among equal logits: in some of them the two best scores are too near for the rough ones."""
    rows = Rows(3000, 500, "same", seed=12, device="cuda")
    for s in (dict(), dict(top_k=100), dict(top_p=0.5), dict(top_k=400, top_p=0.9)):
        assert np.array_equal(rows.draw(1.0, **s), rows.want(1.0, **s)), s
    rows = Rows(400, 20000, "equal", seed=13, device="cuda")
    assert np.array_equal(rows.draw(2.0), rows.want(2.0))
    _sound()


# ----------------------------------------------------------------------------- equal logits that are infinite
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("R, V", [(1, 5000), (1, 60001), (300, 5000)])
def test_ranks_beside_several_infinite_logits(R, V, dtype):
    """Of equal logits the lower id is first, infinite ones too, wherever in the row they are."""
    z = np.random.RandomState(V).randn(V).astype(np.float32)
    at = [0, 7, 1023, 1024, 2047, 4000, V - 1]
    z[at] = np.inf
    x = torch.tensor(z, device="cuda").to(TYPES[dtype]).expand(R, V)
    z = x[0].float().cpu().numpy()
    for t in at + [5, 3000]:
        got = ops.token_logprobs(x, torch.full((R,), t, dtype=torch.int32, device="cuda"), 2)
        lp, rank, ids, lps = want_logprobs(z, t, 2)
        assert got.rank.tolist() == [rank] * R and got.ids.tolist() == [ids] * R
        near(got.logprob.cpu(), [lp] * R)
        near(got.logprobs.cpu(), [lps] * R)
    _sound()


# ----------------------------------------------------------------------------- slots outside the counts
def test_a_slot_outside_the_counts_leaves_a_row_without_penalties():
    """Without any: drafted tokens of the row are not penalised either; its biases and allowed tokens stay."""
    from spark_engine_b200.ops import cuda
    rows = Rows(4, 100, device="cuda")
    i, f = torch.int32, torch.float32
    a = ops.Adjust(counts=torch.full((2, 100), 3, dtype=i, device="cuda"), slots=rows.t([5, -1, 1, 2], i), drafted=rows.t([[3, 3, 60]] * 4, i), repetition=rows.t([1.5] * 4, f),
                   presence=rows.t([0.5] * 4, f), frequency=rows.t([1.0] * 4, f), bias_ids=rows.t([[3, 9]] * 4, i), bias=rows.t([[2.0, -1.0]] * 4, f))
    try:
        got = ops.adjust_logits(rows.logits, a)
        assert cuda.read_status(torch.device("cuda"))[0] != 0
        want = ops.adjust_logits(rows.logits, a._replace(slots=rows.t([-1, -1, 1, -1], i)))
        assert torch.equal(got, want) and not torch.equal(got[2, 10:], rows.logits[2, 10:])
        assert torch.equal(got[0, 10:], rows.logits[0, 10:])
    finally:
        cuda.clear_status(torch.device("cuda"))


# ----------------------------------------------------------------------------- sums that decide
def _borders(z, T, k, n, least):
    """(seed, top_p) of n rows at position 0 whose race has a record at the token that top_p just keeps or just leaves out, as sums are rounded."""
    from spark_engine_b200.spec.sampling import uniform_ref
    from tests.sampling_util import order
    ids = order(z)[:k]
    w = np.exp((z[ids].astype(np.float64) - float(z[ids[0]])) / T)
    before, total = np.cumsum(w) - w, w.sum()
    got, seed = [], 0
    while len(got) < n:
        score = z[ids].astype(np.float64) / T - np.log(-np.log(uniform_ref(seed, 0, len(z)).numpy()[ids]))
        record = np.flatnonzero(score[1:] > np.maximum.accumulate(score)[:-1]) + 1
        got += [(seed, np.float32(before[i] / total)) for i in record if i >= least]
        seed += 1
    return got[:n]


@pytest.mark.parametrize("k, m", [(3000, 0.0), (1500, 0.0), (0, 0.025), (0, 0.0)])
def test_sums_decide_the_same_in_every_batch(k, m):
    """top_p right at the border of a token that wins if it is kept: drawn in one batch of many rows, in batches of few, one by one, and wherever the row begins."""
    V, T, R = 50001, 1.0, 1200
    z = Rows(1, V, "flat", seed=21).z[0]
    n = k or (int((z >= z.max() + T * np.log(m)).sum()) if m else V)
    seeds, p = zip(*_borders(z, T, n, R, 50))
    one = lambda x, d: torch.tensor(np.asarray(x), dtype=d, device="cuda")
    a = dict(temps=one([T] * R, torch.float32), seeds=one(seeds, torch.int64), positions=one([0] * R, torch.int64), top_k=one([k] * R, torch.int32), top_p=one(p, torch.float32),
             min_p=one([m] * R, torch.float32))

    def draws(x, rows, size):
        part = lambda i, j: ops.sample_tokens(x.expand(j - i, V), **{name: y[i:j].contiguous() for name, y in a.items()}).tolist()
        return sum((part(i, min(i + size, rows)) for i in range(0, rows, size)), [])
    every = None
    for shift in range(4):
        x = torch.full((V + 4,), 99.0, device="cuda")[shift: shift + V].unsqueeze(0)
        x.copy_(one(z, torch.float32).unsqueeze(0))
        for rows, size in ((R, R), (R, 200), (R, 60), (R, 8), (100, 1)):
            got = draws(x, rows, size)
            every = every or got
            assert got == every[:rows], (shift, size, sum(g != e for g, e in zip(got, every)))
    _sound()


@pytest.mark.parametrize("V, spread", [(300, 1.0), (4099, 3.0), (50001, 3.0)])
def test_borders_of_short_prefixes_are_the_same_in_every_batch(V, spread):
    """The same where few tokens are kept."""
    T, R = 0.7, 600
    z = (np.random.RandomState(V).randn(V) * spread).astype(np.float32)
    seeds, p = zip(*_borders(z, T, 200, R, 1))
    w = np.exp((np.sort(z.astype(np.float64))[::-1] - float(z.max())) / T)
    p = np.float32(np.asarray(p) * (w[:200].sum() / w.sum()))            # (of the whole row's weight)
    one = lambda x, d: torch.tensor(np.asarray(x), dtype=d, device="cuda")
    f, i = torch.float32, torch.int64
    every = None
    for shift in range(4):
        x = torch.full((V + 4,), 99.0, device="cuda")[shift: shift + V].unsqueeze(0)
        x.copy_(one(z, f).unsqueeze(0))
        for size in (R, 40, 1):
            got = sum((ops.sample_tokens(x.expand(len(seeds[j: j + size]), V), one([T] * len(seeds[j: j + size]), f), one(seeds[j: j + size], i), one([0] * len(seeds[j: j + size]), i),
                                         top_p=one(p[j: j + size], f)).tolist() for j in range(0, R if size > 1 else 100, size)), [])
            every = every or got
            assert got == every[: len(got)], (shift, size, sum(g != e for g, e in zip(got, every)))
    _sound()


# ----------------------------------------------------------------------------- launches
def test_only_kernels_that_run_are_counted():
    from spark_engine_b200.ops import cuda as cu
    i = torch.int32
    c, n = torch.zeros(2, 9, dtype=i, device="cuda"), torch.zeros(2, dtype=i, device="cuda")

    def launches(f):
        cu.reset_launch_count()
        f()
        return cu.launch_count()
    assert launches(lambda: ops.count_tokens(c, c[:, :0], n)) == 0 and launches(lambda: ops.count_tokens(c, c[:0, :3], n[:0])) == 0
    assert launches(lambda: ops.count_tokens(c, c[:, :0], n, reset=True)) == 1 and launches(lambda: ops.count_tokens(c, c[:, :3].clone(), n)) == 1
    x = torch.zeros(0, 9, device="cuda")
    assert launches(lambda: ops.adjust_logits(x, ops.Adjust())) == 0 and launches(lambda: ops.token_logprobs(x, n[:0], 2)) == 0


# ----------------------------------------------------------------------------- cold rows
@pytest.mark.parametrize("R", [1, 40, 300])
@pytest.mark.parametrize("bias", [0.0, 100.0])
def test_cold_rows_with_top_k(R, bias):
    """The k-th token weighs less than 2^-64 of the first: at low temperatures, or beside a strong bias."""
    V = 151936
    rows = Rows(3, V, "peaked", seed=R, device="cuda")
    if bias:
        rows.logits[:, 777] += bias
        rows.z = rows.logits.cpu().numpy()
    z = rows.z
    rows.logits, rows.z, rows.R = rows.logits.repeat(-(-R // 3), 1)[:R].contiguous(), np.tile(z, (-(-R // 3), 1))[:R], R
    rows.seeds, rows.positions = rows.rs.randint(0, 1 << 40, R), rows.rs.randint(0, 1 << 20, R)
    T = rows.rs.choice([0.7] if bias else [0.05, 0.1, 0.2], R)
    s = dict(top_k=rows.rs.choice([20, 40, 64, 3000], R), top_p=rows.rs.choice([1.0, 0.9], R), min_p=rows.rs.choice([0.0, 1e-25], R))
    got = rows.draw(T, **s)
    for r in range(0, R, 1 + R // 40):
        assert got[r] == want_token(rows.z[r], T[r], int(rows.seeds[r]), int(rows.positions[r]), int(s["top_k"][r]), s["top_p"][r], s["min_p"][r])
    _sound()
