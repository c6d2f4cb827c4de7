"""The operators between a round's logits and its tokens on the host: their plain forms against the definitions, and what they refuse."""
import numpy as np
import pytest
import torch

from spark_engine_b200 import ops
from spark_engine_b200.ops import sampling
from spark_engine_b200.spec.sampling import sample
from tests.sampling_util import Rows, Table, near, want_logprobs

SETTINGS = [dict(), dict(top_k=5), dict(top_p=0.8), dict(min_p=0.1), dict(top_k=7, top_p=0.5, min_p=0.01), dict(top_k=1), dict(top_p=0.0), dict(min_p=1.0),
            dict(min_p=3.0), dict(top_k=-1, top_p=1.0, min_p=0.0), dict(top_k=10**6, top_p=0.999999)]


@pytest.mark.parametrize("kind", ["peaked", "flat", "equal", "same", "holes", "one"])
@pytest.mark.parametrize("V", [1, 2, 33, 1000])
def test_draws_follow_the_definition(kind, V):
    rows = Rows(5, V, kind, seed=V)
    for s in SETTINGS:
        for T in (0.7, 0.0, 2.5):
            assert np.array_equal(rows.draw(T, **s), rows.want(T, **s)), (s, T)


def test_without_filters_it_is_the_token_of_perturbed_logits():
    rows = Rows(20, 500, "flat")
    got = rows.draw(0.9)
    for r in range(20):
        assert got[r] == sample(rows.logits[r], 0.9, int(rows.seeds[r]), int(rows.positions[r]))


def test_draws_have_the_kept_tokens_probabilities():
    """40000 draws from six tokens: shares within five standard deviations."""
    z = np.log(np.array([0.4, 0.05, 0.25, 0.1, 0.15, 0.05]))
    n = 40000
    rows = Rows(1, 6)
    rows.logits = torch.tensor(z, dtype=torch.float32).expand(200, 6)
    share = np.zeros(6)
    for i in range(n // 200):
        got = ops.sample_tokens(rows.logits, torch.ones(200), torch.full((200,), 3), torch.arange(200) + 200 * i, top_p=torch.full((200,), 0.75))
        share += np.bincount(got.numpy(), minlength=6)
    want = np.array([0.4, 0, 0.25, 0, 0.15, 0]) / 0.8
    assert (share[want == 0] == 0).all()
    assert (np.abs(share / n - want) <= 5 * np.sqrt(want * (1 - want) / n) + 1e-12).all()


def test_rows_of_nothing_and_of_infinities():
    z = torch.tensor([[-np.inf, np.nan, -np.inf], [1.0, np.inf, np.inf], [3.0, np.nan, 4.0], [0.0, -0.0, -np.inf]])
    one = torch.ones(4)
    seeds = torch.zeros(4, dtype=torch.int64)
    assert ops.sample_tokens(z, one * 0, seeds, seeds).tolist() == [-1, 1, 2, 0]
    got = ops.sample_tokens(z, one, seeds, seeds, top_k=torch.ones(4, dtype=torch.int32))
    assert got.tolist() == [-1, 1, 2, 0]
    r = ops.token_logprobs(z, torch.tensor([0, 2, 1, 3], dtype=torch.int32), top=3)
    assert r.ids.tolist() == [[-1, -1, -1], [1, 2, 0], [2, 0, -1], [0, 1, -1]] and r.rank.tolist() == [1, 2, 3, 0]
    near(r.logprob, [-np.inf, np.log(0.5), -np.inf, -np.inf])


@pytest.mark.parametrize("kind", ["peaked", "equal", "holes", "one"])
def test_logprobs_follow_the_definition(kind):
    rows = Rows(9, 257, kind, seed=3)
    t = rows.rs.randint(-1, 258, 9)
    for top in (0, 1, 20):
        got = ops.token_logprobs(rows.logits, rows.t(t, torch.int32), top)
        for r in range(9):
            lp, rank, ids, lps = want_logprobs(rows.z[r], int(t[r]), top)
            assert got.rank[r] == rank and got.ids[r].tolist() == ids
            near(got.logprob[r: r + 1], [lp])
            near(got.logprobs[r], lps)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_adjustments_follow_the_definition(dtype):
    rows = Rows(12, 301, dtype=dtype, seed=1)
    table = Table(rows, per=3, drafts=3, biases=9, allowed=0.5, dup=True)
    want, tol = table.want()
    got = ops.adjust_logits(rows.logits, table.adjust()).double().numpy()
    assert np.array_equal(np.isfinite(got), np.isfinite(want))
    fine = np.isfinite(want)
    assert (np.abs(got[fine] - want[fine]) <= tol[fine]).all()


def test_slices_of_a_vocabulary_are_adjusted_alike():
    rows = Rows(6, 300, seed=2)
    table = Table(rows, drafts=2, biases=20)
    a = table.adjust()
    whole = ops.adjust_logits(rows.logits, a)
    parts = []
    for o, n in ((0, 130), (130, 170)):
        part = ops.Adjust(counts=a.counts[:, o: o + n], slots=a.slots, drafted=a.drafted, repetition=a.repetition, presence=a.presence, frequency=a.frequency,
                          bias_ids=a.bias_ids, bias=a.bias)
        parts.append(ops.adjust_logits(rows.logits[:, o: o + n], part, offset=o))
    assert torch.equal(torch.cat(parts, 1), whole)


def test_counts_follow_the_tokens():
    counts = torch.full((4, 10), 99, dtype=torch.int32)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)
    ops.count_tokens(counts, i32([3, 3, 9, 12, -1], [1, 2, 3, 4, 5]), i32(5, 2), slots=i32(2, -1), prompt=True, reset=True)
    assert counts[2].tolist() == [0, 0, 0, 1, 0, 0, 0, 0, 0, 1] and (counts[[0, 1, 3]] == 99).all()
    ops.count_tokens(counts, i32([3, 4, 4]), i32(7), slots=i32(2))
    assert counts[2].tolist() == [0, 0, 0, 3, 4, 0, 0, 0, 0, 1]
    ops.count_tokens(counts, i32([0, 0, 0]), i32(0), slots=i32(2))
    ops.count_tokens(counts, i32([0, 0, 0]), i32(-3), slots=i32(2))
    assert counts[2, 0] == 0


def test_a_rounds_calls_together():
    """Counted, adjusted, drawn, scored: the fused draw is the draw from adjusted logits."""
    rows = Rows(8, 200, seed=5)
    table = Table(rows, per=4, drafts=3, biases=5, allowed=0.6)
    a = table.adjust()
    z = ops.adjust_logits(rows.logits, a)
    got = rows.draw(0.8, top_k=20, top_p=0.9, adjust=a)
    assert np.array_equal(got, rows.want(0.8, top_k=20, top_p=0.9, z=z.numpy()))
    lp = ops.token_logprobs(rows.logits, rows.t(got, torch.int32), 2)
    assert (lp.rank[got >= 0] > 0).all() and (lp.rank[got < 0] == 0).all()


# ----------------------------------------------------------------------------- refusals
def _args(R=2, V=8):
    return dict(logits=torch.zeros(R, V), temps=torch.ones(R), seeds=torch.zeros(R, dtype=torch.int64), positions=torch.zeros(R, dtype=torch.int64))


@pytest.mark.parametrize("bad, what", [
    (dict(logits=torch.zeros(2, 8, dtype=torch.float64)), "fp32, bf16 or fp16"), (dict(logits=torch.zeros(8)), r"\[rows, vocabulary\]"),
    (dict(logits=torch.zeros(2, 0)), "1 to"), (dict(logits=torch.zeros(1, 1).expand(2, 800000)), "1 to"), (dict(logits=torch.zeros(1, 8).expand(70000, 8)), "at most"),
    (dict(temps=torch.ones(3)), "temps"), (dict(temps=torch.ones(2, dtype=torch.float64)), "temps"), (dict(seeds=torch.zeros(2, dtype=torch.int32)), "seeds"),
    (dict(positions=torch.zeros(2, 1, dtype=torch.int64)), "positions"), (dict(top_k=torch.zeros(2)), "top_k"), (dict(top_p=torch.ones(4)[::2]), "top_p"),
    (dict(min_p=torch.ones(1)), "min_p"),
])
def test_draws_refuse(bad, what):
    with pytest.raises(ValueError, match=what):
        ops.sample_tokens(**{**_args(), **bad})


@pytest.mark.parametrize("bad, what", [
    (dict(counts=torch.zeros(2, 7, dtype=torch.int32)), "counts"), (dict(counts=torch.zeros(2, 8)), "counts"), (dict(counts=torch.zeros(1, 8, dtype=torch.int32)), "slots"),
    (dict(counts=torch.zeros(1, 8, dtype=torch.int32).expand(2, 8)), "apart"), (dict(slots=torch.zeros(3, dtype=torch.int32)), "slots"),
    (dict(drafted=torch.zeros(2, dtype=torch.int32)), "drafted"), (dict(drafted=torch.zeros(2, 2000, dtype=torch.int32)), "at most"),
    (dict(repetition=torch.ones(3)), "repetition"), (dict(bias=torch.ones(2, 1)), "belong together"),
    (dict(bias=torch.ones(2, 1), bias_ids=torch.zeros(2, 2, dtype=torch.int32)), "same shape"), (dict(allowed=torch.zeros(2, 2, dtype=torch.int32)), "allowed"),
    (dict(allowed=torch.zeros(2, 1, dtype=torch.int64)), "allowed"),
])
def test_adjustments_refuse(bad, what):
    with pytest.raises(ValueError, match=what):
        ops.adjust_logits(torch.zeros(2, 8), ops.Adjust(**bad))


def test_outputs_refuse():
    x = torch.zeros(4, 8)
    for out in (torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(4, 9), torch.zeros(8, 4).t(), torch.zeros(1, 8).expand(4, 8)):
        with pytest.raises(ValueError, match="out must be"):
            ops.adjust_logits(x, ops.Adjust(), out=out)
    both = torch.zeros(40)
    with pytest.raises(ValueError, match="share no memory"):
        ops.adjust_logits(both[:32].view(4, 8), ops.Adjust(), out=both[4:36].view(4, 8))
    with pytest.raises(ValueError, match="31 bits"):
        ops.adjust_logits(x, ops.Adjust(), offset=2**31 - 4)
    assert ops.adjust_logits(x, ops.Adjust(), out=x) is x
    with pytest.raises(ValueError, match="top must be"):
        ops.token_logprobs(x, torch.zeros(4, dtype=torch.int32), 257)
    with pytest.raises(ValueError, match="tokens"):
        ops.token_logprobs(x, torch.zeros(4, dtype=torch.int64), 1)


def test_counts_refuse():
    c, i32 = torch.zeros(2, 8, dtype=torch.int32), torch.int32
    for bad in (dict(counts=c.float()), dict(counts=c.t()), dict(tokens=torch.zeros(2, 3)), dict(tokens=torch.zeros(3, dtype=i32)), dict(n=torch.zeros(3, dtype=i32)),
                dict(slots=torch.zeros(1, dtype=i32)), dict(tokens=torch.zeros(3, 3, dtype=i32), n=torch.zeros(3, dtype=i32))):
        with pytest.raises(ValueError):
            ops.count_tokens(**{**dict(counts=c, tokens=torch.zeros(2, 3, dtype=i32), n=torch.zeros(2, dtype=i32)), **bad})
    with pytest.raises(ValueError, match="slot"):
        ops.count_tokens(c, torch.zeros(1, 1, dtype=i32), torch.ones(1, dtype=i32), slots=torch.full((1,), 2, dtype=i32))


def test_empty_calls():
    x = torch.zeros(0, 8)
    e = torch.zeros(0, dtype=torch.int64)
    assert ops.sample_tokens(x, torch.zeros(0), e, e).shape == (0,)
    assert ops.adjust_logits(x, ops.Adjust()).shape == (0, 8)
    r = ops.token_logprobs(x, torch.zeros(0, dtype=torch.int32), 3)
    assert r.ids.shape == (0, 3) and r.logprob.shape == (0,)


def test_kernels_of_other_sources_are_refused():
    from spark_engine_b200 import build
    mod = sampling._native()
    flag, = build._sampling_layout()
    assert f"={mod.layout()}u" in flag and mod.layout() != 0

    class Lib:
        _name = "libother.so"

    class Fn:
        def __init__(self, value):
            self.value = value

        def __call__(self):
            return self.value
    dll = Lib()
    with pytest.raises(RuntimeError, match="no sampling kernels"):
        sampling._same_layout(mod, dll)
    dll.spark_sampling_layout = Fn(mod.layout() ^ 1)
    with pytest.raises(RuntimeError, match="different sources"):
        sampling._same_layout(mod, dll)


@pytest.mark.parametrize("V, P", [(2**30 + 1, 4), (2**31 - 1, 4), (8, 2**30 + 1), (8, 2**31 - 1)])
def test_counts_refuse_what_32_bit_places_do_not_reach(V, P):
    """A CTA's steps through tokens and columns go beyond their number by up to some thousands."""
    none = lambda *s: torch.empty(*s, dtype=torch.int32, device="meta")
    with pytest.raises(ValueError, match=r"2\^30"):
        ops.count_tokens(none(2, V), none(1, P), none(1))
