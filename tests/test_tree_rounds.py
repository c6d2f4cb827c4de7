"""Drafted trees over paged caches in whole models: every node's logits are those of its path, accepted paths are committed, speculative rounds
are lossless (CPU; on a B200 in bf16 and 32-bit)."""
import debisun_util as U
import pytest
import torch

from spark_engine_b200.models.plan import make_plan
from spark_engine_b200.spec.decoder import SpecDecoder
from spark_engine_b200.spec.tree import Node

CONFIGS = {
    "mixed layers": U.MIXED,
    "dense": dict(layers=[U.layer(U.dense()), U.layer(U.dense(), heads=8, kv_heads=2, dim=64, vdim=32, conv=2, chunk=64)]),
    "one tap": dict(layers=[U.layer(U.dense(), conv=1, chunk=1000), U.layer(conv=7)]),
}
TREE = [-1, 0, 0, 1, 1, 2, 3, 6, 4, -1, 9, 5]          # the last sampled token, drafts below it, and one more root with a draft of its own


def setup(name):
    cfg = U.config(**CONFIGS[name])
    return cfg, U.tensors(cfg)


def path(parents, j):
    line = []
    while j >= 0:
        line.append(j)
        j = parents[j]
    return line[::-1]


def check_nodes_and_commits(name, device, dtype, agree):
    cfg, T = setup(name)
    g = torch.Generator().manual_seed(3)
    tok = lambda n: torch.randint(0, cfg["vocab"], (n,), generator=g).tolist()
    m = U.framework(cfg, T, device, dtype)
    assert m.sparse_ctx_limit() is None
    prompts = {2: tok(61), 0: tok(130)}
    for slot, p in prompts.items():
        m.forward(make_plan([(slot, p, 0)], device=device, all_logits=False))
    said = dict(prompts)
    for rnd, accepted in enumerate((([0, 1, 3, 6], [0]), ([0, 2, 5, 11], [0, 1, 4, 8]), ([9, 10], []))):
        trees = [tok(len(TREE)), tok(9)]
        plan = make_plan([(s, t, len(said[s])) for s, t in zip(said, trees)], device=device, parents=[TREE, TREE[:9]])
        got = m.forward(plan, commit=False).float().cpu()
        for seg, t, par in zip(plan.segs, trees, (TREE, TREE[:9])):
            for j in range(rnd % 2, seg.n, 2):
                line = path(par, j)
                want = U.oracle_logits(cfg, T, said[seg.slot] + [t[i] for i in line])[-1]
                agree(got[seg.r0 + j: seg.r0 + j + 1], want.unsqueeze(0), cfg)
        m.commit([list(a) for a in accepted])
        for s, t, a in zip(list(said), trees, accepted):
            said[s] = said[s] + [t[j] for j in a]
        assert [m.seqs[s].length for s in said] == [len(x) for x in said.values()]
    # what was committed is what a chain would have left: rows of both sequences go on behind it, and a chain's rows are verified again
    nxt = {s: tok(3) for s in said}
    plan = make_plan([(s, nxt[s], len(said[s])) for s in said], device=device)
    got = m.forward(plan, commit=False).float().cpu()
    for seg in plan.segs:
        agree(got[seg.r0: seg.r0 + 3], U.oracle_logits(cfg, T, said[seg.slot] + nxt[seg.slot])[-3:], cfg)
    m.commit([[0, 1], [0]])


def check_rounds(name, device, dtype):
    """Rounds over trees emit what plain greedy decoding of the same model does, in fewer rounds."""
    cfg, T = setup(name)
    prompt = U.prompt(70, cfg["vocab"])
    ref = SpecDecoder(U.framework(cfg, T, device, dtype), lambda s, d: ([], []), depth=0).generate([prompt], 16)[0]
    m = U.framework(cfg, T, device, dtype)
    sd = SpecDecoder(m, lambda s, d: ([], []), depth=0)
    seq = sd.start(1, prompt)
    rounds = 0
    while len(seq.generated) < 16:
        n = len(seq.generated)
        nodes, parent = [], -1
        for t in ref[n: n + 4]:                          # a wrong draft in front of every right one, and one below it
            nodes.append(Node(parent, (t + 1) % cfg["vocab"]))
            nodes.append(Node(parent, t))
            nodes.append(Node(len(nodes) - 2, t))
            parent = len(nodes) - 2
        sd.round_tree([seq], [nodes], budgets=[16 - n])
        rounds += 1
    return ref, seq, rounds


def close(got, want, cfg):
    assert U.error(got, want) < 3e-5


@pytest.mark.parametrize("name", list(CONFIGS))
def test_nodes_see_their_paths(name):
    check_nodes_and_commits(name, "cpu", torch.float32, close)


@pytest.mark.parametrize("name", list(CONFIGS))
def test_tree_rounds_are_lossless(name):
    ref, seq, rounds = check_rounds(name, "cpu", torch.float32)
    assert seq.generated[:16] == ref and rounds <= 5 and seq.accepted >= 10


def test_models_with_other_layers_verify_chains():
    import zapolorn_util as Z
    cfg = Z.config(**Z.MIXED) if not isinstance(Z.MIXED, list) else Z.config(Z.MIXED)
    assert Z.framework(cfg, Z.tensors(cfg)).sparse_ctx_limit() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", list(CONFIGS))
def test_nodes_see_their_paths_on_the_device(name, dtype):
    """bf16 of models with experts: rows whose choice of experts is close may differ by an expert (see test_debisun_gpu); the dense ones are held."""
    def agree(got, want, cfg):
        if dtype == torch.float32:
            assert U.error(got, want) < 3e-5
        elif name != "mixed layers":
            assert U.error(got, want) < 3e-2 * len(cfg["layers"]) ** 0.5
        assert torch.isfinite(got).all()
    check_nodes_and_commits(name, "cuda", dtype, agree)


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(CONFIGS))
def test_tree_rounds_are_lossless_on_the_device(name):
    ref, seq, rounds = check_rounds(name, "cuda", torch.float32)
    assert seq.generated[:16] == ref and rounds <= 5 and seq.accepted >= 10


# ----------------------------------------------------------------------------- trees that are chains
def _family(name):
    import vabunex_util as VU
    import zakusun_util as KU
    import zapolorn_util as ZU
    from test_vabunex import MIXED as vabunex
    u, layers = {"debisun": (U, U.MIXED), "vabunex": (VU, vabunex), "zakusun": (KU, KU.MIXED), "zapolorn": (ZU, ZU.MIXED)}[name]
    cfg = u.config(**layers)
    return u, cfg, u.tensors(cfg)


def check_chains(name, device):
    """A plan whose trees are chains is verified and committed by every paged model as the plan without parents is."""
    u, cfg, T = _family(name)
    g = torch.Generator().manual_seed(4)
    toks = {s: torch.randint(0, cfg["vocab"], (n,), generator=g).tolist() for s, n in ((1, 70), (2, 20))}
    got = []
    for parents in (None, [[-1, 0, 1, 2], [-1, 0]], [None, [-1, 0]]):
        m = u.framework(cfg, T, device)
        for s, t in toks.items():
            m.forward(make_plan([(s, t[:-12], 0)], device=device, all_logits=False))
        outs, at = [], {s: len(t) - 12 for s, t in toks.items()}
        for accepted in ([[0, 1], [0]], [[0, 1, 2], [0, 1]], [[], [0]]):
            plan = make_plan([(s, t[at[s]: at[s] + n], at[s]) for (s, t), n in zip(toks.items(), (4, 2))], device=device, parents=parents)
            outs.append(m.forward(plan, commit=False).float().cpu())
            m.commit([list(a) for a in accepted])
            for s, a in zip(toks, accepted):
                at[s] += len(a)
            assert [m.seqs[s].length for s in toks] == list(at.values())
        got.append(torch.cat(outs))
    for x in got[1:]:
        assert U.error(x, got[0]) < 1e-6


@pytest.mark.parametrize("name", ["debisun", "vabunex", "zakusun", "zapolorn"])
def test_trees_that_are_chains(name):
    check_chains(name, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["debisun", "vabunex", "zakusun", "zapolorn"])
def test_trees_that_are_chains_on_the_device(name):
    check_chains(name, "cuda")


def test_branches_are_refused_where_rows_verify_chains():
    u, cfg, T = _family("zapolorn")
    m = u.framework(cfg, T)
    m.forward(make_plan([(0, [1, 2, 3], 0)], all_logits=False))
    with pytest.raises(AssertionError):
        m.forward(make_plan([(0, [4, 5, 6], 3)], parents=[[-1, 0, 0]]), commit=False)


@pytest.mark.parametrize("kind", ["trees", "chains"])
@pytest.mark.parametrize("extra", [3, 4, 7])
def test_rounds_up_to_the_last_row(kind, extra):
    """A sequence is generated to the end of its pages: drafts that its cache has no rows for are left out."""
    from spark_engine_b200.cache.kv import KvManager
    cfg, T = setup("dense")
    prompt = U.prompt(64 - extra, cfg["vocab"])
    want = SpecDecoder(U.framework(cfg, T), lambda s, d: ([], []), depth=0).generate([prompt], extra + 1)[0]
    m = U.framework(cfg, T)
    assert KvManager(m).assign(1, 64) and m.seqs[1].kv_cap == 64
    sd = SpecDecoder(m, lambda s, d: ([1, 2, 3][:d], [0.9] * min(3, d)), depth=3)
    seq = sd.start(1, prompt)
    while len(seq.generated) < extra + 1:
        left = [extra + 1 - len(seq.generated)]
        if kind == "chains":
            sd.round([seq], left)
        else:
            t = (want[len(seq.generated):] + [1])[0]
            sd.round_tree([seq], [[Node(-1, (t + 1) % cfg["vocab"]), Node(-1, t), Node(0, 3), Node(1, 4), Node(2, 5)]], left)
    assert seq.generated[: extra + 1] == want and m.seqs[1].length <= 64


# ----------------------------------------------------------------------------- the server
class _Guesses:
    """Candidates with the right token best or second best in turn: leaves beside the spine, and down it, are accepted and turned down."""

    def __init__(self, server, texts, vocab):
        self.server, self.texts, self.vocab = server, texts, vocab

    def __call__(self, seq, depth):
        return [], []

    def candidates(self, seq):
        from spark_engine_b200.spec.drafters import Candidates
        i, n = self.server.by_slot[seq.slot].id, len(seq.generated)
        right = (self.texts[i][n: n + 3] + [0, 0, 0])[:3]
        ids = torch.tensor([[(t + 7 + a) % self.vocab if a != (n % 2, 0, 1)[j] else t for a in range(4)] for j, t in enumerate(right)])
        return Candidates(ids=ids, unary=torch.tensor([[4.0, 3.0, 2.0, 1.0]] * 3), edges=torch.zeros(2, 4, 4), path=[0, 0, 0], conf=[0.9] * 3)


def check_server(device):
    """Requests through admission, shared rounds of trees, more requests than slots, prompts and ends at page borders, a continued conversation: the
    text is that of plain decoding."""
    from spark_engine_b200.config import EngineConfig
    from spark_engine_b200.serving.worker import EngineServer
    from test_vabunex import _serve
    cfg, T = setup("dense")
    mc = U.D.read_config(cfg)
    es = EngineServer(mc, U.D.from_tensors(mc, T, device, torch.float32), EngineConfig(max_seqs=2, kv_tokens=1024, prefill_chunk=48, spec="lookup", spec_depth=3,
                                                                                     spec_tree_widths="3,2,2", dtype="float32"), device=device)
    prompts = {i: U.prompt(n, cfg["vocab"], n) for i, n in enumerate((41, 52, 116, 3, 128))}
    texts = {i: U.oracle_greedy(cfg, T, p, 12) for i, p in prompts.items()}
    es.spec.drafter = _Guesses(es, texts, cfg["vocab"])
    done = _serve(es, [{"id": i, "prompt_ids": p, "max_new": 12} for i, p in prompts.items()])
    for i in prompts:
        assert done[i]["token_ids"] == texts[i], i
    p = prompts[0] + done[0]["token_ids"] + [1, 2]
    texts[9] = U.oracle_greedy(cfg, T, p, 9)
    assert _serve(es, [{"id": 9, "prompt_ids": p, "max_new": 9}])[9]["token_ids"] == texts[9]
    assert 0 < es.totals["accepted_drafts"] < es.totals["drafted_tokens"]


def test_server_with_trees():
    check_server("cpu")


@pytest.mark.gpu
def test_server_with_trees_on_the_device():
    check_server("cuda")
