"""Requests with filters, penalties, biases and log-probabilities: in speculative rounds, the server and its HTTP front end, over a sharded vocabulary."""
import json
import threading
import urllib.error
import urllib.request

import numpy as np
import pytest
import torch

from spark_engine_b200.config import EngineConfig, tiny_hybrid
from spark_engine_b200.models.model import Model
from spark_engine_b200.models.weights import init_weights, to_device
from spark_engine_b200.serving.protocol import validate_request
from spark_engine_b200.serving.worker import EngineServer
from spark_engine_b200.spec.decoder import SpecDecoder
from spark_engine_b200.spec.params import SamplingParams
from spark_engine_b200.spec.tree import Node
from tests.sampling_util import want_logprobs, want_token

WILD = SamplingParams(temperature=1.1, seed=5, top_k=40, top_p=0.9, min_p=0.01, repetition=1.3, presence=0.4, frequency=0.2, bias=((7, 3.0), (9, -100.0)), logprobs=3)
SETTINGS = [WILD, SamplingParams(temperature=0.9, seed=8, top_p=0.7), SamplingParams(frequency=1.5, logprobs=0), SamplingParams(temperature=1.3, seed=2)]


def _model(device="cpu", slots=4):
    cfg = tiny_hybrid()
    cfg.mtp_layers, cfg.mtp_depth = 1, 3
    W = init_weights(cfg, seed=0)
    if device != "cpu":
        W = to_device(W, device)
    return cfg, W, Model(cfg, W, device=device, dtype=torch.float32 if device == "cpu" else torch.bfloat16, n_slots=slots, kv_tokens=512 * slots)


def _prompts(cfg, n, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, cfg.vocab, (20 + 9 * i,), generator=g).tolist() for i in range(n)]


def _text(sd, prompts, params, n):
    """Every sequence with settings of its own, n tokens each, and their log-probabilities."""
    seqs = [sd.start(i, p, params=q) for i, (p, q) in enumerate(zip(prompts, params))]
    lps = [list(s.logprobs) for s in seqs]
    while any(len(s.generated) < n for s in seqs):
        live = [s for s in seqs if len(s.generated) < n]
        sd.round(live, [n - len(s.generated) for s in live])
        for s in live:
            lps[seqs.index(s)] += s.logprobs
    return [s.generated for s in seqs], lps


def _by_definition(z, p, seed_pos, prompt, said):
    """Next token from fp32 logits `z` of a row behind prompt + said."""
    z = z.copy()
    f = np.float32
    c = np.bincount(said, minlength=len(z)) if said else np.zeros(len(z), int)
    seen = c > 0
    seen[prompt] = True
    z = np.where(seen, np.where(z > 0, z / f(p.repetition), z * f(p.repetition)), z)
    z = z - f(p.frequency) * c.astype(f) - f(p.presence) * (c > 0).astype(f)
    for t, b in p.bias:
        z[t] += f(b)
    return want_token(z, p.temperature, p.seed, seed_pos, p.top_k, p.top_p, p.min_p)


def test_plain_rounds_draw_by_the_definitions(monkeypatch):
    """One row at a time: every token is the definition's, from the row's own logits and what the request has said."""
    cfg, _, m = _model()
    prompts = _prompts(cfg, 4)
    rows = []
    real = m.draw_rows
    monkeypatch.setattr(m, "draw_rows", lambda lg, *a: rows.append((lg.float().reshape(-1, cfg.vocab).numpy().copy(), a)) or real(lg, *a))
    texts, lps = _text(SpecDecoder(m, lambda s, d: ([], []), depth=0), prompts, SETTINGS, 12)
    logits = {(s, pos): z for lg, (_, slots, positions, *_) in rows for z, s, pos in zip(lg, slots, positions)}
    for i, (p, text) in enumerate(zip(SETTINGS, texts)):
        if not p.shaped:
            continue
        for j, t in enumerate(text):
            z = logits[i, len(prompts[i]) + j]
            assert t == _by_definition(z, p, len(prompts[i]) + j, prompts[i], text[:j]), (i, j)
            if p.logprobs >= 0:
                lp, rank, ids, top = want_logprobs(z, t, p.logprobs)
                got = lps[i][j]
                assert got[1] == rank and [a for a, _ in got[2]] == [int(a) for a in ids]
                assert abs(got[0] - lp) < 1e-5 and all(abs(x - y) < 1e-5 for (_, x), y in zip(got[2], top))
        assert len(lps[i]) == (len(text) if p.logprobs >= 0 else 0)
    assert len(set(map(tuple, texts))) == 4


def check_speculation(device, graphs):
    """Drafts (right, half right, none; chains and trees) change nothing about the text."""
    cfg, W, m = _model(device)
    prompts = _prompts(cfg, 4)
    want, want_lps = _text(SpecDecoder(m, lambda s, d: ([], []), depth=0), prompts, SETTINGS, 14)
    by_slot = dict(enumerate(want))

    def drafter(seq, depth):
        d = by_slot[seq.slot][len(seq.generated): len(seq.generated) + depth]
        if seq.slot == 1:
            d = d[:1] + [(t + 1) % cfg.vocab for t in d[1:]]
        return d, [0.9] * len(d)
    _, _, m2 = _model(device)
    sd = SpecDecoder(m2, drafter, depth=3, graphs=graphs)
    got, lps = _text(sd, prompts, SETTINGS, 14)
    assert got == want and sd.rounds < 14
    assert bool(sd.graphs is not None and sd.graphs.rounds) == graphs
    for a, b in zip(lps, want_lps):
        assert [x[1] for x in a] == [x[1] for x in b]
    if graphs:
        return
    _, _, m3 = _model(device)
    sd = SpecDecoder(m3, lambda s, d: ([], []), depth=0)
    seqs = [sd.start(i, p, params=q) for i, (p, q) in enumerate(zip(prompts, SETTINGS))]
    while any(len(s.generated) < 14 for s in seqs):
        live = [s for s in seqs if len(s.generated) < 14]
        trees = []
        for s in live:
            right = (want[s.slot][len(s.generated): len(s.generated) + 2] + [0, 0])[:2]
            wrong = (right[0] + 1) % cfg.vocab
            trees.append([Node(token=t, parent=a) for t, a in ((wrong, -1), (right[0], -1), (right[1], 0), (right[1], 1))])
        sd.round_tree(live, trees, [14 - len(s.generated) for s in live])
    assert [s.generated for s in seqs] == want


def test_speculation_keeps_the_text():
    check_speculation("cpu", False)


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [False, True])
def test_speculation_keeps_the_text_on_the_device(graphs):
    check_speculation("cuda", graphs)


# ----------------------------------------------------------------------------- the server
def _message(i, prompt, p, n):
    return {"id": i, "prompt_ids": prompt, "max_new": n, "temperature": p.temperature, "seed": p.seed, "top_k": p.top_k, "top_p": p.top_p, "min_p": p.min_p,
            "repetition_penalty": p.repetition, "presence_penalty": p.presence, "frequency_penalty": p.frequency, "logit_bias": [list(b) for b in p.bias], "logprobs": p.logprobs}


def check_server(device):
    """More requests than slots, shared rounds: the text and log-probabilities are those of a request alone."""
    cfg, W, m = _model(device)
    prompts = _prompts(cfg, 4)
    alone, alone_lps = [], []
    for p, q in zip(prompts, SETTINGS):
        t, lp = _text(SpecDecoder(m, lambda s, d: ([], []), depth=0), [p], [q], 10)
        alone += t
        alone_lps += lp
    es = EngineServer(cfg, W, EngineConfig(max_seqs=2, kv_tokens=2048, prefill_chunk=32, spec="mtp", spec_depth=2, cuda_graphs=device != "cpu"), device=device)
    for turn in range(2):                                                # (the second time over used slots and kept prefixes)
        for i, (p, q) in enumerate(zip(prompts, SETTINGS)):
            es.submit(_message(10 * turn + i, p, q, 10))
        while es.sched.has_work():
            es.step()
        out, es.out = es.out, []
        for i, q in enumerate(SETTINGS):
            mine = [x for x in out if x.get("id") == 10 * turn + i]
            assert [x for x in mine if x.get("done")][0]["token_ids"] == alone[i], (turn, i)
            got = sum((x.get("logprobs", []) for x in mine if "delta" in x), [])
            assert len(got) == len(alone_lps[i]) and [x[1] for x in got] == [x[1] for x in alone_lps[i]]


def test_server_draws_as_a_request_alone():
    check_server("cpu")


@pytest.mark.gpu
def test_server_draws_as_a_request_alone_on_the_device():
    check_server("cuda")


@pytest.mark.parametrize("bad", [dict(top_p=1.5), dict(top_p="x"), dict(top_k=1.5), dict(top_k=True), dict(min_p=-0.1), dict(presence_penalty=float("nan")), dict(repetition_penalty=0),
                                 dict(logprobs=21), dict(logit_bias=[[500000, 1.0]]), dict(logit_bias=[[1, 101]]), dict(logit_bias=[[1]]), dict(logit_bias=[[1.5, 1]]),
                                 dict(logit_bias={"1": 2}), dict(logit_bias=[[1, 0.0]] * 1025), dict(frequency_penalty=11)])
def test_requests_are_refused(bad):
    assert validate_request({"prompt_ids": [1], "max_new": 3, **bad}, 1000, 64) != ""
    assert validate_request({"prompt_ids": [1], "max_new": 3, "top_p": 0.5, "top_k": -1, "logit_bias": [[3, -100]], "logprobs": 20}, 1000, 64) == ""


def test_http_front_end(tmp_path):
    from spark_engine_b200.serving.openai_server import serve
    cfg, W, _ = _model()
    sock = str(tmp_path / "e.sock")
    es = EngineServer(cfg, W, EngineConfig(max_seqs=2, kv_tokens=2048, prefill_chunk=32, spec="mtp", spec_depth=2))
    ready = threading.Event()
    threading.Thread(target=es.serve_forever, args=(sock,), kwargs={"ready_cb": ready.set}, daemon=True).start()
    assert ready.wait(30)
    srv, app = serve(sock, "127.0.0.1", 0, "tiny")
    threading.Thread(target=srv.serve_forever, daemon=True).start()

    def post(path, body):
        req = urllib.request.Request(f"http://127.0.0.1:{srv.server_address[1]}{path}", json.dumps(body).encode(), {"Content-Type": "application/json"})
        return urllib.request.urlopen(req, timeout=120).read().decode()
    try:
        ask = {"prompt": "abc", "max_tokens": 6, "temperature": 1.0, "seed": 3, "top_p": 0.8, "top_k": 30, "frequency_penalty": 0.5, "logit_bias": {"65": 2.0}}
        plain = json.loads(post("/v1/completions", ask))["choices"][0]
        assert "logprobs" not in plain
        one = json.loads(post("/v1/completions", {**ask, "logprobs": 2}))["choices"][0]
        assert one["text"] == plain["text"]
        lp = one["logprobs"]
        assert len(lp["tokens"]) == len(lp["token_logprobs"]) == len(lp["top_logprobs"]) == len(lp["text_offset"]) == 6 and all(x <= 0 for x in lp["token_logprobs"])
        chat = {"messages": [{"role": "user", "content": "hi"}], "max_tokens": 5, "temperature": 0.9, "seed": 1, "min_p": 0.01, "logprobs": True, "top_logprobs": 3}
        whole = json.loads(post("/v1/chat/completions", chat))["choices"][0]["logprobs"]["content"]
        assert len(whole) == 5 and all(len(e["top_logprobs"]) == 3 for e in whole)
        lines = [json.loads(x[6:]) for x in post("/v1/chat/completions", {**chat, "stream": True}).split("\n") if x.startswith("data: {")]
        parts = sum((c["logprobs"]["content"] for x in lines for c in x["choices"] if c.get("logprobs")), [])
        assert parts == whole
        for bad in ({"top_p": 2.0}, {"logit_bias": {"x": 1}}, {"logit_bias": [1]}, {"logprobs": 50}):
            with pytest.raises(urllib.error.HTTPError) as e:
                post("/v1/completions", {**ask, **bad})
            assert e.value.code == 400
        with pytest.raises(urllib.error.HTTPError):
            post("/v1/chat/completions", {**chat, "logprobs": False})
    finally:
        srv.shutdown()
        es.shutdown = True


# ----------------------------------------------------------------------------- a sharded vocabulary
def _rank(rank, port, q):
    import os

    import torch.distributed as dist
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=2)
    from spark_engine_b200.models.plan import make_plan
    from spark_engine_b200.parallel.tp import CpuTP, shard_dense_weights
    cfg = tiny_hybrid()
    m = Model(cfg, shard_dense_weights(init_weights(cfg, seed=0), cfg, rank, 2), n_slots=1, kv_tokens=128, tp=CpuTP())
    lg = m.forward(make_plan([(0, list(range(5, 37)), 0)]))
    m.count_prompt(0, list(range(5, 37)))
    got = m.draw_rows(lg, [WILD] * 32, [0] * 32, list(range(32)), [[3, 3]] * 32)
    lps = m.logprobs(lg, got, 3)
    q.put((rank, got, lps, m.tp.gather_vocab(lg).numpy()))
    dist.barrier()
    dist.destroy_process_group()


def test_a_sharded_vocabulary_draws_the_same():
    import torch.multiprocessing as mp
    from test_tp_cpu import _free_port
    ctx = mp.get_context("spawn")
    q, port = ctx.Queue(), _free_port()
    ps = [ctx.Process(target=_rank, args=(r, port, q)) for r in range(2)]
    for p in ps:
        p.start()
    got = sorted((q.get(timeout=120) for _ in ps), key=lambda x: x[0])
    for p in ps:
        p.join(timeout=60)
        assert p.exitcode == 0
    assert got[0][1:3] == got[1][1:3] and np.array_equal(got[0][3], got[1][3])
    z = got[0][3]
    for r in range(32):
        assert got[0][1][r] == _by_definition(z[r], WILD, r, list(range(5, 37)), [3, 3])
        lp, rank, ids, _ = want_logprobs(z[r], got[0][1][r], 3)
        assert got[0][2][r][1] == rank and abs(got[0][2][r][0] - lp) < 1e-5


# ----------------------------------------------------------------------------- numbers that no float holds
HUGE = 10 ** 400


@pytest.mark.parametrize("field", ["top_k", "top_p", "min_p", "presence_penalty", "frequency_penalty", "repetition_penalty", "logprobs", "max_new"])
@pytest.mark.parametrize("value", [HUGE, -HUGE, float("inf"), float("-inf"), float("nan")], ids=["huge", "-huge", "inf", "-inf", "nan"])
def test_numbers_beyond_every_range_are_refused(field, value):
    assert validate_request({"prompt_ids": [1], "max_new": 3, field: value}, 1000, 64) != ""


@pytest.mark.parametrize("pair", [[HUGE, 1.0], [-HUGE, 1.0], [1, HUGE], [1, -HUGE], [1, float("nan")], [1, float("inf")]],
                         ids=["huge id", "-huge id", "huge", "-huge", "nan", "inf"])
def test_biases_beyond_every_range_are_refused(pair):
    assert validate_request({"prompt_ids": [1], "max_new": 3, "logit_bias": [pair]}, 1000, 64) != ""


def test_an_engine_outlives_numbers_beyond_every_range():
    cfg, W, _ = _model()
    es = EngineServer(cfg, W, EngineConfig(max_seqs=1, kv_tokens=512, prefill_chunk=32, spec="none"))
    es.submit({"id": 1, "prompt_ids": [1, 2], "max_new": 2, "top_p": HUGE})
    es.submit({"id": 2, "prompt_ids": [1, 2], "max_new": 2, "top_p": 0.5})
    while es.sched.has_work():
        es.step()
    assert [x["id"] for x in es.out if "error" in x] == [1] and [x["id"] for x in es.out if x.get("done")] == [2]


BAD = [dict(seed=-1), dict(seed=1 << 63), dict(seed=1 << 64), dict(seed=HUGE), dict(seed="x"), dict(seed=None), dict(seed=float("inf")), dict(temperature=HUGE),
       dict(temperature="x"), dict(temperature=None), dict(temperature=[1]), dict(stop_token_ids=[HUGE]), dict(stop_token_ids=["x"]), dict(stop_token_ids=[[1]]), dict(stop_token_ids=5)]


def test_an_engine_outlives_settings_that_it_cannot_hold():
    """Beside a request that goes on, which gets its whole answer; the largest seed and temperatures of every size are served."""
    cfg, W, _ = _model()
    es = EngineServer(cfg, W, EngineConfig(max_seqs=2, kv_tokens=2048, prefill_chunk=32, spec="mtp", spec_depth=2))
    es.submit({"id": 1000, "prompt_ids": [5, 6, 7], "max_new": 40})
    for i, bad in enumerate(BAD):
        es.submit({"id": i, "prompt_ids": [1, 2], "max_new": 2, **bad})
        es.step()
    fine = [dict(seed=(1 << 63) - 1, temperature=0.8), dict(seed=3.0, temperature="0.5"), dict(temperature=1e300), dict(temperature=float("inf")), dict(temperature=float("nan")),
            dict(temperature=-1), dict(stop_token_ids=[-5, 3])]
    for i, good in enumerate(fine):
        es.submit({"id": 100 + i, "prompt_ids": [1, 2], "max_new": 2, **good})
    while es.sched.has_work():
        es.step()
    assert [x["id"] for x in es.out if "error" in x] == list(range(len(BAD)))
    assert sorted(x["id"] for x in es.out if x.get("done")) == [100 + i for i in range(len(fine))] + [1000]
    assert [len(x["token_ids"]) for x in es.out if x.get("done") and x["id"] == 1000] == [40]


# ----------------------------------------------------------------------------- rows without any token
NOTHING = SamplingParams(temperature=0.9, seed=4, top_p=0.8, frequency=0.3, logprobs=2)


def _blind(m, slot, length):
    """The model's logits of a slot's rows are NaN from position `length` on."""
    forward = m.forward

    def blinded(plan, *a, **k):
        logits = forward(plan, *a, **k)
        for i, s in enumerate(plan.segs):
            rows = range(s.r0, s.r0 + s.n) if logits.shape[0] == sum(x.n for x in plan.segs) else [i]
            if s.slot == slot() and s.pos0 + s.n >= length:
                logits[list(rows)] = float("nan")
        return logits
    m.forward = blinded
    return lambda: setattr(m, "forward", forward)


@pytest.mark.parametrize("tree", [False, True])
def test_a_round_without_a_token_ends_its_sequence(tree):
    """Nothing that is no token is emitted, counted or drafted from; the sequences beside it go on."""
    cfg, W, m = _model()
    prompts = _prompts(cfg, 2)
    want, _ = _text(SpecDecoder(m, lambda s, d: ([], []), depth=0), prompts, [NOTHING, WILD], 12)
    _, _, m = _model()
    sd = SpecDecoder(m, lambda s, d: ([], []), depth=0)
    seqs = [sd.start(i, p, params=q) for i, (p, q) in enumerate(zip(prompts, [NOTHING, WILD]))]
    _blind(m, lambda: 0, len(prompts[0]) + 4)
    while any(len(s.generated) < 12 and not s.failed for s in seqs):
        live = [s for s in seqs if len(s.generated) < 12 and not s.failed]
        budgets = [12 - len(s.generated) for s in live]
        if tree:
            sd.round_tree(live, [[Node(token=(want[s.slot] + [0])[len(s.generated)], parent=-1)] for s in live], budgets)
        else:
            sd.round(live, budgets)
    assert seqs[0].failed and seqs[0].generated == want[0][: len(seqs[0].generated)] and 2 <= len(seqs[0].generated) < 6
    assert not seqs[1].failed and seqs[1].generated == want[1]
    assert int((m.token_counts()[0] >> 1).sum()) == len(seqs[0].generated)


def test_a_prompt_without_a_token():
    cfg, W, m = _model()
    prompts = _prompts(cfg, 1)
    sd = SpecDecoder(m, lambda s, d: ([], []), depth=0)
    see = _blind(m, lambda: 0, 0)
    seq = sd.start(0, prompts[0], params=NOTHING)
    assert seq.failed and seq.generated == [] and seq.logprobs == [] and not (m.token_counts()[0] >> 1).any()
    assert sd.generate(prompts, 5, params=NOTHING) == [[]]
    see()
    assert len(sd.generate(prompts, 5, params=NOTHING)[0]) == 5


def check_a_server_ends_requests_without_a_token(after, device, one):
    """With an error and what was said before; the request again (over what its slot was left with) has its whole text, and so have those beside it."""
    cfg, W, m = _model(device)
    prompts = _prompts(cfg, 2)
    alone = []
    for p, q in zip(prompts, [one, WILD]):
        alone += _text(SpecDecoder(m, lambda s, d: ([], []), depth=0), [p], [q], 10)[0]
    es = EngineServer(cfg, W, EngineConfig(max_seqs=2, kv_tokens=2048, prefill_chunk=32, spec="mtp", spec_depth=2, cuda_graphs=False), device=device)
    see = _blind(es.model, lambda: next((s for s, lv in es.by_slot.items() if lv.id == 0), -1), len(prompts[0]) + after)
    for i, q in enumerate([one, WILD]):
        es.submit(_message(i, prompts[i], q, 10))
    while es.sched.has_work():
        es.step()
    see()
    es.submit(_message(2, prompts[0], one, 10))
    while es.sched.has_work():
        es.step()
    mine = [x for x in es.out if x.get("id") == 0]
    said = sum((x["delta"] for x in mine if "delta" in x), [])
    assert "error" in mine[-1] and not any(x.get("done") for x in mine) and said == alone[0][: len(said)] and (len(said) == 0) == (after == 0)
    assert sum(len(x.get("logprobs", [])) for x in mine) == (len(said) if one.logprobs >= 0 else 0)
    done = {x["id"]: x["token_ids"] for x in es.out if x.get("done")}
    assert done == {1: alone[1], 2: alone[0]} and not es.live and not es.by_slot


@pytest.mark.parametrize("after", [0, 4])
def test_a_server_ends_requests_without_a_token(after):
    check_a_server_ends_requests_without_a_token(after, "cpu", NOTHING)


@pytest.mark.gpu
@pytest.mark.parametrize("one", [NOTHING, SamplingParams(temperature=0.9, seed=4), SamplingParams()], ids=["filtered", "plain", "greedy"])
@pytest.mark.parametrize("after", [0, 4])
def test_a_server_ends_requests_without_a_token_on_the_device(after, one):
    """There plain rounds know no token of such rows either."""
    check_a_server_ends_requests_without_a_token(after, "cuda", one)


# ----------------------------------------------------------------------------- the front end alone
class Engine:
    """An engine that answers with the given messages."""
    alive = True

    def __init__(self, messages=()):
        self.messages, self.queues, self.asked, self.cancelled = list(messages), {}, [], []

    def generate(self, ids, max_new, stop, temperature, seed, mm=None, sampling=None):
        import queue
        rid = len(self.asked)
        q = self.queues[rid] = queue.Queue()
        self.asked.append(sampling or {})
        for m in self.messages:
            q.put(dict(m, id=rid))
        return rid, q

    def cancel(self, rid):
        self.cancelled.append(rid)

    def release(self, rid):
        self.queues.pop(rid, None)


def _app(messages=(), tok=None):
    from spark_engine_b200.serving.openai_server import App
    from spark_engine_b200.serving.tokenizer import ByteTokenizer
    return App(Engine(messages), tok or ByteTokenizer(), "tiny")


@pytest.mark.parametrize("top", ["3", "x", [3], 3.5, -1, True, {"a": 1}])
def test_top_logprobs_that_are_no_number_are_refused(top):
    """Before the engine hears of the request."""
    app = _app([{"error": "it has heard of it"}])
    with pytest.raises(ValueError, match="top_logprobs"):
        app.run([1], {"logprobs": True, "top_logprobs": top}, True)
    assert not app.engine.asked and not app.engine.queues


def _byte_level(tmp_path):
    """A tokenizer of the byte-level kind: every byte a token, and a few longer ones of which one ends inside a character."""
    from tokenizers import Tokenizer, decoders, models, pre_tokenizers
    from transformers import PreTrainedTokenizerFast
    from spark_engine_b200.serving.tokenizer import HfTokenizer
    letters = sorted(pre_tokenizers.ByteLevel.alphabet())
    tk = PreTrainedTokenizerFast(tokenizer_object=Tokenizer(models.BPE({c: i for i, c in enumerate(letters)}, [])), eos_token="</s>")
    tk.backend_tokenizer.pre_tokenizer = pre_tokenizers.ByteLevel(add_prefix_space=False, use_regex=False)
    tk.backend_tokenizer.decoder = decoders.ByteLevel()
    tk.save_pretrained(str(tmp_path))
    return HfTokenizer(str(tmp_path))


def _byte_fallback(tmp_path):
    """One of the kind that has a piece <0xXX> for every byte that no other piece covers."""
    from tokenizers import Tokenizer, decoders, models
    from transformers import PreTrainedTokenizerFast
    from spark_engine_b200.serving.tokenizer import HfTokenizer
    vocab = {f"<0x{i:02X}>": i for i in range(256)}
    vocab.update({"h": 256, "i": 257})
    tk = PreTrainedTokenizerFast(tokenizer_object=Tokenizer(models.BPE(vocab, [], byte_fallback=True)), eos_token="</s>")
    tk.backend_tokenizer.decoder = decoders.Sequence([decoders.ByteFallback(), decoders.Fuse()])
    tk.save_pretrained(str(tmp_path))
    return HfTokenizer(str(tmp_path))


TEXT = "hé 你\U0001f600i"


def _toks(kind, tmp_path):
    """(tokenizer, ids of TEXT's bytes one by one)."""
    from spark_engine_b200.serving.tokenizer import ByteTokenizer
    raw = TEXT.encode()
    if kind == "bytes":
        return ByteTokenizer(), list(raw)
    if kind == "fallback":
        return _byte_fallback(tmp_path), list(raw)
    tok = _byte_level(tmp_path)
    ids = tok.encode(TEXT)
    assert len(ids) == len(raw)
    return tok, ids


@pytest.mark.parametrize("kind", ["bytes", "level", "fallback"])
def test_bytes_of_tokens_are_the_tokens_own(kind, tmp_path):
    """A character over several tokens: their bytes together are the text's, and tokens with the same text stay apart."""
    tok, ids = _toks(kind, tmp_path)
    assert tok.decode(ids) == TEXT
    order = list(dict.fromkeys(ids))
    top = [[t, -float(i)] for i, t in enumerate(order)]
    messages = [{"delta": ids[:5], "logprobs": [[-0.5, 1, top]] * 5}, {"delta": ids[5:], "logprobs": [[-0.5, 1, top]] * (len(ids) - 5)},
                {"done": True, "token_ids": ids, "finish_reason": "length"}]
    chat = _app(messages, tok).run([1], {"logprobs": True, "top_logprobs": 20}, True)
    assert chat["content"] == TEXT
    got = chat["logprobs"]["content"]
    assert b"".join(bytes(e["bytes"]) for e in got) == TEXT.encode()
    byte_of = dict(zip(ids, TEXT.encode()))
    for e in got:
        assert [x["bytes"] for x in e["top_logprobs"]] == [[byte_of[t]] for t in order]
        assert len({x["token"] for x in e["top_logprobs"]}) == len(order)
        assert e["token"] == (chr(e["bytes"][0]) if e["bytes"][0] < 128 else "bytes:\\x%02x" % e["bytes"][0])
    plain = _app(messages, tok).run([1], {"logprobs": 20}, False)["logprobs"]
    assert plain["tokens"] == [e["token"] for e in got]
    assert all(list(t.values()) == [x for _, x in top] for t in plain["top_logprobs"])


def test_tokens_of_the_same_text_stay_apart():
    """Ids without text of their own (all of the byte tokenizer's beyond 255) beside one another, and probabilities of nothing."""
    top = [[256, -0.1], [258, -2.0], [300, -3.0], [65, float("-inf")]]
    messages = [{"delta": [256], "logprobs": [[-0.1, 1, top]]}, {"done": True, "token_ids": [256], "finish_reason": "length"}]
    got = _app(messages).run([1], {"logprobs": 4}, False)["logprobs"]
    assert list(got["top_logprobs"][0].values()) == [-0.1, -2.0, -3.0, -9999.0] and got["top_logprobs"][0]["A"] == -9999.0
    json.loads(json.dumps(got, allow_nan=False))


def _answer(parts):
    """An engine's messages for a text in the given pieces (bytes as tokens)."""
    out = [{"delta": list(p), "logprobs": [[-float(b), 1, []] for b in p]} for p in parts]
    return out + [{"done": True, "token_ids": list(b"".join(parts)), "finish_reason": "length"}]


@pytest.mark.parametrize("parts", [[b"one t", b"w", b"o", b" three"], [b"one two", b" three ", b"four"], [bytes([b]) for b in b"one two three"]])
def test_nothing_behind_a_stop_string_is_text(parts):
    """However late the engine hears of it."""
    events = []
    app = _app(_answer(parts))
    r = app.run([1], {"stop": ["two", "xyz"]}, False, lambda *a: events.append(a))
    assert r["content"] == "one " and r["finish"] == "stop" and "".join(e[1] for e in events) == "one " and app.engine.cancelled == [0]


@pytest.mark.parametrize("parts", [[b"one two three"], [b"one t", b"w", b"o three"], [b"one t", b"wo", b" three"], [bytes([b]) for b in b"one two three"]])
@pytest.mark.parametrize("chat", [False, True])
def test_log_probabilities_end_where_the_text_does(parts, chat):
    """At a stop string, however it comes; what was given out before does not have to be taken back, and nothing behind it is text."""
    body = {"stop": ["two", "xyz"], "logprobs": True if chat else 0}
    events = []
    app = _app(_answer(parts))
    r = app.run([1], body, chat, lambda *a: events.append(a))
    assert r["content"] == "one " and r["finish"] == "stop" and app.engine.cancelled == [0]
    flat = lambda x: [e["logprob"] for e in x["content"]] if chat else x["token_logprobs"]
    want = [-float(b) for b in b"one "]
    assert flat(r["logprobs"]) == want
    given = sum((flat(e[2]) for e in events), []) + (flat(r["logprobs_left"]) if r["logprobs_left"] else [])
    assert given == want and "".join(e[1] for e in events) == "one "
    whole = app.run([1], {**body, "stop": ["xyz"]}, chat)
    assert whole["content"] == "one two three" and flat(whole["logprobs"]) == [-float(b) for b in b"one two three"]


def test_offsets_are_where_the_tokens_begin_in_the_text():
    raw = TEXT.encode()
    want = [len(raw[:i].decode(errors="ignore")) for i in range(len(raw))]
    for n in (1, 2, 3, len(raw)):
        got = _app(_answer([raw[i: i + n] for i in range(0, len(raw), n)])).run([1], {"logprobs": 0}, False)
        assert got["content"] == TEXT and got["logprobs"]["text_offset"] == want
    cut = _app(_answer([raw])).run([1], {"logprobs": 0, "stop": "你"}, False)
    assert cut["content"] == "hé " and len(cut["logprobs"]["tokens"]) == len("hé ".encode())


@pytest.mark.parametrize("body", [{"top_p": 2.0}, {"logprobs": True, "top_logprobs": "x"}])
def test_a_stream_that_is_refused_ends_with_an_error(body):
    """As an event of the stream, which begins before the engine answers."""
    from http.server import ThreadingHTTPServer
    from spark_engine_b200.serving.openai_server import make_handler
    app = _app([{"error": "it does not want to"}])
    srv = ThreadingHTTPServer(("127.0.0.1", 0), make_handler(app))
    srv.daemon_threads = True
    threading.Thread(target=srv.serve_forever, daemon=True).start()
    try:
        ask = {"messages": [{"role": "user", "content": "hi"}], "stream": True, **body}
        req = urllib.request.Request(f"http://127.0.0.1:{srv.server_address[1]}/v1/chat/completions", json.dumps(ask).encode(), {"Content-Type": "application/json"})
        lines = [x[6:] for x in urllib.request.urlopen(req, timeout=30).read().decode().split("\n") if x.startswith("data: ")]
        assert lines[-1] == "[DONE]" and json.loads(lines[-2])["error"]["message"] == ("it does not want to" if "top_p" in body else "top_logprobs must be a whole number")
        assert all("choices" in json.loads(x) for x in lines[:-2]) and not app.engine.queues
    finally:
        srv.shutdown()
