"""From a round's logits to its tokens: the operators behind the model's head, each in its plain form and as the framework's call.

  count     tokens of prompts and answers counted per request, which the penalties go by
  adjust    repetition, presence and frequency penalties, biases and allowed tokens applied to logits
  sample    one token per row from temperature, top-k, top-p and min-p, with noise that seed, position and id determine (with `adjust` first)
  logprobs  log-probability and rank of given tokens, and the most probable tokens

A row's tokens are ordered by descending logit, the lower id first where logits are equal.  How many rows a case has of which kind does not depend
on the seed.
"""
import math

import torch

own = False


def listed():
    return [
        # sixteen streams advance by a speculative round's accepted tokens: the smallest call, launches and latency count
        {"name": "count-round-16", "op": "count", "rows": 16, "vocab": 151936, "tokens_min": 1, "tokens_max": 4, "reset": False},
        # prompts of a full batch are admitted: their rows of the table are written anew
        {"name": "count-prompts-64", "op": "count", "rows": 64, "vocab": 151936, "tokens_min": 200, "tokens_max": 32000, "reset": True},
        # four streams of an interactive server, penalties and biases
        {"name": "adjust-4", "op": "adjust", "rows": 4, "vocab": 154880, "dtype": "f32", "logits": "peaked", "drafts": 0, "bias": 8, "allowed": False},
        # a full batch of verified rows: drafted tokens count, a grammar allows some of the vocabulary, bf16 logits
        {"name": "adjust-256-grammar", "op": "adjust", "rows": 256, "vocab": 129280, "dtype": "bf16", "logits": "peaked", "drafts": 3, "bias": 100, "allowed": True},
        # one interactive stream: temperature, top-k and top-p
        {"name": "sample-1", "op": "sample", "rows": 1, "vocab": 151936, "dtype": "f32", "logits": "peaked", "kinds": "kp", "adjust": False},
        # a speculative round of four streams, four rows each: penalties with drafted tokens, biases
        {"name": "sample-16-adjusted", "op": "sample", "rows": 16, "vocab": 151936, "dtype": "f32", "logits": "peaked", "kinds": "kp,chat,minp,k",
         "adjust": True, "drafts": 3, "bias": 8, "allowed": False},
        # a batch of everything that clients ask for, greedy and unfiltered rows among them
        {"name": "sample-256-mixed", "op": "sample", "rows": 256, "vocab": 151936, "dtype": "f32", "logits": "peaked",
         "kinds": "chat,kp,k,minp,greedy,plain,wide,chat", "adjust": False},
        # flat distributions, where many thousands of tokens are kept; bf16 logits, many of them equal
        {"name": "sample-64-flat", "op": "sample", "rows": 64, "vocab": 129280, "dtype": "bf16", "logits": "flat", "kinds": "wide,bigk,chat,plain", "adjust": False},
        # a small vocabulary of odd size, every row behind a grammar
        {"name": "sample-500-small", "op": "sample", "rows": 500, "vocab": 4099, "dtype": "f32", "logits": "peaked", "kinds": "chat,kp,k",
         "adjust": True, "drafts": 0, "bias": 0, "allowed": True},
        # log-probabilities of one stream's token
        {"name": "logprobs-1", "op": "logprobs", "rows": 1, "vocab": 151936, "dtype": "f32", "logits": "peaked", "top": 5},
        # a batch of streams that all want the most the API gives
        {"name": "logprobs-64-top20", "op": "logprobs", "rows": 64, "vocab": 129280, "dtype": "bf16", "logits": "peaked", "top": 20},
        # a prompt scored token by token: the largest call
        {"name": "logprobs-1024", "op": "logprobs", "rows": 1024, "vocab": 151936, "dtype": "f32", "logits": "peaked", "top": 1},
    ]


# --------------------------------------------------------------------------------------------------- drawn cases
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    return work(case)["bytes"]


KINDS = ("greedy", "plain", "chat", "k", "kp", "minp", "wide", "bigk")


def draw(rng):
    op = rng.choice(["count", "adjust", "sample", "sample", "sample", "sample", "logprobs", "logprobs"])
    most = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        case = _drawn(rng, op)
        if _cost(case) <= most and (op != "sample" or case["rows"] * case["vocab"] <= 256 * 151936):
            return case


def _drawn(rng, op):
    case = {"op": op, "rows": _log(rng, 1, 1024), "vocab": rng.choice([151936, 154880, 129280, 65536, 4096, _log(rng, 2, 200000), _log(rng, 2000, 200000)])}
    if op == "count":
        a, b = sorted((_log(rng, 1, 32000), _log(rng, 1, 32000)))
        reset = rng.random() < 0.5
        case.update(rows=_log(rng, 1, 64), tokens_min=a if reset else min(a, 64), tokens_max=b if reset else min(b, 64), reset=reset)
        return case
    case.update(dtype=rng.choice(["f32", "f32", "f32", "bf16", "f16"]), logits=rng.choice(["peaked", "peaked", "flat"]))
    if op == "logprobs":
        case["top"] = rng.choice([0, 1, 5, 20, rng.randint(1, 64)])
        return case
    more = {"drafts": rng.choice([0, 0, 3, 7]), "bias": rng.choice([0, 0, 1, 8, 300]), "allowed": rng.random() < 0.4}
    if op == "adjust":
        return {**case, **more}
    case["kinds"] = ",".join(rng.choice(KINDS) for _ in range(rng.randint(1, 4)))
    case["adjust"] = rng.random() < 0.4
    return {**case, **more} if case["adjust"] else case


# --------------------------------------------------------------------------------------------------- sizes of a case
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
_TYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _counts(case):
    """Tokens of each request: spread evenly over their logarithm."""
    lo, hi, n = case["tokens_min"], case["tokens_max"], case["rows"]
    return [hi] if n == 1 else [int(round(math.exp(math.log(lo) + (math.log(hi) - math.log(lo)) * i / (n - 1)))) for i in range(n)]


def work(case):
    R, V = case["rows"], case["vocab"]
    if case["op"] == "count":
        n = sum(_counts(case))
        # tokens and counts in; a new request's row of the table out, or the entries of the tokens in and out
        return {"bytes": 4 * n + 4 * R + (4 * R * V if case["reset"] else 8 * n), "flops": n}
    e = _BYTES[case["dtype"]]
    adjusted = case["op"] == "adjust" or case.get("adjust")
    more = (4 * -(-R // (case["drafts"] + 1)) * V + R * V / 8 * case["allowed"] + R * (4 * case["drafts"] + 8 * case["bias"])) if adjusted else 0
    if case["op"] == "adjust":
        return {"bytes": R * V * (e + 4) + more, "flops": 5 * R * V}
    if case["op"] == "logprobs":
        return {"bytes": R * V * e + R * (12 + 8 * case["top"]), "flops": 4 * R * V}
    return {"bytes": R * V * e + more + 36 * R, "flops": 4 * R * V + (5 * R * V if adjusted else 0)}


# --------------------------------------------------------------------------------------------------- inputs
class _Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def n(self, *s):
        return torch.randn(*s, device="cuda", generator=self.g)

    def u(self, *s):
        return torch.rand(*s, device="cuda", generator=self.g)

    def i(self, hi, *s):
        return torch.randint(hi, s, device="cuda", generator=self.g)


def _logits(case, r):
    """What a head gives: a bulk of improbable tokens, and some tens that stand out of it; or, for a flat one, the bulk alone."""
    R, V = case["rows"], case["vocab"]
    if case["logits"] == "flat":
        return (r.n(R, V) * 0.8).to(_TYPE[case["dtype"]])
    z = r.n(R, V) * 1.8
    z.scatter_reduce_(1, r.i(V, R, 64), 16.0 - 9.0 * r.u(R, 64) ** 0.5 + 0.5 * r.n(R, 64), "amax")
    return z.to(_TYPE[case["dtype"]])


def _words(r, V, *s):
    """Token ids as text has them: a few very often, most hardly ever."""
    return (torch.exp(r.u(*s) * math.log(V + 1)).long() - 1).clamp(0, V - 1)


def _table(case, r, slots):
    """Counts of requests in their course: prompts of some thousand tokens, answers of some hundred."""
    V = case["vocab"]
    t = torch.zeros(slots, V, dtype=torch.int32, device="cuda")
    t.scatter_(1, _words(r, V, slots, 3000), 1)
    ids = _words(r, V, slots, 400)
    return t.scatter_add_(1, ids, torch.full_like(ids, 2, dtype=torch.int32))


def _adjust(case, r):
    R, V, depth = case["rows"], case["vocab"], case["drafts"]
    k = depth + 1                                                # rows of a request
    slots = -(-R // k)
    a = {"counts": _table(case, r, slots), "slots": (torch.arange(R, device="cuda") // k).to(torch.int32), "drafted": None, "bias_ids": None, "bias": None,
         "allowed": None, "repetition": 1 + 0.3 * r.u(R), "presence": 0.8 * r.u(R), "frequency": 0.4 * r.u(R)}
    if depth:                                                    # row j of a request comes behind j drafts
        ids = _words(r, V, slots, depth).repeat_interleave(k, 0)[:R]
        on = torch.arange(depth, device="cuda") < (torch.arange(R, device="cuda") % k).unsqueeze(1)
        a["drafted"] = torch.where(on, ids, torch.full_like(ids, -1)).to(torch.int32).contiguous()
    if case["bias"]:
        n = case["bias"]                                         # different ids, as a client's table has them; short tables end in -1
        ids = (r.i(V, R, 1) + torch.arange(n, device="cuda") * max(1, V // n)) % V
        short = torch.arange(n, device="cuda") >= torch.clamp(r.i(n + 1, R, 1), min=min(n, V) // 2)
        a["bias_ids"] = torch.where(short | (torch.arange(n, device="cuda") >= V), torch.full_like(ids, -1), ids).to(torch.int32)
        a["bias"] = r.n(R, n) * 3
    if case["allowed"]:                                          # every third row's grammar leaves a few tokens, the others' most, some none at all
        words = -(-V // 32)
        most = r.i(1 << 32, R, words) | r.i(1 << 32, R, words)
        few = torch.zeros(R, words, dtype=torch.int64, device="cuda")
        few.scatter_(1, r.i(words, R, 12), 1 << 5)
        few[:, 0] |= 2
        bits = torch.where((torch.arange(R, device="cuda") % 3 == 0).unsqueeze(1), few, most)
        bits = torch.where((torch.arange(R, device="cuda") % 50 == 49).unsqueeze(1), torch.zeros_like(bits), bits)
        a["allowed"] = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32)
    return a


def _settings(case, r):
    """Temperatures and filters of rows: every row is of one of the case's kinds, its values its client's own."""
    R = case["rows"]
    kinds = (case["kinds"].split(",") * R)[:R]
    of = {  # temperature, top-k, top-p, min-p (lowest, highest)
        "greedy": ((0, 0), (0, 0), (1, 1), (0, 0)), "plain": ((0.7, 1.2), (0, 0), (1, 1), (0, 0)),
        "chat": ((0.6, 1.0), (0, 0), (0.8, 0.97), (0, 0)), "k": ((0.8, 1.1), (20, 100), (1, 1), (0, 0)),
        "kp": ((0.6, 0.9), (20, 64), (0.8, 0.97), (0, 0)), "minp": ((0.9, 1.5), (0, 0), (1, 1), (0.02, 0.15)),
        "wide": ((1.2, 1.6), (0, 0), (0.95, 0.999), (0, 0)), "bigk": ((0.9, 1.2), (2000, 20000), (0.85, 0.99), (0, 0)),
    }
    lo, hi = (torch.tensor([[x[e] for x in of[k]] for k in kinds], dtype=torch.float32, device="cuda") for e in (0, 1))
    t, k, p, m = (lo + (hi - lo) * r.u(R, 4)).unbind(1)
    return {"temps": t.contiguous(), "top_k": k.round().to(torch.int32), "top_p": p.contiguous(), "min_p": m.contiguous(),
            "seeds": r.i(1 << 40, R), "positions": r.i(32000, R)}


def prepare(case, seed):
    r = _Rand(seed)
    s = {"case": case}
    if case["op"] == "count":
        n = torch.tensor(_counts(case), dtype=torch.int32, device="cuda")
        s["n"] = n[torch.argsort(r.u(case["rows"]))].contiguous()
        s["tokens"] = _words(r, case["vocab"], case["rows"], case["tokens_max"]).to(torch.int32)
        s["slots"] = torch.argsort(r.u(case["rows"])).to(torch.int32)
        s["counts"] = _table(case, r, case["rows"])
        return s
    s["logits"] = _logits(case, r)
    if case["op"] == "adjust" or case.get("adjust"):
        s["adjust"] = _adjust(case, r)
    if case["op"] == "sample":
        s["set"] = _settings(case, r)
    if case["op"] == "logprobs":                                 # mostly what was drawn from these logits, sometimes an improbable token
        best = (s["logits"].float() + 2 * r.n(1, case["vocab"])).argmax(1)
        s["tokens"] = torch.where(r.u(case["rows"]) < 0.2, r.i(case["vocab"], case["rows"]), best).to(torch.int32)
    return s


# --------------------------------------------------------------------------------------------------- one pass
def run(state):
    return {"count": _count, "adjust": _adjusted, "sample": _sample, "logprobs": _logprobs}[state["case"]["op"]](state)


def _count(s):
    reset = s["case"]["reset"]
    if own:
        from spark_engine_b200 import ops
        ops.count_tokens(s["counts"], s["tokens"], s["n"], slots=s["slots"], prompt=reset, reset=reset)
        return s["counts"]
    at = s["slots"].long()
    there = torch.arange(s["tokens"].shape[1], device=at.device) < s["n"].unsqueeze(1)
    rows = torch.zeros_like(s["counts"]) if reset else s["counts"][at]
    rows.scatter_add_(1, s["tokens"].long(), torch.where(there, 2, 0).to(torch.int32))
    s["counts"][at] = torch.clamp(rows, max=1) if reset else rows
    return s["counts"]


def _adjusted(s):
    if own:
        from spark_engine_b200 import ops
        return ops.adjust_logits(s["logits"], ops.Adjust(**s["adjust"]))
    return _plain_adjust(s["logits"], s["adjust"])


def _plain_adjust(logits, a):
    z = logits.float()
    R, V = z.shape
    t = a["counts"][a["slots"].long()]
    c, seen = t >> 1, t > 0
    if a["drafted"] is not None:
        on, ids = a["drafted"] >= 0, a["drafted"].clamp(min=0).long()
        more = torch.zeros_like(c).scatter_add_(1, ids, on.to(torch.int32))
        c, seen = c + more, seen | (more > 0)
    rep = a["repetition"].unsqueeze(1)
    z = torch.where(seen, torch.where(z > 0, z / rep, z * rep), z)
    z = z - a["frequency"].unsqueeze(1) * c
    z = z - a["presence"].unsqueeze(1) * (c > 0)
    if a["bias"] is not None:
        on, ids = a["bias_ids"] >= 0, a["bias_ids"].clamp(min=0).long()
        z = z.scatter_add(1, ids, torch.where(on, a["bias"], torch.zeros_like(a["bias"])))
    if a["allowed"] is not None:
        at = torch.arange(V, device=z.device)
        z = torch.where((a["allowed"][:, at // 32] >> (at % 32)) & 1 == 1, z, torch.full_like(z, -math.inf))
    return z


def _mix(x):
    """An integer's bits stirred (products wrap at 64 bits, shifts bring in zeros)."""
    x = (x ^ ((x >> 30) & ((1 << 34) - 1))) * -4658895280553007687
    x = (x ^ ((x >> 27) & ((1 << 37) - 1))) * -7723592293110705685
    return x ^ ((x >> 31) & ((1 << 33) - 1))


def _noise(seeds, positions, ids):
    """g = -log(-log u), u in (0, 1) from the bits of (seed, position, id)."""
    key = (seeds * -7046029254386353131) ^ ((positions + 1) * -4658895280553007687)
    bits = (_mix(ids * -7046029254386353131 + key.unsqueeze(1)) >> 11) & ((1 << 53) - 1)
    u = (bits.double() + 0.5) / float(1 << 53)
    return -torch.log(-torch.log(u))


def _sample(s):
    q = s["set"]
    if own:
        from spark_engine_b200 import ops
        adjust = ops.Adjust(**s["adjust"]) if "adjust" in s else None
        return ops.sample_tokens(s["logits"], q["temps"], q["seeds"], q["positions"], top_k=q["top_k"], top_p=q["top_p"], min_p=q["min_p"], adjust=adjust)
    z = _plain_adjust(s["logits"], s["adjust"]) if "adjust" in s else s["logits"].float()
    z, ids = torch.sort(z, dim=1, descending=True, stable=True)
    V, T = z.shape[1], torch.where(q["temps"] > 0, q["temps"], torch.ones_like(q["temps"])).unsqueeze(1)
    d = (z.double() - z[:, :1].double()) / T.double()            # kept or not is decided in 64 bits: a sum's last bits move the border
    keep = d >= torch.log(q["min_p"].double()).unsqueeze(1)
    k = torch.where(q["top_k"] > 0, q["top_k"], torch.full_like(q["top_k"], V)).unsqueeze(1)
    keep &= torch.arange(V, device=z.device) < k
    w = torch.where(keep, torch.exp(d), torch.zeros_like(d))
    upto = torch.cumsum(w, 1)
    p = q["top_p"].double().unsqueeze(1)
    keep &= (p >= 1) | (upto - w < p * upto[:, -1:])
    keep[:, 0] = True
    score = z / T + _noise(q["seeds"], q["positions"], ids).float()
    score = torch.where(keep, score, torch.full_like(score, -math.inf))
    best = torch.where(score == score.amax(1, keepdim=True), ids, torch.full_like(ids, V)).amin(1)
    best = torch.where(q["temps"] > 0, best, ids[:, 0])
    return torch.where(z[:, 0] == -math.inf, torch.full_like(best, -1), best).to(torch.int32)


def _logprobs(s):
    top = s["case"]["top"]
    if own:
        from spark_engine_b200 import ops
        r = ops.token_logprobs(s["logits"], s["tokens"], top=top)
        return {"logprob": r.logprob, "rank": r.rank, "ids": r.ids, "logprobs": r.logprobs}
    z, t = s["logits"].float(), s["tokens"].long().unsqueeze(1)
    R, V = z.shape
    own_z = z.gather(1, t)
    z0 = z.amax(1, keepdim=True)
    total = torch.exp(z - z0).sum(1, keepdim=True, dtype=torch.float64)
    at = torch.arange(V, device=z.device)
    rank = 1 + ((z > own_z) | ((z == own_z) & (at < t))).sum(1)
    lse = z0.double() + torch.log(total)
    bits = z.view(torch.int32).long()                            # the order as whole numbers: logit descending, id ascending
    key = (torch.where(bits < 0, -(bits & 0x7fffffff), bits) << 32) - at
    n = min(top, V)
    if n:
        first = torch.sort(torch.topk(key, n, dim=1).values, dim=1, descending=True).values
        ids = -first & 0xffffffff
    else:
        ids = torch.empty(R, 0, dtype=torch.int64, device=z.device)
    lp = (z.gather(1, ids).double() - lse).float()
    if n < top:                                                  # fewer tokens than were asked for
        ids = torch.cat((ids, torch.full((R, top - n), -1, device=z.device)), 1)
        lp = torch.cat((lp, torch.full((R, top - n), -math.inf, device=z.device)), 1)
    return {"logprob": (own_z.double() - lse).float()[:, 0], "rank": rank.to(torch.int32), "ids": ids.to(torch.int32), "logprobs": lp}


# --------------------------------------------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    """From the definitions, row by row."""
    if case["op"] in ("count", "sample"):                        # (whole numbers)
        return None
    s = prepare(case, seed)
    rows = [_exact_adjust(s, r) if case["op"] == "adjust" else _exact_logprobs(s, r) for r in range(case["rows"])]
    if case["op"] == "adjust":
        return torch.stack(rows)
    return {"logprob": torch.stack([a for a, _ in rows]), "rank": None, "ids": None, "logprobs": torch.stack([b for _, b in rows])}


def _exact_adjust(s, r):
    a, x = s["adjust"], s["logits"][r].double()
    generated = torch.div(a["counts"][int(a["slots"][r])], 2, rounding_mode="floor").double()
    prompt = a["counts"][int(a["slots"][r])] % 2 == 1
    if a["drafted"] is not None:
        ids = a["drafted"][r][a["drafted"][r] >= 0].long()
        generated = generated + torch.bincount(ids, minlength=x.shape[0]).double()
    factor = torch.where(prompt | (generated > 0), a["repetition"][r].double(), 1.0)
    y = torch.where(x > 0, x / factor, x * factor) - a["frequency"][r].double() * generated - a["presence"][r].double() * (generated > 0)
    if a["bias"] is not None:
        there = a["bias_ids"][r] >= 0
        y = y + torch.bincount(a["bias_ids"][r][there].long(), weights=a["bias"][r][there].double(), minlength=x.shape[0])
    if a["allowed"] is not None:
        bits = torch.stack([(a["allowed"][r] >> b) & 1 for b in range(32)], 1).reshape(-1)[: x.shape[0]]
        y = y.masked_fill(bits == 0, -math.inf)
    return y


def _exact_logprobs(s, r):
    x, top = s["logits"][r].double(), s["case"]["top"]
    lp = torch.log_softmax(x, 0)
    first = torch.sort(lp, descending=True).values[:top]
    return lp[int(s["tokens"][r])], torch.cat((first, torch.full((top - first.shape[0],), -math.inf, dtype=first.dtype, device=first.device)))
