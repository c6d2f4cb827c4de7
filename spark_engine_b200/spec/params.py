"""What a request asks of its draws: temperature and seed, top-k / top-p / min-p, penalties, biases, log-probabilities of the answer."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Any, Dict, Tuple

MAX_BIASES = 1024
MAX_LOGPROBS = 20


@dataclass(frozen=True)
class SamplingParams:
    temperature: float = 0.0
    seed: int = 0
    top_k: int = 0                                 # <= 0: all tokens
    top_p: float = 1.0                             # >= 1: all of their probability
    min_p: float = 0.0                             # <= 0: however improbable
    repetition: float = 1.0                        # divides positive logits of tokens in the prompt or the answer, multiplies others
    presence: float = 0.0                          # off logits of tokens in the answer
    frequency: float = 0.0                         # the same for every time
    bias: Tuple[Tuple[int, float], ...] = ()       # (token id, added to its logit)
    logprobs: int = -1                             # most probable tokens reported with every token of the answer; -1: no log-probabilities

    @property
    def counted(self) -> bool:
        """Whether the request's tokens have to be counted."""
        return self.repetition != 1.0 or self.presence != 0.0 or self.frequency != 0.0

    @property
    def filtered(self) -> bool:
        """Whether its draws are more than a temperature's."""
        return self.counted or bool(self.bias) or self.temperature > 0 and (self.top_k > 0 or self.top_p < 1 or self.min_p > 0)

    @property
    def shaped(self) -> bool:
        """Whether it needs a round's logits as they are (a captured round perturbs them in place)."""
        return self.filtered or self.logprobs >= 0

    @classmethod
    def from_message(cls, msg: Dict[str, Any]) -> "SamplingParams":
        """Of a request of the line protocol (`serving/protocol.py`)."""
        return cls(temperature=float(msg.get("temperature", 0.0)), seed=int(msg.get("seed", 0)), top_k=int(msg.get("top_k", 0)), top_p=float(msg.get("top_p", 1.0)),
                   min_p=float(msg.get("min_p", 0.0)), repetition=float(msg.get("repetition_penalty", 1.0)), presence=float(msg.get("presence_penalty", 0.0)),
                   frequency=float(msg.get("frequency_penalty", 0.0)), bias=tuple((int(i), float(b)) for i, b in msg.get("logit_bias", ())),
                   logprobs=int(msg.get("logprobs", -1)))


def refusal(msg: Dict[str, Any], vocab: int) -> str:
    """Empty string if a request's settings can be served, else the reason."""
    def number(key, lo, hi, default, whole=False):
        v = msg.get(key, default)
        if isinstance(v, bool) or not isinstance(v, int if whole else (int, float)) or not lo <= v <= hi:    # (compared as it is: it may be no float's)
            return f"{key} must be {'an integer' if whole else 'a number'} from {lo} to {hi}"
        return ""
    bad = (number("top_k", -1, 1 << 30, 0, True) or number("top_p", 0.0, 1.0, 1.0) or number("min_p", 0.0, 1.0, 0.0)
           or number("presence_penalty", -10.0, 10.0, 0.0) or number("frequency_penalty", -10.0, 10.0, 0.0)
           or number("repetition_penalty", 0.01, 100.0, 1.0) or number("logprobs", -1, MAX_LOGPROBS, -1, True))
    if bad:
        return bad
    bias = msg.get("logit_bias", ())
    if not isinstance(bias, (list, tuple)) or len(bias) > MAX_BIASES:
        return f"logit_bias must be a list of at most {MAX_BIASES} [token, bias] pairs"
    for pair in bias:
        if not isinstance(pair, (list, tuple)) or len(pair) != 2 or isinstance(pair[0], bool) or not isinstance(pair[0], int) or not 0 <= pair[0] < vocab:
            return "logit_bias must name tokens of the vocabulary"
        if isinstance(pair[1], bool) or not isinstance(pair[1], (int, float)) or not -100.0 <= pair[1] <= 100.0:
            return "a logit_bias must be a number from -100 to 100"
    return ""
