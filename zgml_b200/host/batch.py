"""Tables of the ops that advance many requests in one step (BATCH_APPEND, SHARED_ATTENTION, ADAPTER_LINEAR, LOGIT_RULES, SAMPLE and the ops over pages): what tells the rows apart, as the
words that a program's table buffer is given before every execution.  The kernels check every word once more before it becomes an address; what is
refused here would come back as rows of NaN."""
from dataclasses import dataclass, field
from typing import Dict, List, Optional, Sequence

import numpy as np

from .. import abi


@dataclass(frozen=True)
class BatchRow:
    """A token of some request: the slot of its caches, how many positions of its own sequence (behind the shared prefix) it sees, its own included, and its
    request's adapter (-1: none).  Slot -1: an idle row."""
    slot: int
    length: int = 0
    adapter: int = -1


def table_words(rows: int) -> int:
    """f32 slots of the table buffer of `rows` rows."""
    return abi.BATCH_ROWS + abi.BATCH_WORDS * rows


def rule_words(rows: int) -> int:
    return abi.BATCH_ROWS + abi.RULE_WORDS * rows


def batch_table(entries: Sequence[BatchRow], rows: int, prefix: int = 0, prefix_slot: int = 0, slots: Optional[int] = None, capacity: Optional[int] = None,
                prefix_capacity: Optional[int] = None, adapters: Optional[int] = None) -> np.ndarray:
    """The table of a step whose program takes `rows` rows; the rows behind the last entry are not live.  `slots`, `capacity` (rows of a slot), `prefix_capacity` and
    `adapters`, where given, are checked against."""
    if len(entries) > rows:
        raise ValueError(f"{len(entries)} rows for a step of {rows}")
    if prefix < 0 or prefix_slot < 0 or (prefix_capacity is not None and prefix > prefix_capacity):
        raise ValueError(f"a prefix of {prefix} positions in slot {prefix_slot}")
    t = np.zeros(table_words(rows), np.int32)
    t[0], t[1], t[2] = len(entries), prefix, prefix_slot
    body = t[abi.BATCH_ROWS:].reshape(rows, abi.BATCH_WORDS)
    for i, e in enumerate(entries):
        if e.length < 0 or (slots is not None and e.slot >= slots) or (capacity is not None and e.length > capacity) or (adapters is not None and e.adapter >= adapters):
            raise ValueError(f"row {i}: {e} is outside its buffers")
        body[i, :3] = e.slot, e.length, e.adapter
    return t


@dataclass
class LogitRules:
    """What a request asks of its next token.  A token that its history names has its logit divided (positive) or multiplied (negative) by `repetition`; one that was
    generated (history from the prompt's end on) c times loses presence + frequency * c; `bias` is added; with `allowed` (token ids, or truth values
    over the vocabulary) every other token gets -inf."""
    repetition: float = 1.0
    presence: float = 0.0
    frequency: float = 0.0
    bias: Dict[int, float] = field(default_factory=dict)
    allowed: Optional[np.ndarray] = None

    def __post_init__(self):
        with np.errstate(over="ignore", under="ignore"):            # (what they are to the kernel)
            repetition, *others = (np.float32(x) for x in (self.repetition, self.presence, self.frequency))
            biases = [np.float32(x) for x in self.bias.values()]
        if not (np.isfinite(repetition) and repetition > 0.0):
            raise ValueError("repetition is a factor above zero")
        if not np.isfinite(others).all():
            raise ValueError("presence and frequency are finite")
        if np.isnan(biases).any():
            raise ValueError("a bias is not a number")
        self._check_ids()

    def _check_ids(self):
        if not all(isinstance(k, (int, np.integer)) for k in self.bias):
            raise ValueError("a bias names its token by a whole number")

    @property
    def reads_history(self) -> bool:
        """Whether any history can change a logit, with these numbers as the kernel's f32."""
        with np.errstate(over="ignore", under="ignore"):
            return bool(np.float32(self.repetition) != 1.0 or np.float32(self.presence) != 0.0 or np.float32(self.frequency) != 0.0)

    def mask(self, vocab: int) -> Optional[np.ndarray]:
        """int32 words, bit t % 32 of word t / 32 set where token t is allowed."""
        if self.allowed is None:
            return None
        a = np.asarray(self.allowed)
        if a.dtype == np.bool_:
            if a.shape != (vocab,):
                raise ValueError(f"truth values for {a.shape} tokens over a vocabulary of {vocab}")
            bits = a
        else:
            if a.size and a.dtype.kind not in "iu":
                raise ValueError("allowed tokens are whole numbers, or truth values over the vocabulary")
            ids = a.astype(np.int64).ravel()
            if ids.size and (ids.min() < 0 or ids.max() >= vocab):
                raise ValueError("an allowed token is outside the vocabulary")
            bits = np.zeros(vocab, np.bool_)
            bits[ids] = True
        words = np.packbits(np.concatenate([bits, np.zeros(-vocab % 32, np.bool_)]), bitorder="little")
        return words.view("<i4").astype(np.int32)


def rule_table(rules: Sequence[LogitRules], slots: Sequence[int], lengths: Sequence[int], firsts: Sequence[int], vocab: int, rows: int):
    """(table, bias entries [n, 2], masks [m, words]) of a step: request i's history is the first lengths[i] words of slot slots[i], generated from word firsts[i] on.
    Every array is int32 (biases: the bits of their f32 values)."""
    if not len(rules) == len(slots) == len(lengths) == len(firsts) <= rows:
        raise ValueError("one slot, length and first generated word for each of the step's rules")
    t = np.zeros(rule_words(rows), np.int32)
    t[0] = len(rules)
    body = t[abi.BATCH_ROWS:].reshape(rows, abi.RULE_WORDS)
    entries: List[tuple] = []
    masks: List[np.ndarray] = []
    for i, r in enumerate(rules):
        if lengths[i] < 0 or firsts[i] < 0:
            raise ValueError(f"row {i}: a history of {lengths[i]} words generated from word {firsts[i]} on")
        r._check_ids()
        if any(not 0 <= k < vocab for k in r.bias):
            raise ValueError("a bias names a token outside the vocabulary")
        m = r.mask(vocab)
        body[i, :6] = slots[i], lengths[i], firsts[i], -1 if m is None else len(masks), len(entries), len(r.bias)
        body[i, 6:9] = np.array([r.repetition, r.presence, r.frequency], np.float32).view(np.int32)
        if m is not None:
            masks.append(m)
        entries += list(r.bias.items())
    bias = np.zeros((len(entries), 2), np.int32)
    if entries:
        bias[:, 0] = [k for k, _ in entries]
        bias[:, 1] = np.array([v for _, v in entries], np.float32).view(np.int32)
    return t, bias, np.stack(masks) if masks else np.zeros((0, (vocab + 31) // 32), np.int32)


@dataclass(frozen=True)
class TokenChoice:
    """How a request's next token is drawn: of the softmax of logits / temperature the `top_k` likeliest tokens stay (0: all), of those the fewest whose probability reaches
    `top_p` of theirs, of those the ones with at least `min_p` times the likeliest one's.  Temperature 0: the likeliest token."""
    temperature: float = 1.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0

    def __post_init__(self):
        with np.errstate(over="ignore", under="ignore"):            # (what they are to the kernel)
            temperature, top_p, min_p = (np.float32(x) for x in (self.temperature, self.top_p, self.min_p))
        if not (np.isfinite(temperature) and temperature >= 0.0):
            raise ValueError("a temperature is a finite number, zero or more")
        if not (0.0 <= top_p <= 1.0 and 0.0 <= min_p <= 1.0):
            raise ValueError("top_p and min_p are probabilities")
        if not isinstance(self.top_k, (int, np.integer)) or not 0 <= self.top_k < 1 << 31:
            raise ValueError("top_k is a whole number, zero or more")


def sample_words(rows: int) -> int:
    return abi.BATCH_ROWS + abi.SAMPLE_WORDS * rows


def sample_table(choices: Sequence[Optional[TokenChoice]], draws: Sequence[float], rows: int) -> np.ndarray:
    """The table of a SAMPLE of `rows` rows of logits: a choice (None: the row is idle) and a random number of [0, 1) for each of the first ones, rounded to f32 below 1."""
    if len(choices) != len(draws) or len(choices) > rows:
        raise ValueError(f"{len(choices)} choices and {len(draws)} random numbers for a step of {rows}")
    t = np.zeros(sample_words(rows), np.int32)
    t[0] = len(choices)
    body = t[abi.BATCH_ROWS:].reshape(rows, abi.SAMPLE_WORDS)
    for i, (c, u) in enumerate(zip(choices, draws)):
        if not 0.0 <= u < 1.0:
            raise ValueError(f"row {i}: {u} as a random number of [0, 1)")
        if c is None:
            body[i, 1] = -1
            continue
        u = min(np.float32(u), np.nextafter(np.float32(1.0), np.float32(0.0)))
        body[i, [0, 2, 3, 4]] = np.array([c.temperature, c.top_p, c.min_p, u], np.float32).view(np.int32)
        body[i, 1] = c.top_k
    return t
