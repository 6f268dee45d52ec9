"""Serving session over compiled device programs: the step function every sequence model of the framework is driven by.

A model object provides
  * `vocab`                       — logits per position,
  * `state_specs(max_chunk, max_context)` — the per-sequence device state it carries between steps (host/state.py); a model
                                    that caches every position (`bounded_context`) sizes its caches for `max_context`
                                    positions, and the session refuses to advance a sequence past them,
  * `lower(T, head, pool)`        — the DeviceProgram that advances one sequence by exactly T tokens from the pool's
                                    state (`head` = "none" | "last" | "all": which positions' logits it produces).

`SequenceSession.feed(request, tokens, want)` cuts the request's next tokens into chunks from a fixed menu of program
sizes (powers of two up to `max_chunk`, compiled on first use and kept), writes the control buffer (position, state slot,
previous token, token ids) and executes; the CUDA graph of a program is replayed unchanged from step to step.  How a prompt is cut
changes nothing but rounding: state is carried exactly, and every chunk attends through the same key ring.
`feed(..., rules=LogitRules(...))` asks for the last place's logits as the request's penalties, biases and grammar mask leave them: LOGIT_RULES joins the program that
makes them, over the tokens that the session has fed for the request.
`step(entries, end)` is the batch form (requests are advanced one after the other, each alone in its program, so a
request's logits cannot depend on its neighbours); `generate` is greedy / sampled decoding on top of `feed`.
"""
from dataclasses import dataclass
from typing import Dict, Iterable, List, Optional, Sequence, Tuple

import numpy as np

from .. import abi
from ..backend import CudaBackend, DeviceOp, DeviceProgram, ProgramIO
from .batch import LogitRules, rule_table, rule_words
from .sampling import Sampler
from .state import SequenceStatePool


@dataclass
class LoweredProgram:
    program: DeviceProgram
    buf_ctl: int
    buf_logits: Optional[int]      # None for head == "none"
    logits_rows: int
    layer_bufs: Optional[List[int]] = None   # residual stream after every layer (debug lowering only)
    rule_bufs: Optional[Tuple[int, int, int, int]] = None    # table, history, biases and mask of LOGIT_RULES, which made the logits


def chunk_menu(max_chunk: int) -> List[int]:
    m, out = 1, []
    while m <= max_chunk:
        out.append(m)
        m *= 2
    return out[::-1]


def cut(n: int, menu: Sequence[int]) -> List[int]:
    """Greedy decomposition of n tokens into menu sizes, largest first."""
    out = []
    for m in menu:
        while n >= m:
            out.append(m)
            n -= m
    assert n == 0
    return out


class History:
    """The tokens fed for a request, int32 words that grow in place: `n` of them count, those from `prompt` on as generated."""

    def __init__(self):
        self.words, self.n, self.prompt = np.zeros(64, np.int32), 0, 0

    def put(self, tokens: Sequence[int]):
        """Writes the tokens of a step behind those that count; they do once `advance` is told."""
        need = self.n + len(tokens)
        if need > self.words.size:
            self.words = np.concatenate([self.words[:self.n], np.zeros(max(need, 2 * self.words.size) - self.n, np.int32)])
        self.words[self.n:need] = tokens

    def advance(self, T: int, generated: bool):
        self.n += T
        if not generated:
            self.prompt = self.n


class SequenceSession:
    def __init__(self, be: CudaBackend, model, n_slots: int = 1, max_chunk: int = 256, keep_layers: bool = False,
                 max_context: Optional[int] = None, max_history: Optional[int] = None, max_bias: int = 1024):
        """`max_history` tokens of a request, `max_bias` biases: the most that steps with rules take.  Without a `max_history` the programs with rules have room for
        32768 tokens and are compiled again, for twice as many or more, when a request has more of them."""
        self.max_history, self.max_bias = max_history, max_bias
        self._room = 32768 if max_history is None else max(1, max_history)      # words of a history in the programs with rules
        self._history: Dict[object, History] = {}
        self._uploaded: Dict[tuple, Tuple[History, int]] = {}      # program with rules -> whose tokens its history buffer begins with, and how many
        self.be, self.model, self.keep_layers = be, model, keep_layers
        self.menu = chunk_menu(max_chunk)
        self.max_chunk = self.menu[0]
        self.pool = SequenceStatePool(be, model.state_specs(self.max_chunk, max_context), n_slots)
        self.context_limit = model.capacity(self.max_chunk, max_context) if getattr(model, "bounded_context", False) else None
        self._programs: Dict[Tuple[int, str], tuple] = {}
        self.executions = 0

    # ── programs ──
    def _with_rules(self, lp: LoweredProgram) -> LoweredProgram:
        """The program whose one row of logits passes LOGIT_RULES on its way out."""
        V, p = self.model.vocab, lp.program
        n = p.n_buffers
        table, history, bias, mask, out = range(n, n + 5)
        sizes = list(p.buffer_sizes) + [rule_words(1), self._room, 2 * self.max_bias, (V + 31) // 32, V]
        op = DeviceOp.logit_rules(out, lp.buf_logits, table, 1, V, history=history, history_rows=self._room, bias=bias, masks=mask)
        return LoweredProgram(DeviceProgram(list(p.ops) + [op], sizes, p.initial_uploads, p.qweights, p.externs), lp.buf_ctl, out, lp.logits_rows, lp.layer_bufs,
                              (table, history, bias, mask))

    def _check_history(self, rules: LogitRules, tokens: int):
        if self.max_history is not None and rules.reads_history and tokens > self.max_history:
            raise ValueError(f"rules over {tokens} tokens: the session takes {self.max_history}")

    def _make_room(self, rules: LogitRules, tokens: int):
        if not rules.reads_history or tokens <= self._room:
            return
        self._room = max(tokens, 2 * self._room)
        for key in [k for k in self._programs if len(k) == 3]:
            self.be.free_program(self._programs.pop(key)[1])
        self._uploaded = {}

    def program(self, T: int, head: str, ruled: bool = False):
        key = (T, head, True) if ruled else (T, head)
        if key not in self._programs:
            lp = self.model.lower(T, head, self.pool, keep_layers=self.keep_layers)
            if ruled:
                lp = self._with_rules(lp)
            handle = self.be.compile_program(lp.program)
            if handle is None:
                from ..backend import last_error
                raise RuntimeError(f"compile_program failed for T = {T}, head = {head}: {last_error()}")
            ctl = np.zeros(abi.CTL_IDS + T, np.int32)
            logits = np.zeros((lp.logits_rows, self.model.vocab), np.float32) if lp.buf_logits is not None else None
            self._programs[key] = (lp, handle, ctl, logits)
        return self._programs[key]

    def _run(self, T, head, slot, pos, prev, tokens, past: Optional[History] = None, rule_words=None):
        """With rules: the request's history, this step's tokens behind those that count, and the words of rule_table."""
        lp, handle, ctl, logits = self.program(T, head, rule_words is not None)
        ctl[abi.CTL_POS], ctl[abi.CTL_SLOT], ctl[abi.CTL_PREV] = pos, slot, prev
        ctl[abi.CTL_IDS:] = tokens
        outs = [ProgramIO(lp.buf_logits, logits)] if logits is not None else []
        ins = [ProgramIO(lp.buf_ctl, ctl)]
        if rule_words is not None:
            table, bias, masks = rule_words
            at, history, biases, mask = lp.rule_bufs
            ins += [ProgramIO(b, a) for b, a in ((at, table), (biases, bias.ravel()), (mask, masks.ravel())) if a.size]
            n = int(table[abi.BATCH_ROWS + 1])                      # tokens that the rules read
            if n:                                                   # a history only grows: what the buffer holds of it stays
                owner, there = self._uploaded.pop((T, head), (None, 0))      # (back when this execution is through)
                there = there if owner is past else 0
                ins.append(ProgramIO(history, past.words[there:n], 4 * there))
        self.be.execute_program(handle, ins, outs)
        if rule_words is not None and n:
            self._uploaded[(T, head)] = (past, n)
        self.executions += 1
        return logits

    # ── the step function ──
    def feed(self, request_id, tokens: Sequence[int], want: Iterable[int] = (), rules: Optional[LogitRules] = None, generated: bool = False) -> np.ndarray:
        """Advance `request_id` by `tokens`; returns the logits at the places `want` (indices into `tokens`), in order.  With `rules` (the last place alone may be wanted)
        they are what the rules make of them, over all tokens fed for the request; those fed with `generated` since the last ones without it count as generated."""
        tokens = [int(t) for t in tokens]
        if any(t < 0 or t >= self.model.vocab for t in tokens):
            raise ValueError("token id outside the vocabulary")
        want = [int(w) for w in want]
        if any(w < 0 or w >= len(tokens) for w in want):
            raise ValueError("wanted place outside the step's tokens")
        past = self._history.get(request_id) or History()
        if rules is not None:
            if any(w != len(tokens) - 1 for w in want):
                raise ValueError("rules apply to the logits of a step's last place")
            self._check_history(rules, past.n + len(tokens))
            if len(rules.bias) > self.max_bias:
                raise ValueError(f"{len(rules.bias)} biases: the session takes {self.max_bias}")
            n = past.n + len(tokens) if rules.reads_history else 0
            words = rule_table([rules], [0], [n], [past.prompt if generated and n else n], self.model.vocab, 1)
        slot = self.pool.acquire(request_id)
        if self.context_limit is not None and self.pool.position(request_id) + len(tokens) > self.context_limit:
            raise ValueError(f"request {request_id!r} would reach position {self.pool.position(request_id) + len(tokens)}: the session's caches hold "
                             f"{self.context_limit} positions per sequence")
        self._history[request_id] = past
        if rules is not None:
            self._make_room(rules, past.n + len(tokens))
        plan, at = [], 0
        for T in cut(len(tokens), self.menu):
            local = sorted({w - at for w in want if at <= w < at + T})
            head = "none" if not local else ("last" if local == [T - 1] else "all")
            self.program(T, head, rules is not None and bool(local))     # what cannot be compiled is known before anything runs
            plan.append((at, T, head, local))
            at += T
        rows: Dict[int, np.ndarray] = {}
        for at, T, head, local in plan:
            step = tokens[at:at + T]
            past.put(step)
            logits = self._run(T, head, slot, self.pool.position(request_id), self.pool.last_token(request_id), step, *((past, words) if rules is not None and local else ()))
            for w in local:
                rows[at + w] = logits[0 if head == "last" else w].copy()
            self.pool.advance(request_id, T, step[-1])
            past.advance(T, generated)
        return np.stack([rows[w] for w in want]) if want else np.zeros((0, self.model.vocab), np.float32)

    def release(self, request_id):
        self.pool.release(request_id)
        self._history.pop(request_id, None)

    def step(self, entries: Sequence[dict], end: Iterable = ()) -> List[np.ndarray]:
        """entries: [{"id", "tokens", "want", "rules", "generated"}] (the last three may be absent); `end`: requests whose state is given back after the step."""
        out = [self.feed(e["id"], e["tokens"], e.get("want", ()), e.get("rules"), e.get("generated", False)) for e in entries]
        for r in end:
            self.release(r)
        return out

    def layer_streams(self, T: int, head: str) -> np.ndarray:
        """Residual stream after every layer of the last execution of program (T, head); needs keep_layers."""
        lp, handle, _, _ = self._programs[(T, head)]
        assert lp.layer_bufs is not None
        width = self.model.width
        out = np.zeros((len(lp.layer_bufs), T, width), np.float32)
        for i, b in enumerate(lp.layer_bufs):
            self.be.read_buffer(handle, b, out[i])
        return out

    def generate(self, prompt: Sequence[int], max_new_tokens: int, sampler: Optional[Sampler] = None, request_id="generate",
                 stop: Optional[int] = None, rules: Optional[LogitRules] = None) -> List[int]:
        """Prefill `prompt`, then decode token by token through the same step function; with `rules` the sampler sees logits that have passed them."""
        sampler = sampler or Sampler()
        if rules is not None:                            # what it will look back at has room, or is refused, before the first token
            past = self._history.get(request_id) or History()
            tokens = past.n + len(prompt) + max(0, max_new_tokens - 1)
            self._check_history(rules, tokens)
            self._make_room(rules, min(tokens, past.n + len(prompt) + (1 << 18)))      # (the most that it makes for tokens that may never come)
        logits = self.feed(request_id, prompt, [len(prompt) - 1], rules)[0]
        out: List[int] = []
        try:
            for _ in range(max_new_tokens):
                if rules is not None and logits.max() == -np.inf:
                    raise ValueError(f"the rules leave no token to choose after {len(out)} of them")
                tok = sampler(logits)
                out.append(tok)
                if stop is not None and tok == stop:
                    break
                if len(out) < max_new_tokens:
                    logits = self.feed(request_id, [tok], [0], rules, generated=True)[0]
        finally:
            self.release(request_id)
        return out

    def close(self):
        for _, handle, _, _ in self._programs.values():
            self.be.free_program(handle)
        self._programs = {}
        self.pool.close()
