"""A session's rules on logits without a device: a backend that keeps what it is given and computes LOGIT_RULES from its definition, under a model whose logits are a table."""
import numpy as np
import pytest

import batch_reference as ref
from zgml_b200 import DeviceProgram, abi
from zgml_b200.host.batch import LogitRules
from zgml_b200.host.session import LoweredProgram, SequenceSession

V = 40
LOGITS = np.random.default_rng(0).standard_normal((V, V)).astype(np.float32)      # after a token


class Backend:
    """Programs are dicts of buffers that stay from one execution to the next."""

    def __init__(self):
        self.compiled, self.freed, self.executed, self.refuse, self.uploaded = 0, 0, [], lambda program: False, []

    def compile_program(self, program):
        if self.refuse(program):
            return None
        self.compiled += 1
        return {"program": program, "buffers": [np.zeros(max(1, int(n)), np.int32) for n in program.buffer_sizes]}

    def free_program(self, handle):
        self.freed += 1

    def execute_program(self, handle, inputs, outputs):
        buffers = handle["buffers"]
        for io in inputs:
            words = np.ascontiguousarray(io.host).view(np.int32).ravel()
            assert io.offset % 4 == 0 and io.offset // 4 + words.size <= buffers[io.buf_idx].size
            buffers[io.buf_idx][io.offset // 4:io.offset // 4 + words.size] = words
            self.uploaded.append((io.buf_idx, words.size))
        self.executed.append((buffers[0][abi.CTL_POS], buffers[0][abi.CTL_IDS:].tolist()))
        for op in handle["program"].ops:
            if op.tag == abi.OP_LOGIT_RULES:
                b = op.u.seq.buf
                t = buffers[b[2]][abi.BATCH_ROWS:abi.BATCH_ROWS + abi.RULE_WORDS]
                row = (*t[:6].tolist(), *t[6:9].copy().view(np.float32).tolist())
                bias = buffers[b[4]].reshape(-1, 2)
                bias = list(zip(bias[:, 0].tolist(), bias[:, 1].copy().view(np.float32).tolist()))
                z, _ = ref.rules(np.zeros((1, V)), buffers[b[1]].view(np.float32).reshape(1, V), [row], 1, buffers[b[3]].reshape(1, -1)[:, :op.u.seq.n[4]], bias, buffers[b[5]].reshape(1, -1))
                buffers[b[0]][:] = z.astype(np.float32).view(np.int32).ravel()
            else:
                buffers[1][:] = LOGITS[buffers[0][abi.CTL_IDS:][-1]].view(np.int32)
        for io in outputs:
            io.host[...] = buffers[io.buf_idx].view(np.float32).reshape(io.host.shape)


class Model:
    vocab = V

    def state_specs(self, max_chunk, max_context):
        return []

    def lower(self, T, head, pool, keep_layers=False):
        ops = [] if head == "none" else [abi.ZgOp()]
        return LoweredProgram(DeviceProgram(ops, [abi.CTL_IDS + T, V]), 0, None if head == "none" else 1, 1)


def session(max_chunk=4, **kw):
    be = Backend()
    return SequenceSession(be, Model(), n_slots=2, max_chunk=max_chunk, **kw), be


def want(fed, prompt, rules):
    """The rules' result after the tokens `fed`, of which `prompt` were not generated."""
    masks = None if rules.allowed is None else rules.mask(V)[None]
    line = (0, len(fed), prompt, -1 if masks is None else 0, 0, len(rules.bias), rules.repetition, rules.presence, rules.frequency)
    z, _ = ref.rules(np.zeros((1, V)), LOGITS[fed[-1]][None], [line], 1, np.array([fed]), list(rules.bias.items()), masks)
    return z.astype(np.float32)


RULES = LogitRules(1.5, 0.25, 0.5, {3: 1.0})


def test_rules_over_a_request():
    s, _ = session()
    fed = [1, 2, 3, 4, 5, 6, 7]
    assert np.array_equal(s.feed("a", fed, [6], RULES), want(fed, 7, RULES))
    for t in (9, 9, 3):
        fed.append(t)
        assert np.array_equal(s.feed("a", [t], [0], RULES, generated=True), want(fed, 7, RULES))
    fed += [11, 12]                                     # another turn of the user's
    assert np.array_equal(s.feed("a", [11, 12], [1], RULES), want(fed, len(fed), RULES))


def test_a_request_that_begins_with_generated_tokens():
    s, _ = session()
    assert np.array_equal(s.feed("a", [5, 6, 5], [2], RULES, generated=True), want([5, 6, 5], 0, RULES))


@pytest.mark.parametrize("ruled_only", [True, False])
def test_a_step_that_cannot_be_compiled_leaves_nothing(ruled_only):
    """The request stays where it was, and the same tokens again count once."""
    s, be = session()
    s.feed("a", [1, 2, 2], [2])
    is_ruled = lambda program: any(op.tag == abi.OP_LOGIT_RULES for op in program.ops)
    be.refuse = is_ruled if ruled_only else lambda program: True
    for new in ([2, 7, 7, 7, 8, 7], [9]):
        with pytest.raises(RuntimeError):
            s.feed("a", new, [len(new) - 1], RULES)
        assert s.pool.position("a") == 3 and len(be.executed) == 2
    be.refuse = lambda program: False
    assert np.array_equal(s.feed("a", [2, 7], [1], RULES, generated=True), want([1, 2, 2, 2, 7], 3, RULES))


def test_a_step_that_fails_on_its_way():
    """What had run counts, what had not does not."""
    s, be = session()
    s.feed("a", [1], [0], RULES)
    run, left = be.execute_program, [1]

    def fails(*args):
        if not left:
            raise RuntimeError("no")
        left.pop()
        run(*args)
    be.execute_program = fails
    with pytest.raises(RuntimeError):
        s.feed("a", [2, 3, 4, 5, 6, 7], [5], RULES, generated=True)
    be.execute_program = run
    assert s.pool.position("a") == 5
    assert np.array_equal(s.feed("a", [6, 7], [1], RULES, generated=True), want([1, 2, 3, 4, 5, 6, 7], 1, RULES))


def test_a_history_longer_than_the_first_room():
    """Without a limit of the user's the room grows: programs with rules are made again."""
    s, be = session(max_chunk=32768)
    past = (np.arange(40000) % V).tolist()
    assert np.array_equal(s.feed("a", past, [39999], RULES), want(past, 40000, RULES))
    assert np.array_equal(s.feed("b", [1, 2], [1], RULES), want([1, 2], 2, RULES))
    compiled = be.compiled
    assert np.array_equal(s.feed("a", [7], [0], RULES, generated=True), want(past + [7], 40000, RULES))
    assert be.compiled <= compiled + 1                   # (the step of one token)
    s.close()
    assert be.freed == be.compiled


def test_generate_past_the_first_room():
    """The room is there before the first token: nothing is made again between two tokens."""
    s, be = session(max_chunk=32768)
    prompt = (np.arange(32766) % V).tolist()
    one = LogitRules(presence=100.0, repetition=1.0)
    out = s.generate(prompt, 12, rules=one)
    assert len(set(out)) == 12 and be.freed == 0
    fed = prompt + out[:-1]
    assert out[-1] == int(np.argmax(want(fed, len(prompt), one)))


def test_generate_refuses_at_the_start():
    s, be = session(max_history=10)
    with pytest.raises(ValueError):
        s.generate([1, 2, 3], 9, rules=LogitRules(presence=1.0))
    assert be.executed == [] and not s.pool.has("generate")
    assert len(s.generate([1, 2, 3], 8, rules=LogitRules(presence=1.0))) == 8
    assert s.generate([1, 2, 3], 0, rules=LogitRules(presence=1.0)) == []


@pytest.mark.parametrize("rules", [LogitRules(bias={3: 9.0}), LogitRules(allowed=np.array([5, 6]))])
def test_rules_that_read_no_history_have_no_limit(rules):
    s, be = session(max_history=4)
    fed = [1, 2, 3, 4, 5, 6]
    be.uploaded.clear()
    assert np.array_equal(s.feed("a", fed, [5], rules), want(fed, 6, rules))
    assert s.generate(fed, 20, rules=rules) and all(b != 3 for b, _ in be.uploaded)      # (the history's buffer)
    with pytest.raises(ValueError):
        s.feed("a", [1], [0], LogitRules(frequency=0.5))
    assert s.pool.position("a") == 6


def test_generate_until_a_stop():
    """A number of tokens that is never reached asks for no memory."""
    s, be = session()
    rules = LogitRules(presence=100.0)
    few = s.generate([1, 2], 6, rules=rules)
    assert s.generate([1, 2], 10 ** 12, stop=few[-1], rules=rules) == few
    assert s._room <= 1 << 19


def test_a_history_goes_to_a_program_once():
    """Between two tokens of one request only what is new is uploaded; another request's tokens take its place."""
    s, be = session()
    fed = {"a": [1, 2, 3, 4, 5], "b": [6, 7]}
    for k, t in fed.items():
        s.feed(k, t, [len(t) - 1], RULES)
    words = []
    for step, k in enumerate(["a", "a", "a", "b", "a", "b", "b"]):
        fed[k].append(10 + step)
        be.uploaded.clear()
        prompt = 5 if k == "a" else 2
        assert np.array_equal(s.feed(k, fed[k][-1:], [0], RULES, generated=True), want(fed[k], prompt, RULES))
        words.append(sum(n for b, n in be.uploaded if b == 3))
    assert words == [1, 1, 1, 3, 9, 4, 1]                # (the first steps of one token found the last chunk of the prompt's program, which is theirs too)


def test_rules_that_change_between_tokens():
    """What a request asks is read anew in each step."""
    s, _ = session()
    rules = LogitRules(1.25, bias={1: 1.0})
    fed = [3, 4]
    s.feed("a", fed, [1], rules)
    for t in (5, 6):
        rules.bias = {t: 2.0}
        rules.presence = 0.5
        fed.append(t)
        assert np.array_equal(s.feed("a", [t], [0], rules, generated=True), want(fed, 2, rules))


def test_an_execution_that_fails_behind_its_uploads():
    """What it left in the history's buffer belongs to nobody."""
    s, be = session()
    s.feed("a", [1, 2, 3, 4, 5], [4], RULES)
    run = be.execute_program

    def fails(*args):
        run(*args)
        raise RuntimeError("no")
    be.execute_program = fails
    with pytest.raises(RuntimeError):
        s.feed("b", [9], [0], RULES)
    be.execute_program = run
    assert np.array_equal(s.feed("a", [6], [0], RULES, generated=True), want([1, 2, 3, 4, 5, 6], 5, RULES))
    assert np.array_equal(s.feed("b", [8], [0], RULES, generated=True), want([8], 0, RULES))
    s.release("a")
    assert np.array_equal(s.feed("a", [7], [0], RULES), want([7], 1, RULES))


@pytest.mark.parametrize("make", [lambda: LogitRules(bias={1.5: 2.0}), lambda: LogitRules(bias={"3": 2.0}), lambda: LogitRules(allowed=np.array([1.0, 2.5])).mask(V), lambda: LogitRules(allowed=["1"]).mask(V)])
def test_token_ids_are_whole_numbers(make):
    """2.5 is no token, and not token 2 either."""
    with pytest.raises(ValueError):
        make()


def test_token_ids_of_any_integer_type():
    r = LogitRules(bias={np.int64(3): 2.0, np.uint8(4): 1.0}, allowed=np.array([3, 4], np.uint16))
    assert r.mask(V).tolist() == [24, 0] and LogitRules(allowed=[]).mask(V).tolist() == [0, 0] and LogitRules(allowed=[True] * V).mask(V).tolist() == [-1, 255]


def test_generate_stops_where_no_token_is_left():
    s, be = session()
    with pytest.raises(ValueError):
        s.generate([1, 2], 4, rules=LogitRules(allowed=np.array([], np.int64)))
    assert not s.pool.has("generate") and (s.feed("a", [1], [0], LogitRules(allowed=[])) == -np.inf).all()      # (a row of logits says it by itself)


@pytest.mark.parametrize("option", [["--repetition-penalty", "0"], ["--presence-penalty", "inf"], ["--bias", "3:nan"], ["--bias", "3"], ["--allow", "x"]])
def test_the_command_line_refuses_before_it_loads_a_model(monkeypatch, option):
    from zgml_b200 import cli

    def no_device():
        raise AssertionError("a model would be loaded")
    monkeypatch.setattr(cli, "_backend", no_device)
    with pytest.raises(ValueError):
        cli.main(["generate", "--model", "none", "--prompt", "1,2", "--max-new-tokens", "1", *option])
