"""The batched ops as they are used: a decode loop of several requests behind one prefix through projection, adapters, cache rows, attention, head and rules; steps of two sizes
over the same caches; another stream; a device without room for workspaces; and the sessions' rules on logits against the raw logits."""
import numpy as np
import pytest

import batch_reference as ref
from lududra_models import attention_layer, config, delta_layer, random_weights
from test_gpu_batchops import adapter_case, attend_case, close, table

pytestmark = pytest.mark.gpu


class Loop:
    """A one-layer decoder over `prefix` shared positions, lowered for batches of any size over the same caches, and the same in NumPy."""
    D, H, G, d, V, P, R, A, rank, rot = 64, 4, 2, 16, 50, 20, 8, 3, 8, 8

    def __init__(self, be, slots):
        from zgml_b200 import DeviceBuffer
        r = np.random.default_rng(3)
        self.be, self.slots, self.kv = be, slots, 2 * self.G * self.d
        n_qkv = self.H * self.d + self.kv
        f = lambda *s: (r.standard_normal(s) / np.sqrt(s[-1])).astype(np.float32)
        self.w = dict(qkv=f(n_qkv, self.D), out=f(self.D, self.H * self.d), head=3 * f(self.V, self.D), a=f(self.A, self.rank, self.D), b=f(self.A, n_qkv, self.rank))
        self.emb, self.scales = r.standard_normal((self.V, self.D)).astype(np.float32), np.array([0.5, 1.0, 2.0], np.float32)
        self.pre = r.standard_normal((1, self.P, self.kv)).astype(np.float32)
        self.own = np.zeros((slots, self.R, self.kv))
        self.off, flat, n = {}, [], 0
        for k, v in self.w.items():
            self.off[k] = n
            flat.append(v.ravel())
            n += v.size
        self.n_qkv, self.bufs = n_qkv, {}
        for name, a in (("w", np.concatenate(flat)), ("own", np.zeros(slots * self.R * self.kv, np.float32)), ("pre", self.pre), ("scales", self.scales)):
            self.bufs[name] = DeviceBuffer(be, a.nbytes)
            self.bufs[name].upload(np.ascontiguousarray(a))
        self.programs = {}

    def program(self, B):
        from zgml_b200 import DeviceOp, DeviceProgram, ExternBuffer, abi
        from zgml_b200.host.batch import rule_words, table_words
        if B in self.programs:
            return self.programs[B]
        sizes, ext = [], []

        def buf(n):
            sizes.append(n)
            return len(sizes) - 1
        at = {}
        for k, b in self.bufs.items():
            at[k] = buf(b.elems)
            ext.append(ExternBuffer(at[k], b))
        D, H, G, d, V, kv, q = self.D, self.H, self.G, self.d, self.V, self.kv, self.n_qkv
        for k, n in (("x", B * D), ("qkv", B * q), ("table", table_words(B)), ("turned", B * H * d), ("att", B * H * d), ("y", B * D), ("logits", B * V), ("rules", rule_words(B)), ("history", self.slots * 32),
                     ("bias", 2 * 16), ("masks", B * 2)):
            at[k] = buf(n)
        f32, o = abi.W_F32, self.off
        ops = [DeviceOp.linear(at["qkv"], at["x"], at["w"], o["qkv"], B, q, D, f32),
               DeviceOp.adapter_linear(at["qkv"], at["x"], at["w"], o["a"], o["b"], at["table"], B, q, D, self.rank, self.A, f32, scales=at["scales"]),
               DeviceOp.batch_append(at["own"], at["qkv"], at["table"], H * d, 0, B, kv, q, kv, self.R, key_heads=G, head_dim=d, turn_at=4, rot=self.rot, rot_base=1e4, q_heads=H, turned=at["turned"]),
               DeviceOp.shared_attention(at["att"], at["turned"], at["own"], at["own"], at["pre"], at["pre"], at["table"], 0, 0, G * d, 0, G * d, B, H, G, d, d, H * d, kv, kv, self.R, kv, kv, self.P, d ** -0.5),
               DeviceOp.linear(at["y"], at["att"], at["w"], o["out"], B, D, H * d, f32),
               DeviceOp.linear(at["logits"], at["y"], at["w"], o["head"], B, V, D, f32),
               DeviceOp.logit_rules(at["logits"], at["logits"], at["rules"], B, V, history=at["history"], history_rows=32, bias=at["bias"], masks=at["masks"])]
        h = self.be.compile_program(DeviceProgram(ops, sizes, [], [], ext))
        assert h is not None
        self.programs[B] = (h, at)
        return self.programs[B]

    def step(self, tokens, rows, rules, history):
        """One token of each row's request; -> (logits of the device, of NumPy)."""
        from zgml_b200 import ProgramIO
        from zgml_b200.host.batch import batch_table, rule_table
        B = len(rows)
        h, at = self.program(B)
        x = self.emb[tokens]
        past = np.zeros((self.slots, 32), np.int32)
        for s, t in history.items():
            past[s, :len(t)] = t
        t = batch_table(rows, B, self.P, 0, self.slots, self.R, self.P, self.A)
        rt, bias, masks = rule_table(rules, [r.slot for r in rows], [len(history[r.slot]) for r in rows], [1] * B, self.V, B)
        got = np.zeros((B, self.V), np.float32)
        ins = [("x", x), ("table", t), ("rules", rt), ("history", past), ("bias", bias), ("masks", masks)]
        self.be.execute_program(h, [ProgramIO(at[k], np.ascontiguousarray(v).ravel()) for k, v in ins if v.size], [ProgramIO(at["logits"], got)])
        w = {k: v.astype(np.float64) for k, v in self.w.items()}
        entries = [(r.slot, r.length, r.adapter) for r in rows]
        qkv, _ = ref.adapt(np.zeros((B, self.n_qkv)), x.astype(np.float64) @ w["qkv"].T, x, self.w["a"], self.w["b"], self.scales, entries, B)
        H, G, d = self.H, self.G, self.d
        self.own, turned = ref.append(self.own, qkv, entries, B, self.P, H * d, 0, self.kv, G, d, 4, self.rot, 1e4, "pairs", H, 0, np.zeros((B, H * d)))
        heads = lambda c, col: c[:, :, col:col + G * d].reshape(c.shape[0], c.shape[1], G, d)
        att, _ = ref.attend(np.zeros((B, H, d)), turned.reshape(B, H, d), heads(self.own, 0), heads(self.own, G * d), heads(self.pre, 0), heads(self.pre, G * d), entries, B, self.P, 0, d ** -0.5)
        logits = att.reshape(B, H * d) @ w["out"].T @ w["head"].T
        lines = []
        for i, (r, q) in enumerate(zip(rows, rules)):
            lines.append((r.slot, len(history[r.slot]), 1, -1 if q.allowed is None else i, 0, 0, q.repetition, q.presence, q.frequency))
        want, _ = ref.rules(np.zeros((B, self.V)), logits, lines, B, past, [], np.stack([q.mask(self.V) if q.allowed is not None else np.zeros(2, np.int32) for q in rules]))
        for i, q in enumerate(rules):
            for k, v in q.bias.items():
                want[i, k] += v
        return got, want

    def close(self):
        for h, _ in self.programs.values():
            self.be.free_program(h)
        for b in self.bufs.values():
            b.free()


def test_decode_loop(cuda_backend):
    """Seven steps of five requests with adapters and rules of their own, two of which pause every third step (a smaller program over the same caches).  The longest chain has
    sums of 64, 8, 28, 64 and 64 terms: 228 roundings of 2^-24, which weights of about one pass on; four times that is allowed."""
    from zgml_b200.host.batch import BatchRow, LogitRules
    L = Loop(cuda_backend, 6)
    slots, adapters, length, token = [4, 0, 2, 5, 1], [0, -1, 2, 1, 2], [0] * 5, [3, 9, 11, 30, 49]
    history = {s: [t] for s, t in zip(slots, token)}
    rules = [LogitRules(), LogitRules(1.3, 0.5, 0.25), LogitRules(bias={7: 2.5, 8: -1.0}), LogitRules(repetition=2.0, allowed=np.arange(0, 50, 3)), LogitRules(presence=1.0)]
    for step in range(7):
        alive = [0, 1, 2, 3, 4] if step % 3 != 2 else [4, 1, 0]
        for i in alive:
            length[i] += 1
        got, want = L.step([token[i] for i in alive], [BatchRow(slots[i], length[i], adapters[i]) for i in alive], [rules[i] for i in alive], history)
        scale = np.abs(want[np.isfinite(want)]).max()
        close(got, want, 4 * 228 * 2.0 ** -24 * scale, step)
        for i, z in zip(alive, got):
            token[i] = int(np.argmax(z))
            history[slots[i]].append(token[i])
    assert all(t % 3 == 0 for t in history[5][1:])
    L.close()


def test_on_another_stream():
    import torch
    from zgml_b200 import CudaBackend
    be = CudaBackend(0)
    stream = torch.cuda.Stream()
    be.set_stream(stream.cuda_stream)
    attend_case(be, 40, 8, 2, 64, 64, 300, 17, [(i, 1 + i % 17, 0) for i in range(40)])
    adapter_case(be, "bf16", 300, 136, 64, 16, 3, [(0, 0, i // 70 - 1) for i in range(300)])
    be.close()


def test_without_workspaces(cuda_backend, monkeypatch):
    """Where there is no room for records and parts the ops run in forms that need none."""
    monkeypatch.setenv("ZG_CUDA_SCRATCH_MB", "0")
    attend_case(cuda_backend, 40, 8, 2, 64, 64, 300, 17, [(i, 1 + i % 17, 0) for i in range(40)])
    attend_case(cuda_backend, 1, 1, 1, 64, 64, 4000, 17, [(0, 17, 0)])
    adapter_case(cuda_backend, "f32", 300, 136, 64, 16, 3, [(0, 0, i // 70 - 1) for i in range(300)])


def test_few_rows_over_many_keys(cuda_backend):
    """More shares than a cluster has CTAs: records and a second launch."""
    attend_case(cuda_backend, 1, 1, 1, 64, 64, 9000, 100, [(0, 77, 0)])
    attend_case(cuda_backend, 2, 3, 1, 128, 96, 5000, 3, [(1, 0, 0), (0, 3, 0)], sink="f32")
    attend_case(cuda_backend, 3, 2, 1, 64, 64, 3000, 10, [(0, 3, 0), (-1, 0, 0), (1, 11, 0)])


def test_two_programs_at_once(cuda_backend):
    """Replays of two programs in turns, each with workspaces of its own."""
    from zgml_b200 import DeviceOp, DeviceProgram, ProgramIO
    r = np.random.default_rng(0)
    handles = []
    for seed in range(2):
        q, own, pre = r.standard_normal((48, 8 * 64)).astype(np.float32), r.standard_normal((48, 5, 256)).astype(np.float32), r.standard_normal((1, 1100, 256)).astype(np.float32)
        t = table([(i, 1 + i % 5, 0) for i in range(48)], 48, 1100)
        op = DeviceOp.shared_attention(0, 1, 2, 2, 3, 3, 4, 0, 0, 128, 0, 128, 48, 8, 2, 64, 64, 512, 256, 256, 5, 256, 256, 1100, 0.125)
        h = cuda_backend.compile_program(DeviceProgram([op], [48 * 512, q.size, own.size, pre.size, t.size]))
        first = np.zeros((48, 512), np.float32)
        cuda_backend.execute_program(h, [ProgramIO(1, q.ravel()), ProgramIO(2, own.ravel()), ProgramIO(3, pre.ravel()), ProgramIO(4, t)], [ProgramIO(0, first)])
        handles.append((h, first))
    for _ in range(3):
        for h, first in handles:
            cuda_backend.lib.zg_cuda_execute_device(cuda_backend.ctx, h.ptr)
    for h, first in handles:
        got = np.zeros_like(first)
        cuda_backend.read_buffer(h, 0, got)
        assert np.array_equal(got, first)                # the same sums in the same order, whenever they run
        cuda_backend.free_program(h)


def test_bits_do_not_change(cuda_backend):
    """Adapters and rules give the same bits in every run."""
    from zgml_b200 import DeviceOp, DeviceProgram, ProgramIO, abi
    r = np.random.default_rng(1)
    for B in (7, 300):
        x, w = r.standard_normal((B, 256)).astype(np.float32), r.standard_normal(3 * 16 * (256 + 72)).astype(np.float32)
        t = table([(0, 0, i // 50 % 3) for i in range(B)], B)
        h = cuda_backend.compile_program(DeviceProgram([DeviceOp.adapter_linear(0, 1, 2, 0, 3 * 16 * 256, 3, B, 72, 256, 16, 3, abi.W_F32, base=4)], [B * 72, x.size, w.size, t.size, B * 72]))
        runs = []
        for _ in range(3):
            got = np.zeros((B, 72), np.float32)
            cuda_backend.execute_program(h, [ProgramIO(1, x.ravel()), ProgramIO(2, w), ProgramIO(3, t)], [ProgramIO(0, got)])
            runs.append(got)
        assert np.array_equal(runs[0], runs[1]) and np.array_equal(runs[0], runs[2])
        cuda_backend.free_program(h)


# ── rules in sessions ────────────────────────────────────────────────────────────────────────────────────────────────
def sessions(be, n, **kw):
    from zgml_b200.host.lududra import LududraConfig, LududraModel
    from zgml_b200.host.session import SequenceSession
    cfg = config([delta_layer(), attention_layer()], vocab=97)
    W = random_weights(cfg, seed=2)
    model = LududraModel(be, LududraConfig.from_dict(cfg), lambda name: W[name], "float32")
    return [SequenceSession(be, model, n_slots=2, max_chunk=8, **kw) for _ in range(n)]


def test_session_rules(cuda_backend):
    """Two requests in turns, prompts cut into chunks: the logits are those of a session without rules, passed through the definition."""
    from zgml_b200.host.batch import LogitRules
    ruled, raw = sessions(cuda_backend, 2)
    rules = {"a": LogitRules(1.7, 0.5, 0.25, {3: 1.5, 96: -2.0}), "b": LogitRules(0.6, allowed=np.arange(97) % 5 != 1)}
    r = np.random.default_rng(0)
    fed, prompt = {"a": [], "b": []}, {"a": 13, "b": 5}
    for step in range(5):
        for k in ("a", "b"):
            new = r.integers(0, 97, prompt[k] if step == 0 else 1).tolist()
            z = raw.feed(k, new, [len(new) - 1])
            got = ruled.feed(k, new, [len(new) - 1], rules[k], generated=step > 0)
            fed[k] += new
            q = rules[k]
            masks = None if q.allowed is None else q.mask(97)[None]
            line = (0, len(fed[k]), prompt[k], -1 if masks is None else 0, 0, len(q.bias), q.repetition, q.presence, q.frequency)
            want, tol = ref.rules(np.zeros((1, 97)), z, [line], 1, np.array([fed[k]]), list(q.bias.items()), masks)
            close(got, want, tol, (step, k))
    assert np.array_equal(ruled.feed("a", [4], [0]), raw.feed("a", [4], [0]))             # without rules in this step
    with pytest.raises(ValueError):
        ruled.feed("b", [1, 2], [0], rules["b"])
    with pytest.raises(ValueError):
        ruled.feed("b", [1], [0], LogitRules(bias={97: 1.0}))
    assert ruled.pool.position("b") == raw.pool.position("b")                              # refused before anything ran
    a, b = (s.step([{"id": "a", "tokens": [9], "want": [0], **x}], ["b"])[0] for s, x in ((ruled, {"rules": LogitRules(bias={5: 2.0}), "generated": True}), (raw, {})))
    assert a[0, 5] == b[0, 5] + np.float32(2.0) and np.array_equal(np.delete(a, 5), np.delete(b, 5)) and not ruled.pool.has("b")
    ruled.release("a")
    assert np.array_equal(ruled.feed("a", [7, 8], [1], LogitRules(repetition=1.0)), sessions(cuda_backend, 1)[0].feed("a", [7, 8], [1]))      # a new request, nothing kept of the old one
    for s in (ruled, raw):
        s.close()


def test_generate_with_rules(cuda_backend):
    from zgml_b200.host.batch import LogitRules
    s, = sessions(cuda_backend, 1)
    prompt = [5, 6, 7]
    plain = s.generate(prompt, 12)
    assert s.generate(prompt, 12, rules=LogitRules()) == plain
    only = s.generate(prompt, 12, rules=LogitRules(allowed=np.array([11, 12, 80])))
    assert set(only) <= {11, 12, 80}
    once = s.generate(prompt, 20, rules=LogitRules(presence=1e6))
    assert len(set(once)) == 20                          # a token that was generated is never the best again
    first = s.generate(prompt, 3, rules=LogitRules(bias={42: 1e6}))
    assert first == [42, 42, 42]
    small, = sessions(cuda_backend, 1, max_history=4)
    with pytest.raises(ValueError):
        small.generate(prompt, 4, rules=LogitRules(presence=1.0))
    for x in (s, small):
        x.close()
