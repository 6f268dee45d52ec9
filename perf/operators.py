"""The operators of a batched decode step as cases that can be timed and checked: rows of many sequences join their caches, attend over a
prefix that all share and over what is their own, pass their request's low-rank adapter, and their logits pass the request's penalties,
biases and grammar mask.

`run` computes each case in plain torch, or (`own`) executes the compiled DeviceProgram that a user of the framework runs; both work on the
same tensors in HBM.  `exact` restates each operator in 64 bits."""
import math

import numpy as np
import torch

own = False

HEAD, ROW, RULE = 8, 4, 12          # words before the rows of a table, per row of a batch table, per row of a rule table

# What each listed case stands for:
LISTED = [
    # one sequence decoded alone, 32 query and 8 key heads of 128: latency of the smallest step
    {"name": "append_one", "kind": "append", "rows": 1, "idle": 0, "heads": 32, "kv_heads": 8, "dk": 128, "dv": 128, "turn_at": 0, "rot": 128, "layout": "halves", "prefix": 2048, "capacity": 512, "latent": False},
    # a batch of 256 sequences behind a prefix of 100000 positions, half of every head turned, a few rows of the batch idle
    {"name": "append_batch", "kind": "append", "rows": 256, "idle": 6, "heads": 32, "kv_heads": 8, "dk": 128, "dv": 128, "turn_at": 0, "rot": 64, "layout": "pairs", "prefix": 100000, "capacity": 32, "latent": False},
    # one sequence of a SmolLM-135M-shape model behind a 512-token prompt prefix: latency
    {"name": "attend_one", "kind": "attend", "seqs": 1, "tokens": 1, "idle": 0, "heads": 9, "kv_heads": 3, "dk": 64, "dv": 64, "prefix": 512, "own": 64, "latent": False, "cap": 0.0, "sink": False},
    # 32 sequences of an 8B-size model decoded behind one 8192-token prefix, up to 512 tokens each of their own
    {"name": "attend_decode", "kind": "attend", "seqs": 32, "tokens": 1, "idle": 0, "heads": 32, "kv_heads": 8, "dk": 128, "dv": 128, "prefix": 8192, "own": 512, "latent": False, "cap": 0.0, "sink": False},
    # 9 sequences that each bring 7 tokens (drafts to verify), capped scores and sinks, a few rows idle
    {"name": "attend_drafts", "kind": "attend", "seqs": 9, "tokens": 7, "idle": 5, "heads": 16, "kv_heads": 4, "dk": 128, "dv": 128, "prefix": 1777, "own": 333, "latent": False, "cap": 30.0, "sink": True},
    # 16 sequences over a latent that serves as key and value (absorbed form)
    {"name": "attend_latent", "kind": "attend", "seqs": 16, "tokens": 1, "idle": 0, "heads": 16, "kv_heads": 1, "dk": 576, "dv": 512, "prefix": 4096, "own": 256, "latent": True, "cap": 0.0, "sink": False},
    # 128 sequences behind a 32768-token document
    {"name": "attend_long", "kind": "attend", "seqs": 128, "tokens": 1, "idle": 0, "heads": 32, "kv_heads": 8, "dk": 128, "dv": 128, "prefix": 32768, "own": 512, "latent": False, "cap": 0.0, "sink": False},
    # one token through one f32 adapter of a small model: latency
    {"name": "adapter_one", "kind": "adapter", "rows": 1, "idle": 0, "run": 1, "inputs": 2048, "outputs": 2048, "rank": 8, "adapters": 4, "dtype": "f32"},
    # 64 requests decoded together, each with an adapter of its own
    {"name": "adapter_decode", "kind": "adapter", "rows": 64, "idle": 0, "run": 1, "inputs": 4096, "outputs": 4096, "rank": 16, "adapters": 64, "dtype": "bf16"},
    # prompts of four requests, 2048 tokens in all, through the adapters of a feed-forward's wide product
    {"name": "adapter_prompts", "kind": "adapter", "rows": 2048, "idle": 40, "run": 500, "inputs": 4096, "outputs": 14336, "rank": 64, "adapters": 4, "dtype": "bf16"},
    # one request's logits of a SmolLM-size vocabulary: penalties and a few biases
    {"name": "rules_one", "kind": "rules", "rows": 1, "idle": 0, "vocab": 49152, "history": 600, "bias": 16, "masked": False},
    # 64 requests over a vocabulary of 128256, up to 4096 tokens of history, every second one under a grammar
    {"name": "rules_batch", "kind": "rules", "rows": 64, "idle": 1, "vocab": 128256, "history": 4096, "bias": 64, "masked": True},
]


def listed():
    return [dict(c) for c in LISTED]


def _log(rng, lo, hi, step=1):
    """A whole number spread over the logarithm of [lo, hi], a multiple of `step`."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))
    return max(lo, min(hi, (v + step // 2) // step * step))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "adapter", "adapter", "rules", "rules"])
    if kind == "append":
        rows, kv = _log(rng, 1, 256), rng.choice([1, 2, 3, 4, 8])
        latent = rng.random() < 0.2
        dk = 576 if latent else rng.choice([32, 64, 80, 96, 128])
        rot = 64 if latent else rng.choice([dk, dk // 2, 16])
        return {"kind": kind, "rows": rows, "idle": rng.choice([0, 0, rows // 5]), "heads": 16 if latent else kv * rng.choice([1, 2, 4]), "kv_heads": 1 if latent else kv, "dk": dk, "dv": 0 if latent else rng.choice([dk, 64, 128]),
                "turn_at": 512 if latent else rng.choice([0, 0, dk - rot]), "rot": rot, "layout": rng.choice(["pairs", "halves"]), "prefix": rng.choice([0, _log(rng, 16, 200000)]),
                "capacity": _log(rng, 8, 64), "latent": latent}
    if kind == "attend":
        latent = rng.random() < 0.2
        tokens = rng.choice([1, 1, 1, rng.randint(2, 16)])
        seqs = _log(rng, 1, 24 if latent else 128 if tokens == 1 else 16)
        kv = 1 if latent else rng.choice([1, 2, 3, 4, 8])
        heads = 16 if latent else kv * rng.choice([1, 2, 3, 4, 8]) if kv < 8 else kv * rng.choice([1, 4])
        dk = 576 if latent else rng.choice([32, 64, 80, 96, 112, 128, 128])
        prefix = rng.choice([0, _log(rng, 1, 32768), _log(rng, 256, 32768), _log(rng, 1024, 16384)])
        if latent:
            prefix = min(prefix, 8192)
        return {"kind": kind, "seqs": seqs, "tokens": tokens, "idle": rng.choice([0, 0, rng.randint(1, 9)]), "heads": heads, "kv_heads": kv, "dk": dk, "dv": 512 if latent else dk, "prefix": prefix,
                "own": max(tokens, _log(rng, 1, 512)), "latent": latent, "cap": 0.0 if latent else rng.choice([0.0, 0.0, 0.0, 30.0]), "sink": rng.random() < 0.25}
    if kind == "adapter":
        dtype, step = rng.choice(["bf16", "bf16", "f32"]), rng.choice([8, 8, 1])
        rows = rng.choice([_log(rng, 1, 8), _log(rng, 1, 256), _log(rng, 64, 2048 if dtype == "bf16" else 512)])
        return {"kind": kind, "rows": rows, "idle": rng.choice([0, 0, rows // 9]), "run": rng.choice([1, 1, rng.randint(2, 40), rows]) if rows <= 256 else rng.randint(33, rows), "inputs": _log(rng, 256, 4096, step),
                "outputs": _log(rng, 256, 8192, step), "rank": rng.choice([4, 8, 16, 16, 24, 32, 64, 7]), "adapters": _log(rng, 1, 64 if rows <= 256 else 8), "dtype": dtype}
    rows, vocab = _log(rng, 1, 64), rng.choice([32000, 49152, _log(rng, 1000, 128256), _log(rng, 30000, 128256)])
    return {"kind": kind, "rows": rows, "idle": rng.choice([0, rows // 6]), "vocab": vocab, "history": _log(rng, 1, 4096), "bias": rng.choice([0, _log(rng, 1, 300)]), "masked": rng.random() < 0.5}


# ── inputs: made on the GPU from the seed alone, the same tensors for `prepare` and `exact` ──────────────────────────
class _Random:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(0xBA7C4 + seed)

    def normal(self, *shape, scale=1.0):
        return torch.randn(*shape, generator=self.g, device="cuda", dtype=torch.float32) * scale

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.g, device="cuda", dtype=torch.float32)

    def order(self, n):
        return torch.randperm(n, generator=self.g, device="cuda")


def _device(values, dtype=torch.int32):
    return torch.tensor(np.asarray(values), dtype=dtype, device="cuda")


def _table(rows, live, prefix, slots, lengths, adapters=None):
    """A batch table: live rows, prefix length, prefix slot, and {slot, length, adapter, 0} for every row."""
    t = torch.zeros(HEAD + ROW * rows, dtype=torch.int32, device="cuda")
    t[:2] = _device([live, prefix])
    body = t[HEAD:].view(rows, ROW)
    body[:, 0], body[:, 1], body[:, 2] = slots, lengths, -1 if adapters is None else adapters
    return t


def _spread(n, lo, hi):
    """n whole numbers spread over [lo, hi], the first one hi."""
    return [lo + int(round((hi - lo) * (1.0 - i * 0.6180339887 % 1.0))) for i in range(n)]


def _inputs_append(c, r):
    B, H, G, dk, dv, R = (c[k] for k in ("rows", "heads", "kv_heads", "dk", "dv", "capacity"))
    cols = G * dk if c["latent"] else G * (dk + dv)
    return {"src": r.normal(B, H * dk + cols), "cache": r.normal(B, R, cols), "turned": torch.zeros(B, H * dk, device="cuda"),
            "table": _table(B, B - c["idle"], c["prefix"], r.order(B), _device(_spread(B, 1, R)))}


def _lengths(c):
    """Positions of its own that every row sees: the tokens of a sequence see one more each."""
    ends = _spread(c["seqs"], c["tokens"], c["own"])
    return [[e - c["tokens"] + 1 + t for t in range(c["tokens"])] for e in ends]


def _inputs_attend(c, r):
    S, T, H, G, dk, dv, P, R = (c[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dk", "dv", "prefix", "own"))
    B, width = S * T + c["idle"], G * dk if c["latent"] else G * (dk + dv)
    slots, lengths = torch.zeros(B, dtype=torch.int64, device="cuda"), torch.zeros(B, dtype=torch.int64, device="cuda")
    slots[:S * T], lengths[:S * T] = r.order(S).repeat_interleave(T), _device(_lengths(c), torch.int64).reshape(-1)
    scale = 1.5 if not c["latent"] else 0.6
    return {"q": r.normal(B, H * dk, scale=scale), "own": r.normal(S, R, width), "prefix": r.normal(1, P + 5, width), "sink": r.normal(H) if c["sink"] else None,
            "dst": torch.zeros(B, H * dv, device="cuda"), "table": _table(B, S * T, P, slots, lengths)}


def _adapters(c):
    """Every row's adapter; each seventh run of rows has none."""
    runs = [r // c["run"] for r in range(c["rows"])]
    return [-1 if n % 7 == 6 else (n * 5 + 2) % c["adapters"] for n in runs]


def _inputs_adapter(c, r):
    B, K, N, rank, A = (c[k] for k in ("rows", "inputs", "outputs", "rank", "adapters"))
    a, b = r.normal(A, rank, K, scale=K ** -0.5), r.normal(A, N, rank, scale=rank ** -0.5)
    if c["dtype"] == "bf16":
        a, b = a.to(torch.bfloat16), b.to(torch.bfloat16)
    zeros = torch.zeros(B, dtype=torch.int64, device="cuda")
    return {"x": r.normal(B, K), "base": r.normal(B, N), "weights": torch.cat([a.reshape(-1), b.reshape(-1), a.new_zeros(-(a.numel() + b.numel()) % 8)]), "scales": 0.25 + r.uniform(A), "dst": torch.zeros(B, N, device="cuda"),
            "table": _table(B, B - c["idle"], 0, zeros, zeros, _device(_adapters(c)))}


def _inputs_rules(c, r):
    B, V, L, n = (c[k] for k in ("rows", "vocab", "history", "bias"))
    lengths = _device(_spread(B, (L + 1) // 2, L))
    t = torch.zeros(HEAD + RULE * B, dtype=torch.int32, device="cuda")
    t[0] = B - c["idle"]
    rows = torch.arange(B, device="cuda")
    body = t[HEAD:].view(B, RULE)
    body[:, 0], body[:, 1], body[:, 2] = r.order(B), lengths, lengths // 3
    body[:, 3] = torch.where(rows % 2 == 0, rows // 2, -1) if c["masked"] else -1
    body[:, 4], body[:, 5] = rows * n, n
    body[:, 6:9] = torch.stack([1.0 + 0.5 * r.uniform(B), r.uniform(B), 0.5 * r.uniform(B)], 1).view(torch.int32)
    history = (V * r.uniform(B, L) ** 3).to(torch.int32).clamp_(max=V - 1)                   # few tokens often, many once
    bias = torch.zeros(max(1, B * n), 2, dtype=torch.int32, device="cuda")
    if n:
        bias[:, 0] = ((r.uniform(B, 1) * V).long() + torch.arange(n, device="cuda") * 7).remainder(V).reshape(-1).to(torch.int32)
        bias[:, 1] = r.normal(B * n, scale=4.0).view(torch.int32)
    masks = None
    if c["masked"]:                                                                            # one word in eight allows tokens
        words = (r.uniform((B + 1) // 2, (V + 31) // 32, 2) * 65536).to(torch.int32)
        masks = torch.where(r.uniform(*words.shape[:2]) < 0.125, words[..., 0] * 65536 + words[..., 1], 0).to(torch.int32)
    return {"logits": r.normal(B, V, scale=3.0), "history": history, "bias": bias, "masks": masks, "dst": torch.zeros(B, V, device="cuda"), "table": t}


# ── the framework's calls ────────────────────────────────────────────────────────────────────────────────────────────
_BACKEND = []


class _Memory:
    """A tensor's memory as a program's external buffer."""

    def __init__(self, t):
        self.t, self.ptr, self.elems = t, t.data_ptr(), t.numel() * t.element_size() // 4


class _Program:
    """A compiled one-op program over tensors of the caller."""

    def __init__(self, make, tensors):
        from zgml_b200.backend import CudaBackend, DeviceProgram, ExternBuffer, last_error
        if not _BACKEND:
            _BACKEND.append(CudaBackend(0))
        self.be = _BACKEND[0]
        given = [(k, _Memory(t)) for k, t in tensors.items() if t is not None]
        at = {k: None for k in tensors}
        at.update({k: i for i, (k, _) in enumerate(given)})
        program = DeviceProgram([make(at)], [m.elems for _, m in given], externs=[ExternBuffer(i, m) for i, (_, m) in enumerate(given)])
        self.handle = self.be.compile_program(program)
        if self.handle is None:
            raise RuntimeError("the program did not compile: " + last_error())

    def execute(self):
        self.be.lib.zg_cuda_execute_device(self.be.ctx, self.handle.ptr)

    def __del__(self):
        if getattr(self, "handle", None) is not None:
            self.be.sync()
            self.be.free_program(self.handle)


def _op_append(c, at):
    from zgml_b200.backend import DeviceOp
    B, H, G, dk, dv = (c[k] for k in ("rows", "heads", "kv_heads", "dk", "dv"))
    cols = G * dk if c["latent"] else G * (dk + dv)
    return DeviceOp.batch_append(at["cache"], at["src"], at["table"], H * dk, 0, B, cols, H * dk + cols, cols, c["capacity"], key_heads=G, head_dim=dk, turn_at=c["turn_at"], rot=c["rot"],
                                 rot_base=10000.0, rot_layout=c["layout"], q_heads=H, q_col=0, turned=at["turned"])


def _op_attend(c, at):
    from zgml_b200.backend import DeviceOp
    H, G, dk, dv = (c[k] for k in ("heads", "kv_heads", "dk", "dv"))
    width, v_col = (G * dk, 0) if c["latent"] else (G * (dk + dv), G * dk)
    return DeviceOp.shared_attention(at["dst"], at["q"], at["own"], at["own"], at["prefix"], at["prefix"], at["table"], 0, 0, v_col, 0, v_col, c["seqs"] * c["tokens"] + c["idle"], H, G, dk, dv, H * dk,
                                     width, width, c["own"], width, width, c["prefix"] + 5, dk ** -0.5, softcap=c["cap"], sink=at["sink"])


def _op_adapter(c, at):
    from zgml_b200 import abi
    from zgml_b200.backend import DeviceOp
    K, N, rank, A = (c[k] for k in ("inputs", "outputs", "rank", "adapters"))
    return DeviceOp.adapter_linear(at["dst"], at["x"], at["weights"], 0, A * rank * K, at["table"], c["rows"], N, K, rank, A, abi.W_BF16 if c["dtype"] == "bf16" else abi.W_F32, base=at["base"], scales=at["scales"])


def _op_rules(c, at):
    from zgml_b200.backend import DeviceOp
    return DeviceOp.logit_rules(at["dst"], at["logits"], at["table"], c["rows"], c["vocab"], history=at["history"], history_rows=c["history"], bias=at["bias"], masks=at["masks"])


def prepare(case, seed):
    kind = case["kind"]
    tensors = globals()["_inputs_" + kind](case, _Random(seed))
    program = None
    if own:                                      # compiled once, executed every step
        torch.cuda.synchronize()
        program = _Program(lambda at: globals()["_op_" + kind](case, at), tensors)
    return {"case": case, "tensors": tensors, "program": program}


def run(state):
    case, t = state["case"], state["tensors"]
    if own:
        state["program"].execute()
    else:
        globals()["_plain_" + case["kind"]](case, t)
    return [t["cache"], t["turned"]] if case["kind"] == "append" else [t["dst"]]


def exact(case, seed):
    return globals()["_exact_" + case["kind"]](case, _Random(seed))


def work(case):
    return globals()["_work_" + case["kind"]](case)


# ── rows join their caches ───────────────────────────────────────────────────────────────────────────────────────────
def _plain_append(c, t):
    H, G, dk, at, rot, live = c["heads"], c["kv_heads"], c["dk"], c["turn_at"], c["rot"], c["rows"] - c["idle"]
    rows = t["table"][HEAD:].view(-1, ROW)[:live]
    angle = (c["prefix"] + rows[:, 1].double() - 1)[:, None] * 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    src = t["src"][:live]
    heads = src[:, :(H + G) * dk].reshape(live, H + G, dk).clone()
    part = heads[..., at:at + rot]
    x, y = (part[..., 0::2], part[..., 1::2]) if c["layout"] == "pairs" else (part[..., :rot // 2], part[..., rot // 2:])
    turned = [x * cos - y * sin, x * sin + y * cos]
    heads[..., at:at + rot] = torch.stack(turned, -1).flatten(-2) if c["layout"] == "pairs" else torch.cat(turned, -1)
    t["turned"][:live] = heads[:, :H].flatten(1)
    t["cache"][rows[:, 0].long(), rows[:, 1].long() - 1] = torch.cat([heads[:, H:].flatten(1), src[:, (H + G) * dk:]], 1)


def _exact_append(c, r):
    t = _inputs_append(c, r)
    H, G, dk, at, rot, live = c["heads"], c["kv_heads"], c["dk"], c["turn_at"], c["rot"], c["rows"] - c["idle"]
    src, cache, out = t["src"].double(), t["cache"].double(), t["turned"].double()
    body = t["table"][HEAD:].view(-1, ROW).long()
    j = torch.arange(rot // 2, device="cuda")
    first, second = (2 * j, 2 * j + 1) if c["layout"] == "pairs" else (j, j + rot // 2)
    first, second = first + at, second + at
    heads = src[:, :(H + G) * dk].reshape(-1, H + G, dk)
    phase = torch.exp(-2.0 * j.double() / rot * math.log(10000.0)) * (c["prefix"] + body[:, 1:2] - 1).double()
    z = torch.complex(heads[..., first], heads[..., second]) * torch.polar(torch.ones_like(phase), phase)[:, None]
    full = heads.clone()
    full[..., first], full[..., second] = z.real, z.imag
    out[:live] = full[:live, :H].flatten(1)
    cache[body[:live, 0], body[:live, 1] - 1] = torch.cat([full[:, H:].flatten(1), src[:, (H + G) * dk:]], 1)[:live]
    return [cache, out]


def _work_append(c):
    values = c["heads"] * c["dk"] + (c["kv_heads"] * c["dk"] if c["latent"] else c["kv_heads"] * (c["dk"] + c["dv"]))
    live = c["rows"] - c["idle"]
    return {"bytes": 4 * live * (2 * values + ROW), "flops": 3 * live * (c["heads"] + c["kv_heads"]) * c["rot"]}


# ── attention over a shared prefix and what is a row's own ───────────────────────────────────────────────────────────
def _split(c, cache):
    """Keys and values [.., positions, kv heads, dim] of cache rows."""
    G, dk, dv = c["kv_heads"], c["dk"], c["dv"]
    if c["latent"]:
        return cache[..., None, :], cache[..., None, :dv]
    return cache[..., :G * dk].unflatten(-1, (G, dk)), cache[..., G * dk:].unflatten(-1, (G, dv))


def _plain_attend(c, t):
    S, T, H, G, dk, dv, P, R = (c[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dk", "dv", "prefix", "own"))
    rows = t["table"][HEAD:].view(-1, ROW)[:S * T]
    q = t["q"][:S * T].view(S, T, G, H // G, dk) * dk ** -0.5
    kp, vp = _split(c, t["prefix"][0, :P])
    ko, vo = _split(c, t["own"][rows[::T, 0].long()])
    shared = (q.permute(2, 0, 1, 3, 4).reshape(G, S * T * H // G, dk) @ kp.permute(1, 2, 0)).view(G, S, T, H // G, P)
    mine = (q.permute(2, 0, 1, 3, 4).reshape(G, S, T * H // G, dk) @ ko.permute(2, 0, 3, 1)).view(G, S, T, H // G, R)
    if c["cap"]:
        shared, mine = c["cap"] * torch.tanh(shared / c["cap"]), c["cap"] * torch.tanh(mine / c["cap"])
    hidden = torch.arange(R, device="cuda") >= rows[:, 1].view(1, S, T, 1, 1)
    mine = mine.masked_fill(hidden, -math.inf)
    top = mine.amax(-1, keepdim=True)
    if P:
        top = torch.maximum(top, shared.amax(-1, keepdim=True))
    shared, mine = torch.exp(shared - top), torch.exp(mine - top)
    total = shared.sum(-1, keepdim=True) + mine.sum(-1, keepdim=True)
    if c["sink"]:
        total = total + torch.exp(t["sink"].view(G, 1, 1, H // G, 1) - top)
    o = (shared.reshape(G, S * T * H // G, P) @ vp.permute(1, 0, 2)).view(G, S, T, H // G, dv) + (mine.reshape(G, S, T * H // G, R) @ vo.permute(2, 0, 1, 3)).view(G, S, T, H // G, dv)
    t["dst"][:S * T] = (o / total).permute(1, 2, 0, 3, 4).reshape(S * T, H * dv)


def _exact_attend(c, r):
    t = _inputs_attend(c, r)
    S, T, H, G, dk, dv, P = (c[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dk", "dv", "prefix"))
    body, out = t["table"][HEAD:].view(-1, ROW).long(), t["dst"].double()
    lengths = _lengths(c)
    slots = body[:S * T:T, 0].tolist()
    kp, vp = (x.double() for x in _split(c, t["prefix"][0, :P]))
    for g in range(G):
        q = t["q"][:S * T].view(S, T, G, H // G, dk)[:, :, g].double()
        shared = torch.einsum("sthd,pd->sthp", q, kp[:, g])
        for s in range(S):
            k, v = (x.double() for x in _split(c, t["own"][slots[s], :lengths[s][-1]]))
            score = torch.cat([shared[s], torch.einsum("thd,jd->thj", q[s], k[:, g])], -1) / math.sqrt(dk)
            if c["cap"]:
                score = c["cap"] * torch.tanh(score / c["cap"])
            seen = torch.arange(P + lengths[s][-1], device="cuda") < P + _device(lengths[s]).view(T, 1, 1)
            score = torch.where(seen, score, -math.inf)
            if c["sink"]:
                score = torch.cat([score, t["sink"].double().view(G, H // G)[g].view(1, -1, 1).expand(T, -1, 1)], -1)
            p = torch.softmax(score, -1)[..., :P + lengths[s][-1]]
            out.view(-1, G, H // G, dv)[s * T:(s + 1) * T, g] = p @ torch.cat([vp[:, g], v[:, g]])
    return [out]


def _work_attend(c):
    S, T, H, G, dk, dv, P = (c[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dk", "dv", "prefix"))
    lengths = _lengths(c)
    width = dk if c["latent"] else G * (dk + dv)
    return {"bytes": 4 * (P + sum(x[-1] for x in lengths)) * width + 4 * S * T * H * (dk + dv), "flops": 2 * H * (dk + dv) * sum(P + n for x in lengths for n in x)}


# ── adapters of many requests ────────────────────────────────────────────────────────────────────────────────────────
def _plain_adapter(c, t):
    K, N, rank, A, live = c["inputs"], c["outputs"], c["rank"], c["adapters"], c["rows"] - c["idle"]
    a, b = t["weights"][:A * rank * K].view(A * rank, K), t["weights"][A * rank * K:A * rank * (K + N)].view(A, N, rank)
    which = t["table"][HEAD:].view(-1, ROW)[:live, 2]
    mine = (which[:, None] == torch.arange(A, device="cuda")) * t["scales"]                   # [rows, adapters]
    h = (t["x"][:live] @ a.float().T).view(live, A, rank) * mine[..., None]
    t["dst"][:live] = t["base"][:live] + h.view(live, A * rank) @ b.float().permute(0, 2, 1).reshape(A * rank, N)


def _exact_adapter(c, r):
    t = _inputs_adapter(c, r)
    K, N, rank, A, live = c["inputs"], c["outputs"], c["rank"], c["adapters"], c["rows"] - c["idle"]
    a, b = t["weights"][:A * rank * K].double().view(A, rank, K), t["weights"][A * rank * K:A * rank * (K + N)].double().view(A, N, rank)
    out, which = t["dst"].double(), _device(_adapters(c)[:live])
    out[:live] = t["base"][:live].double()
    for i in sorted(set(_adapters(c)[:live]) - {-1}):
        at = (which == i).nonzero()[:, 0]
        out[at] += t["scales"][i].double() * torch.einsum("nj,jk,rk->rn", b[i], a[i], t["x"][at].double()) if len(at) < rank else t["scales"][i].double() * ((t["x"][at].double() @ a[i].T) @ b[i].T)
    return [out]


def _work_adapter(c):
    K, N, rank, live = c["inputs"], c["outputs"], c["rank"], c["rows"] - c["idle"]
    which = [i for i in _adapters(c)[:live] if i >= 0]
    size = 2 if c["dtype"] == "bf16" else 4
    return {"bytes": 4 * (len(which) * K + 2 * live * N) + size * len(set(which)) * rank * (K + N), "flops": 2 * len(which) * rank * (K + N)}


# ── rules on logits ──────────────────────────────────────────────────────────────────────────────────────────────────
def _plain_rules(c, t):
    V, L, n, live = c["vocab"], c["history"], c["bias"], c["rows"] - c["idle"]
    body = t["table"][HEAD:].view(-1, RULE)[:live]
    rep, presence, frequency = body[:, 6:9].contiguous().view(torch.float32).split(1, 1)
    tokens, place = t["history"][body[:, 0].long()].long(), torch.arange(L, device="cuda")
    zeros = torch.zeros(live, V, device="cuda")
    seen = zeros.scatter_add(1, tokens, (place < body[:, 1:2]).float()) > 0
    count = zeros.scatter_add(1, tokens, ((place < body[:, 1:2]) & (place >= body[:, 2:3])).float())
    z = t["logits"][:live]
    z = torch.where(seen, torch.where(z > 0, z / rep, z * rep), z)
    z = z - presence * (count > 0) - frequency * count
    if n:
        entries = t["bias"][:live * n].view(live, n, 2)
        z = z + zeros.scatter_add(1, entries[..., 0].long(), entries[..., 1].contiguous().view(torch.float32))
    if c["masked"]:
        bits = (t["masks"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32) & 1).flatten(1)[:, :V]
        allowed = (bits[body[:, 3].long().clamp(min=0)] != 0) | (body[:, 3:4] < 0)
        z = z.masked_fill(~allowed, -math.inf)
    t["dst"][:live] = z


def _exact_rules(c, r):
    t = _inputs_rules(c, r)
    V, n = c["vocab"], c["bias"]
    out = t["dst"].double()
    for i, w in enumerate(t["table"][HEAD:].view(-1, RULE)[:c["rows"] - c["idle"]].tolist()):
        rep, presence, frequency = np.array(w[6:9], np.int32).view(np.float32).astype(np.float64)
        tokens = t["history"][w[0], :w[1]].long()
        count = torch.bincount(tokens[w[2]:], minlength=V).double()
        z = t["logits"][i].double()
        past = torch.unique(tokens)
        z[past] = z[past].clamp(min=0) / rep + z[past].clamp(max=0) * rep
        z -= presence * count.clamp(max=1) + frequency * count
        if n:
            e = t["bias"][w[4]:w[4] + n]
            z.index_add_(0, e[:, 0].long(), e[:, 1].contiguous().view(torch.float32).double())
        if w[3] >= 0:
            words = t["masks"][w[3]].cpu().numpy().view(np.uint8)
            z[torch.from_numpy(np.unpackbits(words, bitorder="little")[:V] == 0).cuda()] = -math.inf
        out[i] = z
    return [out]


def _work_rules(c):
    V, live = c["vocab"], c["rows"] - c["idle"]
    lengths = _spread(c["rows"], (c["history"] + 1) // 2, c["history"])[:live]
    masks = ((live + 1) // 2) * ((V + 31) // 32) if c["masked"] else 0
    return {"bytes": 4 * (2 * live * V + sum(lengths) + masks + 2 * live * c["bias"]), "flops": 4 * live * V}
