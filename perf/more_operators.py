"""The operators of a decode step over paged caches in 8 bits, as cases that can be timed and checked: rows of many sequences join the pages of their caches (and are read
back from them), attend over them, pages are copied, and the next tokens are sampled from the rows' logits.

`run` computes each case in plain torch, or (`own`) executes the compiled DeviceProgram that a user of the framework runs; both work on
tensors in HBM that hold the same values.  `exact` restates each operator in 64 bits."""
import math

import numpy as np
import torch

own = False

HEAD, ROW, MOVE, CHOICE = 8, 4, 4, 8          # words before the rows of a table, per row of a batch table, per move of pages, per row of a sampling table

# What each listed case stands for:
LISTED = [
    # one sequence decoded alone, 32 query and 8 key heads of 128: latency of the smallest step
    {"name": "append_one", "kind": "append", "seqs": 1, "tokens": 1, "idle": 0, "heads": 32, "kv_heads": 8, "dk": 128, "dv": 128, "turn_at": 0, "rot": 128, "layout": "halves", "prefix": 0, "longest": 700, "page": 16},
    # a batch of 256 sequences, half of every head turned, a few rows of the batch idle
    {"name": "append_batch", "kind": "append", "seqs": 256, "tokens": 1, "idle": 6, "heads": 32, "kv_heads": 8, "dk": 128, "dv": 128, "turn_at": 0, "rot": 64, "layout": "pairs", "prefix": 1000, "longest": 4096, "page": 16},
    # prompts of four requests, 2048 tokens in all, behind what their caches hold already
    {"name": "append_prompts", "kind": "append", "seqs": 4, "tokens": 512, "idle": 0, "heads": 32, "kv_heads": 8, "dk": 128, "dv": 128, "turn_at": 0, "rot": 128, "layout": "halves", "prefix": 0, "longest": 1333, "page": 64},
    # one sequence of a SmolLM-135M-shape model behind 576 tokens: latency
    {"name": "attend_one", "kind": "attend", "seqs": 1, "tokens": 1, "idle": 0, "heads": 9, "kv_heads": 3, "dk": 64, "dv": 64, "longest": 576, "page": 16, "window": 0, "cap": 0.0, "sink": False},
    # 64 sequences of an 8B-size model decoded together, up to 4096 tokens each
    {"name": "attend_decode", "kind": "attend", "seqs": 64, "tokens": 1, "idle": 3, "heads": 32, "kv_heads": 8, "dk": 128, "dv": 128, "longest": 4096, "page": 16, "window": 0, "cap": 0.0, "sink": False},
    # 9 sequences that each bring 7 tokens (drafts to verify), capped scores and sinks, heads of an odd size, a window
    {"name": "attend_drafts", "kind": "attend", "seqs": 9, "tokens": 7, "idle": 5, "heads": 16, "kv_heads": 4, "dk": 80, "dv": 80, "longest": 2111, "page": 32, "window": 1500, "cap": 30.0, "sink": True},
    # 16 sequences over documents of up to 65536 tokens
    {"name": "attend_long", "kind": "attend", "seqs": 16, "tokens": 1, "idle": 0, "heads": 32, "kv_heads": 8, "dk": 128, "dv": 128, "longest": 65536, "page": 64, "window": 0, "cap": 0.0, "sink": False},
    # a request is forked: the page that both write on in is copied
    {"name": "copy_fork", "kind": "copy", "moves": 1, "idle": 0, "kv_heads": 8, "dk": 128, "dv": 128, "page": 16, "pages": 64},
    # a pool is compacted: every second page moves
    {"name": "copy_compact", "kind": "copy", "moves": 4096, "idle": 17, "kv_heads": 8, "dk": 128, "dv": 128, "page": 16, "pages": 8192},
    # one request's next token over a SmolLM-size vocabulary
    {"name": "sample_one", "kind": "sample", "rows": 1, "idle": 0, "vocab": 49152, "form": "both", "spread": 3.0},
    # 64 requests over a vocabulary of 128256, each with choices of its own
    {"name": "sample_batch", "kind": "sample", "rows": 64, "idle": 1, "vocab": 128256, "form": "mixed", "spread": 3.0},
    # 32 requests that keep 0.95 of flat distributions: tens of thousands of tokens each
    {"name": "sample_flat", "kind": "sample", "rows": 32, "idle": 0, "vocab": 128256, "form": "top_p", "spread": 1.0},
]


def listed():
    return [dict(c) for c in LISTED]


def _log(rng, lo, hi, step=1):
    """A whole number spread over the logarithm of [lo, hi], a multiple of `step`."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))
    return max(lo, min(hi, (v + step // 2) // step * step))


def draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "copy", "sample", "sample"])
    kv, dk, page = rng.choice([1, 2, 3, 4, 8]), rng.choice([32, 64, 80, 96, 128, 128, 192, 44]), rng.choice([16, 16, 32, 64])
    dv = rng.choice([dk, dk, 64, 128])
    if kind == "append":
        tokens = rng.choice([1, 1, _log(rng, 2, 512)])
        rot = rng.choice([dk, dk // 2 // 2 * 2, 16])
        return {"kind": kind, "seqs": _log(rng, 1, max(1, 256 if tokens == 1 else 2048 // tokens)), "tokens": tokens, "idle": rng.choice([0, 0, rng.randint(1, 9)]), "heads": kv * rng.choice([1, 2, 4]), "kv_heads": kv, "dk": dk,
                "dv": dv, "turn_at": rng.choice([0, 0, dk - rot]), "rot": rot, "layout": rng.choice(["pairs", "halves"]), "prefix": rng.choice([0, _log(rng, 16, 100000)]), "longest": tokens + _log(rng, 1, 4096), "page": page}
    if kind == "attend":
        tokens = rng.choice([1, 1, 1, rng.randint(2, 16)])
        seqs = _log(rng, 1, 128 if tokens == 1 else 16)
        group = rng.choice([1, 2, 3, 4, 4, 8] if kv < 8 else [1, 4])
        most = min(65536, (1 << 31) // (seqs * kv * (dk + dv) * max(1, tokens * group // 4)))
        longest = max(tokens, rng.choice([_log(rng, 1, 300), _log(rng, 64, most), _log(rng, 1024, most)]))
        return {"kind": kind, "seqs": seqs, "tokens": tokens, "idle": rng.choice([0, 0, rng.randint(1, 9)]), "heads": kv * group, "kv_heads": kv, "dk": dk, "dv": dv, "longest": longest,
                "page": page, "window": rng.choice([0, 0, 0, _log(rng, 1, 4096)]), "cap": rng.choice([0.0, 0.0, 0.0, 30.0]), "sink": rng.random() < 0.25}
    if kind == "copy":
        moves = _log(rng, 1, 2048)
        return {"kind": kind, "moves": moves, "idle": rng.choice([0, moves // 5]), "kv_heads": kv, "dk": dk, "dv": dv, "page": page, "pages": 2 * moves + _log(rng, 1, 500)}
    return {"kind": kind, "rows": _log(rng, 1, 64), "idle": rng.choice([0, 0, 1]), "vocab": rng.choice([32000, 49152, _log(rng, 1000, 128256), _log(rng, 30000, 128256)]), "form": rng.choice(["both", "mixed", "mixed", "top_p", "top_k"]),
            "spread": rng.choice([1.0, 3.0, 3.0, 6.0])}


# ── inputs: made on the GPU from the seed alone, the same values for `prepare` and `exact` ───────────────────────────
class _Random:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(0x9A6ED + seed)

    def normal(self, *shape, scale=1.0):
        return torch.randn(*shape, generator=self.g, device="cuda", dtype=torch.float32) * scale

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.g, device="cuda", dtype=torch.float32)

    def order(self, n):
        return torch.randperm(n, generator=self.g, device="cuda")

    def codes(self, *shape):
        """Codes of 8 bits as caches hold them, most of them small."""
        return self.normal(*shape, scale=38.0).round_().clamp_(-127, 127).to(torch.int8)

    def scales(self, *shape):
        return torch.exp2(-5.0 - (3 * self.uniform(*shape)).floor_())


def _device(values, dtype=torch.int32):
    return torch.tensor(np.asarray(values), dtype=dtype, device="cuda")


def _spread(n, lo, hi):
    """n whole numbers spread over [lo, hi], the first one hi."""
    return [lo + int(round((hi - lo) * (1.0 - i * 0.6180339887 % 1.0))) for i in range(n)]


def _ends(c):
    """How many positions each sequence has after the step."""
    return _spread(c["seqs"], max(c["tokens"], c["longest"] // 8), c["longest"])


def _table(rows, live, prefix, slots, lengths):
    """A batch table: live rows, prefix length, and {slot, length, -1, 0} for every row."""
    t = torch.zeros(HEAD + ROW * rows, dtype=torch.int32, device="cuda")
    t[:2] = _device([live, prefix])
    body = t[HEAD:].view(rows, ROW)
    body[:len(slots), 0], body[:len(slots), 1], body[:, 2] = slots, lengths, -1
    return t


def _steps_rows(c, r):
    """Slot and length of every live row: a sequence's tokens one after the other."""
    ends = _device(_ends(c), torch.int64)
    lengths = ends[:, None] - c["tokens"] + 1 + torch.arange(c["tokens"], device="cuda")
    return r.order(c["seqs"]).repeat_interleave(c["tokens"]), lengths.flatten()


def _inputs_append(c, r):
    S, T, H, G, dk, dv, page = (c[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dk", "dv", "page"))
    rows, width, most = S * T + c["idle"], G * (dk + dv), -(-c["longest"] // page)
    slots, lengths = _steps_rows(c, r)
    by_slot = torch.empty(S, dtype=torch.int64, device="cuda")
    by_slot[slots[::T]] = _device(_ends(c), torch.int64)
    # pages that the step writes on, in a pool of their own and as many others: the first one of a sequence may hold tokens already
    first, count = (by_slot - T) // page, (by_slot - 1) // page - (by_slot - T) // page + 1
    total = int(count.sum())
    seq = torch.arange(S, device="cuda").repeat_interleave(count)
    nth = first[seq] + torch.arange(total, device="cuda") - (count.cumsum(0) - count)[seq]
    pages = 2 * total
    ids = r.order(pages)[:total]
    page_table = torch.full((S, most), pages - 1, dtype=torch.int32, device="cuda")
    page_table[seq, nth] = ids.to(torch.int32)
    # what is read back: every position that those pages hold after the step
    at = nth[:, None] * page + torch.arange(page, device="cuda")
    held = at < by_slot[seq][:, None]
    read_slots, read_lengths = seq[:, None].expand(-1, page)[held], at[held] + 1
    freqs = 10000.0 ** (-torch.arange(0, c["rot"], 2, device="cuda", dtype=torch.float64) / max(1, c["rot"]))
    return {"src": r.normal(rows, H * dk + width), "keys": r.codes(pages, G, page, dk), "values": r.codes(pages, G, page, dv), "scales": r.scales(pages, G, 2), "page_table": page_table,
            "table": _table(rows, S * T, c["prefix"], slots, lengths), "freqs": freqs.float(), "turned": torch.zeros(rows, H * dk, device="cuda"),
            "read": _table(len(read_slots), len(read_slots), 0, read_slots, read_lengths), "dst": torch.zeros(len(read_slots), width, device="cuda"), "written": ids}


def _inputs_attend(c, r):
    S, T, H, G, dk, dv, page = (c[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dk", "dv", "page"))
    rows, most = S * T + c["idle"], -(-c["longest"] // page)
    slots, lengths = _steps_rows(c, r)
    pages = S * most
    return {"q": r.normal(rows, H * dk, scale=1.5), "keys": r.codes(pages, G, page, dk), "values": r.codes(pages, G, page, dv), "scales": r.scales(pages, G, 2), "page_table": r.order(pages).to(torch.int32).view(S, most),
            "table": _table(rows, S * T, 0, slots, lengths), "sink": r.normal(H) if c["sink"] else None, "dst": torch.zeros(rows, H * dv, device="cuda")}


def _page_words(c):
    """32-bit words of a page of all key heads: two scales and two words beside them, keys in rows of 32 values, values in rows of 16."""
    return c["kv_heads"] * (16 + c["page"] * (-(-c["dk"] // 32) * 32 + -(-c["dv"] // 16) * 16)) // 4


def _inputs_copy(c, r):
    ids = r.order(c["pages"])
    moves = torch.zeros(HEAD + MOVE * c["moves"], dtype=torch.int32, device="cuda")
    moves[0] = c["moves"] - c["idle"]
    body = moves[HEAD:].view(-1, MOVE)
    body[:, 0], body[:, 1] = ids[:c["moves"]], ids[c["moves"]:2 * c["moves"]]
    return {"pages": torch.randint(-2 ** 31, 2 ** 31, (c["pages"], _page_words(c)), generator=r.g, device="cuda", dtype=torch.int32), "moves": moves}


def _inputs_sample(c, r):
    B, V = c["rows"], c["vocab"]
    i = torch.arange(B, device="cuda")
    t = torch.zeros(HEAD + CHOICE * B, dtype=torch.int32, device="cuda")
    t[0] = B - c["idle"] if B > c["idle"] else B
    body = t[HEAD:].view(B, CHOICE)
    temperature, top_p = 0.6 + 0.6 * r.uniform(B), 0.85 + 0.14 * r.uniform(B)
    top_k = _device([40, 5, 1000, 200, 1], torch.int64)[i % 5].clamp(max=V)
    min_p = torch.zeros(B, device="cuda")
    if c["form"] == "both":                          # a few tokens and most of what they have
        pass
    elif c["form"] == "top_p":
        top_k, top_p = torch.zeros_like(top_k), torch.full_like(top_p, 0.95)
    elif c["form"] == "top_k":
        top_p = torch.ones_like(top_p)
    else:                                            # in turns: both, one of them, the likeliest token, all of the distribution, a least probability
        turn = i % 6
        top_k = torch.where((turn == 1) | (turn == 3) | (turn == 4), 0, top_k)
        top_p = torch.where((turn == 2) | (turn == 3) | (turn == 4), 1.0, top_p)
        temperature = torch.where(turn == 3, 0.0, temperature)
        min_p = torch.where(turn >= 4, torch.where(turn == 5, 0.05, 0.0), min_p)
    body[:, 0], body[:, 1] = temperature.view(torch.int32), top_k.to(torch.int32)
    body[:, 2], body[:, 3], body[:, 4] = top_p.view(torch.int32), min_p.view(torch.int32), r.uniform(B).view(torch.int32)
    return {"logits": r.normal(B, V, scale=c["spread"]), "table": t, "dst": torch.zeros(B, dtype=torch.int32, device="cuda"), "probability": torch.zeros(B, device="cuda")}


# ── the framework's calls ────────────────────────────────────────────────────────────────────────────────────────────
_BACKEND = []


class _Memory:
    """A tensor's memory as a program's external buffer."""

    def __init__(self, t):
        self.t, self.ptr, self.elems = t, t.data_ptr(), t.numel() * t.element_size() // 4


class _Program:
    """A compiled program over tensors of the caller."""

    def __init__(self, make, tensors):
        from zgml_b200.backend import CudaBackend, DeviceProgram, ExternBuffer, last_error
        if not _BACKEND:
            _BACKEND.append(CudaBackend(0))
        self.be = _BACKEND[0]
        given = [(k, _Memory(t)) for k, t in tensors.items() if t is not None]
        at = {k: None for k in tensors}
        at.update({k: i for i, (k, _) in enumerate(given)})
        program = DeviceProgram(make(at), [m.elems for _, m in given], externs=[ExternBuffer(i, m) for i, (_, m) in enumerate(given)])
        self.handle = self.be.compile_program(program)
        if self.handle is None:
            raise RuntimeError("the program did not compile: " + last_error())

    def execute(self):
        self.be.lib.zg_cuda_execute_device(self.be.ctx, self.handle.ptr)

    def __del__(self):
        if getattr(self, "handle", None) is not None:
            self.be.sync()
            self.be.free_program(self.handle)


def _packed(c, t):
    """The framework's pages of the same caches: codes of a head behind its scales, offset by 128; keys in tiles of 8 tokens by 32 values, values in tiles of 16 by 16."""
    keys, values, scales = t["keys"], t["values"], t["scales"]
    P, G, page, dk = keys.shape
    dv = values.shape[-1]
    tiled = torch.zeros(P, G, page, -(-dk // 32) * 32, dtype=torch.int8, device="cuda")
    tiled[..., :dk] = keys
    k = (tiled.view(torch.uint8) ^ 128).view(P, G, page // 8, 8, -1, 32).transpose(3, 4).reshape(P, G, -1)
    tiled = torch.zeros(P, G, page, -(-dv // 16) * 16, dtype=torch.int8, device="cuda")
    tiled[..., :dv] = values
    v = (tiled.view(torch.uint8) ^ 128).view(P, G, page // 16, 2, 4, 2, -1, 2, 8).permute(0, 1, 2, 6, 8, 4, 7, 3, 5).reshape(P, G, -1)
    head = torch.zeros(P, G, 4, device="cuda")
    head[..., :2] = scales
    return torch.cat([head.view(torch.uint8), k, v], -1).view(torch.int32)


def _ops_append(c, at):
    from zgml_b200.backend import DeviceOp
    S, T, H, G, dk, dv, page = (c[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dk", "dv", "page"))
    most = -(-c["longest"] // page)
    return [DeviceOp.page_append(at["pages"], at["src"], at["page_table"], at["table"], H * dk, H * dk + G * dk, S * T + c["idle"], G, dk, dv, H * dk + G * (dk + dv), page, most, turn_at=c["turn_at"], rot=c["rot"],
                                 rot_layout=c["layout"], freqs=at["freqs"], q_heads=H, q_col=0, turned=at["turned"]),
            DeviceOp.page_read(at["dst"], at["pages"], at["page_table"], at["read"], c["read"], G, dk, dv, page, most)]


def _ops_attend(c, at):
    from zgml_b200.backend import DeviceOp
    S, T, H, G, dk, dv, page = (c[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dk", "dv", "page"))
    return [DeviceOp.paged_attention(at["dst"], at["q"], at["pages"], at["page_table"], at["table"], S * T + c["idle"], H, G, dk, dv, H * dk, page, -(-c["longest"] // page), dk ** -0.5, window=c["window"],
                                     softcap=c["cap"], sink=at["sink"])]


def _ops_copy(c, at):
    from zgml_b200.backend import DeviceOp
    from zgml_b200.host.pages import page_words
    return [DeviceOp.page_copy(at["pages"], at["moves"], c["moves"], page_words(c["kv_heads"], c["dk"], c["dv"], c["page"]))]


def _ops_sample(c, at):
    from zgml_b200.backend import DeviceOp
    return [DeviceOp.sample(at["dst"], at["logits"], at["table"], c["rows"], c["vocab"], probability=at["probability"])]


def prepare(case, seed):
    kind = case["kind"]
    tensors = globals()["_inputs_" + kind](case, _Random(seed))
    program = None
    if own:                                      # compiled once, executed every step; caches are kept as pages
        given = {k: t for k, t in tensors.items() if k not in ("keys", "values", "scales", "written")}
        if kind in ("append", "attend"):
            tensors = {**{k: t for k, t in tensors.items() if k not in ("keys", "values", "scales")}, "pages": _packed(case, tensors)}
            given["pages"] = tensors["pages"]
        sizes = dict(case, read=(given["read"].numel() - HEAD) // ROW) if kind == "append" else case
        torch.cuda.synchronize()
        program = _Program(lambda at: globals()["_ops_" + kind](sizes, at), given)
    return {"case": case, "tensors": tensors, "program": program}


def run(state):
    case, t = state["case"], state["tensors"]
    if own:
        state["program"].execute()
    else:
        globals()["_plain_" + case["kind"]](case, t)
    return [t[k] for k in {"append": ("dst", "turned"), "attend": ("dst",), "copy": ("pages",), "sample": ("dst", "probability")}[case["kind"]]]


def exact(case, seed):
    return globals()["_exact_" + case["kind"]](case, _Random(seed))


def work(case):
    return globals()["_work_" + case["kind"]](case)


# ── rows join their pages, and pages are read ────────────────────────────────────────────────────────────────────────
# A page holds `page` tokens of every key head: whole numbers of -127 to 127, and for its keys and for its values of each head one power of two that they are multiples of.
# Tokens that need a larger one than the page has make the page's other values, multiples of the smaller, into the nearest of the larger (halves to even numbers).
def _power(most):
    """The smallest power of two (2^-126 at least) of which 127 times reach `most`."""
    mantissa, exponent = torch.frexp(most)
    exponent = torch.where(most > 0, exponent - 7 + (mantissa > 127 / 128), -126)
    return torch.exp2(exponent.clamp(min=-126).double()).float()


def _turned(heads, c, t, live):
    """Heads [live, heads, dk] in 64 bits at their rows' positions, rounded once."""
    at, rot = c["turn_at"], c["rot"]
    rows = t["table"][HEAD:].view(-1, ROW)[:live]
    angle = (c["prefix"] + rows[:, 1:2].double() - 1) * t["freqs"].double()
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    heads = heads.double()
    part = heads[..., at:at + rot]
    x, y = (part[..., 0::2], part[..., 1::2]) if c["layout"] == "pairs" else (part[..., :rot // 2], part[..., rot // 2:])
    both = [x * cos - y * sin, x * sin + y * cos]
    heads[..., at:at + rot] = torch.stack(both, -1).flatten(-2) if c["layout"] == "pairs" else torch.cat(both, -1)
    return heads.float()


def _plain_append(c, t):
    S, T, H, G, dk, dv, page = (c[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dk", "dv", "page"))
    live = S * T
    rows, src, written = t["table"][HEAD:].view(-1, ROW)[:live].long(), t["src"][:live], t["written"]
    heads = _turned(src[:, :(H + G) * dk].reshape(live, H + G, dk), c, t, live)
    t["turned"][:live] = heads[:, :H].flatten(1)
    place = torch.empty(len(t["keys"]), dtype=torch.int64, device="cuda")
    place[written] = torch.arange(len(written), device="cuda")
    at = place[t["page_table"][rows[:, 0], (rows[:, 1] - 1) // page].long()]
    token = (rows[:, 1] - 1) % page
    fresh = torch.zeros(len(written), 1, device="cuda").index_put_((at,), (token == 0).float()[:, None], accumulate=True) > 0
    for name, which, new in (("keys", 0, heads[:, H:]), ("values", 1, src[:, (H + G) * dk:].view(live, G, dv))):
        most = torch.zeros(len(written), G, device="cuda").scatter_reduce_(0, at[:, None].expand(-1, G), new.abs().amax(-1), "amax")
        before = torch.where(fresh, 0.0, t["scales"][written, :, which])
        after = torch.maximum(_power(most), before)
        codes = torch.round(t[name][written].float() * (before / after)[:, :, None, None])
        codes[at, :, token] = torch.round(new / after[at][:, :, None])
        t[name][written], t["scales"][written, :, which] = codes.to(torch.int8), after
    # read back
    rows = t["read"][HEAD:].view(-1, ROW).long()
    at, token = t["page_table"][rows[:, 0], (rows[:, 1] - 1) // page].long(), (rows[:, 1] - 1) % page
    scales = t["scales"][at]
    t["dst"][:, :G * dk] = (t["keys"][at, :, token].float() * scales[:, :, :1]).flatten(1)
    t["dst"][:, G * dk:] = (t["values"][at, :, token].float() * scales[:, :, 1:]).flatten(1)


def _exact_append(c, r):
    t = _inputs_append(c, r)
    S, T, H, G, dk, dv, page, at, rot = (c[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dk", "dv", "page", "turn_at", "rot"))
    body, src, out = t["table"][HEAD:].view(-1, ROW).long(), t["src"].double(), t["turned"].double()
    j = torch.arange(rot // 2, device="cuda")
    first, second = (2 * j + at, 2 * j + 1 + at) if c["layout"] == "pairs" else (j + at, j + rot // 2 + at)
    full = src[:, :(H + G) * dk].reshape(-1, H + G, dk).clone()
    phase = t["freqs"].double() * (c["prefix"] + body[:, 1:2] - 1).double()
    z = torch.complex(full[..., first], full[..., second]) * torch.polar(torch.ones_like(phase), phase)[:, None]
    full[..., first], full[..., second] = z.real, z.imag
    out[:S * T] = full[:S * T, :H].flatten(1)
    # page by page, on the host
    keys, values, scales = (t[k].cpu().numpy().astype(np.float64) for k in ("keys", "values", "scales"))
    new = [full[:, H:].float().double().cpu().numpy(), src[:, (H + G) * dk:].reshape(-1, G, dv).cpu().numpy()]
    held, table, lines = t["page_table"].cpu().numpy(), body[:S * T].cpu().numpy(), {}
    for row, (slot, length) in enumerate(table[:, :2]):
        lines.setdefault(int(held[slot, (length - 1) // page]), []).append((row, (length - 1) % page))
    for p, joined in lines.items():
        rows, tokens = [x for x, _ in joined], [y for _, y in joined]
        for which, codes in enumerate((keys, values)):
            now = new[which][rows]
            for g in range(G):
                old = 0.0 if 0 in tokens else scales[p, g, which]
                most = np.abs(now[:, g]).max()
                need = 2.0 ** -126 if most == 0 else 2.0 ** max(-126, math.ceil(math.log2(most / 127) - 1e-12))
                while most > 127 * need:
                    need *= 2
                grown = max(old, need)
                codes[p, g] = np.rint(codes[p, g] * (old / grown))
                codes[p, g, tokens] = np.rint(now[:, g] / grown)
                scales[p, g, which] = grown
    back = t["read"][HEAD:].view(-1, ROW).cpu().numpy().astype(np.int64)
    p, token = held[back[:, 0], (back[:, 1] - 1) // page], (back[:, 1] - 1) % page
    dst = np.concatenate([(keys[p, :, token] * scales[p][:, :, :1]).reshape(len(p), -1), (values[p, :, token] * scales[p][:, :, 1:]).reshape(len(p), -1)], 1)
    return [torch.from_numpy(dst).cuda(), out]


def _work_append(c):
    S, T, H, G, dk, dv, page = (c[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dk", "dv", "page"))
    width, rows = G * (dk + dv), S * T
    read = sum(e - (e - T) // page * page for e in _ends(c))                                  # positions of the pages that the step writes on
    return {"bytes": 4 * rows * (2 * H * dk + width + ROW) + rows * width + read * (5 * width + 4 * ROW), "flops": 3 * rows * (H + G) * c["rot"] + 2 * (rows + read) * width}


# ── attention over pages ─────────────────────────────────────────────────────────────────────────────────────────────
def _plain_attend(c, t):
    S, T, H, G, dk, dv, page = (c[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dk", "dv", "page"))
    rows = t["table"][HEAD:].view(-1, ROW)[:S * T]
    at = t["page_table"][rows[::T, 0].long()].long()                                          # [S, pages]
    scales = t["scales"][at]
    L = at.shape[1] * page
    k = (t["keys"][at].float() * scales[..., 0, None, None]).transpose(1, 2).reshape(S, G, L, dk)
    q = (t["q"][:S * T].view(S, T, G, H // G, dk) * dk ** -0.5).permute(0, 2, 1, 3, 4).reshape(S, G, T * H // G, dk)
    score = (q @ k.transpose(2, 3)).view(S, G, T, H // G, L)
    del k
    if c["cap"]:
        score = c["cap"] * torch.tanh(score / c["cap"])
    place, length = torch.arange(L, device="cuda"), rows[:, 1].view(S, 1, T, 1, 1)
    hidden = place >= length
    if c["window"]:
        hidden = hidden | (place < length - c["window"])
    score = score.masked_fill(hidden, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    if c["sink"]:
        total = total + torch.exp(t["sink"].view(1, G, 1, H // G, 1) - top)
    v = (t["values"][at].float() * scales[..., 1, None, None]).transpose(1, 2).reshape(S, G, L, dv)
    o = (p.view(S, G, T * H // G, L) @ v).view(S, G, T, H // G, dv) / total
    t["dst"][:S * T] = o.permute(0, 2, 1, 3, 4).reshape(S * T, H * dv)


def _exact_attend(c, r):
    t = _inputs_attend(c, r)
    S, T, H, G, dk, dv, page = (c[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dk", "dv", "page"))
    out, rows = t["dst"].double(), t["table"][HEAD:].view(-1, ROW)[:S * T].tolist()
    for s in range(S):
        end = rows[s * T + T - 1][1]
        ids = t["page_table"][rows[s * T][0], :-(-end // page)].long()
        for g in range(G):
            k = (t["keys"][ids, g].double() * t["scales"][ids, g, 0].double()[:, None, None]).reshape(-1, dk)[:end]
            v = (t["values"][ids, g].double() * t["scales"][ids, g, 1].double()[:, None, None]).reshape(-1, dv)[:end]
            for i in range(T):
                length = rows[s * T + i][1]
                lo = max(0, length - c["window"]) if c["window"] else 0
                score = torch.einsum("hd,jd->hj", t["q"][s * T + i].view(G, H // G, dk)[g].double(), k[lo:length]) / math.sqrt(dk)
                if c["cap"]:
                    score = c["cap"] * torch.tanh(score / c["cap"])
                if c["sink"]:
                    score = torch.cat([score, t["sink"].double().view(G, H // G)[g][:, None]], 1)
                out.view(-1, G, H // G, dv)[s * T + i, g] = torch.softmax(score, -1)[:, :length - lo] @ v[lo:length]
    return [out]


def _work_attend(c):
    T, H, G, dk, dv, W = (c[k] for k in ("tokens", "heads", "kv_heads", "dk", "dv", "window"))
    ends = _ends(c)
    seen = sum(min(e - T + 1 + i, W or e) for e in ends for i in range(T))
    held = sum(min(e, W + T - 1) if W else e for e in ends)
    return {"bytes": held * G * (dk + dv) + -(-held // c["page"]) * (8 * G + 4) + 4 * len(ends) * T * H * (dk + dv), "flops": 2 * H * (dk + dv) * seen}


# ── pages are copied ─────────────────────────────────────────────────────────────────────────────────────────────────
def _plain_copy(c, t):
    body = t["moves"][HEAD:].view(-1, MOVE)[:c["moves"] - c["idle"]].long()
    t["pages"][body[:, 1]] = t["pages"][body[:, 0]]


def _exact_copy(c, r):
    t = _inputs_copy(c, r)
    pages = t["pages"].clone()
    for source, to in t["moves"][HEAD:].view(-1, MOVE)[:c["moves"] - c["idle"], :2].tolist():
        pages[to] = t["pages"][source]
    return [pages]


def _work_copy(c):
    return {"bytes": (c["moves"] - c["idle"]) * (8 * _page_words(c) + 4 * MOVE), "flops": 0}


# ── the next tokens ──────────────────────────────────────────────────────────────────────────────────────────────────
# Of e^((z - largest z) / temperature): the top_k largest stay, of those the fewest of the largest whose sum reaches top_p of theirs, of those the ones that are at least min_p.
# The token is the first, in the vocabulary's order, up to which what stays sums to more than u of all that stays; its probability is its share of that sum.  Equal logits: the
# lower token goes first.  Temperature 0: the largest logit, with probability 1.
def _plain_sample(c, t):
    V, body = c["vocab"], t["table"][HEAD:].view(-1, CHOICE)[:_choices(c)]
    temperature, top_p, min_p, u = (body[:, i].contiguous().view(torch.float32)[:, None].double() for i in (0, 2, 3, 4))
    top_k = body[:, 1:2].long()
    z, order = t["logits"][:len(body)].sort(dim=1, descending=True, stable=True)
    greedy = temperature == 0
    e = torch.exp((z.double() - z[:, :1].double()) / torch.where(greedy, 1.0, temperature))
    kept = e * ((torch.arange(V, device="cuda") < top_k) | (top_k <= 0))
    below = kept.cumsum(1) - kept
    kept = torch.where((below < top_p * kept.sum(1, keepdim=True)) | (top_p >= 1), kept, 0.0)
    kept = torch.where(kept >= min_p, kept, 0.0)
    kept = torch.zeros_like(kept).scatter_(1, order, kept)
    sums = kept.cumsum(1)
    token = (sums <= u * sums[:, -1:]).sum(1, keepdim=True)
    t["dst"][:len(body)] = torch.where(greedy, order[:, :1], token)[:, 0].to(torch.int32)
    t["probability"][:len(body)] = torch.where(greedy, 1.0, kept.gather(1, token) / sums[:, -1:])[:, 0].float()


def _choices(c):
    return c["rows"] - c["idle"] if c["rows"] > c["idle"] else c["rows"]


def _exact_sample(c, r):
    t = _inputs_sample(c, r)
    out, share = t["dst"].cpu().numpy(), np.zeros(c["rows"])
    logits, body = t["logits"].cpu().numpy().astype(np.float64), t["table"][HEAD:].view(-1, CHOICE).cpu().numpy()
    for i in range(_choices(c)):
        temperature, top_p, min_p, u = body[i, [0, 2, 3, 4]].copy().view(np.float32).astype(np.float64)
        if temperature == 0:
            out[i], share[i] = int(np.argmax(logits[i])), 1.0
            continue
        e = np.exp((logits[i] - logits[i].max()) / temperature)
        order = np.argsort(-logits[i], kind="stable")
        order = order[:body[i, 1]] if body[i, 1] > 0 else order
        if top_p < 1:
            sums = np.cumsum(e[order])
            order = order[:1 + int(np.searchsorted(sums, top_p * sums[-1], side="left"))]
        stays = np.sort(order[e[order] >= min_p])
        sums = np.cumsum(e[stays])
        out[i] = stays[np.searchsorted(sums, u * sums[-1], side="right")]
        share[i] = e[out[i]] / sums[-1]
    return [torch.from_numpy(out).cuda(), torch.from_numpy(share).cuda()]


def _work_sample(c):
    return {"bytes": _choices(c) * (4 * c["vocab"] + 4 * CHOICE + 8), "flops": 4 * _choices(c) * c["vocab"]}
