"""The ops of a batched step in one-op programs against NumPy in 64 bits: sizes that end inside vectors and tiles, rows that are idle, see nothing or name places that
do not exist, stale memory behind a sequence's end, the same program replayed with another table, and one decode loop in which they run together.  Tolerances come from
the number of roundings (tests/batch_reference.py)."""
import numpy as np
import pytest

import batch_reference as ref

pytestmark = pytest.mark.gpu
NAN = np.float32("nan")


class Prog:
    """One program over named arrays: those in `sizes` are its own buffers, DeviceBuffers are shared."""

    def __init__(self, be, make, arrays, extern=()):
        from zgml_b200 import DeviceBuffer, DeviceProgram, ExternBuffer
        from zgml_b200.backend import last_error
        self.be, self.at, self.shared, self.shape = be, {}, {}, {}
        sizes, externs = [], []
        for name, a in arrays.items():
            a = np.ascontiguousarray(a)
            self.at[name], self.shape[name] = len(sizes), a.shape
            if name in extern:
                b = DeviceBuffer(be, a.nbytes + 16)
                b.upload(a)
                self.shared[name] = b
                externs.append(ExternBuffer(len(sizes), b))
                sizes.append(b.elems)
            else:
                sizes.append(max(1, (a.nbytes + 3) // 4))
        self.h = be.compile_program(DeviceProgram(make(self.at), sizes, [], [], externs))
        assert self.h is not None, last_error()
        self.arrays = {k: np.ascontiguousarray(a) for k, a in arrays.items() if k not in self.shared}

    def run(self, out, **given):
        from zgml_b200 import ProgramIO
        ins = {**self.arrays, **{k: np.ascontiguousarray(v) for k, v in given.items()}}
        outs = {k: np.zeros(self.shape[k], np.float32) for k in out}
        self.be.execute_program(self.h, [ProgramIO(self.at[k], v.view(np.float32).ravel() if v.nbytes % 4 == 0 else v) for k, v in ins.items()], [ProgramIO(self.at[k], v) for k, v in outs.items()])
        return outs[out[0]] if len(out) == 1 else [outs[k] for k in out]

    def close(self):
        self.be.free_program(self.h)
        for b in self.shared.values():
            b.free()


def table(entries, rows, prefix=0, prefix_slot=0, live=None):
    """Without the host's checks: the kernels have checks of their own."""
    t = np.zeros(8 + 4 * rows, np.int32)
    t[:3] = len(entries) if live is None else live, prefix, prefix_slot
    for i, e in enumerate(entries):
        t[8 + 4 * i:11 + 4 * i] = e
    return t


def close(got, want, tol, what=""):
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    inf = np.isinf(want)
    assert np.array_equal(np.isinf(got), inf) and np.array_equal(got[inf], want[inf]), what
    ok = np.isfinite(want)
    off = np.abs(got[ok] - want[ok]) - (tol[ok] if isinstance(tol, np.ndarray) else tol)
    assert not ok.any() or off.max() <= 0.0, (what, off.max(), np.abs(want[ok]).max())


# ── BATCH_APPEND ─────────────────────────────────────────────────────────────────────────────────────────────────────
# Angles are reduced in 64 bits, so a turned value is off by the roundings of its angle (2^-24 pi), of sine and cosine (2 ulp) and of two products and a sum.
TURN = 12 * 2.0 ** -24


@pytest.mark.parametrize("B,heads,kv,dim,turn_at,rot,layout,extra,pad", [(1, 2, 1, 8, 0, 8, "pairs", 8, 0), (5, 4, 2, 16, 4, 12, "halves", 32, 3), (33, 3, 3, 80, 0, 40, "pairs", 7, 1), (3, 2, 1, 576, 512, 64, "halves", 0, 0),
                                                                         (4, 2, 2, 7, 1, 6, "halves", 5, 2), (6, 1, 2, 32, 0, 0, "pairs", 4, 0), (2, 1, 1, 64, 0, 2, "pairs", 1, 0)])
@pytest.mark.parametrize("prefix,tabled", [(0, False), (131071, False), (99, True)])
def test_batch_append(cuda_backend, B, heads, kv, dim, turn_at, rot, layout, extra, pad, prefix, tabled):
    from zgml_b200 import DeviceOp
    r = np.random.default_rng(B + dim)
    slots, R, cols = B + 1, 4, kv * dim + extra
    rs, width, trs = heads * dim + cols + pad, cols + 2 * pad, heads * dim + pad
    src, cache = r.standard_normal((B, rs)).astype(np.float32), r.standard_normal((slots, R, width)).astype(np.float32)
    freqs = r.uniform(0.01, 1.0, max(1, rot // 2)).astype(np.float32)
    make = lambda at: [DeviceOp.batch_append(at["cache"], at["src"], at["table"], heads * dim, pad, B, cols, rs, width, R, key_heads=kv, head_dim=dim, turn_at=turn_at, rot=rot, rot_base=1e4,
                                             rot_layout=layout, freqs=at["freqs"] if tabled else None, q_heads=heads, turned=at["turned"], turned_col=pad, turned_rs=trs)]
    turned = r.standard_normal((B, trs)).astype(np.float32)
    p = Prog(cuda_backend, make, dict(cache=cache, src=src, table=np.zeros(8 + 4 * B, np.int32), freqs=freqs, turned=turned))
    perm = r.permutation(slots)[:B]
    full = [(int(perm[i]), 1 + i % R, 0) for i in range(B)]
    odd = [(-1, 1, 0), (slots, 1, 0), (0, R + 1, 0), (1, -1, 0), (0, 0, 0), (int(perm[0]), R, 0)][:B]
    odd += full[len(odd):]
    same = [(0, 2, 0)] * B                              # one place for all: the last one stays
    for entries, live in ((full, B), (odd, B), (same, B), (full, B - 1), (full, B + 7), (full, -3)):
        got, got_t = p.run(["cache", "turned"], table=table(entries, B, prefix, live=live))
        want, want_t = ref.append(cache, src, entries, max(0, live), prefix, heads * dim, pad, cols, kv, dim, turn_at, rot, 1e4, layout, heads, 0, turned[:, pad:], freqs if tabled else None)
        close(got, want, TURN * (np.abs(src).max() + 1))
        close(got_t[:, pad:], want_t, TURN * (np.abs(src).max() + 1))
        assert np.array_equal(got_t[:, :pad], turned[:, :pad]) and np.array_equal(got[:, :, :pad], cache[:, :, :pad])
    p.close()


def test_batch_append_twice_into_one_row(cuda_backend):
    """Keys with their turn, values without, into the two halves of a cache row; no query heads."""
    from zgml_b200 import DeviceOp
    r = np.random.default_rng(0)
    B, kv, dim, R = 3, 2, 8, 3
    src = r.standard_normal((B, 2 * kv * dim)).astype(np.float32)
    make = lambda at: [DeviceOp.batch_append(at["cache"], at["src"], at["table"], 0, 0, B, kv * dim, 2 * kv * dim, 2 * kv * dim, R, key_heads=kv, head_dim=dim, rot=dim, rot_base=100.0),
                       DeviceOp.batch_append(at["cache"], at["src"], at["table"], kv * dim, kv * dim, B, kv * dim, 2 * kv * dim, 2 * kv * dim, R)]
    p = Prog(cuda_backend, make, dict(cache=np.zeros((B, R, 2 * kv * dim), np.float32), src=src, table=np.zeros(8 + 4 * B, np.int32)))
    entries = [(2, 3, 0), (0, 1, 0), (1, 2, 0)]
    got = p.run(["cache"], table=table(entries, B, 5))
    want, _ = ref.append(np.zeros((B, R, 2 * kv * dim)), src, entries, B, 5, 0, 0, 2 * kv * dim, kv, dim, 0, dim, 100.0, "pairs", 0, 0, np.zeros((B, 0)))
    close(got, want, TURN * np.abs(src).max())
    p.close()


# ── SHARED_ATTENTION ─────────────────────────────────────────────────────────────────────────────────────────────────
def attend_case(be, B, H, G, dk, dv, prefix, R, entries, *, cap=0.0, sink=None, pad=0, latent=False, prefix_slots=2, prefix_slot=1, live=None, seed=0, spare=None, scale=None, loud=1.0, graph=True, v_shift=0):
    from zgml_b200 import DeviceOp, abi
    r = np.random.default_rng(seed)
    slots = max([e[0] for e in entries if e[0] < 100] + [0]) + 1
    width = pad + G * dk + (0 if latent else G * dv) + pad
    v_col = pad + v_shift if latent else pad + G * dk
    if spare is None:                                   # many query rows: a capacity that asks for the tensor cores
        spare = max(3, (3 << 17) // (B * H) + 1 - prefix) if prefix and B * H // G >= 32 and max(dk, dv) <= 128 else 3
    Rp = prefix + spare
    def cache(n, rows):
        c = r.standard_normal((n, rows, width)).astype(np.float32)
        c[:, :, pad:pad + G * dk] *= loud
        return c
    own, pre = cache(slots, R), cache(prefix_slots, Rp)
    seen = np.zeros((slots, R), bool)
    for s, n, _ in entries[:B if live is None else max(live, 0)]:
        if 0 <= s < slots and 0 <= n <= R:
            seen[s, :n] = True
    own[~seen] = NAN                                    # what no row sees may hold anything
    pre[:, prefix:] = NAN
    pre[[i for i in range(prefix_slots) if i != prefix_slot]] = NAN
    if not prefix:
        pre[:] = NAN
    qrs, drs = H * dk + 2 * pad, H * dv + 2 * pad
    q, dst = r.standard_normal((B, qrs)).astype(np.float32), r.standard_normal((B, drs)).astype(np.float32)
    scale = dk ** -0.5 if scale is None else scale
    arrays = dict(dst=dst, q=q, table=table(entries, B, prefix, prefix_slot, live), own=own, pre=pre)
    if sink is not None:
        s32 = (np.round(r.standard_normal(H) * 16) / 8).astype(np.float32)                                   # bfloat16-exact
        bits = (np.concatenate([np.zeros(1, np.float32), s32, np.zeros(H % 2 + 1, np.float32)]).view(np.uint32) >> 16).astype(np.uint16)
        arrays["sink"] = s32 if sink == "f32" else bits
    make = lambda at: [DeviceOp.shared_attention(at["dst"], at["q"], at["own"], at["own"], at["pre"], at["pre"], at["table"], pad, pad, v_col, pad, v_col, B, H, G, dk, dv, qrs, width, width, R, width, width, Rp,
                                                 scale, softcap=cap, sink=at.get("sink"), sink_off=0 if sink != "bf16" else 1, sink_wdt=abi.W_BF16 if sink == "bf16" else abi.W_F32, dst_rs=drs, dst_col=pad)]
    be.set_graph_mode(graph)
    p = Prog(be, make, arrays, extern=("own", "pre"))
    def heads(c, col, d):
        return c[:, :, col:col + G * d].reshape(c.shape[0], c.shape[1], G, d)
    want, tol = ref.attend(dst[:, pad:pad + H * dv].reshape(B, H, dv), q[:, pad:pad + H * dk].reshape(B, H, dk), heads(own, pad, dk), heads(own, v_col, dv), heads(pre, pad, dk), heads(pre, v_col, dv),
                           entries, B if live is None else max(0, live), prefix, prefix_slot, scale, cap, s32 if sink is not None else None)
    for _ in range(2):                                  # the second run replays the graph
        got = p.run(["dst"])
        close(got[:, pad:pad + H * dv].reshape(B, H, dv), want, tol, (B, H, G, dk, dv, prefix))
        assert np.array_equal(got[:, :pad], dst[:, :pad]) and np.array_equal(got[:, pad + H * dv:], dst[:, pad + H * dv:])
    be.set_graph_mode(True)
    p.close()
    return got


@pytest.mark.parametrize("prefix", [0, 1, 63, 64, 129, 700])
@pytest.mark.parametrize("H,G,dk,dv", [(1, 1, 64, 64), (4, 2, 128, 128), (9, 3, 64, 64), (8, 1, 32, 48), (6, 2, 7, 5), (3, 3, 96, 80)])
def test_shared_attention(cuda_backend, prefix, H, G, dk, dv):
    attend_case(cuda_backend, 4, H, G, dk, dv, prefix, 70, [(2, 1, 0), (0, 70, 0), (3, 33, 0), (1, 0, 0)], seed=prefix + H)


@pytest.mark.parametrize("B", [1, 2, 17, 40, 130])
def test_batches(cuda_backend, B):
    attend_case(cuda_backend, B, 8, 2, 128, 128, 300, 20, [(i, 1 + i * 7 % 20, 0) for i in range(B)], seed=B)


@pytest.mark.parametrize("B,H,G,dk,dv,prefix", [(20, 32, 4, 64, 64, 513), (9, 16, 1, 128, 128, 1000), (70, 4, 2, 128, 64, 129), (33, 12, 3, 80, 112, 260), (16, 8, 1, 32, 128, 77), (40, 4, 1, 16, 24, 200), (48, 8, 2, 100, 60, 300)])
def test_many_query_rows(cuda_backend, B, H, G, dk, dv, prefix):
    """Rows times heads of a key head that fill, and end inside, a tile."""
    attend_case(cuda_backend, B, H, G, dk, dv, prefix, 9, [(i, i % 10, 0) for i in range(B)], seed=B + prefix)


@pytest.mark.parametrize("B", [3, 40])
@pytest.mark.parametrize("cap,sink", [(0.0, "f32"), (0.0, "bf16"), (5.0, None), (2.0, "bf16")])
def test_caps_and_sinks(cuda_backend, B, cap, sink):
    attend_case(cuda_backend, B, 8, 2, 64, 64, 90, 33, [(i, (5 + 7 * i) % 34, 0) for i in range(B)], cap=cap, sink=sink)
    attend_case(cuda_backend, B, 8, 2, 64, 64, 0, 33, [(i, (5 + 7 * i) % 34 if i else 0, 0) for i in range(B)], cap=cap, sink=sink, seed=1)


@pytest.mark.parametrize("B,prefix,R", [(2, 100, 30), (12, 530, 40)])
def test_latent(cuda_backend, B, prefix, R):
    attend_case(cuda_backend, B, 16, 1, 576, 512, prefix, R, [(i, 1 + i * 3 % R, 0) for i in range(B)], latent=True, scale=0.03)


def test_large_heads(cuda_backend):
    for dk, dv in ((640, 640), (700, 1024), (1024, 512), (300, 200)):
        attend_case(cuda_backend, 2, 6, 2, dk, dv, 40, 20, [(0, 20, 0), (1, 3, 0)])


@pytest.mark.parametrize("pad", [1, 2, 3, 4])
@pytest.mark.parametrize("B", [3, 36])
def test_columns_and_strides(cuda_backend, pad, B):
    attend_case(cuda_backend, B, 8, 2, 64, 64, 150, 21, [(i, 1 + i % 21, 0) for i in range(B)], pad=pad)


def test_rows_of_one_sequence(cuda_backend):
    """Drafts: tokens of a sequence that see one position more each; two rows that are alike."""
    attend_case(cuda_backend, 9, 8, 2, 128, 128, 333, 50, [(0, 11 + t, 0) for t in range(4)] + [(1, 1 + t, 0) for t in range(4)] + [(0, 12, 0)])


@pytest.mark.parametrize("big", [False, True])
def test_idle_rows_and_rows_out_of_range(cuda_backend, big):
    """Idle rows and those behind the live ones stay as they were; a slot or length that does not exist makes NaN of its own row alone."""
    more = [(i, 3, 0) for i in range(4, 40)] if big else []
    entries = [(0, 5, 0), (-1, 5, 0), (100, 5, 0), (1, 41, 0), (2, -1, 0), (-7, 100, 0), (3, 40, 0)] + more
    for live in (None, 4, 0, -1):
        got = attend_case(cuda_backend, len(entries), 8, 2, 64, 64, 200, 40, entries, live=live)
        if live is None:
            assert np.isnan(got[2]).all() and np.isnan(got[3]).all() and np.isnan(got[4]).all() and np.isfinite(got[[0, 1, 5, 6]]).all()


@pytest.mark.parametrize("R", [10, 1300])
@pytest.mark.parametrize("prefix,slot", [(1301, 0), (5, 2), (5, -1), (-1, 0), (2 ** 31 - 1, 0)])
@pytest.mark.parametrize("B", [2, 40])
def test_prefix_out_of_range(cuda_backend, prefix, slot, B, R):
    from zgml_b200 import DeviceOp
    one = np.ones((B, 8 * 64), np.float32)
    make = lambda at: [DeviceOp.shared_attention(at["dst"], at["q"], at["own"], at["own"], at["pre"], at["pre"], at["table"], 0, 0, 0, 0, 0, B, 8, 1, 64, 64, 512, 64, 64, 4, 64, 64, R, 0.1)]
    p = Prog(cuda_backend, make, dict(dst=one, q=one, own=np.ones((B, 4, 64), np.float32), pre=np.ones((2, R, 64), np.float32), table=np.zeros(8 + 4 * B, np.int32)))
    assert np.isnan(p.run(["dst"], table=table([(i, 1, 0) for i in range(B)], B, prefix, slot))).all()
    assert (p.run(["dst"], table=table([(i, 1, 0) for i in range(B)], B, 10, 1)) == 1.0).all()          # the same program, another table
    assert (p.run(["dst"], table=table([(i, 0, 0) for i in range(B)], B, 0, -5)) == 0.0).all()          # no prefix: its slot is not looked at; nothing seen: zeros
    p.close()


def test_without_prefix_buffers(cuda_backend):
    from zgml_b200 import DeviceOp
    r = np.random.default_rng(2)
    q, own = r.standard_normal((3, 4 * 16)).astype(np.float32), r.standard_normal((3, 9, 2 * 16)).astype(np.float32)
    make = lambda at: [DeviceOp.shared_attention(at["dst"], at["q"], at["own"], at["own"], None, None, at["table"], 0, 0, 0, 0, 0, 3, 4, 2, 16, 16, 64, 32, 32, 9, 0, 0, 0, 0.25)]
    p = Prog(cuda_backend, make, dict(dst=np.zeros((3, 64), np.float32), q=q, own=own, table=np.zeros(20, np.int32)))
    entries = [(1, 9, 0), (0, 0, 0), (2, 4, 0)]
    kv = own.reshape(3, 9, 2, 16)
    want, tol = ref.attend(np.zeros((3, 4, 16)), q.reshape(3, 4, 16), kv, kv, None, None, entries, 3, 0, 0, 0.25)
    close(p.run(["dst"], table=table(entries, 3)).reshape(3, 4, 16), want, tol)
    assert np.isnan(p.run(["dst"], table=table(entries, 3, 1))).all()
    p.close()


@pytest.mark.parametrize("B,loud", [(2, 1e4), (40, 1e4), (40, 1e-6), (40, 30.0)])
def test_magnitudes(cuda_backend, B, loud):
    """Scores far apart (one key takes all the weight) and all but equal."""
    attend_case(cuda_backend, B, 8, 2, 64, 64, 333, 17, [(i, 1 + i % 17, 0) for i in range(B)], loud=loud, seed=5)


@pytest.mark.parametrize("B", [2, 40])
def test_eager_launches(cuda_backend, B):
    attend_case(cuda_backend, B, 8, 2, 128, 128, 400, 17, [(i, 1 + i % 17, 0) for i in range(B)], graph=False)


# ── ADAPTER_LINEAR ───────────────────────────────────────────────────────────────────────────────────────────────────
def bf16_bits(a):
    """bfloat16 bit patterns of values that bfloat16 holds."""
    a = np.ascontiguousarray(a, np.float32).ravel()
    bits = (a.view(np.uint32) >> 16).astype(np.uint16)
    assert np.array_equal((bits.astype(np.uint32) << 16).view(np.float32), a)
    return np.concatenate([bits, np.zeros(-bits.size % 2, np.uint16)])


def exact16(r, *shape, scale=1.0):
    v = (r.standard_normal(shape) * scale).astype(np.float32)
    return (v.view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)


def adapter_case(be, fmt, B, N, K, rank, A, entries, *, pad=0, offset=0, scaled=True, in_place=False, live=None, seed=0, form="auto"):
    from zgml_b200 import DeviceOp, abi
    r = np.random.default_rng(seed)
    a, b = exact16(r, A, rank, K, scale=K ** -0.5), exact16(r, A, N, rank, scale=rank ** -0.5)
    flat = np.concatenate([np.zeros(offset, np.float32), a.ravel(), b.ravel()])
    x, base, dst = (r.standard_normal((B, n + pad)).astype(np.float32) for n in (K, N, N))
    scales = r.uniform(0.2, 2.0, A).astype(np.float32)
    arrays = dict(dst=base if in_place else dst, x=x, w=bf16_bits(flat) if fmt == "bf16" else flat, scales=scales, table=table(entries, B, live=live))
    if not in_place:
        arrays["base"] = base
    make = lambda at: [DeviceOp.adapter_linear(at["dst"], at["x"], at["w"], offset, offset + A * rank * K, at["table"], B, N, K, rank, A, abi.W_BF16 if fmt == "bf16" else abi.W_F32, form=form, base=at.get("base"),
                                               base_off=0 if in_place else pad, base_rs=N + pad, scales=at["scales"] if scaled else None, src_off=pad, src_rs=K + pad, dst_off=0 if in_place else pad, dst_rs=N + pad)]
    p = Prog(be, make, arrays)
    c = 0 if in_place else pad
    want, tol = ref.adapt((base if in_place else dst)[:, c:c + N], base[:, c:c + N], x[:, pad:], a, b, scales if scaled else None, entries, B if live is None else max(0, live))
    for _ in range(2):
        got = p.run(["dst"])
        close(got[:, c:c + N], want, tol, (fmt, B, N, K, rank, A))
        if pad:
            keep = (base if in_place else dst)
            assert np.array_equal(got[:, :c], keep[:, :c]) and np.array_equal(got[:, c + N:], keep[:, c + N:])
    p.close()


@pytest.mark.parametrize("fmt", ["f32", "bf16"])
@pytest.mark.parametrize("B,N,K,rank,A", [(1, 8, 8, 1, 1), (1, 300, 257, 8, 3), (5, 64, 512, 16, 2), (9, 1000, 96, 7, 4), (64, 256, 320, 24, 64), (33, 130, 1000, 64, 5), (3, 40, 2000, 200, 2)])
def test_adapter_linear(cuda_backend, fmt, B, N, K, rank, A):
    adapter_case(cuda_backend, fmt, B, N, K, rank, A, [(0, 0, i * 5 % (A + 1) - 1) for i in range(B)], seed=B + K)
    adapter_case(cuda_backend, fmt, B, N, K, rank, A, [(0, 0, (i // 3) % A) for i in range(B)], pad=3, seed=K, scaled=False)


@pytest.mark.parametrize("fmt", ["f32", "bf16"])
@pytest.mark.parametrize("B,run", [(200, 200), (300, 70), (515, 33), (260, 1), (640, 256)])
def test_adapters_of_prompts(cuda_backend, fmt, B, run):
    adapter_case(cuda_backend, fmt, B, 200, 264, 16, 4, [(0, 0, (i // run) % 5 - 1) for i in range(B)], seed=B)


@pytest.mark.parametrize("fmt", ["f32", "bf16"])
@pytest.mark.parametrize("B,N,K,rank", [(300, 136, 1032, 64), (270, 72, 200, 33), (257, 513, 129, 8), (256, 1024, 512, 130)])
def test_adapters_of_prompts_sizes(cuda_backend, fmt, B, N, K, rank):
    adapter_case(cuda_backend, fmt, B, N, K, rank, 3, [(0, 0, (i // 90) % 3) for i in range(B)], seed=B)


@pytest.mark.parametrize("fmt", ["f32", "bf16"])
@pytest.mark.parametrize("B", [6, 300])
def test_adapter_rows_left_alone_and_out_of_range(cuda_backend, fmt, B):
    entries = [(0, 0, 1), (-1, 0, 1), (0, 0, 2), (5, -9, -1), (0, 0, -7), (0, 0, 0)] + [(0, 0, i % 4 - 1) for i in range(B - 6)]      # adapter 2 does not exist
    for live in (None, 4, B - 1, 0, -2):
        adapter_case(cuda_backend, fmt, B, 72, 40, 8, 2, entries, live=live)


@pytest.mark.parametrize("fmt", ["f32", "bf16"])
@pytest.mark.parametrize("offset,pad", [(1, 0), (4, 1), (8, 2), (3, 5)])
@pytest.mark.parametrize("B", [4, 260])
def test_adapter_alignment(cuda_backend, fmt, offset, pad, B):
    adapter_case(cuda_backend, fmt, B, 96, 64, 16, 3, [(0, 0, i % 3) for i in range(B)], offset=offset, pad=pad)


@pytest.mark.parametrize("B", [3, 300])
def test_adapter_in_place(cuda_backend, B):
    adapter_case(cuda_backend, "bf16", B, 96, 64, 16, 3, [(0, 0, i // 50 % 4 - 1) for i in range(B)], in_place=True)


# ── LOGIT_RULES ──────────────────────────────────────────────────────────────────────────────────────────────────────
def rules_case(be, B, V, rows, *, history=None, bias=(), masks=None, pad=0, in_place=False, live=None, logits=None, seed=0):
    from zgml_b200 import DeviceOp
    r = np.random.default_rng(seed)
    z = r.standard_normal((B, V + pad)).astype(np.float32) * 4
    if logits is not None:
        z[:, pad:] = logits
    dst = z if in_place else r.standard_normal((B, V + pad)).astype(np.float32)
    t = np.zeros(8 + 12 * B, np.int32)
    t[0] = len(rows) if live is None else live
    for i, w in enumerate(rows):
        t[8 + 12 * i:14 + 12 * i] = w[:6]
        t[14 + 12 * i:17 + 12 * i] = np.array(w[6:], np.float32).view(np.int32)
    arrays = dict(dst=dst, table=t)
    if not in_place:
        arrays["src"] = z
    if history is not None:
        arrays["history"] = np.asarray(history, np.int32)
    if len(bias):
        e = np.zeros((len(bias), 2), np.int32)
        e[:, 0], e[:, 1] = [k for k, _ in bias], np.array([v for _, v in bias], np.float32).view(np.int32)
        arrays["bias"] = e
    if masks is not None:
        arrays["masks"] = masks
    c = pad
    make = lambda at: [DeviceOp.logit_rules(at["dst"], at.get("src", at["dst"]), at["table"], B, V, history=at.get("history"), history_rows=0 if history is None else np.asarray(history).shape[1], bias=at.get("bias"),
                                            masks=at.get("masks"), src_off=c, src_rs=V + pad, dst_off=c, dst_rs=V + pad)]
    p = Prog(be, make, arrays)
    want, tol = ref.rules(dst[:, c:], z[:, c:], rows, B if live is None else max(0, live), None if history is None else np.asarray(history), list(bias), masks)
    for _ in range(2):
        got = p.run(["dst"])
        close(got[:, c:], want, tol, (B, V))
        assert np.array_equal(got[:, :c], dst[:, :c])
    p.close()
    return got[:, c:]


@pytest.mark.parametrize("B,V,L", [(1, 1, 1), (1, 33, 7), (3, 1000, 300), (2, 49152, 600), (5, 8191, 1025), (4, 20000, 5000), (2, 128256, 2000)])
@pytest.mark.parametrize("pad", [0, 1, 4])
def test_logit_rules(cuda_backend, B, V, L, pad):
    r = np.random.default_rng(V)
    history = (V * r.random((B + 1, L)) ** 3).astype(np.int32)
    bias = [(int(t), float(v)) for t, v in zip(r.integers(0, V, 40 * B), r.standard_normal(40 * B) * 3)]
    masks = r.integers(-2 ** 31, 2 ** 31, (2, (V + 31) // 32)).astype(np.int32)
    rows = [((i + 1) % (B + 1), L - i % L, L // 3, i % 3 - 1, 40 * i, 40 if i % 2 == 0 else 3, 1.3, 0.4, 0.2) for i in range(B)]
    rules_case(cuda_backend, B, V, rows, history=history, bias=bias, masks=masks, pad=pad)
    rules_case(cuda_backend, B, V, rows, history=history, bias=bias, masks=masks, pad=pad, in_place=True)


def test_rules_that_ask_for_nothing(cuda_backend):
    """Without history, biases and masks a row is copied bit for bit, infinities and NaN among it."""
    z = np.random.default_rng(0).standard_normal((3, 70)).astype(np.float32)
    z[0, 3], z[1, 69], z[2, 0], z[2, 1] = np.inf, -np.inf, NAN, -0.0
    got = rules_case(cuda_backend, 3, 70, [(0, 0, 0, -1, 0, 0, 1.0, 0.0, 0.0)] * 3, logits=z)
    assert np.array_equal(got, z, equal_nan=True)


def test_rules_on_infinities(cuda_backend):
    z = np.zeros((1, 64), np.float32)
    z[0, :4] = np.inf, -np.inf, NAN, 3.4e38
    h = [[0, 1, 2, 3, 0, 1]]
    rules_case(cuda_backend, 1, 64, [(0, 6, 4, -1, 0, 0, 2.0, 0.5, 0.25)], history=h, logits=z)
    m = np.zeros((1, 2), np.int32)
    got = rules_case(cuda_backend, 1, 64, [(0, 6, 4, 0, 0, 0, 2.0, 0.5, 0.25)], history=h, logits=z, masks=m)
    assert (got == -np.inf).all()                       # a mask that allows nothing


def test_biases_of_one_token_add_up(cuda_backend):
    bias = [(5, 1.0), (6, -2.0)] * 40 + [(5, 0.5)]
    got = rules_case(cuda_backend, 1, 40, [(0, 0, 0, -1, 0, 81, 1.0, 0.0, 0.0)], bias=bias, logits=np.zeros((1, 40), np.float32))
    assert got[0, 5] == 40.5 and got[0, 6] == -80.0


def test_tokens_outside_the_vocabulary(cuda_backend):
    h = [[-1, 5, 70, 2 ** 31 - 1, -2 ** 31, 5, 69]]
    rules_case(cuda_backend, 1, 70, [(0, 7, 0, -1, 0, 0, 1.5, 0.5, 0.25)], history=h)


def test_rule_rows_left_alone_and_out_of_range(cuda_backend):
    """What a row asks of memory that is not there makes NaN of it."""
    h, bias, masks = np.zeros((2, 9), np.int32), [(1, 1.0)] * 4, np.full((2, 3), -1, np.int32)
    good = (1, 9, 2, 1, 1, 3, 1.0, 0.0, 0.0)
    bad = [(2, 1, 0, -1, 0, 0, 1.0, 0.0, 0.0), (0, 10, 0, -1, 0, 0, 1.0, 0.0, 0.0), (0, -1, 0, -1, 0, 0, 1.0, 0.0, 0.0), (0, 1, -1, -1, 0, 0, 1.0, 0.0, 0.0), (0, 0, 0, 2, 0, 0, 1.0, 0.0, 0.0),
           (0, 0, 0, -1, 2, 3, 1.0, 0.0, 0.0), (0, 0, 0, -1, -1, 1, 1.0, 0.0, 0.0), (0, 0, 0, -1, 0, -1, 1.0, 0.0, 0.0), (0, 0, 0, -1, 2 ** 31 - 1, 2 ** 31 - 1, 1.0, 0.0, 0.0)]
    for w in bad:
        from zgml_b200 import DeviceOp
        t = np.zeros(8 + 36, np.int32)
        t[0] = 3
        for i, x in enumerate((good, w, (-1,) + good[1:])):
            t[8 + 12 * i:14 + 12 * i] = x[:6]
            t[14 + 12 * i:17 + 12 * i] = np.array(x[6:], np.float32).view(np.int32)
        e = np.array([[1, 0x3f800000]] * 4, np.int32)
        p = Prog(cuda_backend, lambda at: [DeviceOp.logit_rules(at["dst"], at["src"], at["table"], 3, 90, history=at["h"], history_rows=9, bias=at["e"], masks=at["m"])],
                 dict(dst=np.full((3, 90), 7.0, np.float32), src=np.ones((3, 90), np.float32), table=t, h=h, e=e, m=masks))
        got = p.run(["dst"])
        assert np.isfinite(got[0]).all() and np.isnan(got[1]).all() and (got[2] == 7.0).all(), w
        p.close()


@pytest.mark.parametrize("wdt", ["bf16", "f32"])
@pytest.mark.parametrize("rank", [8, 24, 64])
@pytest.mark.parametrize("B,N,runs", [(300, 976, 1), (584, 640, 1), (700, 128, 1), (300, 976, 2), (1400, 300, 3)])
def test_adapters_of_one_tile(cuda_backend, wdt, rank, B, N, runs):
    """As many CTAs as tiles: a CTA has one product to do, or as many as its block has runs.  Other programs run between, so that nothing right lies in shared memory yet."""
    for seed in range(3):
        adapter_case(cuda_backend, wdt, B, N, 440, rank, 4, [(0, 0, (i * runs // B + seed) % 4) for i in range(B)], seed=seed)
        attend_case(cuda_backend, 3, 8, 2, 64, 64, 90, 33, [(i, 5, 0) for i in range(3)], loud=1e4)


@pytest.mark.parametrize("wdt", ["bf16", "f32"])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("form", ["runs", "blocks"])
def test_adapters_in_blocks_and_by_runs(cuda_backend, wdt, in_place, form):
    """Blocks of 128 rows with long runs, with runs of one to nine rows, without any adapter, with a bad one, and the last one cut short."""
    which = [i // 64 for i in range(128)] + [i % 5 - 1 for i in range(128)] + [-1] * 128 + [i // 9 % 4 for i in range(100)] + [7] * 28 + [2] * 33 + [i // 31 % 3 for i in range(110)]
    entries = [(-1 if i % 50 == 49 else 0, 0, w) for i, w in enumerate(which)]
    adapter_case(cuda_backend, wdt, len(entries), 328, 200, 24, 4, entries, in_place=in_place, form=form)
    adapter_case(cuda_backend, wdt, len(entries), 328, 200, 24, 4, entries, in_place=in_place, live=500, form=form)


@pytest.mark.parametrize("wdt", ["bf16", "f32"])
@pytest.mark.parametrize("rank", [8, 16, 24, 40, 64, 128, 136])
def test_adapters_of_many_outputs(cuda_backend, wdt, rank):
    """Runs of one row and of more, weights beyond what is fetched ahead, outputs that end inside a warp's."""
    for N in (9003, 333):
        for form in ("runs", "blocks"):
            adapter_case(cuda_backend, wdt, 13, N, 72, rank, 3, [(0, 0, w) for w in (0, 1, 1, 2, 2, 2, 2, 0, 0, 0, 0, 0, 1)], form=form)


# ── wide heads with many query rows over a long prefix: tensor cores ─────────────────────────────────────────────────
def wide_entries(B, R):
    return [(i, (5 + 7 * i) % (R + 1), 0) for i in range(B)]


@pytest.mark.parametrize("B,H,G,dk,dv,prefix,R", [(12, 16, 1, 576, 512, 700, 20), (64, 16, 1, 576, 512, 2500, 5), (40, 8, 2, 192, 136, 1000, 9), (33, 4, 2, 132, 128, 1100, 3), (34, 4, 2, 64, 260, 1000, 3),
                                                  (40, 6, 1, 1024, 640, 900, 7), (9, 16, 1, 320, 1024, 1025, 4)])
def test_wide_heads(cuda_backend, B, H, G, dk, dv, prefix, R):
    attend_case(cuda_backend, B, H, G, dk, dv, prefix, R, wide_entries(B, R), latent=G == 1 and dv <= dk, seed=B)


@pytest.mark.parametrize("shift", [0, 8, 64, 4])
def test_wide_values_inside_keys(cuda_backend, shift):
    """Values that are columns of the keys' rows, from the first or a later one on (4: no multiple of 16 bytes of half-precision pairs)."""
    attend_case(cuda_backend, 12, 16, 1, 576, 512, 800, 11, wide_entries(12, 11), latent=True, v_shift=shift, pad=4)


@pytest.mark.parametrize("cap,sink,scale", [(0.0, "f32", None), (5.0, None, None), (2.0, "bf16", None), (0.0, None, -0.05), (3.0, None, -0.1)])
def test_wide_caps_and_sinks(cuda_backend, cap, sink, scale):
    attend_case(cuda_backend, 40, 8, 2, 160, 160, 500, 33, wide_entries(40, 33), cap=cap, sink=sink, scale=scale)


def test_wide_idle_rows(cuda_backend):
    """Rows without a sequence, bad slots and lengths, rows behind the last, a prefix shorter than its cache, and none."""
    e = wide_entries(40, 9)
    e[3], e[7], e[11] = (-1, 0, 0), (200, 1, 0), (2, 10, 0)
    attend_case(cuda_backend, 40, 8, 2, 160, 160, 500, 9, e, live=37)
    attend_case(cuda_backend, 40, 8, 2, 160, 160, 100, 9, e, spare=900)
    attend_case(cuda_backend, 40, 8, 2, 160, 160, 0, 9, wide_entries(40, 9), spare=900)
    attend_case(cuda_backend, 40, 8, 2, 160, 160, 1, 9, wide_entries(40, 9), spare=900)


@pytest.mark.parametrize("loud", [1e-12, 300.0, 3e4])
def test_wide_magnitudes(cuda_backend, loud):
    attend_case(cuda_backend, 40, 8, 2, 160, 160, 500, 9, wide_entries(40, 9), loud=loud)


@pytest.mark.parametrize("what", ["column", "keys", "query nan", "key inf", "value inf", "value nan"])
def test_wide_what_pairs_cannot_hold(cuda_backend, what):
    """Columns of values and values of keys that are small beside the others; what is not finite."""
    from zgml_b200 import DeviceOp
    B, H, G, d, P, R = 40, 8, 2, 160, 500, 4
    r = np.random.default_rng(5)
    q, own, pre = r.standard_normal((B, H * d)).astype(np.float32), r.standard_normal((B, R, 2 * G * d)).astype(np.float32), r.standard_normal((1, P, 2 * G * d)).astype(np.float32)
    v = G * d
    if what == "column":
        pre[:, :, v + 7] *= 1e-9
        own[:, :, v + 7] *= 1e-9
    elif what == "keys":                                # the ones that count have small values, others that do not have large ones
        pre[:, ::2, v:] *= 1e-8
        own[:, :, v:] *= 1e-8
        pre[:, ::2, :v], pre[:, 1::2, :v] = 2 * q[0, :1], -30 * np.sign(q[0, :1])
        q[:] = q[0, 0]
    elif what == "query nan":
        q[17, 5] = NAN
    elif what == "key inf":
        pre[0, 333, 11] = np.inf
    else:
        pre[0, 333, v + 11] = np.inf if what == "value inf" else NAN
    entries = wide_entries(B, R)
    t = table(entries, B, P)
    op = DeviceOp.shared_attention(0, 1, 2, 2, 3, 3, 4, 0, 0, v, 0, v, B, H, G, d, d, H * d, 2 * v, 2 * v, R, 2 * v, 2 * v, P, 0.05)
    heads = lambda c, col: c[:, :, col:col + v].reshape(c.shape[0], c.shape[1], G, d)
    with np.errstate(all="ignore"):
        want, tol = ref.attend(np.zeros((B, H, d), np.float32), q.reshape(B, H, d), heads(own, 0), heads(own, v), heads(pre, 0), heads(pre, v), entries, B, P, 0, 0.05)
    p = Prog(cuda_backend, lambda at: [op], dict(dst=np.zeros((B, H * d), np.float32), q=q, own=own, pre=pre, table=t))
    got = p.run(["dst"]).reshape(B, H, d)
    p.close()
    if what in ("column", "keys"):
        relative = want[:, :, 7] if what == "column" else want      # small beside the rest, and as exact as if it were alone
        mine = got[:, :, 7] if what == "column" else got
        assert np.abs(mine - relative).max() <= 1e-4 * np.abs(relative).max()
        return
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    assert (np.abs(got[fine] - want[fine]) <= np.where(np.isfinite(tol), tol, 1e-4)[fine]).all()


@pytest.mark.parametrize("prefix,slot", [(501, 0), (500, 2), (500, -1), (-1, 0), (2 ** 31 - 1, 0)])
def test_wide_prefix_out_of_range(cuda_backend, prefix, slot):
    from zgml_b200 import DeviceOp
    B, d = 40, 160
    one = np.ones((B, 8 * d), np.float32)
    make = lambda at: [DeviceOp.shared_attention(at["dst"], at["q"], at["own"], at["own"], at["pre"], at["pre"], at["table"], 0, 0, 0, 0, 0, B, 8, 1, d, d, 8 * d, d, d, 4, d, d, 500, 0.1)]
    p = Prog(cuda_backend, make, dict(dst=one, q=one, own=np.ones((B, 4, d), np.float32), pre=np.ones((2, 500, d), np.float32), table=np.zeros(8 + 4 * B, np.int32)))
    assert np.isnan(p.run(["dst"], table=table([(i, 1, 0) for i in range(B)], B, prefix, slot))).all()
    assert np.abs(p.run(["dst"], table=table([(i, 1, 0) for i in range(B)], B, 500, 1)) - 1.0).max() <= 2.0 ** -20          # the same program, another table: a mean of ones
    assert (p.run(["dst"], table=table([(i, 0, 0) for i in range(B)], B, 0, -5)) == 0.0).all()
    p.close()


def test_no_wait_ran_out(cuda_backend):
    """The kernels that wait on barriers count waits that gave up."""
    from zgml_b200 import DeviceOp, DeviceProgram
    h = cuda_backend.compile_program(DeviceProgram([DeviceOp.logit_rules(0, 0, 1, 1, 4)], [4, 20]))
    assert cuda_backend.lib.zg_cuda_program_stats(h.ptr, 5) == 0
    cuda_backend.free_program(h)
