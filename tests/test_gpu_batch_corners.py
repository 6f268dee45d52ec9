"""The batched ops where their documentation allows more than their other tests use: caches of keys and values in buffers of their own, several ops that share one workspace in one
program, launches outside a graph, and elements beyond 2^32 of a buffer."""
import numpy as np
import pytest

import batch_reference as ref
from test_gpu_batchops import Prog, adapter_case, attend_case, close, table, wide_entries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,H,G,dk,dv,P,Rp", [(3, 8, 2, 64, 48, 40, 60), (40, 8, 2, 64, 48, 500, 1300), (40, 8, 2, 128, 64, 500, 1300), (40, 8, 2, 160, 136, 500, 1300), (40, 8, 1, 64, 256, 500, 1300)])
def test_keys_and_values_in_buffers_of_their_own(cuda_backend, B, H, G, dk, dv, P, Rp):
    """Rows of other widths, other numbers of slots: a slot that only one of the two caches has does not exist."""
    from zgml_b200 import DeviceOp
    r = np.random.default_rng(B + dk)
    R, slots, kw, vw, pkw, pvw = 9, B, G * dk + 4, G * dv + 12, G * dk + 8, G * dv
    f = lambda *s: r.standard_normal(s).astype(np.float32)
    q, kc, vc, kp, vp = f(B, H * dk), f(slots + 1, R, kw), f(slots, R, vw), f(2, Rp, pkw), f(3, Rp, pvw)
    entries = [(i, (5 + 7 * i) % (R + 1), 0) for i in range(B)]
    entries[1] = (slots, 1, 0)                          # keys are there, values are not
    op = DeviceOp.shared_attention(0, 1, 2, 3, 4, 5, 6, 0, 4, 8, 8, 0, B, H, G, dk, dv, H * dk, kw, vw, R, pkw, pvw, Rp, dk ** -0.5)
    p = Prog(cuda_backend, lambda at: [op], dict(dst=np.zeros((B, H * dv), np.float32), q=q, kc=kc, vc=vc, kp=kp, vp=vp, table=np.zeros(8 + 4 * B, np.int32)))
    heads = lambda c, col, d: c[:, :, col:col + G * d].reshape(c.shape[0], c.shape[1], G, d)
    for slot in (1, 2):                                 # of the prefix: the second one has values only
        got = p.run(["dst"], table=table(entries, B, P, slot)).reshape(B, H, dv)
        want, tol = ref.attend(np.zeros((B, H, dv)), q.reshape(B, H, dk), heads(kc[:slots], 4, dk), heads(vc, 8, dv), heads(kp, 8, dk), heads(vp[:2], 0, dv), entries, B, P, slot, dk ** -0.5)
        close(got, want, tol, slot)
        assert np.isnan(want[1]).all() and np.isnan(want).all() == (slot == 2)
    p.close()


def test_ops_that_share_a_workspace(cuda_backend):
    """Attention over narrow heads, over wide ones, and adapters of many rows, twice each in one program, in turns: to the bit what each gives alone, again and again."""
    from zgml_b200 import DeviceOp, DeviceProgram, ProgramIO, abi
    r = np.random.default_rng(4)
    f = lambda *s: r.standard_normal(s).astype(np.float32)
    B, H, G, P, Rp, R = 40, 8, 2, 500, 1300, 4
    t = table(wide_entries(B, R), B, P)
    bufs, makers, inputs = [], [], {}

    def buf(a):
        bufs.append(a)
        return len(bufs) - 1
    at_t = buf(t)
    outs = []
    for turn in range(2):
        for d in (64, 160):
            w = 2 * G * d
            o, q, own, pre = buf(np.zeros(B * H * d, np.float32)), buf(f(B, H * d)), buf(f(B, R, w)), buf(f(1, Rp, w))
            makers.append(DeviceOp.shared_attention(o, q, own, own, pre, pre, at_t, 0, 0, G * d, 0, G * d, B, H, G, d, d, H * d, w, w, R, w, w, Rp, d ** -0.5))
            outs.append(o)
        rows, N, K, rank, A = 300, 200, 264, 16, 3
        o, x, w, base, at = buf(np.zeros(rows * N, np.float32)), buf(f(rows, K)), buf(f(A * rank * (K + N))), buf(f(rows, N)), buf(table([(0, 0, i // 70 % 4 - 1) for i in range(rows)], rows))
        makers.append(DeviceOp.adapter_linear(o, x, w, 0, A * rank * K, at, rows, N, K, rank, A, abi.W_F32, base=base))
        outs.append(o)
    ins = [ProgramIO(i, np.ascontiguousarray(a).view(np.float32).ravel()) for i, a in enumerate(bufs) if i not in outs]

    def run(ops, wanted, times):
        h = cuda_backend.compile_program(DeviceProgram(ops, [b.size for b in bufs]))
        got = []
        for _ in range(times):
            got.append([np.zeros(bufs[o].size, np.float32) for o in wanted])
            cuda_backend.execute_program(h, ins, [ProgramIO(o, g) for o, g in zip(wanted, got[-1])])
        cuda_backend.free_program(h)
        return got
    alone = [run([op], [o], 1)[0][0] for op, o in zip(makers, outs)]
    for got in run(makers, outs, 5):
        assert all(np.array_equal(g, a) for g, a in zip(got, alone)) and all(np.isfinite(a).all() for a in alone)


@pytest.mark.parametrize("fmt", ["f32", "bf16"])
def test_launches_outside_a_graph(cuda_backend, fmt):
    attend_case(cuda_backend, 40, 8, 2, 160, 160, 500, 9, wide_entries(40, 9), graph=False)
    cuda_backend.set_graph_mode(False)
    for B, form in ((9, "runs"), (300, "blocks")):
        adapter_case(cuda_backend, fmt, B, 200, 264, 16, 4, [(0, 0, (i // 70) % 5 - 1) for i in range(B)], form=form)
    cuda_backend.set_graph_mode(True)


@pytest.mark.parametrize("G,d,B", [(2, 64, 4), (2, 64, 40), (2, 160, 40)])
def test_beyond_2_to_the_32_elements(cuda_backend, G, d, B):
    """Caches of more than 2^32 values: the rows that are used lie at their very ends."""
    from zgml_b200 import DeviceBuffer, DeviceOp, DeviceProgram, ExternBuffer, ProgramIO
    r = np.random.default_rng(B)
    H, P, Rp, R = 4 * G, 500, 1 << 16, 64
    w = 2 * G * d
    slots, pslots = (1 << 32) // (R * w) + B + 1, (1 << 32) // (Rp * w) + 2
    own = DeviceBuffer(cuda_backend, 4 * slots * R * w)
    pre = DeviceBuffer(cuda_backend, 4 * pslots * Rp * w)
    first = slots - B                                   # the requests' slots
    k = r.standard_normal((B, R, w)).astype(np.float32)
    kp = r.standard_normal((1, Rp, w)).astype(np.float32)
    own.upload(k, 4 * first * R * w)
    pre.upload(kp, 4 * (pslots - 1) * Rp * w)
    q, new = r.standard_normal((B, H * d)).astype(np.float32), r.standard_normal((B, w)).astype(np.float32)
    entries = [(i, 1 + (9 * i) % R, 0) for i in range(B)]
    t = table([(first + s, n, a) for s, n, a in entries], B, P, pslots - 1)
    ops = [DeviceOp.batch_append(0, 4, 5, 0, 0, B, w, w, w, R), DeviceOp.shared_attention(2, 3, 0, 0, 1, 1, 5, 0, 0, G * d, 0, G * d, B, H, G, d, d, H * d, w, w, R, w, w, Rp, d ** -0.5)]
    h = cuda_backend.compile_program(DeviceProgram(ops, [own.elems, pre.elems, B * H * d, q.size, new.size, t.size], [], [], [ExternBuffer(0, own), ExternBuffer(1, pre)]))
    got = np.zeros((B, H, d), np.float32)
    cuda_backend.execute_program(h, [ProgramIO(3, q.ravel()), ProgramIO(4, new.ravel()), ProgramIO(5, t)], [ProgramIO(2, got)])
    cuda_backend.free_program(h)
    for i, (s, n, _) in enumerate(entries):
        k[s, n - 1] = new[i]
    assert np.array_equal(own.download(byte_offset=4 * first * R * w, count=k.size).reshape(k.shape), k)
    heads = lambda c, col: c[:, :, col:col + G * d].reshape(c.shape[0], c.shape[1], G, d)
    want, tol = ref.attend(np.zeros((B, H, d)), q.reshape(B, H, d), heads(k, 0), heads(k, G * d), heads(kp, 0), heads(kp, G * d), entries, B, P, 0, d ** -0.5)
    own.free()
    pre.free()
    close(got, want, tol)
