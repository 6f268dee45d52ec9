"""The ops over paged 8-bit caches in small programs against NumPy in 64 bits: heads and pages of every form, rows that are idle, see nothing or name places and pages that do not exist, tokens
of one step in one page, scales that grow, values that are not finite, and a decode loop in which the ops run together.  Tolerances come from the number of roundings (tests/page_reference.py)."""
import numpy as np
import pytest

import page_reference as ref
from test_gpu_batchops import Prog, close, table
from zgml_b200.host.pages import PagePool, move_words, pack_pages, page_moves, page_words, unpack_pages

pytestmark = pytest.mark.gpu
i32 = lambda a: np.ascontiguousarray(a).view(np.int32)


def pool(r, pages, G, dk, dv, page, lo=-9, hi=-4):
    keys, values = r.integers(-127, 128, (pages, G, page, dk)).astype(np.int8), r.integers(-127, 128, (pages, G, page, dv)).astype(np.int8)
    return keys, values, (2.0 ** r.integers(lo, hi, (pages, G, 2))).astype(np.float32)


# ── PAGE_APPEND ──────────────────────────────────────────────────────────────────────────────────────────────────────
class Append:
    def __init__(self, be, B, G, dk, dv, page, *, H=0, turn_at=0, rot=0, layout="pairs", tabled=False, pad=0, slots=4, most=3, pages=16, seed=0, lo=-9, hi=-4):
        from zgml_b200 import DeviceOp
        r = self.r = np.random.default_rng(seed)
        self.a = dict(B=B, G=G, dk=dk, dv=dv, page=page, turn_at=turn_at, rot=rot, layout=layout, q_heads=H)
        self.cols = (pad + G * dv, pad, pad + G * (dk + dv))             # values before keys, queries last
        rs, trs = self.cols[2] + H * dk + pad, H * dk + 2 * pad
        self.pool = pool(r, pages, G, dk, dv, page, lo, hi)
        self.src, self.turned, self.pad = r.standard_normal((B, rs)).astype(np.float32), r.standard_normal((B, max(1, trs))).astype(np.float32), pad
        self.page_table = r.permutation(pages)[:slots * most].reshape(slots, most).astype(np.int32)
        freqs = r.uniform(0.01, 1.0, max(1, rot // 2)).astype(np.float32)
        self.freqs = freqs.astype(np.float64) if tabled else 1e4 ** (-2.0 * np.arange(rot // 2) / max(1, rot))
        make = lambda at: [DeviceOp.page_append(at["pages"], at["src"], at["page_table"], at["table"], self.cols[0], self.cols[1], B, G, dk, dv, rs, page, most, turn_at=turn_at, rot=rot, rot_base=1e4, rot_layout=layout,
                                                freqs=at["freqs"] if tabled else None, q_heads=H, q_col=self.cols[2], turned=at["turned"], turned_col=pad, turned_rs=trs)]
        arrays = dict(pages=pack_pages(*self.pool), src=self.src, page_table=self.page_table, table=np.zeros(8 + 4 * B, np.int32), freqs=freqs, turned=self.turned)
        self.p = Prog(be, make, arrays)

    def check(self, entries, live=None, prefix=0, src=None, page_table=None, state=None):
        a, H, dk = self.a, self.a["q_heads"], self.a["dk"]
        src, page_table, state = self.src if src is None else src, self.page_table if page_table is None else page_table, state or self.pool
        live = len(entries) if live is None else live
        words, turned = self.p.run(["pages", "turned"], table=table(entries, a["B"], prefix, live=live), src=src, page_table=page_table, pages=pack_pages(*state))
        k, v, s = unpack_pages(i32(words), a["G"], dk, a["dv"], a["page"])
        wk, wv, ws, wt = ref.append(*state, src, page_table, entries, live, prefix, self.cols, freqs=self.freqs, turned=self.turned[:, self.pad:self.pad + H * dk], **a)
        assert np.array_equal(s, ws.astype(np.float32), equal_nan=True)
        fine = ~np.isnan(s)
        assert np.array_equal(k[fine[..., 0]], wk[fine[..., 0]]) and np.array_equal(v[fine[..., 1]], wv[fine[..., 1]])
        if H:
            close(turned[:, self.pad:self.pad + H * dk], wt, 2.0 ** -24 * np.abs(wt) + 1e-12)
        rest = np.ones(turned.shape[1], bool)
        rest[self.pad:self.pad + H * dk] = False
        assert np.array_equal(turned[:, rest], self.turned[:, rest])
        return k, v, s

    def close(self):
        self.p.close()


@pytest.mark.parametrize("B,H,G,dk,dv,page,turn_at,rot,layout,pad,tabled", [(1, 2, 1, 128, 128, 16, 0, 128, "halves", 0, False), (5, 4, 2, 16, 8, 16, 4, 12, "halves", 3, True), (33, 3, 3, 80, 64, 32, 0, 40, "pairs", 1, False),
                                                                            (4, 0, 2, 7, 33, 64, 1, 6, "pairs", 2, False), (6, 1, 2, 32, 1, 16, 0, 0, "pairs", 0, False), (9, 8, 1, 256, 256, 64, 0, 256, "halves", 1, True), (2, 9, 3, 250, 17, 32, 200, 50, "pairs", 5, False)])
@pytest.mark.parametrize("prefix", [0, 131071])
def test_page_append(cuda_backend, B, H, G, dk, dv, page, turn_at, rot, layout, pad, tabled, prefix):
    a = Append(cuda_backend, B, G, dk, dv, page, H=H, turn_at=turn_at, rot=rot, layout=layout, tabled=tabled, pad=pad, seed=B + dk)
    full = [(i % 4, 1 + (7 * i) % (3 * page), 0) for i in range(B)]      # (some in one page, some twice in one place)
    odd = [(-1, 1, 0), (4, 1, 0), (0, 3 * page + 1, 0), (1, -1, 0), (0, 0, 0), (2, 3 * page, 0)][:B]
    odd += full[len(odd):]
    for entries, live in ((full, B), (odd, B), ([(0, 2, 0)] * B, B), (full, B - 1), (full, B + 7), (full, -3)):
        a.check(entries, live, prefix)
    bad = a.page_table.copy()
    bad[0, :], bad[1, 1] = [-1, 16, 1 << 30], -7
    a.check(full, B, prefix, page_table=bad)
    a.check(full, B, -1)
    a.close()


@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("first,tokens", [(0, 1), (5, 1), (0, 70), (3, 64), (15, 2), (63, 66), (16, 16), (1, 15)])
def test_a_sequences_tokens_at_once(cuda_backend, page, first, tokens):
    """Prompts and drafts: a page that had tokens, whole pages, a page that is begun; in any order of rows, among other sequences."""
    a = Append(cuda_backend, 2 * tokens + 1, 2, 48, 40, page, H=2, rot=48, slots=3, most=9, pages=40, seed=first)
    rows = [(0, first + 1 + i, 0) for i in range(tokens)] + [(2, first + 1 + i, 0) for i in range(tokens)] + [(1, 1, 0)]
    a.check(rows)
    a.check([rows[i] for i in a.r.permutation(len(rows))])
    a.close()


@pytest.mark.parametrize("B,G", [(5000, 8), (2100, 8), (300, 1), (90, 20)])
def test_prompts_and_single_tokens_at_once(cuda_backend, B, G):
    """Long runs of rows in one page beside short ones and single rows, in order and shuffled by blocks and row by row."""
    a = Append(cuda_backend, B, G, 8, 4, 16, H=1, rot=8, slots=100, most=40, pages=4000, seed=B)
    r, rows = a.r, []
    for slot in r.permutation(100):
        if len(rows) < B:
            first, tokens = int(r.integers(0, 30)), int(r.choice([1, 1, 2, 4, 5, 6, 40, 600]))
            rows += [(int(slot), first + 1 + i, 0) for i in range(tokens)]
    rows = rows[:B]
    rows += [(-1, 1, 0)] * (B - len(rows))
    a.check(rows)
    blocks = [rows[i:i + 7] for i in range(0, B, 7)]
    a.check([x for i in r.permutation(len(blocks)) for x in blocks[i]])
    a.check([rows[i] for i in r.permutation(B)])
    a.close()


def test_scales_grow_and_stay(cuda_backend):
    """Token after token in one page, ever larger and then small again: each code is what the definition makes of the last state."""
    a = Append(cuda_backend, 1, 1, 8, 8, 16, slots=1, most=1, pages=2)
    state = tuple(x.copy() for x in a.pool)
    state[2][:] = np.nan                                 # (what a page held does not count when its first token comes)
    held = np.zeros((16, 16))
    for t in range(16):
        src = (a.r.standard_normal(a.src.shape) * 2.0 ** (min(t, 24 - 2 * t) - 3)).astype(np.float32)
        held[t] = np.concatenate([src[0, a.cols[0]:a.cols[0] + 8], src[0, a.cols[1]:a.cols[1] + 8]])
        state = a.check([(0, t + 1, 0)], src=src, state=state)
        k, v, s = state
        p = a.page_table[0, 0]
        for codes, which, cols in ((k, 0, slice(0, 8)), (v, 1, slice(8, 16))):
            assert np.abs(codes[p, 0, :t + 1] * float(s[p, 0, which]) - held[:t + 1, cols]).max() < s[p, 0, which]
    a.close()


@pytest.mark.parametrize("value,needs", [(0.0, 2.0 ** -126), (127.0, 1.0), (127.5, 2.0), (np.nextafter(np.float32(127), np.float32(128)), 2.0), (1e-45, 2.0 ** -126), (127 * 2.0 ** -126, 2.0 ** -126), (2.0 ** -119, 2.0 ** -125), (3.4e38, 2.0 ** 122), (-64.0, 2.0 ** -0),
                                         (63.5, 0.5), (np.inf, np.nan), (-np.inf, np.nan), (np.nan, np.nan)])
def test_scales(cuda_backend, value, needs):
    a = Append(cuda_backend, 2, 1, 4, 4, 16, slots=2, most=1, pages=2)
    src = np.zeros_like(a.src)
    src[0, a.cols[0] + 2], src[1, a.cols[1] + 3] = value, value
    k, v, s = a.check([(0, 1, 0), (1, 1, 0)], src=src)
    x, y = a.page_table[:, 0]
    assert np.array_equal(s[[x, y], 0], np.array([[needs, 2.0 ** -126], [2.0 ** -126, needs]], np.float32), equal_nan=True)
    # a page that holds tokens: the larger of both, and a scale that is not a number stays
    state = (k, v, s)
    src[:] = 0.25
    k, v, s2 = a.check([(0, 2, 0), (1, 2, 0)], src=src, state=state)
    assert np.isnan(s2[x, 0, 0]) == np.isnan(needs) and np.isnan(s2[y, 0, 1]) == np.isnan(needs)
    a.check([(0, 1, 0), (1, 1, 0)], src=src, state=(k, v, s2))           # until the page begins anew
    a.close()


def test_a_pool_of_zeros(cuda_backend):
    """Pages that nothing wrote, appended to in the middle."""
    a = Append(cuda_backend, 1, 2, 20, 12, 32, slots=1, most=1, pages=1)
    words = a.p.run(["pages"], table=table([(0, 9, 0)], 1), pages=np.zeros((1, page_words(2, 20, 12, 32)), np.int32))
    k, v, s = unpack_pages(i32(words), 2, 20, 12, 32)
    new = a.src[0, a.cols[0]:a.cols[0] + 40].reshape(2, 20)
    assert np.array_equal(s[0, :, 0], [ref.scale_for(np.abs(x).max()) for x in new])
    assert np.array_equal(k[0, :, 8], np.rint(new / s[0, :, :1])) and not np.delete(k[0], 8, 1).any() and not np.delete(v[0], 8, 1).any()
    a.close()


# ── PAGE_READ, PAGE_COPY ─────────────────────────────────────────────────────────────────────────────────────────────
@pytest.mark.parametrize("B,G,dk,dv,page,k_col,v_col,pad", [(1, 1, 128, 128, 16, 0, None, 0), (40, 3, 44, 7, 16, 2, 200, 3), (100, 2, 64, 64, 64, 128, 0, 0), (17, 1, 1, 255, 32, 0, None, 1), (65, 8, 16, 16, 32, 0, None, 4)])
def test_page_read(cuda_backend, B, G, dk, dv, page, k_col, v_col, pad):
    from zgml_b200 import DeviceOp
    r = np.random.default_rng(B)
    keys, values, scales = pool(r, 13, G, dk, dv, page)
    scales[3, 0, 0] = np.nan
    page_table = r.permutation(13)[:12].reshape(4, 3).astype(np.int32)
    page_table[3, 1], page_table[3, 2] = 13, -1
    v_at = k_col + G * dk if v_col is None else v_col
    rs = max(k_col + G * dk, v_at + G * dv) + pad
    dst = r.standard_normal((B, rs)).astype(np.float32)
    make = lambda at: [DeviceOp.page_read(at["dst"], at["pages"], at["page_table"], at["table"], B, G, dk, dv, page, 3, k_col=k_col, v_col=v_col, dst_rs=rs)]
    p = Prog(cuda_backend, make, dict(dst=dst, pages=pack_pages(keys, values, scales), page_table=page_table, table=np.zeros(8 + 4 * B, np.int32)))
    run = [(0, 1 + i % (3 * page), 0) for i in range(B)]
    mixed = [(int(r.integers(-1, 6)), int(r.integers(-1, 3 * page + 2)), 0) for _ in range(B)]
    mine = np.r_[np.arange(k_col, k_col + G * dk), np.arange(v_at, v_at + G * dv)]
    for entries, live in ((run, B), (mixed, B), (run[::-1], B - 1), (run, B + 3), (run, -1)):
        got = p.run(["dst"], table=table(entries, B, live=live))
        assert np.array_equal(got[:, mine], ref.read(keys, values, scales, page_table, entries, live, B, dst[:, mine]).astype(np.float32), equal_nan=True)
        assert np.array_equal(np.delete(got, mine, 1), np.delete(dst, mine, 1))
    p.close()


@pytest.mark.parametrize("words", [1, 5, 4, 1028, 8224, 8223])
def test_page_copy(cuda_backend, words):
    from zgml_b200 import DeviceOp
    r = np.random.default_rng(words)
    pages = r.integers(-2 ** 31, 2 ** 31, (9, words)).astype(np.int32)
    p = Prog(cuda_backend, lambda at: [DeviceOp.page_copy(at["pages"], at["moves"], 4, words)], dict(pages=pages, moves=np.zeros(move_words(4), np.int32)))
    for moves in ([(8, 0), (7, 2), (8, 3)], [], [(0, 1), (2, 3), (4, 5), (6, 7)]):
        want = pages.copy()
        for a, b in moves:
            want[b] = pages[a]
        assert np.array_equal(i32(p.run(["pages"], moves=page_moves(moves, 4, 9))), want)
    t = page_moves([(8, 0)], 4, 9)
    for bad in ((9, 1), (1, 9), (-1, 1), (1, -1), (3, 3), (2 ** 31 - 1, 0)):      # (behind the host's back)
        t[0], t[12:14] = 2, bad
        want = pages.copy()
        want[0] = pages[8]
        assert np.array_equal(i32(p.run(["pages"], moves=t)), want)
    t[0] = 9                                             # more than the table has: the two moves behind are (0, 0)
    t[12:14] = (7, 1)
    want[1] = pages[7]
    assert np.array_equal(i32(p.run(["pages"], moves=t)), want)
    p.close()


# ── PAGED_ATTENTION ──────────────────────────────────────────────────────────────────────────────────────────────────
def attend_case(be, B, H, G, dk, dv, page, most, entries, *, window=0, cap=0.0, sink=None, bf16=False, pad=0, slots=3, pages=None, live=None, seed=0, loud=1.0, lo=-7, hi=-4, scale=None, change=None, graph=True, spare=0):
    """spare: columns of the page table behind those that any row uses."""
    from zgml_b200 import DeviceOp, abi
    r = np.random.default_rng(seed)
    pages = slots * most + 1 if pages is None else pages
    keys, values, scales = pool(r, pages, G, dk, dv, page, lo, hi)
    page_table = np.full((slots, most + spare), -1, np.int32)
    page_table[:, :most] = r.permutation(pages)[:slots * most].reshape(slots, most)
    most += spare
    qrs, drs, scale = H * dk + 2 * pad, H * dv + pad, dk ** -0.5 if scale is None else scale
    q, dst = (loud * r.standard_normal((B, qrs))).astype(np.float32), r.standard_normal((B, drs)).astype(np.float32)
    s = None if sink is None else np.full(H, sink, np.float32) if np.ndim(sink) == 0 else np.asarray(sink, np.float32)
    if change is not None:
        change(q, keys, values, scales, page_table)
    stored = None if s is None else (s.view(np.uint32) >> 16).astype(np.uint16) if bf16 else s
    if bf16:
        s = (stored.astype(np.uint32) << 16).view(np.float32)
    make = lambda at: [DeviceOp.paged_attention(at["dst"], at["q"], at["pages"], at["page_table"], at["table"], B, H, G, dk, dv, qrs, page, most, scale, q_col=pad, window=window, softcap=cap,
                                                sink=at["sink"] if s is not None else None, sink_wdt=abi.W_BF16 if bf16 else abi.W_F32, dst_rs=drs, dst_col=pad)]
    be.set_graph_mode(graph)
    p = Prog(be, make, dict(dst=dst, q=q, pages=pack_pages(keys, values, scales), page_table=page_table, table=np.zeros(8 + 4 * B, np.int32), sink=np.zeros(2, np.float32) if s is None else stored if not bf16 else np.r_[stored, stored].view(np.float32)))
    live = len(entries) if live is None else live
    got = p.run(["dst"], table=table(entries, B, live=live))
    again = p.run(["dst"], table=table(entries, B, live=live))
    be.set_graph_mode(True)
    want, tol = ref.attend(dst[:, pad:].reshape(B, H, dv), q[:, pad:pad + H * dk].reshape(B, H, dk), keys, values, scales, page_table, entries, live, B, scale, window, cap, s)
    p.close()
    assert np.array_equal(got, again, equal_nan=True) and np.array_equal(got[:, :pad], dst[:, :pad])
    close(got[:, pad:].reshape(B, H, dv), want, tol)
    return got[:, pad:].reshape(B, H, dv), want


LENGTHS = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191]


@pytest.mark.parametrize("H,G,dk,dv", [(1, 1, 128, 128), (8, 2, 128, 128), (9, 3, 64, 64), (6, 2, 80, 48), (16, 1, 96, 112), (5, 5, 33, 17), (4, 1, 256, 256), (24, 2, 192, 128), (40, 1, 64, 64), (3, 1, 1, 1), (7, 7, 16, 250), (17, 1, 250, 16), (32, 1, 128, 256)])
@pytest.mark.parametrize("page", [16, 32, 64])
def test_heads_and_lengths(cuda_backend, H, G, dk, dv, page):
    most = 192 // page
    entries = [(i % 3, n, 0) for i, n in enumerate(LENGTHS)]
    attend_case(cuda_backend, len(entries) + 2, H, G, dk, dv, page, most, entries, pad=(dk + H) % 3, seed=H)


@pytest.mark.parametrize("window", [1, 5, 16, 40, 64, 100, 1000, 2 ** 32 - 1])
@pytest.mark.parametrize("page", [16, 64])
def test_windows(cuda_backend, window, page):
    entries = [(i % 3, n, 0) for i, n in enumerate(LENGTHS)]
    attend_case(cuda_backend, len(entries), 8, 2, 64, 80, page, 192 // page, entries, window=window, seed=window % 7)


@pytest.mark.parametrize("cap,sink,bf16", [(30.0, None, False), (2.0, 0.5, False), (0.0, 1.5, True), (50.0, -np.inf, False), (0.0, 40.0, False), (0.0, -90.0, False), (0.25, 0.0, True)])
def test_caps_and_sinks(cuda_backend, cap, sink, bf16):
    entries = [(0, 150, 0), (1, 1, 0), (2, 64, 0), (0, 0, 0)]
    attend_case(cuda_backend, 4, 6, 2, 64, 64, 16, 12, entries, cap=cap, sink=sink, bf16=bf16, loud=3.0, scale=0.3)


@pytest.mark.parametrize("tokens", [2, 3, 7, 16, 40])
@pytest.mark.parametrize("H,G", [(4, 4), (8, 2), (12, 1), (3, 1)])
def test_drafts(cuda_backend, tokens, H, G):
    """Tokens of one sequence in a row, each sees one more; other orders of the rows, two sequences in turns."""
    for slots in ([0] * tokens + [1] * tokens, [0, 1] * tokens, [0] * (tokens - 1) + [-1] + [0] * tokens):
        n = {}
        entries = []
        for s in slots:
            n[s] = n.get(s, 180 - tokens if s else 90) + 1
            entries.append((s, n[s], 0))
        attend_case(cuda_backend, len(entries), H, G, 64, 64, 32, 8, entries, seed=tokens)
    attend_case(cuda_backend, tokens, H, G, 64, 64, 32, 8, [(2, 200 - 3 * i, 0) for i in range(tokens)], window=50)


@pytest.mark.parametrize("B,H,G,length,page", [(1, 8, 8, 5000, 16), (1, 32, 8, 3001, 64), (2, 4, 1, 9999, 32), (1, 1, 1, 20011, 16), (40, 8, 2, 700, 16), (3, 16, 1, 4097, 64)])
def test_long_sequences(cuda_backend, B, H, G, length, page):
    """Positions over many CTAs, rows of very different lengths among them."""
    most = -(-length // page)
    entries = [(i % 3, max(1, length - i * 611 % length), 0) for i in range(B)]
    attend_case(cuda_backend, B, H, G, 64, 64, page, most, entries)
    if B > 1:
        attend_case(cuda_backend, B, H, G, 64, 64, page, most, [(i % 3, 1 if i else length, 0) for i in range(B)], sink=0.0)


def test_rows_that_are_not_there(cuda_backend):
    def change(q, keys, values, scales, page_table):
        page_table[1, 2], page_table[2, 0] = -1, 10 ** 6
    entries = [(-1, 5, 0), (3, 1, 0), (0, 0, 0), (0, 193, 0), (0, -1, 0), (1, 32, 0), (1, 33, 0), (2, 192, 0), (2 ** 31 - 1, 3, 0), (0, 2 ** 31 - 1, 0), (0, 192, 0)]
    got, _ = attend_case(cuda_backend, 13, 4, 2, 64, 64, 16, 12, entries, change=change)
    assert np.isnan(got[[1, 3, 4, 6, 7, 8, 9]]).all() and np.isfinite(np.delete(got, [1, 3, 4, 6, 7, 8, 9], 0)).all()
    attend_case(cuda_backend, 13, 4, 2, 64, 64, 16, 12, entries, change=change, window=20)      # a page before the window does not count
    for live in (0, 5, -1, 99):
        attend_case(cuda_backend, 11, 4, 2, 64, 64, 16, 12, entries, live=live)


def test_what_lies_behind_a_sequence(cuda_backend):
    """Scales that are not numbers on pages that no row sees, and codes beyond a row's length on pages that it does see, change nothing."""
    def change(q, keys, values, scales, page_table):
        scales[page_table[0, 2:]] = np.nan
        scales[page_table[1, :1]] = np.nan
        keys[page_table[2, 3], :, 1:], values[page_table[2, 3], :, 1:] = 127, -127
    entries = [(0, 32, 0), (0, 31, 0), (1, 40, 0), (2, 49, 0)]
    got, _ = attend_case(cuda_backend, 4, 4, 2, 64, 64, 16, 12, entries, change=change, window=24)
    assert np.isfinite(got).all()
    got, _ = attend_case(cuda_backend, 4, 4, 2, 64, 64, 16, 12, entries, change=change)
    assert np.isnan(got[2]).all() and np.isfinite(got[[0, 1, 3]]).all()


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_queries_that_are_not_finite(cuda_backend, value):
    def change(q, keys, values, scales, page_table):
        q[1, 64:128] = value                             # of one head
    got, want = attend_case(cuda_backend, 3, 4, 2, 64, 64, 16, 12, [(0, 100, 0), (1, 100, 0), (2, 100, 0)], change=change)
    assert np.isnan(got[1, 1]).all() and np.isfinite(np.delete(got.reshape(12, 64), 5, 0)).all()


@pytest.mark.parametrize("lo,hi", [(-120, 100), (-60, -20), (20, 60), (100, 118), (-126, -125)])
def test_scales_far_apart(cuda_backend, lo, hi):
    """Pages of very different magnitudes; keys that small have scores near 0, so that every value counts."""
    def change(q, keys, values, scales, page_table):
        scales[..., 0] = 2.0 ** -20
    attend_case(cuda_backend, 3, 4, 2, 64, 64, 16, 12, [(0, 190, 0), (1, 100, 0), (2, 3, 0)], change=change, lo=lo, hi=hi)


@pytest.mark.parametrize("loud", [1e-30, 1e-8, 300.0, 1e5])
def test_scores_of_any_size(cuda_backend, loud):
    attend_case(cuda_backend, 3, 4, 2, 64, 64, 16, 12, [(0, 190, 0), (1, 100, 0), (2, 3, 0)], loud=loud)


def test_queries_with_outliers(cuda_backend):
    """One element of a query far above the others, which still count where it meets codes of 0."""
    def change(q, keys, values, scales, page_table):
        q[:, 5] = 3e4
        keys[..., 5] = 0
    attend_case(cuda_backend, 3, 4, 2, 64, 64, 16, 12, [(0, 190, 0), (1, 100, 0), (2, 3, 0)], change=change)


@pytest.mark.parametrize("H,G,dk,dv", [(16, 2, 128, 128), (10, 2, 80, 96), (16, 2, 64, 64), (12, 2, 33, 48), (11, 1, 128, 64), (20, 2, 192, 256), (9, 3, 64, 64)])
@pytest.mark.parametrize("page", [16, 64])
def test_tables_of_long_sequences(cuda_backend, H, G, dk, dv, page):
    """Page tables that could hold far more than they do: sizes go by them, answers by the rows."""
    entries = [(i % 3, n, 0) for i, n in enumerate(LENGTHS)]
    for window in (0, 40, 1 << 18):
        attend_case(cuda_backend, len(entries) + 1, H, G, dk, dv, page, 192 // page, entries, spare=(1 << 19) // page, window=window, pad=2)
    attend_case(cuda_backend, 40, H, G, dk, dv, page, 192 // page, [(i // 15, 180 - 40 + i, 0) for i in range(40)], spare=(1 << 19) // page)      # runs of one slot


def test_many_rows(cuda_backend):
    """More rows than a warp reads at once, most of them short, runs of one slot across its blocks of 32, rows that are idle among them."""
    r = np.random.default_rng(0)
    for H, G in ((4, 4), (4, 1)):
        for window in (0, 20):
            attend_case(cuda_backend, 700, H, G, 32, 32, 16, 12, [(int(r.integers(-1, 3)), int(r.integers(0, 60)), 0) for _ in range(690)], window=window, spare=3000)
        attend_case(cuda_backend, 400, H, G, 32, 32, 16, 12, [(i // 37 % 3, 1 + i % 192, 0) for i in range(400)], slots=3)
        attend_case(cuda_backend, 300, H, G, 32, 32, 16, 4, [(i, 1 + i % 64, 0) for i in range(300)], slots=300)
    for first in (0, 1, 33):                             # a chunk of one sequence's prompt, one launch and two
        for spare in (0, 3000):
            attend_case(cuda_backend, 140, 2, 1, 32, 32, 16, 13, [(1, 5, 0)] * first + [(0, 1 + i, 0) for i in range(139 - first)], slots=2, spare=spare)


@pytest.mark.parametrize("H,G,dk,dv", [(8, 2, 128, 128), (9, 3, 64, 64), (6, 1, 80, 48), (4, 1, 256, 192), (5, 5, 33, 17)])
def test_without_a_workspace(cuda_backend, monkeypatch, H, G, dk, dv):
    """No room for records: a CTA takes whole sequences, of thousands of tiles as well."""
    monkeypatch.setenv("ZG_CUDA_SCRATCH_MB", "0")
    entries = [(i % 3, n, 0) for i, n in enumerate(LENGTHS)] + [(-1, 1, 0), (0, 0, 0), (3, 1, 0), (0, 193, 0)]
    for window in (0, 50):
        attend_case(cuda_backend, len(entries) + 1, H, G, dk, dv, 16, 12, entries, window=window, sink=0.5, spare=4000)
    attend_case(cuda_backend, 30, H, G, dk, dv, 32, 8, [(0, 100 + i, 0) for i in range(15)] + [(1, 90 + i, 0) for i in range(15)], spare=4000)
    if dk != 256:
        attend_case(cuda_backend, 1, G, G, dk, dv, 64, 2400, [(0, 150011, 0)], slots=1, loud=0.1)


def test_outside_a_graph(cuda_backend):
    attend_case(cuda_backend, 5, 8, 2, 128, 128, 16, 40, [(i % 3, 640 - 100 * i, 0) for i in range(5)], graph=False)


# ── beyond 2^32 ──────────────────────────────────────────────────────────────────────────────────────────────────────
def test_pages_beyond_4_gb(cuda_backend):
    """Append, read, attend and copy where pages lie more than 4 GB into their pool."""
    from zgml_b200 import DeviceBuffer, DeviceOp, DeviceProgram, ExternBuffer, ProgramIO
    r = np.random.default_rng(4)
    G, H, dk, dv, page, most, B = 8, 16, 128, 128, 64, 2, 3
    words = page_words(G, dk, dv, page)
    count = (9 << 30) // (4 * words)
    memory = DeviceBuffer(cuda_backend, 4 * words * count, zero=False)
    used = [count - 1, count // 2 + 7, count - 5, 3, count - 2, count - 9]
    state = pool(r, 6, G, dk, dv, page)
    for i, p in enumerate(used):
        memory.upload(pack_pages(*(x[i:i + 1] for x in state)), 4 * words * p)
    near = np.array([[0, 1], [2, 3], [4, 5]], np.int32)
    far = np.array(used, np.int32)[near]
    entries = [(0, 100, 0), (1, 64, 0), (2, 3, 0)]
    src, q = r.standard_normal((B, G * (dk + dv))).astype(np.float32), r.standard_normal((B, H * dk)).astype(np.float32)
    sizes = [memory.elems, src.size, far.size, 8 + 4 * B, q.size, B * H * dv, B * G * (dk + dv), move_words(2)]
    ops = [DeviceOp.page_append(0, 1, 2, 3, 0, G * dk, B, G, dk, dv, G * (dk + dv), page, most), DeviceOp.paged_attention(5, 4, 0, 2, 3, B, H, G, dk, dv, H * dk, page, most, dk ** -0.5),
           DeviceOp.page_read(6, 0, 2, 3, B, G, dk, dv, page, most), DeviceOp.page_copy(0, 7, 2, words)]
    h = cuda_backend.compile_program(DeviceProgram(ops, sizes, externs=[ExternBuffer(0, memory)]))
    out, back = np.zeros((B, H, dv), np.float32), np.zeros((B, G * (dk + dv)), np.float32)
    moves = [(used[0], count - 20), (used[3], count - 21)]
    f = lambda a: np.ascontiguousarray(a).view(np.float32).ravel()
    cuda_backend.execute_program(h, [ProgramIO(1, f(src)), ProgramIO(2, f(far)), ProgramIO(3, f(table(entries, B))), ProgramIO(4, f(q)), ProgramIO(7, f(page_moves(moves, 2, count)))], [ProgramIO(5, out), ProgramIO(6, back)])
    k, v, s, _ = ref.append(*state, src, near, entries, B, 0, (0, G * dk, 0), B, G, dk, dv, page)
    want, tol = ref.attend(np.zeros((B, H, dv)), q.reshape(B, H, dk), k, v, s, near, entries, B, B, dk ** -0.5)
    close(out, want, tol)
    assert np.array_equal(back, ref.read(k, v, s, near, entries, B, B, np.zeros((B, G * (dk + dv)))).astype(np.float32))
    for source, to in moves:
        a, b = (memory.download(np.int32, 4 * words * p, words) for p in (source, to))
        assert np.array_equal(a, b)
    assert np.array_equal(memory.download(np.int32, 4 * words * used[0], words)[:4].view(np.float32)[:2], s[0, 0].astype(np.float32))
    cuda_backend.free_program(h)
    memory.free()


# ── two at once ──────────────────────────────────────────────────────────────────────────────────────────────────────
def test_two_programs_over_one_pool(cuda_backend):
    """Programs of their own workspaces over one pool, run by turns: what one leaves in its workspace is not the other's."""
    from zgml_b200 import DeviceBuffer, DeviceOp, DeviceProgram, ExternBuffer, ProgramIO
    r = np.random.default_rng(8)
    G, H, d, page, most = 2, 8, 64, 16, 200
    state = pool(r, 2 * most, G, d, d, page)
    words = np.ascontiguousarray(pack_pages(*state))
    memory = DeviceBuffer(cuda_backend, words.nbytes, zero=False)
    memory.upload(words, 0)
    page_table = r.permutation(2 * most).reshape(2, most).astype(np.int32)
    f = lambda x: np.ascontiguousarray(x).view(np.float32).ravel()
    programs = []
    for B in (1, 3, 40):
        entries = [(i % 2, 1 + (997 * (i + B)) % (most * page), 0) for i in range(B)]
        q = r.standard_normal((B, H, d)).astype(np.float32)
        h = cuda_backend.compile_program(DeviceProgram([DeviceOp.paged_attention(4, 1, 0, 2, 3, B, H, G, d, d, H * d, page, most, d ** -0.5)], [memory.elems, q.size, page_table.size, 8 + 4 * B, q.size], externs=[ExternBuffer(0, memory)]))
        programs.append((h, entries, q, *ref.attend(np.zeros((B, H, d)), q, *state, page_table, entries, B, B, d ** -0.5)))
    first = {}
    for turn in range(3):
        for i, (h, entries, q, want, tol) in enumerate(programs):
            out = np.zeros(q.shape, np.float32)
            cuda_backend.execute_program(h, [ProgramIO(1, f(q)), ProgramIO(2, f(page_table)), ProgramIO(3, f(table(entries, len(entries))))], [ProgramIO(4, out)])
            close(out, want, tol)
            assert np.array_equal(out, first.setdefault(i, out))
    for h, *_ in programs:
        cuda_backend.free_program(h)
    memory.free()


def test_on_another_stream():
    import torch
    from zgml_b200 import CudaBackend
    be = CudaBackend(0)
    stream = torch.cuda.Stream()
    be.set_stream(stream.cuda_stream)
    a = Append(be, 90, 2, 32, 16, 16, H=3, rot=32, slots=6, most=3, pages=20)
    a.check([(i % 6, 1 + i // 6 * 2 + i % 2, 0) for i in range(90)])
    a.close()
    for spare in (0, 4000):
        attend_case(be, 20, 8, 2, 64, 64, 16, 12, [(i % 3, LENGTHS[i % len(LENGTHS)], 0) for i in range(20)], spare=spare)
    be.close()


# ── together ─────────────────────────────────────────────────────────────────────────────────────────────────────────
def test_a_decode_loop(cuda_backend):
    """Requests come with prompts, decode, fork, drop drafts, end, and their pages are compacted: one program of copies, appends, attention and reads, replayed with other tables, over one pool that the
    programs share."""
    from zgml_b200 import DeviceOp
    r = np.random.default_rng(11)
    G, H, dk, dv, page, most, slots, pages, B = 2, 6, 40, 24, 16, 6, 5, 24, 24
    words, rs = page_words(G, dk, dv, page), H * dk + G * (dk + dv)
    make = lambda at: [DeviceOp.page_copy(at["pages"], at["moves"], 8, words),
                       DeviceOp.page_append(at["pages"], at["src"], at["page_table"], at["table"], H * dk, H * dk + G * dk, B, G, dk, dv, rs, page, most, rot=dk, rot_base=1e4, rot_layout="halves", q_heads=H, turned=at["turned"]),
                       DeviceOp.paged_attention(at["dst"], at["turned"], at["pages"], at["page_table"], at["table"], B, H, G, dk, dv, H * dk, page, most, dk ** -0.5),
                       DeviceOp.page_read(at["back"], at["pages"], at["page_table"], at["table"], B, G, dk, dv, page, most)]
    zeros = lambda *s: np.zeros(s, np.float32)
    p = Prog(cuda_backend, make, dict(pages=np.zeros((pages, words), np.int32), src=zeros(B, rs), page_table=np.zeros((slots, most), np.int32), table=np.zeros(8 + 4 * B, np.int32), moves=np.zeros(move_words(8), np.int32),
                                      turned=zeros(B, H * dk), dst=zeros(B, H * dv), back=zeros(B, G * (dk + dv))), extern=("pages",))
    state = tuple(np.zeros(s) for s in ((pages, G, page, dk), (pages, G, page, dv), (pages, G, 2)))
    host = PagePool(pages, page, slots, most)

    def step(new, moves=()):
        nonlocal state
        moves, entries = list(moves), []
        for slot, tokens in new:
            moves += host.extend(slot, tokens)
            entries += [(slot, host.lengths[slot] - tokens + 1 + i, 0) for i in range(tokens)]
        src = r.standard_normal((B, rs)).astype(np.float32)
        got, back = p.run(["dst", "back"], src=src, page_table=host.table, table=table(entries, B), moves=page_moves(moves, 8, pages))
        for x in state:
            x[[d for _, d in moves]] = x[[s for s, _ in moves]]
        k, v, s, turned = ref.append(*state, src, host.table, entries, len(entries), 0, (H * dk, H * dk + G * dk, 0), B, G, dk, dv, page, 0, dk, 1e4 ** (-2.0 * np.arange(dk // 2) / dk), "halves", H, np.zeros((B, H * dk)))
        state = (k, v, s)
        want, tol = ref.attend(zeros(B, H, dv), turned.astype(np.float32).reshape(B, H, dk), k, v, s, host.table, entries, len(entries), B, dk ** -0.5)
        n = len(entries)
        close(got.reshape(B, H, dv)[:n], want[:n], tol[:n])
        assert np.array_equal(back[:n], ref.read(k, v, s, host.table, entries, n, B, np.zeros((B, G * (dk + dv))))[:n].astype(np.float32))
    step([(0, 20)])
    step([(0, 1), (1, 23)])
    host.fork(0, 2)
    host.fork(0, 3, 17)
    step([(0, 1), (1, 1), (2, 1), (3, 1)])
    step([(0, 4), (2, 4), (3, 4)])
    host.shrink(2, host.lengths[2] - 3)
    host.shrink(3, 16)
    step([(2, 1), (3, 1), (1, 2)])
    host.release(0)
    step([(4, 3), (2, 1)], host.compact())
    for _ in range(4):
        step([(i, 1) for i in (1, 2, 3, 4)])
    p.close()
