"""Host side of paged caches and of the choice of tokens, without a device: pools, tables, the bytes of a page, and what the ops' static checks refuse."""
import numpy as np
import pytest

from zgml_b200 import DeviceOp, abi
from zgml_b200.backend import seq_check
from zgml_b200.host.batch import TokenChoice, sample_table, sample_words, table_words
from zgml_b200.host.pages import PagePool, move_words, pack_pages, page_moves, page_words, unpack_pages


@pytest.mark.parametrize("G,dk,dv,page", [(1, 1, 1, 16), (2, 44, 7, 16), (3, 128, 128, 64), (1, 33, 256, 32)])
def test_page_bytes(G, dk, dv, page):
    r = np.random.default_rng(dk)
    k, v, s = r.integers(-127, 128, (3, G, page, dk)).astype(np.int8), r.integers(-127, 128, (3, G, page, dv)).astype(np.int8), r.random((3, G, 2)).astype(np.float32)
    w = pack_pages(k, v, s)
    assert w.shape == (3, page_words(G, dk, dv, page)) and w.dtype == np.int32
    for a, b in zip(unpack_pages(w, G, dk, dv, page), (k, v, s)):
        assert np.array_equal(a, b)
    # the places that the header names
    by, kp, vp = w.view(np.uint8).reshape(3, G, -1), -(-dk // 32) * 32, -(-dv // 16) * 16
    t = np.arange(page)[:, None]
    d = np.arange(dk)
    assert np.array_equal(by[:, :, 16 + ((t // 8) * (kp // 32) + d // 32) * 256 + t % 8 * 32 + d % 32].astype(int) - 128, k)
    d = np.arange(dv)
    at = 16 + page * kp + ((t // 16) * (vp // 16) + d // 16) * 256 + (4 * (d % 8) + t % 8 // 2) * 8 + 4 * (d // 8 % 2) + 2 * (t // 8 % 2) + t % 2
    assert np.array_equal(by[:, :, at].astype(int) - 128, v)


@pytest.mark.parametrize("G,dk,dv,page", [(0, 8, 8, 16), (1, 0, 8, 16), (1, 8, 0, 16), (1, 257, 8, 16), (1, 8, 257, 16), (1, 8, 8, 8), (1, 8, 8, 48), (1, 8, 8, 128)])
def test_pages_that_do_not_exist(G, dk, dv, page):
    with pytest.raises(ValueError):
        page_words(G, dk, dv, page)


def test_pool_extends_and_gives_back():
    p = PagePool(6, 16, 3, 4)
    assert p.extend(0, 16) == [] and p.extend(1, 1) == [] and p.extend(0, 1) == []
    assert p.page_ids(0) == [0, 2] and p.page_ids(1) == [1] and p.table.tolist() == [[0, 2, 0, 0], [1, 0, 0, 0], [0] * 4]
    assert p.extend(0, 15) == [] and p.lengths == [32, 1, 0] and p.free_pages == 3
    assert p.extend(0, 0) == []
    with pytest.raises(ValueError):
        p.extend(0, 33)                                  # beyond its page table
    with pytest.raises(ValueError):
        p.extend(0, -1)
    p.extend(2, 48)
    with pytest.raises(RuntimeError):
        p.extend(1, 16)
    assert p.lengths == [32, 1, 48] and p.free_pages == 0 and p.page_ids(1) == [1]
    p.extend(1, 15)                                      # room in the page that it has
    p.release(0)
    assert p.free_pages == 2 and p.page_ids(0) == [] and p.table[0].tolist() == [0] * 4
    p.shrink(2, 17)
    assert p.page_ids(2) == [3, 4] and p.free_pages == 3
    assert p.extend(2, 16) == [] and p.page_ids(2) == [3, 4, 0]
    with pytest.raises(ValueError):
        p.shrink(2, 34)


def test_pool_forks_by_copying_what_is_written():
    p = PagePool(8, 16, 4, 4)
    p.extend(0, 40)
    p.fork(0, 1)
    p.fork(0, 2, 32)
    assert p.page_ids(1) == [0, 1, 2] and p.page_ids(2) == [0, 1] and p.free_pages == 5
    assert p.extend(1, 1) == [(2, 3)] and p.page_ids(1) == [0, 1, 3]      # the page with positions 32 to 39
    assert p.extend(0, 1) == []                          # now it has that page alone
    assert p.extend(2, 1) == [] and p.page_ids(2) == [0, 1, 4]      # a page of its own, nothing to copy
    p.shrink(2, 20)                                      # back into a page that all share
    assert p.extend(2, 1) == [(1, 4)] and p.page_ids(2) == [0, 4]
    p.shrink(1, 16)
    assert p.extend(1, 20) == []                         # whole pages of its own
    p.fork(1, 3, 0)
    assert p.page_ids(3) == []
    for args in ((1, 1), (0, 2), (1, 3, 50), (1, 3, -1)):
        with pytest.raises(ValueError):
            p.fork(*args)
    for s in range(4):
        p.release(s)
    assert p.free_pages == 8


def test_pool_that_cannot_copy_changes_nothing():
    p = PagePool(2, 16, 2, 4)
    p.extend(0, 20)
    p.fork(0, 1)
    with pytest.raises(RuntimeError):
        p.extend(1, 1)
    assert p.lengths == [20, 20] and p.page_ids(1) == [0, 1] and p.free_pages == 0
    p.release(0)
    assert p.extend(1, 1) == []


def test_pool_compacts():
    p = PagePool(10, 16, 3, 5)
    for s in (0, 1, 2):
        p.extend(s, 48)
    p.release(1)
    p.extend(0, 17)
    before = [p.page_ids(s) for s in range(3)]
    holds = {page: page for page in range(10)}
    moves = p.compact()
    page_moves(moves, 10, 10)
    for source, to in moves:
        holds[to] = source
    assert sorted(p.page_ids(0) + p.page_ids(2)) == list(range(8)) and p.free_pages == 2
    assert [[holds[x] for x in p.page_ids(s)] for s in range(3)] == before
    assert [p.table[s, :len(p.page_ids(s))].tolist() for s in range(3)] == [p.page_ids(s) for s in range(3)]
    assert p.compact() == []


def test_pool_at_random():
    """Every position's page holds what was written for it, whatever was forked, cut off, copied and compacted."""
    r = np.random.default_rng(5)
    p, page, slots = PagePool(40, 16, 6, 8), 16, 6
    memory, want = np.full((40, page), -1), [[] for _ in range(slots)]
    stamp = 0
    for _ in range(3000):
        s, act = r.integers(slots), r.integers(6)
        moves = []
        if act <= 2:
            n = int(r.integers(0, 20))
            try:
                moves = p.extend(s, n)
            except (RuntimeError, ValueError):
                n = 0
            page_moves(moves, 40, 40)
            memory[[d for _, d in moves]] = memory[[a for a, _ in moves]]
            for _ in range(n):
                at = len(want[s])
                memory[p.table[s, at // page], at % page] = stamp
                want[s].append(stamp)
                stamp += 1
        elif act == 3 and want[s]:
            n = int(r.integers(0, len(want[s]) + 1))
            p.shrink(s, n)
            del want[s][n:]
        elif act == 4:
            to = int(r.integers(slots))
            if to != s and not p.page_ids(to):
                n = int(r.integers(0, len(want[s]) + 1))
                p.fork(s, to, n)
                want[to] = want[s][:n]
        elif act == 5:
            moves = p.compact()
            page_moves(moves, 40, 40)
            memory[[d for _, d in moves]] = memory[[a for a, _ in moves]]
        for i in range(slots):
            assert [memory[p.table[i, j // page], j % page] for j in range(len(want[i]))] == want[i]
        assert p.free_pages == 40 - len({x for i in range(slots) for x in p.page_ids(i)})


@pytest.mark.parametrize("args", [(0, 16, 1, 1), (4, 15, 1, 1), (4, 16, 0, 1), (4, 16, 1, 0)])
def test_pools_refuse(args):
    with pytest.raises(ValueError):
        PagePool(*args)


def test_page_moves():
    t = page_moves([(3, 0), (4, 1)], 3, 5)
    assert t.size == move_words(3) and t[0] == 2 and t[8:].reshape(3, 4).tolist() == [[3, 0, 0, 0], [4, 1, 0, 0], [0] * 4]
    assert page_moves([], 1, 5)[0] == 0
    page_moves([(3, 0), (3, 1)], 3, 5)                   # one page to two places
    for moves in ([(3, 0), (4, 0)], [(3, 4), (4, 1)], [(3, 3)], [(5, 0)], [(0, 5)], [(-1, 0)], [(0, 1)] * 4):
        with pytest.raises(ValueError):
            page_moves(moves, 3, 5)


def test_sample_table():
    t = sample_table([TokenChoice(0.5, 7, 0.25, 0.125), None, TokenChoice()], [0.75, 0.0, 1 - 1e-12], 4)
    assert t.size == sample_words(4) and t[0] == 3
    body = t[8:].reshape(4, 8)
    assert body[:, 1].tolist() == [7, -1, 0, 0]
    f = body.copy().view(np.float32)
    assert f[0, [0, 2, 3, 4]].tolist() == [0.5, 0.25, 0.125, 0.75] and f[2, [0, 2, 3]].tolist() == [1.0, 1.0, 0.0] and 0.99 < f[2, 4] < 1.0


@pytest.mark.parametrize("kw", [dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=float("inf")), dict(temperature=1e60), dict(top_k=-1), dict(top_k=1.5), dict(top_k=1 << 31), dict(top_p=1.5), dict(top_p=-0.1),
                                dict(top_p=float("nan")), dict(min_p=2.0), dict(min_p=float("nan"))])
def test_choices_refuse(kw):
    with pytest.raises(ValueError):
        TokenChoice(**kw)


@pytest.mark.parametrize("choices,draws", [([TokenChoice()] * 3, [0.0] * 3), ([TokenChoice()], []), ([TokenChoice()], [1.0]), ([TokenChoice()], [-0.1]), ([TokenChoice()], [float("nan")])])
def test_sample_tables_refuse(choices, draws):
    with pytest.raises(ValueError):
        sample_table(choices, draws, 2)


WORDS = page_words(2, 24, 20, 16)
APPEND = dict(pages=0, src=1, page_table=2, table=3, k_col=96, v_col=144, B=3, G=2, dk=24, dv=20, src_rs=190, page_tokens=16, most=5, turn_at=4, rot=16, rot_base=1e4, q_heads=4, q_col=0, turned=4, turned_rs=100)
APPEND_SIZES = [WORDS, 2 * 190 + 184, 5, table_words(3), 2 * 100 + 96]
ATTEND = dict(dst=0, q=1, pages=2, page_table=3, table=4, B=3, H=4, G=2, dk=24, dv=20, q_rs=99, page_tokens=16, most=5, scale=0.5, q_col=2, sink=5, dst_rs=90, dst_col=3)
ATTEND_SIZES = [2 * 90 + 83, 2 * 99 + 98, WORDS, 5, table_words(3), 4]
READ = dict(dst=0, pages=1, page_table=2, table=3, B=3, G=2, dk=24, dv=20, page_tokens=16, most=5, k_col=1, v_col=50, dst_rs=91)
READ_SIZES = [2 * 91 + 90, WORDS, 5, table_words(3)]
COPY = dict(pages=0, moves=1, B=3, page_words=WORDS)
COPY_SIZES = [WORDS, move_words(3)]
SAMPLE = dict(dst=0, logits=1, table=2, B=3, V=50, probability=3, dst_off=1, logits_off=2, logits_rs=60, probability_off=3)
SAMPLE_SIZES = [4, 2 + 2 * 60 + 50, sample_words(3), 6]


@pytest.mark.parametrize("make,kw,sizes", [(DeviceOp.page_append, APPEND, APPEND_SIZES), (DeviceOp.paged_attention, ATTEND, ATTEND_SIZES), (DeviceOp.page_read, READ, READ_SIZES), (DeviceOp.page_copy, COPY, COPY_SIZES),
                                           (DeviceOp.sample, SAMPLE, SAMPLE_SIZES)])
def test_what_the_checks_take(make, kw, sizes):
    assert seq_check(make(**kw), sizes) is None
    for i in range(len(sizes)):                          # every operand is as small as it may be
        short = list(sizes)
        short[i] -= 1
        assert seq_check(make(**kw), short), i


def refused(make, standard, sizes, **kw):
    return seq_check(make(**dict(standard, **kw)), sizes + [1 << 20])


@pytest.mark.parametrize("kw", [dict(B=0), dict(B=65537), dict(G=0), dict(dk=0), dict(dk=257), dict(dv=257), dict(page_tokens=8), dict(page_tokens=24), dict(most=0), dict(rot=15), dict(rot=22), dict(turn_at=9), dict(rot_base=0.0),
                                dict(rot_base=float("inf")), dict(src_rs=183), dict(turned_rs=95), dict(q_heads=5), dict(turned=0), dict(turned=1), dict(turned=2), dict(turned=3), dict(src=0), dict(table=0), dict(page_table=0),
                                dict(freqs=2, freqs_off=2), dict(freqs=4), dict(turned_col=5)])
def test_page_append_refuses(kw):
    assert refused(DeviceOp.page_append, APPEND, APPEND_SIZES, **kw)


@pytest.mark.parametrize("kw", [dict(B=0), dict(H=0), dict(H=5), dict(G=0), dict(dk=257), dict(dv=0), dict(page_tokens=128), dict(most=0), dict(q_rs=97), dict(dst_rs=82), dict(dst=1), dict(dst=2), dict(dst=3), dict(dst=4), dict(dst=5),
                                dict(scale=float("nan")), dict(scale=float("inf")), dict(softcap=-1.0), dict(softcap=float("nan")), dict(sink_wdt=2), dict(sink_off=1), dict(B=65536)])
def test_paged_attention_refuses(kw):
    assert refused(DeviceOp.paged_attention, ATTEND, ATTEND_SIZES, **kw)


@pytest.mark.parametrize("kw", [dict(B=0), dict(dk=0), dict(page_tokens=17), dict(most=0), dict(dst_rs=89), dict(v_col=48), dict(k_col=49), dict(dst=1), dict(dst=2), dict(dst=3)])
def test_page_read_refuses(kw):
    assert refused(DeviceOp.page_read, READ, READ_SIZES, **kw)


@pytest.mark.parametrize("kw", [dict(B=0), dict(page_words=0), dict(page_words=(1 << 24) + 1), dict(moves=0)])
def test_page_copy_refuses(kw):
    assert refused(DeviceOp.page_copy, COPY, COPY_SIZES, **kw)


@pytest.mark.parametrize("kw", [dict(B=0), dict(V=0), dict(logits_rs=49), dict(dst=1), dict(dst=2), dict(dst=3), dict(probability=0), dict(probability=1), dict(probability=2), dict(V=(1 << 18) + (1 << 17))])
def test_sample_refuses(kw):
    big = [1 << 20 if i == 1 and kw.get("V", 0) > 60 else n for i, n in enumerate(SAMPLE_SIZES)]
    assert refused(DeviceOp.sample, SAMPLE, big, **kw)


def test_sizes_that_do_not_fit_the_words_of_an_op():
    with pytest.raises(ValueError):
        DeviceOp.page_read(**dict(READ, dst_rs=1 << 32))


def test_tags():
    assert abi.OP_END == abi.OP_SAMPLE + 1 == 47
