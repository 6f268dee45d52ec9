"""Copies of pages that several calls of a step ask for, made by one PAGE_COPY, whose moves all run at once."""
import numpy as np
import pytest

from zgml_b200.host.pages import PagePool, page_moves


def at_once(moves, memory):
    page_moves(moves, len(moves), len(memory))           # (refuses pages that one move writes and another touches)
    memory[[d for _, d in moves]] = memory[[s for s, _ in moves]]


def test_a_copy_of_a_page_that_is_about_to_move():
    p = PagePool(8, 16, 3, 4)
    p.extend(0, 40)
    p.extend(1, 20)
    p.fork(1, 2)
    p.release(0)
    moves = p.compact()
    assert moves == [(3, 0), (4, 1)]
    moves += p.extend(2, 1, moves)                       # its last page is 4, soon 1
    assert moves[2][0] == 4
    memory = np.arange(8)
    at_once(moves, memory)
    assert [memory[x] for x in p.page_ids(1)] == [3, 4] and [memory[x] for x in p.page_ids(2)] == [3, 4]
    assert len(set(p.page_ids(1) + p.page_ids(2))) == 3


def test_a_page_that_is_about_to_be_copied_is_not_written():
    p = PagePool(6, 16, 4, 2)
    p.extend(0, 10)
    p.extend(1, 10)
    p.fork(0, 2)
    p.fork(1, 3)
    moves = p.extend(2, 1)
    p.release(0)
    assert moves == [(0, 2)] and p.free_pages == 4       # page 0 is free, and read by the copy that has not run
    moves += p.extend(3, 1, moves)
    memory = np.arange(6)
    at_once(moves, memory)
    assert [memory[p.page_ids(s)[0]] for s in (1, 2, 3)] == [1, 0, 1]


def test_without_a_page_for_the_copy_nothing_changes():
    p = PagePool(3, 16, 4, 2)
    p.extend(0, 10)
    p.extend(1, 10)
    p.fork(0, 2)
    p.fork(1, 3)
    moves = p.extend(2, 1)
    p.release(0)
    with pytest.raises(RuntimeError):
        p.extend(3, 1, moves)                            # page 0 is free, but the copy that has not run reads it
    assert p.lengths == [0, 10, 11, 10] and p.page_ids(3) == [1] and p.free_pages == 1
    assert p.extend(3, 1) == [(1, 0)]                    # once it has run


def test_compacting_leaves_pages_that_copies_touch():
    p = PagePool(6, 16, 3, 3)
    p.extend(0, 10)
    p.extend(1, 30)
    p.fork(0, 2)
    moves = p.extend(2, 1)
    p.release(0)
    assert moves == [(0, 3)]
    moves += p.compact(moves)                            # page 0 has to stay until it is read
    assert p.page_ids(1) == [1, 2] and p.page_ids(2) == [3]
    memory = np.arange(6)
    at_once(moves, memory)
    assert memory[p.page_ids(2)[0]] == 0
    assert p.compact() == [(3, 0)] and p.free_pages == 3


@pytest.mark.parametrize("seed", range(4))
def test_steps_at_random(seed):
    """Sequences are cut off, forked, ended, extended and compacted in any order, all copies of a step run at once, then the step writes."""
    r = np.random.default_rng(seed)
    pages, page, slots = 30, 16, 6
    p = PagePool(pages, page, slots, 8)
    memory, want = np.full((pages, page), -1), [[] for _ in range(slots)]
    stamp, joined, early = 0, 0, 0
    for _ in range(800):
        moves, fresh = [], {}                            # positions that the step will write
        for _ in range(r.integers(1, 9)):
            s, act = int(r.integers(slots)), int(r.integers(8))
            if act <= 3 and s not in fresh:
                n = int(r.integers(0, 20))
                try:
                    moves += p.extend(s, n, moves)
                except ValueError:
                    continue
                except RuntimeError:
                    before = (list(p.lengths), p.table.copy(), p.free_pages)
                    at_once(moves, memory)               # the copies so far first
                    moves, early = [], early + 1
                    try:
                        moves += p.extend(s, n, moves)
                    except RuntimeError:
                        assert before[0] == p.lengths and np.array_equal(before[1], p.table) and before[2] == p.free_pages
                        continue
                fresh[s] = n
            elif act == 4 and s not in fresh:
                n = int(r.integers(0, len(want[s]) + 1))
                p.shrink(s, n)
                del want[s][n:]
            elif act == 5 and s not in fresh:
                to = int(r.integers(slots))
                if to != s and not p.page_ids(to) and to not in fresh:
                    n = int(r.integers(0, len(want[s]) + 1))
                    p.fork(s, to, n)
                    want[to] = want[s][:n]
            elif act == 6:
                moves += p.compact(moves)
            elif act == 7 and s not in fresh:
                p.release(s)
                want[s] = []
        joined += len(moves) > 1
        at_once(moves, memory)
        for s, n in fresh.items():
            for _ in range(n):
                memory[p.table[s, len(want[s]) // page], len(want[s]) % page] = stamp
                want[s].append(stamp)
                stamp += 1
        for i in range(slots):
            assert [memory[p.table[i, j // page], j % page] for j in range(len(want[i]))] == want[i]
        assert p.free_pages == pages - len({x for i in range(slots) for x in p.page_ids(i)})
    assert joined > 50
    p.compact()
    assert sorted({x for i in range(slots) for x in p.page_ids(i)}) == list(range(pages - p.free_pages))
