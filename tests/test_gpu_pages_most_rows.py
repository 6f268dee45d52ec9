"""The ops over pages with as many rows as they take, against NumPy in 64 bits."""
import numpy as np
import pytest

from test_gpu_batchops import table
from test_gpu_pages import Append, attend_case
from zgml_b200 import DeviceOp
from zgml_b200.host.pages import page_moves

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("slots,spare", [(4000, 0), (4000, 3000), (70000, 0)])
def test_attention(cuda_backend, slots, spare):
    """65535 rows: runs of one slot, idle rows and rows that see nothing among them; with and without room for longer sequences."""
    r = np.random.default_rng(slots)
    entries = [(int(s), int(n), 0) for s, n in zip(np.repeat(r.integers(-1, slots, 32768), 2), r.integers(0, 33, 65535))][:65535]
    attend_case(cuda_backend, 65535, 1, 1, 8, 8, 16, 2, entries, slots=slots, pages=9000 if slots < 9000 else 2 * slots, spare=spare, seed=1)


def test_append(cuda_backend):
    """65536 rows, of which two at a time come to one page, those of a block of 64 side by side and those of others far apart."""
    a = Append(cuda_backend, 65536, 1, 8, 4, 16, H=1, rot=8, slots=32768, most=1, pages=32768, seed=9)
    slot = np.arange(65536) // 2
    slot[32768:] = np.r_[slot[32768:][0::2], slot[32768:][1::2]]
    count = np.zeros(32768, int)
    rows = []
    for s in slot:
        count[s] += 1
        rows.append((int(s), 3 + int(count[s]), 0))
    a.check(rows)
    a.close()


def test_read_and_copy(cuda_backend):
    """More rows and moves than a grid's second dimension takes."""
    from test_gpu_batchops import Prog
    from zgml_b200.host.pages import move_words, pack_pages
    import page_reference as ref
    r = np.random.default_rng(2)
    keys, values, scales = r.integers(-127, 128, (50, 1, 16, 4)).astype(np.int8), r.integers(-127, 128, (50, 1, 16, 3)).astype(np.int8), (2.0 ** r.integers(-9, -4, (50, 1, 2))).astype(np.float32)
    page_table, B = r.permutation(50)[:48].reshape(16, 3).astype(np.int32), 70001
    p = Prog(cuda_backend, lambda at: [DeviceOp.page_read(at["dst"], at["pages"], at["page_table"], at["table"], B, 1, 4, 3, 16, 3)],
             dict(dst=np.zeros((B, 7), np.float32), pages=pack_pages(keys, values, scales), page_table=page_table, table=np.zeros(8 + 4 * B, np.int32)))
    entries = [(int(a), int(b), 0) for a, b in zip(r.integers(-1, 17, B), r.integers(0, 50, B))]
    got = p.run(["dst"], table=table(entries, B))
    p.close()
    assert np.array_equal(got, ref.read(keys, values, scales, page_table, entries, B, B, np.zeros((B, 7))).astype(np.float32), equal_nan=True)
    pages = r.integers(-2 ** 31, 2 ** 31, (140000, 5)).astype(np.int32)
    order = r.permutation(140000)
    moves = list(zip(order[:70000].tolist(), order[70000:].tolist()))
    p = Prog(cuda_backend, lambda at: [DeviceOp.page_copy(at["pages"], at["moves"], 70000, 5)], dict(pages=pages, moves=np.zeros(move_words(70000), np.int32)))
    want = pages.copy()
    want[order[70000:]] = pages[order[:70000]]
    assert np.array_equal(np.ascontiguousarray(p.run(["pages"], moves=page_moves(moves, 70000, 140000))).view(np.int32), want)
    p.close()
