"""PAGED_ATTENTION over sequences in which few keys outweigh very many others: what small weights add up to, in the outputs and in the softmax's sum, against NumPy in 64 bits within a bound that does not grow with the
number of keys.

The bound, in units of 2^-23 of the sum of weight * 127 * scale of the values over the sum of weights (the largest that a page of such scales can give): 8 for weights rounded to whole numbers (less than 2^-20 of what all
weigh is lost), and roundings of half a unit each: of the outputs 4 where digits are joined, 3 where products are put away, 7 where warps' records are joined (by eights, these one after the other, four warps) and 1 of
the quotient; of the softmax's sum 2 of a tile's four, 2 of all tiles, 3 of a warp's lanes, 7 of records: 22.5, taken as 24.  Beside it the exponentials (2^-22 and the rounding of their argument: 0.7 * 2^-20 up to 32, where the
largest weights are whole numbers, and more below them) and the scores' own roundings, weight by weight."""
import numpy as np
import pytest

from test_gpu_batchops import Prog, close, table
from zgml_b200.host.pages import pack_pages

pytestmark = pytest.mark.gpu
FORMS = {"a warp takes whole sequences": (256, 16, 16, 32, 16, 65536, 64), "one sequence for all warps": (1, 8, 8, 32, 16, 65536, 64), "one launch": (2, 16, 16, 32, 16, 1024, 16),
         "eight queries": (300, 32, 4, 64, 32, 40000, 32), "128 dims": (500, 4, 4, 128, 128, 20000, 32), "256 dims": (600, 2, 2, 256, 256, 20000, 64)}


def weigh(be, B, H, G, dk, dv, N, page, far, large, cap=0.0, grown=0):
    """One sequence that all rows read: key head g has the keys at `large` and all others `far[g]` quarter powers of two below them.  Values: the large keys' are 0, 1 and random by turns of three dims, the others' 1,
    1 and random.  grown: powers of two by which the scales of the large keys' pages are larger."""
    from zgml_b200 import DeviceOp
    r = np.random.default_rng(G + N)
    count = -(-N // page)
    keys = np.zeros((count, G, page, dk), np.int8)
    values = r.integers(-127, 128, (count, G, page, dv)).astype(np.int8)
    values[..., 0::3], values[..., 1::3] = 64, 64
    scales = np.full((count, G, 2), 0.25, np.float32)
    scales[..., 1] = 2.0 ** -6
    keys[..., 0] = (124 - np.asarray(far))[None, :, None]
    at = np.asarray(large)
    scales[at // page, :, 1] *= 2.0 ** grown
    keys[at // page, :, at % page, 0] = 124
    values[at // page, :, at % page, 0::3] = 0
    q = np.zeros((B, H * dk), np.float32)
    q[:, 0::dk] = 1.0
    scale = float(np.float32(np.log(2.0)))
    page_table = np.tile(r.permutation(count).astype(np.int32), (B, 1))
    inverse = np.argsort(page_table[0])
    make = lambda at: [DeviceOp.paged_attention(at["dst"], at["q"], at["pages"], at["page_table"], at["table"], B, H, G, dk, dv, H * dk, page, count, scale, softcap=cap)]
    p = Prog(be, make, dict(dst=np.zeros((B, H * dv), np.float32), q=q, pages=pack_pages(keys[inverse], values[inverse], scales[inverse]), page_table=page_table, table=np.zeros(8 + 4 * B, np.int32)))
    got = p.run(["dst"], table=table([(i, N, 0) for i in range(B)], B)).reshape(B, G, H // G, dv)
    p.close()
    want, tol = np.zeros((G, dv)), np.zeros((G, dv))
    for g in range(G):
        s = keys[:, g, :, 0].reshape(-1)[:N] * 0.25 * scale
        e = np.repeat(scales[:, g, 1].astype(np.float64), page)[:N]
        v = values[:, g].reshape(-1, dv)[:N] * e[:, None]
        off = 2.0 ** -21 * np.abs(s)                     # score and its product with log2 e, in 32 bits
        if cap:
            s = cap * np.tanh(s / cap)
            off += 2.0 ** -20 * np.abs(s)                # (the cap's own)
        w = np.exp(s - s.max())
        error = off + 2.0 ** -20 + 2.0 ** -23 * (s.max() - s)
        want[g] = w @ v / w.sum()
        tol[g] = (w * (error + w @ error / w.sum())) @ np.abs(v) / w.sum() + 24 * 2.0 ** -23 * 127.0 * (w @ e) / w.sum()
    return got, *(np.broadcast_to(x[None, :, None], got.shape) for x in (want, tol))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("where", ["first", "middle", "last", "often"])
def test_many_small_weights(cuda_backend, form, where):
    B, H, G, dk, dv, N, page = FORMS[form]
    large = {"first": [0], "middle": [N // 2 + 3], "last": [N - 1], "often": list(range(5, N, 3001))}[where]
    for base in (100, 115):                              # 25 bits below, and 28.75
        got, want, tol = weigh(cuda_backend, B, H, G, dk, dv, N, page, [base + 1 + 13 * g // G for g in range(G)], large)
        close(got, want, tol)


@pytest.mark.parametrize("far", [[4], [40], [100], [113], [118], [119], [120], [124], [140], [200]])
def test_without_a_workspace(cuda_backend, monkeypatch, far):
    """A warp takes an eighth of a sequence, however long."""
    monkeypatch.setenv("ZG_CUDA_SCRATCH_MB", "0")
    for large in ([0], [131071, 200000]):
        close(*weigh(cuda_backend, 1, 2, 1, 32, 16, 262144, 64, far, large))


@pytest.mark.parametrize("grown", [1, 5, 12])
def test_pages_of_larger_values(cuda_backend, grown):
    """The pages of the large keys have larger scales too, which the frame of the weights follows."""
    close(*weigh(cuda_backend, 256, 16, 16, 32, 16, 30000, 32, [60 + 4 * g for g in range(16)], [0, 20000], grown=grown))


def test_capped(cuda_backend):
    close(*weigh(cuda_backend, 256, 16, 16, 32, 16, 30000, 32, [100 + g for g in range(16)], [7, 20000], cap=40.0))


@pytest.mark.parametrize("N", [4096, 65536, 262144])
def test_equal_weights(cuda_backend, monkeypatch, N):
    """All keys alike, with values that do not cancel: sums of very many equal parts, by warps that share a sequence and by those that have it to themselves."""
    close(*weigh(cuda_backend, 1, 4, 2, 32, 16, N, 64, [0, 50], [N - 1]))
    monkeypatch.setenv("ZG_CUDA_SCRATCH_MB", "0")
    close(*weigh(cuda_backend, 1, 4, 2, 32, 16, N, 64, [1, 50], [N - 1]))
