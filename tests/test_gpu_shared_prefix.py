"""SHARED_ATTENTION's prefix on the tensor cores, heads up to 128 (and one wider size beside them): what half-precision pairs cannot hold, and magnitudes near the
ends of f32, against NumPy in 64 bits."""
import numpy as np
import pytest

import batch_reference as ref
from test_gpu_batchops import NAN, Prog, table

pytestmark = pytest.mark.gpu
# 40 rows of 8 heads over a prefix that may hold 1300 rows: the tensor cores' side of the rule on rows x heads x keys (3 * 2^17)
B, H, G, R, P, RP, SCALE = 40, 8, 2, 4, 500, 1300, 0.05


def entries():
    return [(i, (5 + 7 * i) % (R + 1), 0) for i in range(B)]


def inputs(d, seed=5):
    r = np.random.default_rng(seed)
    q, own, pre = r.standard_normal((B, H, d)).astype(np.float32), r.standard_normal((B, R, 2, G, d)).astype(np.float32), r.standard_normal((1, RP, 2, G, d)).astype(np.float32)
    pre[:, P:] = NAN                                    # what no row sees may hold anything
    return q, own, pre


def exact(q, own, pre, cap=0.0, P=P, scale=SCALE, rows=None):
    """-> (want, how far a result may be off), [B, H, d] each"""
    with np.errstate(all="ignore"):
        return ref.attend(np.zeros((B, H, own.shape[4]), np.float32), q, own[:, :, 0], own[:, :, 1], pre[:, :, 0], pre[:, :, 1], rows or entries(), B, P, 0, scale, cap)


def attend(be, q, own, pre, cap=0.0, P=P, scale=SCALE, rows=None):
    from zgml_b200 import DeviceOp
    d = q.shape[2]
    w = G * d
    op = DeviceOp.shared_attention(0, 1, 2, 2, 3, 3, 4, 0, 0, w, 0, w, B, H, G, d, d, H * d, 2 * w, 2 * w, R, 2 * w, 2 * w, RP, scale, softcap=cap)
    p = Prog(be, lambda at: [op], dict(dst=np.zeros((B, H * d), np.float32), q=q, own=own, pre=pre, table=table(rows or entries(), B, P)))
    got = p.run(["dst"]).reshape(B, H, d)
    p.close()
    return got


@pytest.mark.parametrize("size", [1e35, 1e30, 1e-30, 1e-33])
@pytest.mark.parametrize("d", [64, 80, 128, 160])
def test_values_near_the_ends_of_f32(cuda_backend, d, size):
    """Finite results, whatever form takes the prefix: the sum of weights is below 500, so no sum of weights times values passes f32's range."""
    q, own, pre = inputs(d)
    own[:, :, 1] *= np.float32(size)
    pre[:, :, 1] *= np.float32(size)
    got = attend(cuda_backend, q, own, pre)
    want, tol = exact(q, own, pre)
    assert np.isfinite(got).all() and (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("size", [1e-9, 1e-5, 3e-5, 1e-4])
@pytest.mark.parametrize("d", [64, 80, 128, 160])
def test_a_small_column_of_values(cuda_backend, d, size):
    """A column that is small beside the others is as exact as if it were alone."""
    q, own, pre = inputs(d)
    for c in (own, pre):
        c[:, :, 1, :, 7] *= np.float32(size)
    got = attend(cuda_backend, q, own, pre)
    with np.errstate(all="ignore"):                     # (the column alone: its own magnitude is what the tolerance counts)
        want, tol = ref.attend(np.zeros((B, H, 1), np.float32), q, own[:, :, 0], own[:, :, 1, :, 7:8], pre[:, :, 0], pre[:, :, 1, :, 7:8], entries(), B, P, 0, SCALE)
    assert (np.abs(got[:, :, 7:8] - want) <= tol).all()
    want, tol = exact(q, own, pre)
    assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("size", [1e-8, 1e-6, 1e-5, 1e-4])
@pytest.mark.parametrize("d", [64, 80, 128, 160])
def test_keys_with_small_values(cuda_backend, d, size):
    """The keys that count have small values, others, whose scores lie 200 and more below theirs, large ones: nothing of these is left in f32 (e^-200) or in the tolerance."""
    q, own, pre = inputs(d)
    r = np.random.default_rng(9)
    u = np.sign(r.standard_normal(d)).astype(np.float32)
    q[:] = u + 0.1 * q
    pre[:, :, 0] = 0.3 * pre[:, :, 0]
    pre[:, 1:P:2, 0] -= np.float32(6000.0 / d) * u      # scores of 0.05 * 6000 * 0.9 less at least
    pre[:, 0:P:2, 1] *= np.float32(size)
    own[:, :, 1] *= np.float32(size)
    got = attend(cuda_backend, q, own, pre)
    want, _ = exact(q, own, pre)
    # the tolerance of the keys that count alone, their scores off by what the loudest key of all allows
    few = np.concatenate([pre[:, 0:P:2], np.full((1, RP - P // 2, 2, G, d), NAN)], 1).astype(np.float32)
    alone, tol = exact(q, own, few, P=P // 2)
    assert (np.abs(alone - want) <= 1e-12 * np.abs(alone).max()).all()
    top = np.abs(pre[:, :P, 0]).max()
    off = SCALE * (d * 2.0 ** -24 + 3 * 2.0 ** -22) * top * np.abs(q).sum(2, keepdims=True)
    mean = np.zeros_like(want)
    kv = [own[:, :, 0], np.abs(own[:, :, 1]), few[:, :, 0], np.abs(few[:, :, 1])]
    mean, _ = ref.attend(mean, q, *kv, entries(), B, P // 2, 0, SCALE)
    assert (np.abs(got - want) <= tol + 2 * off * mean).all()


@pytest.mark.parametrize("what", ["query nan", "query inf", "key nan", "key inf", "value inf", "value nan"])
@pytest.mark.parametrize("d", [64, 80, 128, 160])
def test_what_is_not_finite(cuda_backend, d, what):
    """It reaches the results that the definition gives it to, and no others."""
    q, own, pre = inputs(d)
    want, tol = exact(q, own, pre)
    x = np.float32("inf") if what.endswith("inf") else NAN
    if what.startswith("query"):
        q[17, 5, 3] = x
    else:
        pre[0, 333, 0 if what.startswith("key") else 1, 0, 11] = x
    dirty, _ = exact(q, own, pre)
    if what == "key inf":                               # where its score is -inf: as without this key
        less, off = exact(q, own, np.delete(pre, 333, 1), P=P - 1)
        want[:, :H // G], tol[:, :H // G] = less[:, :H // G], off[:, :H // G]
    got = attend(cuda_backend, q, own, pre)
    ok = np.isfinite(dirty)
    assert (np.abs(dirty[ok] - want[ok]) <= 1e-12).all() and 0 < (~ok).sum() < ok.size
    assert np.array_equal(np.isnan(got), np.isnan(dirty)) and np.array_equal(got[np.isinf(dirty)], dirty[np.isinf(dirty)])
    assert (np.abs(got[ok] - want[ok]) <= tol[ok]).all()


@pytest.mark.parametrize("bits,cap", [(20, 0.0), (20, 2.0 ** 22), (22, 0.0)])
@pytest.mark.parametrize("d", [64, 128, 160])
def test_loud_scores(cuda_backend, d, bits, cap):
    """Scores around 2^17 or 2^19 that f32 holds exactly and that differ by a few units, so that many keys share the weight: whole numbers in queries and keys, a scale of 2^-3, no
    keys of a row's own.  A cap far above them leaves a thousandth part less of a difference: the slope at 2^-5 is 1 - 2^-10."""
    q, own, pre = inputs(d)
    r = np.random.default_rng(2)
    u = np.sign(r.standard_normal(d)).astype(np.float32)
    q[:] = u
    pre[:, :, 0] = np.float32(2 ** bits // d) * u + r.integers(-10, 11, (1, RP, G, d))
    rows, scale = [(i, 0, 0) for i in range(B)], 0.125
    got = attend(cuda_backend, q, own, pre, cap, scale=scale, rows=rows)
    want, _ = exact(q, own, pre, cap, scale=scale, rows=rows)
    mean, _ = ref.attend(np.zeros_like(want), q, own[:, :, 0], own[:, :, 1], pre[:, :, 0], np.abs(pre[:, :, 1]), rows, B, P, 0, scale, cap)
    # Plain f32 (keys of 2^14 and more) works on the scores as they are.  Pairs hold these keys and scores exactly too, but a share of the prefix names its largest score in units of
    # ln 2 and is joined in units of one: one rounding, of 2^17 at most.  A cap: its tanh and the two roundings beside it, 2 + 2 units of 2^-24 of a score.
    plain = 2 ** bits // d >= 2 ** 14
    off = (4.0 * 1.01 if cap else 0.0 if plain else 1.0) * 2.0 ** (bits - 3 - 24)
    assert (np.abs(got - want) <= (2 * off + (64 + 32) * 2.0 ** -24 + 4 * 2.0 ** -22) * (mean + np.abs(pre[:, :P, 1]).max() * 2.0 ** -14)).all()


@pytest.mark.parametrize("H,dk,dv", [(16, 160, 160), (16, 160, 300), (16, 128, 128)])
def test_sums_over_many_tiles_do_not_drift(cuda_backend, H, dk, dv):
    """Sums on the tensor cores are cut at 24 bits, always towards zero.  Positive values over some twenty tiles a CTA: eight products of full size make a tile's sum, each cut by less
    than 2^-23 of it (the others' sums are 2^-11 as large, and come first); tiles, shares and the sum of weights are rounded, which has no direction.  So the mean error over all
    results is below 8 * 2^-23 of them, however many tiles there are, and 2^-23 for what roundings leave of a mean."""
    from zgml_b200 import DeviceOp
    r = np.random.default_rng(3)
    B, G, P = 128, 2, 20000
    q = r.standard_normal((B, H, dk)).astype(np.float32)
    k, v = r.standard_normal((P, G, dk)).astype(np.float32), r.uniform(1.0, 2.0, (P, G, dv)).astype(np.float32)
    pre = np.concatenate([k.reshape(P, -1), v.reshape(P, -1)], 1)
    w, scale = pre.shape[1], 0.3 * dk ** -0.5
    op = DeviceOp.shared_attention(0, 1, 2, 2, 3, 3, 4, 0, 0, G * dk, 0, G * dk, B, H, G, dk, dv, H * dk, w, w, 1, w, w, P, scale)
    p = Prog(cuda_backend, lambda at: [op], dict(dst=np.zeros((B, H * dv), np.float32), q=q, own=np.zeros((1, 1, w), np.float32), pre=pre, table=table([(0, 0, 0)] * B, B, P)))
    got = p.run(["dst"]).reshape(B, H, dv)
    p.close()
    for g in range(G):
        z = q[:, g * (H // G):(g + 1) * (H // G)].reshape(-1, dk).astype(np.float64)
        s = np.exp(scale * (z @ k[:, g].astype(np.float64).T))
        want = s @ v[:, g].astype(np.float64) / s.sum(1, keepdims=True)
        off = got[:, g * (H // G):(g + 1) * (H // G)].reshape(-1, dv) / want - 1.0
        assert abs(off.mean()) <= 9 * 2.0 ** -23 and np.abs(off).max() <= 2.0 ** -16, (off.mean(), np.abs(off).max())
