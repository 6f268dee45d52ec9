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


def attend(be, q, own, pre, cap=0.0, P=P):
    """-> (got, want, how far a result may be off), [B, H, d] each"""
    from zgml_b200 import DeviceOp
    d = q.shape[2]
    w = G * d
    op = DeviceOp.shared_attention(0, 1, 2, 2, 3, 3, 4, 0, 0, w, 0, w, B, H, G, d, d, H * d, 2 * w, 2 * w, R, 2 * w, 2 * w, RP, SCALE, softcap=cap)
    p = Prog(be, lambda at: [op], dict(dst=np.zeros((B, H * d), np.float32), q=q, own=own, pre=pre, table=table(entries(), B, P)))
    got = p.run(["dst"]).reshape(B, H, d)
    p.close()
    with np.errstate(all="ignore"):
        want, tol = ref.attend(np.zeros((B, H, d), np.float32), q, own[:, :, 0], own[:, :, 1], pre[:, :, 0], pre[:, :, 1], entries(), B, P, 0, SCALE, cap)
    return got, want, tol


@pytest.mark.parametrize("size", [1e35, 1e30, 1e-30, 1e-33])
@pytest.mark.parametrize("d", [64, 80, 128, 160])
def test_values_near_the_ends_of_f32(cuda_backend, d, size):
    """Finite results, whatever form takes the prefix: the sum of weights is below 500, so no sum of weights times values passes f32's range."""
    q, own, pre = inputs(d)
    own[:, :, 1] *= np.float32(size)
    pre[:, :, 1] *= np.float32(size)
    got, want, tol = attend(cuda_backend, q, own, pre)
    assert np.isfinite(got).all() and (np.abs(got - want) <= tol).all()
