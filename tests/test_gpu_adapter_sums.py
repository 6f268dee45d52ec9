"""ADAPTER_LINEAR of many rows over long inputs: sums on the tensor cores are cut at 24 bits, always towards zero, and may not grow with the inputs."""
import numpy as np
import pytest

from test_gpu_batchops import Prog, bf16_bits, table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("runs", [1, 5])
@pytest.mark.parametrize("fmt", ["bf16", "f32"])
def test_sums_over_long_inputs_do_not_drift(cuda_backend, fmt, runs):
    """Positive inputs and weights.  256 inputs make a sum of 48 products (f32 weights: 96), each cut by less than 2^-23 of what the sum is by then, half of it on average; further sums
    are rounded, which has no direction.  The second product adds at most 12 (24) cuts.  So the mean error is below 24.5 + 12 (48.5 + 24) of 2^-23, and 2^-23 for
    what roundings leave of a mean, however long the inputs are."""
    from zgml_b200 import DeviceOp, abi
    r = np.random.default_rng(1)
    B, N, K, rank, A = 256, 64, 32768, 8, 5
    exact = lambda *s: (r.uniform(0.5, 1.0, s).astype(np.float32).view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)      # bfloat16-exact
    a, b = (exact(A, rank, K), exact(A, N, rank)) if fmt == "bf16" else (r.uniform(0.5, 1.0, s).astype(np.float32) for s in ((A, rank, K), (A, N, rank)))
    x = r.uniform(1.0, 2.0, (B, K)).astype(np.float32)
    which = [i * runs // B for i in range(B)]
    flat = np.concatenate([a.ravel(), b.ravel()])
    op = DeviceOp.adapter_linear(0, 1, 2, 0, A * rank * K, 3, B, N, K, rank, A, abi.W_BF16 if fmt == "bf16" else abi.W_F32, base=4, form="blocks")
    p = Prog(cuda_backend, lambda at: [op], dict(dst=np.zeros((B, N), np.float32), x=x, w=bf16_bits(flat) if fmt == "bf16" else flat, table=table([(0, 0, w) for w in which], B), base=np.zeros((B, N), np.float32)))
    got = p.run(["dst"])
    p.close()
    want = np.stack([b[w].astype(np.float64) @ (a[w].astype(np.float64) @ x[i].astype(np.float64)) for i, w in enumerate(which)])
    off = got / want - 1.0
    assert abs(off.mean()) <= (37.5 if fmt == "bf16" else 73.5) * 2.0 ** -23 and np.abs(off).max() <= 2.0 ** -15, (off.mean(), np.abs(off).max())
