"""SAMPLE against NumPy in 64 bits: vocabularies that end inside vectors and slices, equal logits, rows without tokens, every kind of choice at its ends, and rules and choices in one program."""
import numpy as np
import pytest

import page_reference as ref
from test_gpu_batchops import Prog
from zgml_b200.host.batch import LogitRules, TokenChoice, rule_table, sample_table, sample_words

pytestmark = pytest.mark.gpu
# a probability is rounded once, behind a quotient in 64 bits whose denominator is off by half of 2^-43 a token at most
SHARE = 2.0 ** -24 + 2.0 ** 19 * 2.0 ** -44


def program(be, B, V, *, pad=0, off=0, probability=True):
    from zgml_b200 import DeviceOp
    make = lambda at: [DeviceOp.sample(at["dst"], at["logits"], at["table"], B, V, probability=at["p"] if probability else None, dst_off=off, logits_off=off, logits_rs=V + pad, probability_off=off)]
    return Prog(be, make, dict(dst=np.full(B + off, 77, np.int32), logits=np.zeros(off + B * (V + pad), np.float32), table=np.zeros(sample_words(B), np.int32), p=np.full(B + off, 5.0, np.float32)))


def check(p, logits, choices, draws, *, pad=0, off=0, probability=True, words=None):
    B, V = logits.shape
    held = np.full((B, V + pad), np.inf, np.float32)
    held[:, :V] = logits
    t = sample_table([TokenChoice(*c) for c in choices], draws, B) if words is None else words
    got, share = p.run(["dst", "p"], logits=np.concatenate([np.full(off, np.nan, np.float32), held.ravel()]), table=t)
    got = got.view(np.int32)
    assert (got[:off] == 77).all() and (share[:off] == 5.0).all()
    for i in range(len(choices)):
        token, prob = ref.sample(logits[i], choices[i], min(np.float32(draws[i]), np.nextafter(np.float32(1), np.float32(0))))
        assert got[off + i] == token, (i, choices[i], draws[i], got[off + i], token)
        if not probability:
            assert share[off + i] == 5.0
        else:
            assert np.isnan(share[off + i]) == np.isnan(prob) and (np.isnan(prob) or abs(share[off + i] - prob) <= SHARE * prob), (share[off + i], prob)
    return got[off:], share[off:]


CHOICES = [(1.0, 0, 1.0, 0.0), (0.7, 5, 1.0, 0.0), (1.3, 0, 0.9, 0.0), (1.0, 40, 0.8, 0.0), (0.0, 3, 0.5, 0.5), (0.9, 0, 1.0, 0.1), (0.8, 300, 0.95, 0.02), (2.0, 1, 0.9, 0.0), (1.0, 10 ** 6, 0.5, 0.0), (0.25, 700, 0.999, 0.0),
           (5.0, 0, 0.99, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.0), (1e-3, 50, 0.9, 0.0), (1e4, 0, 0.9, 0.0), (1e-38, 0, 0.9, 0.0)]


@pytest.mark.parametrize("V,pad,off", [(1, 0, 0), (2, 3, 1), (31, 0, 0), (33, 1, 3), (512, 0, 4), (1000, 0, 0), (1024, 4, 0), (1025, 0, 1), (4099, 2, 0), (32000, 0, 0), (49152, 0, 4), (128256, 0, 0), (327680, 0, 0)])
def test_choices(cuda_backend, V, pad, off):
    r = np.random.default_rng(V)
    B = len(CHOICES)
    p = program(cuda_backend, B, V, pad=pad, off=off)
    for spread in (3.0, 1.0):
        check(p, (spread * r.standard_normal((B, V))).astype(np.float32), CHOICES, r.random(B), pad=pad, off=off)
    check(p, r.standard_normal((B, V)).astype(np.float32), CHOICES, np.zeros(B), pad=pad, off=off)
    check(p, r.standard_normal((B, V)).astype(np.float32), CHOICES, np.full(B, 1 - 1e-9), pad=pad, off=off)
    p.close()


@pytest.mark.parametrize("V", [40, 3000, 50000])
def test_equal_logits(cuda_backend, V):
    """Lower tokens first: all equal, few different values, and a largest value that many share; zeros of both signs are one value."""
    r = np.random.default_rng(V)
    B = len(CHOICES)
    p = program(cuda_backend, B, V)
    check(p, np.full((B, V), -1.5, np.float32), CHOICES, r.random(B))
    check(p, r.integers(-2, 3, (B, V)).astype(np.float32), CHOICES, r.random(B))
    check(p, np.minimum(r.standard_normal((B, V)), 0.5).astype(np.float32), CHOICES, r.random(B))
    check(p, np.where(r.random((B, V)) < 0.5, 0.0, -0.0).astype(np.float32), CHOICES, r.random(B))
    p.close()


@pytest.mark.parametrize("V", [100, 20000])
def test_tokens_that_are_excluded(cuda_backend, V):
    r = np.random.default_rng(V)
    B = len(CHOICES)
    p = program(cuda_backend, B, V)
    few = np.where(r.random((B, V)) < 0.01, r.standard_normal((B, V)), -np.inf).astype(np.float32)
    few[:, V // 3] = 0.0
    check(p, few, CHOICES, r.random(B))
    one = np.full((B, V), -np.inf, np.float32)
    one[np.arange(B), r.integers(0, V, B)] = -3e38
    check(p, one, CHOICES, r.random(B))
    got, share = check(p, np.full((B, V), -np.inf, np.float32), CHOICES, r.random(B))
    assert (got == -1).all() and np.isnan(share).all()
    lost = r.standard_normal((B, V)).astype(np.float32)
    lost[::2, V - 1] = np.nan
    check(p, lost, CHOICES, r.random(B))
    sure = r.standard_normal((B, V)).astype(np.float32)
    sure[:, [3, V - 2]] = np.inf                        # what is infinitely likely shares all
    check(p, sure, CHOICES, r.random(B))
    p.close()


@pytest.mark.parametrize("kind", ["far", "ladder", "near"])
def test_logits_far_apart_and_near(cuda_backend, kind):
    """Distributions that bins of one width do not part: one logit far above, a ladder of magnitudes, differences of single bits."""
    r = np.random.default_rng(3)
    V, B = 30000, len(CHOICES)
    z = r.standard_normal((B, V))
    if kind == "far":
        z[:, 77] = 1e30
    elif kind == "ladder":
        z = -(10.0 ** r.uniform(-30, 30, (B, V)))
    else:
        z = 1.0 + r.integers(0, 2000, (B, V)) * 2.0 ** -23
    p = program(cuda_backend, B, V)
    check(p, z.astype(np.float32), CHOICES, r.random(B))
    check(p, (1e-3 * z).astype(np.float32), [(c[0] and 1e-3, *c[1:]) for c in CHOICES], r.random(B))
    p.close()


@pytest.mark.parametrize("B,V", [(3, 6000), (3, 9000), (40, 9000), (200, 6000), (300, 2500), (70, 40000), (160, 66000), (130, 70001)])
def test_rows_that_fill_the_gpu(cuda_backend, B, V):
    """Rows by fewer CTAs each, and rows that are read again."""
    r = np.random.default_rng(B + V)
    p = program(cuda_backend, B, V)
    choices = [CHOICES[i % len(CHOICES)] for i in range(B)]
    check(p, ((1 + 2 * (np.arange(B)[:, None] % 2)) * r.standard_normal((B, V))).astype(np.float32), choices, r.random(B))
    p.close()


@pytest.mark.parametrize("V", [300, 9000])
def test_least_share_of_logits_near_zero(cuda_backend, V):
    """The largest logit over the temperature is all but -ln(min_p): what is let through ends within a range of tiny numbers of either sign, most of which are one exponent in 64 bits."""
    T = np.arange(1 << 22, 1 << 23, dtype=np.float64)
    M = np.round(T * np.log(2.0))
    gap = M / T - np.log(2.0)
    r = np.random.default_rng(V)
    p = program(cuda_backend, 8, V)
    logits, choices = np.empty((8, V), np.float32), []
    for i in range(8):
        near = np.where((np.abs(gap) > 1e-13 * (1 + i)) & ((gap > 0) == (i % 2 == 0)), np.abs(gap), 1)
        at = near.argmin()
        end = gap[at] * T[at]                          # what is let through ends here
        logits[i] = end * (1 + r.uniform(0.05, 3, V) * r.choice([-1, 1], V)) * 10.0 ** r.choice([0, 0, -20, -38], V)
        logits[i] = np.where(np.abs(logits[i] - end) < 0.04 * abs(end), 0, logits[i])
        logits[i, V // 2] = M[at]
        choices.append((T[at], 0, 1.0, 0.5))
    check(p, logits, choices, r.random(8))
    p.close()


def test_many_draws(cuda_backend):
    """One distribution, 2000 random numbers: the shares of the tokens are their probabilities."""
    r = np.random.default_rng(9)
    B, V = 2000, 50
    z = np.repeat(r.standard_normal((1, V)), B, 0).astype(np.float32)
    u = (np.arange(B) + 0.5) / B
    p = program(cuda_backend, B, V)
    got, _ = check(p, z, [(1.0, 0, 1.0, 0.0)] * B, u)
    want = np.exp(z[0].astype(np.float64))
    want /= want.sum()
    assert np.abs(np.bincount(got, minlength=V) / B - want).max() <= 1.0 / B + 1e-7
    p.close()


def test_rows_that_are_idle_or_wrong(cuda_backend):
    r = np.random.default_rng(1)
    B, V = 9, 1500
    z = r.standard_normal((B, V)).astype(np.float32)
    p = program(cuda_backend, B, V, probability=False)
    t = sample_table([TokenChoice(0.0)] * 4 + [None] + [TokenChoice(0.0)] * 4, [0.0] * B, B)
    for live in (9, 5, 0, -2, 99):
        t[0] = live
        got, share = p.run(["dst", "p"], logits=z.ravel(), table=t)
        want = np.array([77 if i == 4 or i >= min(9, max(0, live)) else z[i].argmax() for i in range(B)])
        assert np.array_equal(got.view(np.int32), want) and (share == 5.0).all()
    p.close()
    p = program(cuda_backend, B, V)
    t = sample_table([TokenChoice()] * B, [0.5] * B, B)
    body = t[8:].reshape(B, 8).view(np.float32)
    body[0, 0], body[1, 0], body[2, 0], body[3, 2], body[4, 2], body[5, 3], body[6, 4], body[7, 4] = -1.0, np.nan, np.inf, 1.5, np.nan, -0.5, 1.0, np.nan
    got, share = p.run(["dst", "p"], logits=z.ravel(), table=t)
    assert (got.view(np.int32)[:8] == -1).all() and np.isnan(share[:8]).all() and got.view(np.int32)[8] == ref.sample(z[8], (1.0, 0, 1.0, 0.0), 0.5)[0]
    p.close()


def test_rules_then_a_choice(cuda_backend):
    """LOGIT_RULES and SAMPLE in one program, in place, and again to the bit outside a graph."""
    from zgml_b200 import DeviceOp
    r = np.random.default_rng(2)
    B, V, L = 3, 700, 20
    z, history = r.standard_normal((B, V)).astype(np.float32), r.integers(0, V, (B, L)).astype(np.int32)
    rules = [LogitRules(1.5, 0.2, 0.1), LogitRules(allowed=np.arange(0, V, 7)), LogitRules(bias={5: 9.0})]
    t, bias, masks = rule_table(rules, [0, 1, 2], [L] * B, [5] * B, V, B)
    choices = [TokenChoice(0.8, 50, 0.9), TokenChoice(1.0, 0, 0.95), TokenChoice(1.0, 20)]
    make = lambda at: [DeviceOp.logit_rules(at["z"], at["z"], at["rules"], B, V, history=at["history"], history_rows=L, bias=at["bias"], masks=at["masks"]),
                       DeviceOp.sample(at["dst"], at["z"], at["table"], B, V, probability=at["p"])]
    for graph in (True, False):
        cuda_backend.set_graph_mode(graph)
        p = Prog(cuda_backend, make, dict(dst=np.zeros(B, np.int32), z=z, rules=t, history=history, bias=bias, masks=masks, table=sample_table(choices, [0.3, 0.6, 0.9], B), p=np.zeros(B, np.float32)))
        got, ruled = p.run(["dst", "z"])
        for i, c in enumerate(choices):
            assert got.view(np.int32)[i] == ref.sample(ruled[i], (c.temperature, c.top_k, c.top_p, c.min_p), (0.3, 0.6, 0.9)[i])[0]
        assert got.view(np.int32)[1] % 7 == 0
        p.close()
    cuda_backend.set_graph_mode(True)


def test_on_another_stream():
    import torch
    from zgml_b200 import CudaBackend
    be = CudaBackend(0)
    stream = torch.cuda.Stream()
    be.set_stream(stream.cuda_stream)
    r = np.random.default_rng(5)
    p = program(be, len(CHOICES), 20000)
    check(p, (3 * r.standard_normal((len(CHOICES), 20000))).astype(np.float32), CHOICES, r.random(len(CHOICES)))
    p.close()
    be.close()
