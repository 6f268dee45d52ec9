"""Rules over long histories on the device: LOGIT_RULES beyond 65535 words, where counts are whole words, and sessions whose histories outgrow their room."""
import numpy as np
import pytest

from test_gpu_batchops import rules_case
from test_gpu_batchsteps import sessions

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pad", [0, 1])
@pytest.mark.parametrize("L", [65535, 65536, 70001])
def test_long_histories(cuda_backend, L, pad):
    """One token makes up most of the history: its count passes 16 bits, before `first` and behind it."""
    r = np.random.default_rng(L)
    history = np.where(r.random((3, L)) < 0.99, 7, r.integers(0, 5000, (3, L))).astype(np.int32)
    rows = [(0, L, 0, -1, 0, 0, 1.5, 0.25, 2.0 ** -10), (2, L, L - 3, -1, 0, 0, 1.25, 0.5, 0.25), (1, L - 1, L, -1, 0, 0, 2.0, 0.5, 0.25)]
    rules_case(cuda_backend, 3, 5000, rows, history=history, pad=pad)


def test_a_session_whose_history_outgrows_its_room(cuda_backend):
    """Programs that are made again for more tokens give what a session with room for all gives, to the bit."""
    from zgml_b200.host.batch import LogitRules
    grown, roomy = sessions(cuda_backend, 1)[0], sessions(cuda_backend, 1, max_history=64)[0]
    grown._room = 8
    rules = LogitRules(1.7, 0.5, 0.25, {3: 1.5})
    r = np.random.default_rng(0)
    for step in range(12):
        for k in ("a", "b"):
            new = r.integers(0, 97, 3 if step == 0 else 1 + step % 3).tolist()
            x, y = (s.feed(k, new, [len(new) - 1], rules, generated=step > 0) for s in (grown, roomy))
            assert np.array_equal(x, y), (step, k)
    assert grown._room >= 3 + sum(1 + step % 3 for step in range(1, 12))
    for s in (grown, roomy):
        for k in ("a", "b"):
            s.release(k)
    rules = LogitRules(1.1, presence=2.0, frequency=0.5)
    assert grown.generate([5, 6, 7], 60, rules=rules) == roomy.generate([5, 6, 7], 60, rules=rules)
    for s in (grown, roomy):
        s.close()
