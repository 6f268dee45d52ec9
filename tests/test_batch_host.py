"""Host side of the batched step, without a device: the tables and rules a user builds, and what the ops' static checks refuse."""
import numpy as np
import pytest

from zgml_b200 import DeviceOp, abi
from zgml_b200.backend import seq_check
from zgml_b200.host.batch import BatchRow, LogitRules, batch_table, rule_table, rule_words, table_words


def test_table_words():
    t = batch_table([BatchRow(3, 5, 2), BatchRow(-1), BatchRow(0, 0)], 4, prefix=17, prefix_slot=1, slots=4, capacity=5, prefix_capacity=17, adapters=3)
    assert t.dtype == np.int32 and t.size == table_words(4) == 24
    assert list(t[:3]) == [3, 17, 1]
    assert t[abi.BATCH_ROWS:].reshape(4, 4).tolist() == [[3, 5, 2, 0], [-1, 0, -1, 0], [0, 0, -1, 0], [0, 0, 0, 0]]


@pytest.mark.parametrize("kw,rows", [(dict(slots=3), [BatchRow(3, 1)]), (dict(capacity=4), [BatchRow(0, 5)]), (dict(adapters=2), [BatchRow(0, 1, 2)]), ({}, [BatchRow(0, -1)]), (dict(prefix=-1), []),
                                     (dict(prefix=9, prefix_capacity=8), []), (dict(prefix_slot=-1), []), ({}, [BatchRow(0, 1)] * 3)])
def test_tables_refuse(kw, rows):
    with pytest.raises(ValueError):
        batch_table(rows, 2, **kw)


def test_rule_table():
    rules = [LogitRules(1.5, 0.25, 0.5, {7: 1.0, 3: -2.0}), LogitRules(allowed=np.array([0, 33])), LogitRules(allowed=np.arange(40) % 2 == 0, bias={39: 4.0})]
    t, bias, masks = rule_table(rules, [2, 0, 1], [10, 0, 4], [6, 0, 4], 40, 4)
    assert t.size == rule_words(4) and t[0] == 3
    body = t[abi.BATCH_ROWS:].reshape(4, abi.RULE_WORDS)
    assert body[:, :6].tolist() == [[2, 10, 6, -1, 0, 2], [0, 0, 0, 0, 2, 0], [1, 4, 4, 1, 2, 1], [0] * 6]
    assert body[:3, 6:9].copy().view(np.float32).tolist() == [[1.5, 0.25, 0.5], [1.0, 0.0, 0.0], [1.0, 0.0, 0.0]]
    assert bias[:, 0].tolist() == [7, 3, 39] and bias[:, 1].copy().view(np.float32).tolist() == [1.0, -2.0, 4.0]
    assert masks.tolist() == [[1, 2], [0x55555555, 0x55]]


@pytest.mark.parametrize("kw", [dict(repetition=0.0), dict(repetition=-1.0), dict(repetition=float("nan")), dict(repetition=float("inf")), dict(presence=float("inf")), dict(frequency=float("nan")),
                                dict(repetition=1e-60), dict(repetition=1e60), dict(presence=1e60), dict(bias={3: float("nan")})])
def test_rules_refuse(kw):
    with pytest.raises(ValueError):
        LogitRules(**kw)


@pytest.mark.parametrize("rules", [LogitRules(bias={40: 1.0}), LogitRules(bias={-1: 1.0}), LogitRules(allowed=np.array([40])), LogitRules(allowed=np.ones(39, bool))])
def test_rule_table_refuses(rules):
    with pytest.raises(ValueError):
        rule_table([rules], [0], [0], [0], 40, 1)


def test_sizes_that_do_not_fit_the_words_of_an_op():
    with pytest.raises(ValueError):
        DeviceOp.adapter_linear(0, 1, 2, 0, 1 << 32, 3, 1, 8, 8, 4, 2, abi.W_F32)


APPEND = dict(cache=0, src=1, table=2, src_col=16, cache_col=0, B=3, cols=16, src_rs=32, width=16, rows=5, key_heads=1, head_dim=8, rot=8, rot_base=1e4, q_heads=2, q_col=0, turned=3)
APPEND_SIZES = [2 * 5 * 16, 3 * 32, table_words(3), 3 * 16]
ATTEND = dict(dst=0, q=1, k_cache=2, v_cache=2, k_prefix=3, v_prefix=3, table=4, q_col=0, k_col=0, v_col=16, k_prefix_col=0, v_prefix_col=16, B=3, H=4, G=2, dk=8, dv=4, q_rs=32, k_width=24, v_width=24,
              rows=5, k_prefix_width=24, v_prefix_width=24, prefix_rows=7, scale=0.5, sink=5)
ATTEND_SIZES = [3 * 16, 3 * 32, 2 * 5 * 24, 7 * 24, table_words(3), 4]
ADAPTER = dict(dst=0, src=1, w=2, a_off=0, b_off=2 * 4 * 8, table=3, B=3, N=6, K=8, rank=4, adapters=2, wdt=abi.W_F32, base=4, scales=5)
ADAPTER_SIZES = [3 * 6, 3 * 8, 2 * 4 * 14, table_words(3), 3 * 6, 2]
RULES = dict(dst=0, src=1, table=2, B=3, V=40, history=3, history_rows=9, bias=4, masks=5)
RULES_SIZES = [3 * 40, 3 * 40, rule_words(3), 2 * 9, 2, 2]


@pytest.mark.parametrize("make,kw,sizes", [(DeviceOp.batch_append, APPEND, APPEND_SIZES), (DeviceOp.shared_attention, ATTEND, ATTEND_SIZES), (DeviceOp.adapter_linear, ADAPTER, ADAPTER_SIZES),
                                           (DeviceOp.logit_rules, RULES, RULES_SIZES)])
def test_what_the_checks_take(make, kw, sizes):
    assert seq_check(make(**kw), sizes) is None
    for i in range(len(sizes)):                        # every operand is as small as it may be
        short = list(sizes)
        short[i] = 1 if make in (DeviceOp.logit_rules,) and i in (3, 4, 5) else {2 * 5 * 16: 5 * 16, 2 * 5 * 24: 5 * 24}.get(sizes[i], sizes[i]) - 1
        assert seq_check(make(**kw), short), i


def change(make, standard, sizes, **kw):
    return seq_check(make(**dict(standard, **kw)), sizes)


@pytest.mark.parametrize("kw", [dict(B=0), dict(cols=0), dict(width=15), dict(rows=0), dict(key_heads=3), dict(rot=7), dict(rot=10), dict(turn_at=1), dict(rot_base=0.0), dict(rot_base=-1.0), dict(src_rs=31),
                                dict(turned=0), dict(turned=1), dict(turned=2), dict(turned_rs=15), dict(cache=1), dict(cache=2), dict(q_heads=5), dict(head_dim=0), dict(freqs=2, freqs_off=1000)])
def test_batch_append_refuses(kw):
    assert change(DeviceOp.batch_append, APPEND, APPEND_SIZES, **kw)


@pytest.mark.parametrize("kw", [dict(B=0), dict(H=3), dict(H=0), dict(G=0), dict(dk=0), dict(dv=0), dict(dk=1025), dict(q_rs=31), dict(dst_rs=15), dict(k_width=15), dict(v_width=23), dict(rows=0), dict(k_prefix=None),
                                dict(v_prefix=None), dict(k_prefix=None, v_prefix=None), dict(prefix_rows=0), dict(prefix_rows=8), dict(v_prefix_width=23), dict(sink_wdt=2), dict(sink_off=1),
                                dict(scale=float("nan")), dict(scale=float("inf")), dict(softcap=-1.0), dict(softcap=float("nan")), dict(dst=1), dict(dst=2), dict(dst=3), dict(dst=4), dict(dst=5), dict(table=9)])
def test_shared_attention_refuses(kw):
    assert change(DeviceOp.shared_attention, ATTEND, ATTEND_SIZES, **kw)


def test_shared_attention_without_a_prefix():
    assert change(DeviceOp.shared_attention, ATTEND, ATTEND_SIZES, k_prefix=None, v_prefix=None, prefix_rows=0, k_prefix_width=0, v_prefix_width=0) is None


@pytest.mark.parametrize("kw", [dict(B=0), dict(N=0), dict(K=0), dict(rank=0), dict(adapters=0), dict(adapters=3), dict(rank=1025), dict(src_rs=7), dict(dst_rs=5), dict(base_rs=5), dict(wdt=2), dict(b_off=65),
                                dict(a_off=60), dict(scales_off=1), dict(dst=1), dict(dst=2), dict(dst=3), dict(dst=5), dict(base=0, base_off=1), dict(base=0, base_rs=7)])
def test_adapter_linear_refuses(kw):
    assert change(DeviceOp.adapter_linear, ADAPTER, ADAPTER_SIZES, **kw)


@pytest.mark.parametrize("kw", [dict(adapters=1 << 31, K=1 << 31, N=1 << 31), dict(adapters=1 << 30, K=1 << 24, N=1 << 24)])
def test_adapter_linear_refuses_products_that_pass_64_bits(kw):
    """Buffers as large as the rows ask for, and weights whose size is a multiple of 2^64."""
    sizes = [1 << 33, 1 << 33, 2 * 4 * 14, table_words(1), 1 << 33, 2]
    assert change(DeviceOp.adapter_linear, ADAPTER, sizes, **dict(kw, B=1, rank=1024, scales=None, a_off=0, b_off=0))


def test_adapter_linear_forms():
    for form in ("auto", "runs", "blocks"):
        assert change(DeviceOp.adapter_linear, ADAPTER, ADAPTER_SIZES, form=form) is None
    with pytest.raises(ValueError):
        DeviceOp.adapter_linear(**ADAPTER, form="rows")
    op = DeviceOp.adapter_linear(**ADAPTER)
    op.u.seq.n[9] = 3
    assert seq_check(op, ADAPTER_SIZES)


def test_adapter_linear_in_place():
    assert change(DeviceOp.adapter_linear, ADAPTER, ADAPTER_SIZES, base=None) is None


@pytest.mark.parametrize("kw", [dict(B=0), dict(V=0), dict(src_rs=39), dict(dst_rs=39), dict(V=41), dict(history_rows=0), dict(history_rows=19), dict(dst=2), dict(dst=3), dict(dst=4), dict(dst=5),
                                dict(src=0, src_off=1), dict(src=0, src_rs=41)])
def test_logit_rules_refuses(kw):
    assert change(DeviceOp.logit_rules, RULES, RULES_SIZES, **kw)


def test_logit_rules_in_place_and_without_operands():
    assert change(DeviceOp.logit_rules, RULES, RULES_SIZES, src=0) is None
    assert change(DeviceOp.logit_rules, RULES, RULES_SIZES, history=None, bias=None, masks=None) is None


def test_check_of_other_things():
    assert seq_check(DeviceOp.softmax(0, 0, 1, 4), [4]) and seq_check(DeviceOp.activation(0, 1, 4, "relu"), [4]) and seq_check(DeviceOp.activation(0, 1, 4, "relu"), [4, 4]) is None


def test_rules_of_the_command_line():
    from argparse import Namespace
    from zgml_b200.cli import _rules
    a = dict(repetition_penalty=1.0, presence_penalty=0.0, frequency_penalty=0.0, bias="", allow="")
    assert _rules(Namespace(**a)) is None
    r = _rules(Namespace(**dict(a, repetition_penalty=1.2, bias="3:1.5,7:-2", allow="1,2")))
    assert r.repetition == 1.2 and r.bias == {3: 1.5, 7: -2.0} and list(r.allowed) == [1, 2]
    with pytest.raises(ValueError):
        _rules(Namespace(**dict(a, repetition_penalty=0.0)))
