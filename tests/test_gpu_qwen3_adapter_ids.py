"""GPU: a serving layer's adapter ids: inputs without them, ids that name none, and the counter of what a step left out."""
import numpy as np
import pytest
from helpers import randn, to_dev, to_np
from test_gpu_qwen3_serving import Case

from acestep_ops.device import DTensor
from acestep_ops.qwen3 import decode_mask

pytestmark = pytest.mark.gpu


def test_prompt_inputs_that_say_nothing_of_adapters(dev):
    c = Case("small")
    hidden = to_dev(randn((2, 5, c.H), seed=11))
    inp = c.layer.prefill_inputs([3, 0], 5, c.s0)
    want = to_np(c.layer.prefill_run(hidden, inp))
    del inp["adapter_ids"]
    assert np.array_equal(to_np(c.layer.prefill_run(hidden, inp)), want)


@pytest.mark.parametrize("only", [("qkv", "o", "gu", "down"), ("o",), ()])
def test_what_a_decode_step_leaves_out_is_counted(dev, only):
    """An id past the last adapter once for each adapted product, a slot and a set that are not there for K and V."""
    c, N = Case("small", only=only), 4
    hidden, mask = to_dev(randn((N, c.H), seed=6)), decode_mask(np.array([3, 9, 0, 12], np.int32), c.max_seq)
    sets = np.arange(c.s0, c.s0 + N, dtype=np.int32)
    err = DTensor.zeros((1,), "i32")

    def step(pos, sets, ids):
        return to_np(c.layer.forward(hidden, to_dev(np.array(pos, np.int32)), to_dev(sets), c.s0, c.max_seq, mask,
                                     adapter_ids=to_dev(np.array(ids, np.int32)), err=err))

    want = step([3, 9, 0, 12], sets, [2, -1, 0, -1])
    assert err.item() == 0
    got = step([3, 9, 0, 12], sets, [2, 4, 0, 1 << 20])
    assert err.item() == 2 * len(only) and np.array_equal(got, want)
    sets[1] = 99
    step([3, 9, 0, c.max_seq], sets, [2, -1, 0, -1])
    assert err.item() == 2 * len(only) + 2 * 2 * c.Nkv


def test_what_a_prompt_leaves_out_is_counted(dev):
    c = Case("small")
    hidden, err = to_dev(randn((2, 5, c.H), seed=11)), DTensor.zeros((1,), "i32")
    c.layer.prefill(hidden, [3, 0], c.s0, adapter_ids=[1, -3], err=err)
    assert err.item() == 0
    inp = c.layer.prefill_inputs([3, 0], 5, c.s0, adapter_ids=[1, -1])
    inp["adapter_ids"] = to_dev(np.repeat(np.array([9, -1], np.int32), 5))
    inp["sets"] = to_dev(np.array([c.s0, 77], np.int32))
    c.layer.prefill_run(hidden, inp, err=err)
    assert err.item() == 4 * 5 + 2 * 5 * c.Nkv


def test_adapters_given_to_a_layer_later(dev):
    c, later = Case("small"), Case("small", only=())
    later.layer.adapters.update(c.layer.adapters)
    hidden = to_dev(randn((2, 5, c.H), seed=11))
    got = [to_np(x.layer.prefill(hidden, [3, 0], x.s0, adapter_ids=[1, 3])) for x in (c, later)]
    assert np.array_equal(*got)
    with pytest.raises(ValueError):
        later.layer.prefill(hidden, [3, 0], later.s0, adapter_ids=[1, 4])
