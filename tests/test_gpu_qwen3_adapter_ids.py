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
