"""CPU: what Qwen3Layer refuses of adapters and their ids, before anything is uploaded."""
import numpy as np
import pytest

from acestep_ops.device import DTensor
from acestep_ops.qwen3 import Qwen3Layer


class Mem:
    ptr, nbytes = 1 << 20, 1 << 30


def _t(*shape, dtype="bf16"):
    return DTensor(Mem(), shape, dtype)


def _layer(adapters, scales=None):
    return Qwen3Layer(*[None] * 8, 64, 2, 1, 64, 96, 128, 2, "f16", adapters=adapters, adapter_scales=scales)


@pytest.mark.parametrize("adapters,scales", [
    ({"o": (_t(3, 8, 64), _t(4, 64, 8))}, None),
    ({"o": (_t(3, 8, 64), _t(3, 64, 8)), "down": (_t(2, 8, 96), _t(2, 64, 8))}, None),
    ({"o": (_t(3, 8, 64), _t(3, 64, 8))}, _t(4, dtype="f32")),
    ({"gate": (_t(3, 8, 64), _t(3, 64, 8))}, None)])
def test_stacks_that_do_not_agree(adapters, scales):
    with pytest.raises(ValueError, match="adapters"):
        _layer(adapters, scales)


@pytest.mark.parametrize("ids", [[0, 3], [1 << 32, 0], [0], [0, 1, 2]])
def test_ids_of_a_prompt(ids):
    layer = Qwen3Layer.__new__(Qwen3Layer)
    layer.kv_type, layer.k_cache = "f16", _t(2, 1, 128, 64, dtype="f16")
    layer.adapters = {"o": (_t(3, 8, 64), _t(3, 64, 8))}
    with pytest.raises(ValueError, match="adapter id"):
        layer.prefill_inputs(np.array([0, 5]), 4, 0, adapter_ids=ids)
