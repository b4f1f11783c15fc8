"""GPU: adapters and logits from columns of a buffer to other columns of it: the bits of the call on buffers of
their own, and every other byte as it was."""
import numpy as np
import pytest
from helpers import randn, to_dev, to_np
from test_gpu_logits import _case as logits_case, _ref as logits_ref
from test_gpu_lora import _case, _run

from acestep_ops import ops
from acestep_ops.device import DTensor

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n", [(2, 96), (24, 130), (1505, 1002)])
def test_adapters(dev, m, n):
    k = 64
    x, y0, a, _, b, _, ids, scales = _case(m, k, n, 16, 4, "bf16", seed=m)
    want = _run(x, y0, a, b, ids, scales)
    wide = randn((m, 2 * n + k + 30), seed=9)
    wide[:, 5:5 + n], wide[:, 2 * n + 11:2 * n + 11 + k] = y0, x
    wd = to_dev(wide)
    ops.lora_add(wd[:, 5:5 + n], wd[:, 2 * n + 11:2 * n + 11 + k], a, b, to_dev(ids), to_dev(scales), out=wd[:, 5 + n:5 + 2 * n])
    wide[:, 5 + n:5 + 2 * n] = want
    assert np.array_equal(to_np(wd), wide)


def test_logits(dev):
    m, V = 5, 5001
    hist, lens, pen, bias, allowed, state = logits_case(m, V, 300, 3, seed=4)
    wide = randn((m, 2 * V + 9), seed=5)
    wd = to_dev(wide)
    ops.logits_adjust(wd[:, V + 3:2 * V + 3], *(to_dev(t) for t in (hist, lens, pen, bias, allowed, state)), out=wd[:, 2:V + 2])
    wide[:, 2:V + 2] = logits_ref(wide[:, V + 3:2 * V + 3].copy(), hist, lens, pen, bias, allowed, state)
    assert np.array_equal(to_np(wd), wide)
