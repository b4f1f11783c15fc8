"""GPU: adapters whose first launch did not take place add nothing: y, here y0 itself, stays as it was."""
import numpy as np
import pytest
from helpers import to_dev, to_np
from test_gpu_lora import _case, _check

from acestep_ops import MiError, ops
from acestep_ops.device import DTensor, hip

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n", [(8, 192), (1505, 1002)])
def test_y_stays_after_an_error(dev, m, n):
    x, y0, a, ah, b, bh, ids, scales = _case(m, 64, n, 16, 4, "bf16", seed=m)
    yd, xd, idd, sd = to_dev(y0), to_dev(x), to_dev(ids), to_dev(scales)
    ws = DTensor.full_byte((ops.lora_add_workspace(xd, a, b),), 0xFF)
    assert hip().hipSetDevice(1 << 20) != 0  # a pending error, as a refused launch leaves it
    with pytest.raises(MiError):
        ops.lora_add(yd, xd, a, b, idd, sd, out=yd, workspace=ws)
    assert np.array_equal(to_np(yd), y0)
    ops.lora_add(yd, xd, a, b, idd, sd, out=yd, workspace=ws)
    _check(to_np(yd), y0, x, ah, bh, ids, scales)
