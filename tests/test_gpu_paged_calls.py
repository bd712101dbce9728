"""GPU: calls of the paged 8-bit cache that its documentation allows and that are easily missed: odd strides, limits in replays, batches that are dropped, graphs of long rows."""
import gc

import pytest
import torch

import paged_rows as plain
from test_gpu_paged_cache import DEV, _cache, _check_attend, _filled, _holds, _pages_add_up, _queries, _rows

pytestmark = pytest.mark.gpu


def test_strides_of_single_rows_mean_nothing():
    """Dimensions of one with strides that are no multiple of 8: one token, one head, one row."""
    k, v = _rows(1, 1, 1, 70, torch.float16)
    c = _filled(k, v, [70], "int8")
    q = _queries(1, 1, 4, 1, torch.float16)
    odd = torch.zeros(4 * 128, dtype=torch.float16, device=DEV).as_strided((1, 4, 1, 128), (3, 128, 5, 1)).copy_(q)
    assert torch.equal(c.attend(0, odd), c.attend(0, q.to(DEV)))
    c.extend(1)
    one = torch.zeros(128, dtype=torch.float16, device=DEV).as_strided((1, 1, 1, 128), (9, 7, 5, 1))
    one.copy_(k[:, :, :1])
    c.write(0, one, one)
    _holds(c, 0, [tuple(torch.cat([x[0], k[0, :, :1]], dim=1) for x in (k, v))], "int8")
