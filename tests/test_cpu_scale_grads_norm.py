"""scale_grads refuses a norm that lies in what it writes (host tensors: checked where the table is formed)."""

import numpy as np
import pytest
import torch

from apexw_amd import _lib
from apexw_amd._plan import _host


def table(grads, total, out=None, writes=True):
    t = np.zeros(len(grads), dtype=_lib.CLIP_TENSOR_DTYPE)
    _host().clip_table(grads, grads if out is None else out, t.ctypes.data, "scale", writes, total.data_ptr())


def test_norm_among_the_gradients():
    base = torch.zeros(100)
    grads = [base[:40], base[41:60], base[60:]]
    table(grads, torch.zeros(()))
    table(grads, base[40])                                            # between two of them
    for at in (0, 39, 41, 99):
        with pytest.raises(ValueError, match="holds total_norm"):
            table(grads, base[at])
    table(grads, base[0], writes=False)
    table(grads, base[0], out=[torch.zeros(40), torch.zeros(19), torch.zeros(40)])   # only read
    to = torch.zeros(100)
    with pytest.raises(ValueError, match="tensor 1"):
        table(grads, to[45], out=[to[:40], to[41:60], to[60:]])
