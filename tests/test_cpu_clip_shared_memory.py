"""Lists of tensors that share memory: a clip refuses them where it would write them.  No GPU is needed: the table
of a clip is formed from host tensors here."""

import numpy as np
import pytest
import torch

from apexw_amd import _lib
from apexw_amd._plan import _host


def table(grads, out=None, writes=True):
    t = np.zeros(max(len(grads), 1), dtype=_lib.CLIP_TENSOR_DTYPE)
    _host().clip_table(grads, grads if out is None else out, t.ctypes.data, "clip", writes)
    return t


def refused(grads, out=None, match="share memory"):
    with pytest.raises(ValueError, match=match):
        table(grads, out)


def test_in_place():
    base = torch.zeros(1000)
    a, b, c = base[:300], base[300:301], base[301:]
    for grads in ([a, b, c], [c, a, b], [b, c, a], [a, base[0:0], b], [base[5:5], base]):
        assert table(grads)["n"].tolist()[:len(grads)] == [g.numel() for g in grads]
    refused([a, b, a], match="tensors 0 and 2")
    refused([c, b, a, base[299:300]], match="tensors 2 and 3")
    refused([base[301:700], a, base[600:601]], match="tensors 0 and 2")
    refused([base, a])
    refused([a, base.view(torch.bfloat16)[:2]])
    refused([base[:6].view(2, 3), base[:6].view(2, 3).t()])


def test_copies():
    base, to = torch.zeros(1000), torch.zeros(2000, dtype=torch.bfloat16)
    a, b, c = base[:300], base[300:600], base[600:]
    x, y, z = to[:300], to[300:600], to[600:1000]
    table([a, b, c], [x, y, z])
    table([c, a, b], [z, x, y])
    table([a, b, a], [x, y, to[600:900]])                   # read twice
    table([a, b, base[250:350]], [x, y, to[600:700]])       # overlapping, only read
    table([a, b], [a, y])                                   # one in place, one not
    refused([a, b], [x, x], match="tensors 0 and 1")
    refused([a, b], [x, to[299:599]])
    refused([a, b], [b, torch.zeros(300)], match="tensors 0 and 1")
    refused([a, b], [b, a])
    refused([a, a], [a, x])                                  # scaled in place, and read for a copy
    refused([a], [base[1:301]], match="tensors 0 and 0")
    refused([a], [base.view(torch.bfloat16)[:300]])          # over itself in another type
    refused([a.bfloat16(), b], [base.view(torch.bfloat16)[599:899], torch.zeros(300)], match="tensors 0 and 1")


def test_nothing_written():
    """A norm alone reads what it is given."""
    base = torch.zeros(100)
    table([base, base, base[3:7]], writes=False)


def test_many():
    base = torch.zeros(100000)
    order = torch.randperm(1000, generator=torch.Generator().manual_seed(0)).tolist()
    grads = [base[100 * i:100 * i + 100] for i in order]
    table(grads)
    refused(grads + [base[54321:54322]])
