"""What a clip writes gets a new version, as from torch's in-place operations (host tensors here: the versions are
counted where the clip's table is formed)."""

import torch

from test_cpu_clip_shared_memory import table


def test_versions():
    a, b, x, y = (torch.zeros(5) for _ in range(4))
    before = [t._version for t in (a, b, x, y)]
    table([a, b], writes=False)
    assert [t._version for t in (a, b, x, y)] == before
    table([a, b])
    assert [t._version for t in (a, b)] == [before[0] + 1, before[1] + 1]
    table([a, b], [x, y])
    assert [t._version for t in (a, b, x, y)] == [n + 1 for n in before]
    view = x[1:3]
    table([view])
    assert x._version == before[2] + 2          # shared with its base


def test_refused_lists_keep_their_versions():
    a, b = torch.zeros(5), torch.zeros(5)
    before = a._version, b._version
    for bad in ([a, b, a], [a, b, torch.zeros(3, dtype=torch.float64)]):
        try:
            table(bad)
        except (ValueError, TypeError):
            pass
    assert (a._version, b._version) == before


def test_inference_tensors():
    with torch.inference_mode():
        t = torch.zeros(4)
    table([t])
