"""What the tokens' operators, the embedding and the linear cross entropy refuse before anything is launched: no GPU
is needed."""

import pytest
import torch

import apexw_amd
from apexw_amd import _lib


def order(tokens=2, k=2):
    place = torch.arange(tokens * k, dtype=torch.int32).view(tokens, k)
    return apexw_amd.ExpertOrder(place.view(-1), place, torch.tensor([tokens * k], dtype=torch.int32))


def test_expert_order_refuses():
    with pytest.raises(ValueError, match="GPU"):
        apexw_amd.expert_order(torch.tensor([0, 1]), 2)
    with pytest.raises(TypeError, match="int32 or int64"):
        apexw_amd.expert_order(torch.tensor([0.0]), 2)


def test_dispatch_and_combine_refuse():
    x = torch.randn(2, 8)
    for call in (lambda t: apexw_amd.expert_dispatch_forward(t, order()), lambda t: apexw_amd.expert_combine_forward(t, order()),
                 lambda t: apexw_amd.expert_combine_backward(t, t, order(), torch.ones(2, 2)), lambda t: apexw_amd.expert_dispatch(t, order())):
        with pytest.raises(ValueError, match="GPU"):
            call(x)
        with pytest.raises(TypeError, match="float64"):
            call(x.double())
        with pytest.raises(ValueError, match="shape"):
            call(x[0])
        with pytest.raises(ValueError, match="shape"):
            call(x[:, :0])


def test_embedding_refuses():
    ids, w = torch.tensor([0, 1]), torch.randn(4, 8)
    with pytest.raises(ValueError, match="GPU"):
        apexw_amd.embedding(ids, w)
    with pytest.raises(TypeError, match="int32 or int64"):
        apexw_amd.embedding_forward(ids.float(), w)
    with pytest.raises(ValueError, match="GPU"):
        apexw_amd.embedding_weight_grad(torch.randn(2, 8), ids, 4)


def test_linear_cross_entropy_refuses():
    x, w, t = torch.randn(3, 8).bfloat16(), torch.randn(5, 8).bfloat16(), torch.tensor([0, 1, 2])
    f = apexw_amd.linear_cross_entropy_forward
    with pytest.raises(ValueError, match="GPU"):
        f(x, w, t)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        f(x.float(), w.float(), t)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        f(x, w.half(), t)
    with pytest.raises(ValueError, match="width"):
        f(x, w[:, :4], t)
    with pytest.raises(ValueError, match="width"):
        f(x, w[:0], t)
    with pytest.raises(ValueError, match="target"):
        f(x, w, t[:2])
    with pytest.raises(TypeError, match="int32 or int64"):
        f(x, w, t.float())
    with pytest.raises(ValueError, match="reduction"):
        apexw_amd.linear_cross_entropy(x, w, t, reduction="max")
    with pytest.raises(ValueError, match="dloss"):
        apexw_amd.linear_cross_entropy_backward(torch.ones(2), x, w, t, torch.ones(3))
    with pytest.raises(ValueError, match="lse"):
        apexw_amd.linear_cross_entropy_backward(torch.ones(3), x, w, t, torch.ones(3).double())


def test_entry_points_refuse_without_launching():
    lib, ok = _lib.load(), 4096        # an aligned address that no call here reaches
    F32, BF16, F16, MOST = _lib.F32, _lib.BF16, _lib.F16, 16776960
    order, dispatch, combine, back = (lib.apexw_expert_order, lib.apexw_expert_dispatch, lib.apexw_expert_combine,
                                      lib.apexw_expert_combine_backward)
    assert order(ok, 8, 4, 2, ok, ok, None, None, None) == 1
    assert order(None, 8, 4, 2, ok, ok, ok, None, None) == 1
    assert order(ok, 2, 4, 2, ok, ok, ok, None, None) == 1
    assert order(ok, 8, 4, 0, ok, ok, ok, None, None) == 1
    assert order(ok, 8, -1, 2, ok, ok, ok, None, None) == 1
    assert order(ok, 8, 2 ** 31 - 1, 2, ok, ok, ok, ok, None) == 1
    assert order(ok + 4, 8, 4, 2, ok, ok, ok, None, None) == 4
    assert order(ok, 8, 4, 2, ok + 2, ok, ok, None, None) == 4
    assert order(ok, 8, 4, 1000, ok, ok, ok, None, None) == 1           # two passes, no workspace
    assert order(ok, 8, 5000, 2, ok, ok, ok, None, None) == 1
    assert lib.apexw_expert_order_workspace(4096, 511) == 0 and lib.apexw_expert_order_workspace(4096, 512) > 0
    assert lib.apexw_expert_order_workspace(4097, 8) > 0
    assert lib.apexw_expert_order_workspace(-1, 8) == -1 and lib.apexw_expert_order_workspace(5, 0) == -1
    assert dispatch(None, 8, 4, 2, 8, BF16, ok, ok, ok, None) == 1
    assert dispatch(ok, -8, 4, 2, 8, BF16, ok, ok, ok, None) == 1
    assert dispatch(ok, 8, 4, 0, 8, BF16, ok, ok, ok, None) == 1
    assert dispatch(ok, 8, 4, 2, 0, BF16, ok, ok, ok, None) == 1
    assert dispatch(ok, 8, 4, 2, MOST + 1, BF16, ok, ok, ok, None) == 1
    assert dispatch(ok, 8, 2 ** 30, 4, 8, BF16, ok, ok, ok, None) == 1
    assert dispatch(ok, 8, 4, 2, 8, 7, ok, ok, ok, None) == 2
    assert dispatch(ok + 2, 8, 4, 2, 8, F32, ok, ok, ok, None) == 4
    assert dispatch(ok, 8, 4, 2, 8, F32, ok + 1, ok, ok, None) == 4
    assert combine(ok, 8, 4, 2, 8, BF16, None, ok, BF16, ok, None) == 1
    assert combine(ok, 8, 4, 2, 8, BF16, ok, ok, F16, ok, None) == 2
    assert combine(ok, 8, 4, 2, 8, BF16, ok, ok + 2, F32, ok, None) == 4
    assert back(ok, 8, ok, 8, 4, 2, 8, BF16, ok, ok, None, BF16, ok, ok, None) == 1
    assert back(ok, 8, None, 8, 4, 2, 8, BF16, ok, ok, ok, BF16, ok, ok, None) == 1
    assert back(ok, 8, ok, 8, 4, 2, 8, F32, ok, ok, ok, BF16, ok, ok, None) == 2
    assert back(ok, 8, ok, 8, 4, 2, 8, BF16, ok, ok, ok, BF16, ok + 1, ok, None) == 4

    fwd, grad = lib.apexw_embedding_forward, lib.apexw_embedding_weight_grad
    assert fwd(None, 8, 4, ok, 8, 10, 8, BF16, 1.0, ok, None) == 1
    assert fwd(ok, 1, 4, ok, 8, 10, 8, BF16, 1.0, ok, None) == 1
    assert fwd(ok, 8, 4, ok, 8, 0, 8, BF16, 1.0, ok, None) == 1
    assert fwd(ok, 8, 4, ok, 8, 2 ** 31, 8, BF16, 1.0, ok, None) == 1
    assert fwd(ok, 8, 4, ok, 8, 10, 8, 9, 1.0, ok, None) == 2
    assert fwd(ok + 4, 8, 4, ok, 8, 10, 8, BF16, 1.0, ok, None) == 4
    assert grad(ok, 8, ok, 8, 4, 10, 8, BF16, 1.0, None, BF16, ok, None) == 1
    assert grad(ok, 8, ok, 8, 4, 10, 8, BF16, 1.0, ok, BF16, None, None) == 1
    assert grad(ok, 8, ok, 8, 4, 10, 8, BF16, 1.0, ok, F16, ok, None) == 2
    assert grad(ok, 8, ok, 8, 4, 10, 8, F32, 1.0, ok, BF16, ok, None) == 2
    assert grad(ok, 8, ok, 8, 4, 10, 8, BF16, 1.0, ok + 2, F32, ok, None) == 4
    assert grad(ok, 8, ok, 8, 4, 10, 8, BF16, 1.0, ok, BF16, ok + 8, None) == 4
    assert lib.apexw_embedding_weight_grad_workspace(5, 0, 8) == -1
    assert lib.apexw_embedding_weight_grad_workspace(5, 10, MOST + 1) == -1

    fwd, back = lib.apexw_linear_cross_entropy_forward, lib.apexw_linear_cross_entropy_backward
    space = lib.apexw_linear_cross_entropy_workspace
    call = dict(x=ok, xs=8, n=4, width=8, w=ok, ws=8, vocab=10, dtype=BF16, t=ok, ids=8, ignore=-100, loss=ok, lse=ok,
                reduction=0, total=None, space=ok, stream=None)
    for change, status in (({"x": None}, 1), ({"w": None}, 1), ({"t": None}, 1), ({"loss": None}, 1), ({"space": None}, 1),
                           ({"n": -1}, 1), ({"width": 0}, 1), ({"width": 2 ** 23}, 1), ({"vocab": 0}, 1), ({"ids": 2}, 1),
                           ({"xs": -1}, 1), ({"reduction": 3}, 1), ({"reduction": 1}, 1), ({"dtype": F32}, 2),
                           ({"x": ok + 1}, 4), ({"t": ok + 4}, 4), ({"lse": ok + 2}, 4), ({"space": ok + 8}, 4),
                           ({"n": 2 ** 31 - 70000, "vocab": 2 ** 31 - 70000}, 5)):
        assert fwd(*{**call, **change}.values()) == status, change
    call = dict(d=ok, ds=1, mean=0, x=ok, xs=8, n=4, width=8, w=ok, ws=8, vocab=10, dtype=BF16, t=ok, ids=8, ignore=-100,
                lse=ok, dx=ok, dw=ok, space=ok, stream=None)
    for change, status in (({"d": None}, 1), ({"ds": -1}, 1), ({"lse": None}, 1), ({"dtype": F32}, 2), ({"dx": ok + 1}, 4),
                           ({"d": ok + 2}, 4), ({"dx": None, "dw": None}, 0)):
        assert back(*{**call, **change}.values()) == status, change
    assert space(ok, 8, 4, 0, 10, 0) == -1 and space(ok, 8, 400, 8, 1000, 3) > space(ok, 8, 400, 8, 1000, 0) > 0


def test_sizes_that_no_launch_holds():
    lib = _lib.load()
    assert lib.apexw_embedding_weight_grad_workspace(5, 2 ** 29, 1) > 0
    assert lib.apexw_embedding_weight_grad_workspace(5, 2 ** 29 + 1, 1) == -_lib.ERR_SIZE
    ok = 2 ** 40
    assert lib.apexw_embedding_weight_grad(ok, 8, ok, 8, 4, 2 ** 30, 8, 1, 1.0, ok, 1, ok, None) == _lib.ERR_SIZE
    space = lib.apexw_linear_cross_entropy_workspace
    assert space(ok, 8, 2 ** 26 - 1, 8, 1000, 0) > 0 and space(ok, 8, 2 ** 26, 8, 1000, 0) == -_lib.ERR_SIZE
    assert space(ok, 8, 2 ** 25, 8, 2 ** 30, 3) == -_lib.ERR_SIZE
