"""Refusals of the row operators and their 64-bit reference -- no GPU needed."""

import ctypes

import numpy as np
import pytest

from tests import rows_reference as ref

P = ctypes.c_void_p
I64 = ctypes.c_int64
INVALID, SHAPE, UNAVAILABLE = 2, 6, 7
AT = 4096  # a well-aligned address that is never followed: every call here is refused


def _has_gpu():
    import torch

    return torch.cuda.is_available()


def _refusals(call, good, bad):
    for i, value, status in bad:
        args = list(good)
        args[i] = value
        assert call(*args) == status, (i, value)
    if not _has_gpu():
        assert call(*good) == UNAVAILABLE  # valid arguments, no device: no CPU fallback


def test_sample_rows_refusals(ovvs):
    res = ovvs.Resources()
    good = [res._h, AT, 0, 4, 100, 100, AT, AT, AT, AT, AT, 2, AT, AT, AT, None]
    _refusals(ovvs.lib().ovvsSampleRowsDevice, good, [
        (0, None, INVALID), (1, None, INVALID), (10, None, INVALID), (12, None, INVALID),
        (2, 1 + 16, INVALID), (2, -1, INVALID), (2, 2, INVALID),
        (3, 0, INVALID), (3, -4, INVALID), (4, 0, INVALID), (5, 99, INVALID), (11, 0, INVALID),
        (1, AT + 2, INVALID), (12, AT + 4, INVALID), (10, AT + 1, INVALID), (6, AT + 2, INVALID),
        (7, AT + 2, INVALID), (8, AT + 2, INVALID), (9, AT + 2, INVALID), (13, AT + 2, INVALID),
        (14, AT + 2, INVALID),
        (5, 1 << 60, SHAPE), (3, 1 << 40, SHAPE), (11, 1 << 60, SHAPE)])
    wide = list(good)
    wide[4] = wide[5] = 1 << 31
    assert ovvs.lib().ovvsSampleRowsDevice(*wide) == SHAPE
    if not _has_gpu():  # the optional arrays
        for i in (6, 7, 8, 9, 13, 14):
            args = list(good)
            args[i] = None
            assert ovvs.lib().ovvsSampleRowsDevice(*args) == UNAVAILABLE
        half = list(good)
        half[1], half[2] = AT + 2, 16
        assert ovvs.lib().ovvsSampleRowsDevice(*half) == UNAVAILABLE


def test_route_topk_refusals(ovvs):
    res = ovvs.Resources()
    good = [res._h, AT, 0, 4, 64, 64, AT, 1, 8, 4, 1, 6, 1, 1.0, AT, AT, AT, None]
    _refusals(ovvs.lib().ovvsRouteTopkDevice, good, [
        (0, None, INVALID), (1, None, INVALID), (14, None, INVALID), (15, None, INVALID),
        (2, 7, INVALID), (3, 0, INVALID), (4, 0, INVALID), (5, 63, INVALID), (7, 2, INVALID),
        (7, -1, INVALID), (8, 0, INVALID), (8, 7, INVALID), (9, 0, INVALID), (9, 9, INVALID),
        (10, 2, INVALID), (11, 0, INVALID), (6, AT + 1, INVALID), (14, AT + 2, INVALID),
        (15, AT + 2, INVALID), (16, AT + 2, INVALID),
        (11, 33, SHAPE), (8, 64, SHAPE), (5, 1 << 60, SHAPE), (3, 1 << 40, SHAPE)])
    many = list(good)
    many[4] = many[5] = 1032
    assert ovvs.lib().ovvsRouteTopkDevice(*many) == SHAPE
    few = list(good)
    few[4] = few[5] = 8
    few[11] = 9
    assert ovvs.lib().ovvsRouteTopkDevice(*few) == SHAPE


def test_route_topk_backward_refusals(ovvs):
    res = ovvs.Resources()
    good = [res._h, AT, 16, 4, 64, 64, AT, 6, 0, 1, 1.0, AT, AT, AT, 64, None]
    _refusals(ovvs.lib().ovvsRouteTopkBackwardDevice, good, [
        (0, None, INVALID), (1, None, INVALID), (6, None, INVALID), (11, None, INVALID),
        (13, None, INVALID), (2, 3, INVALID), (3, 0, INVALID), (4, -1, INVALID),
        (5, 60, INVALID), (14, 60, INVALID), (7, 0, INVALID), (8, 3, INVALID),
        (13, AT + 1, INVALID), (6, AT + 1, INVALID), (11, AT + 2, INVALID),
        (12, AT + 2, INVALID), (7, 33, SHAPE), (14, 1 << 60, SHAPE)])


def test_route_plan_refusals(ovvs):
    res = ovvs.Resources()
    good = [res._h, AT, 100, 8, 16, AT, AT, 220, AT, None]
    _refusals(ovvs.lib().ovvsRoutePlanDevice, good, [
        (0, None, INVALID), (1, None, INVALID), (5, None, INVALID), (6, None, INVALID),
        (8, None, INVALID), (2, 0, INVALID), (3, 0, INVALID), (4, 0, INVALID), (7, 0, INVALID),
        (1, AT + 2, INVALID), (5, AT + 2, INVALID), (6, AT + 2, INVALID), (8, AT + 2, INVALID),
        (7, 219, SHAPE), (3, 1025, SHAPE), (2, 1 << 31, SHAPE), (7, 1 << 31, SHAPE),
        (4, 0x7FFFFFFF, SHAPE)])


def test_forced_cpu_refuses(ovvs):
    res = ovvs.Resources()
    res.set_policy("force_cpu")
    assert ovvs.lib().ovvsRoutePlanDevice(res._h, AT, 100, 8, 16, AT, AT, 220, AT,
                                          None) == UNAVAILABLE


def test_binding_refuses_host_tensors_and_wrong_shapes(ovvs):
    import torch

    res = ovvs.Resources()
    x = torch.zeros(4, 8)
    u = torch.zeros(4)
    with pytest.raises(ValueError, match="is on cpu"):
        res.sample_rows(x, u, torch.zeros(4, dtype=torch.int64), stream=0)
    with pytest.raises(ValueError, match="2-D"):
        res.sample_rows(u, u, torch.zeros(4, dtype=torch.int64), stream=0)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        res.sample_rows(x.double(), u, torch.zeros(4, dtype=torch.int64), stream=0)
    with pytest.raises(ValueError, match="next to each other"):
        res.sample_rows(x.T, torch.zeros(8), torch.zeros(8, dtype=torch.int64), stream=0)
    with pytest.raises(ValueError, match="overlapping"):
        res.sample_rows(x[:1].expand(4, 8), u, torch.zeros(4, dtype=torch.int64), stream=0)


def test_reference_sample_by_hand():
    x = np.log(np.array([1.0, 4.0, 2.0, 1.0]))
    u = np.array([0.0, 0.124, 0.126, 0.624, 0.626, 0.874, 0.876], np.float32)
    ids, p, kept = ref.sample_row(x, u)
    assert ids.tolist() == [0, 0, 1, 1, 2, 2, 3] and kept == 4
    assert np.allclose(p, np.array([1, 1, 4, 4, 2, 2, 1]) / 8)
    assert ref.sample_row(x, u, top_k=3)[2] == 3  # column 0 before column 3
    assert ref.sample_row(x, u, top_p=0.74)[2] == 2
    assert ref.sample_row(x, u, top_p=0.76)[2] == 3
    assert ref.sample_row(x, u, min_p=0.4)[2] == 2
    assert ref.sample_row(x, u, top_k=3, top_p=0.6)[2] == 2  # 4 of 7 is below 0.6
    assert ref.sample_row(x, u, temperature=0.0)[0].tolist() == [1] * 7


def test_reference_route_gradient_is_the_slope():
    """The written-out gradient against differences of the forward formula with the ids fixed."""
    rng = np.random.default_rng(5)
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            x = rng.standard_normal(12) * 2
            x[4] = -np.inf
            dw, ds = rng.standard_normal(3), rng.standard_normal(12)
            ids = ref.route_row(x, 3, score=score)[0]

            def loss(x):
                s = ref.scores_row(x, score)
                w = ref.ratio_row(x, ids, score) if renormalize else s[ids]
                return (dw * w * 1.7).sum() + (ds * s).sum()

            grad, _ = ref.route_backward_row(x, ids, dw, score=score, renormalize=renormalize,
                                             scale=1.7, dscores=ds)
            for e in range(12):
                h = 1e-6
                up, down = x.copy(), x.copy()
                up[e] += h
                down[e] -= h
                slope = (loss(up) - loss(down)) / (2 * h)
                assert abs(slope - grad[e]) < 1e-8, (score, renormalize, e)
