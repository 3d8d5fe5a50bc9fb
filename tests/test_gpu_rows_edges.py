"""Row operators on the GPU where a kernel's shortcut could show: biases of any size, ids at the
ends of a packed key, gradients that are not finite, weights and scores held to the accuracy that
is stated for them, places near 2^31."""

import numpy as np
import pytest

from tests import rows_reference as ref
from tests.test_gpu_rows import TYPES, check_route, logits, run_backward, torch  # noqa: F401

pytestmark = pytest.mark.gpu


# ---- routing: biases of any size ------------------------------------------------------------------

def biases(experts, groups):
    """name -> bias [experts]: what a router's balance bias may come to, and what blocks or forces
    an expert."""
    rng = np.random.default_rng(experts)
    per = experts // groups
    normal = lambda mean, std: rng.normal(mean, std, experts).astype(np.float32)  # noqa: E731
    out = {"wide": normal(0, 2), "drifted": normal(6, 1), "off_centre": normal(2, 1),
           "drifted_narrow": normal(6, 0.1), "far_below": normal(-40, 3)}
    # one large value against a group of middling ones: their sums, not their parts, decide
    one = np.zeros(experts, np.float32)
    one[0] = 10.0
    one[per:2 * per] = 3.0
    out["one_of_ten"] = one
    for v in (3.0, 5.0, 1e4, 3e38, np.inf):
        for sign in (1, -1):
            b = normal(0, 0.1)
            b[rng.integers(0, experts, 3)] = sign * v
            out[f"few_at_{sign * v:g}"] = b
    alone = np.full(experts, -1e9, np.float32)  # every group but one expert disabled
    alone[::per] = normal(0, 0.5)[::per]
    out["one_left_a_group"] = alone
    mixed = normal(0, 0.1)
    mixed[::2] = -5.0
    mixed[1::4] = -1e9
    out["disabled_beside_low"] = mixed
    return out


@pytest.mark.parametrize("experts,groups,topk_groups,k", [
    (64, 8, 1, 4), (64, 8, 3, 8), (128, 8, 4, 6), (256, 8, 4, 8), (256, 32, 9, 8), (512, 16, 5, 8),
    (1024, 32, 7, 8), (160, 8, 3, 6)])
def test_route_groups_with_any_bias(experts, groups, topk_groups, k, gpu, torch):  # noqa: F811
    """A group's value is the sum of its two best s + b whatever the size of the biases."""
    for i, (name, bias) in enumerate(biases(experts, groups).items()):
        x = logits(torch, 70, experts, TYPES[i % 3], experts + i, 1.5)
        x[0] = 0.0
        x[1, ::3] = -float("inf")
        for score in ("sigmoid", "softmax"):
            for rule in ("top2", "max"):
                check_route(torch, gpu, x, k, bias=bias, score=score, groups=groups,
                            topk_groups=topk_groups, group_rule=rule, renormalize=i % 2 == 0)


def test_route_any_bias_without_groups(gpu, torch):  # noqa: F811
    for experts in (64, 128, 256, 1024):
        for i, bias in enumerate(biases(experts, 8).values()):
            x = logits(torch, 70, experts, TYPES[i % 3], experts + i, 1.5)
            for score in ("sigmoid", "softmax"):
                check_route(torch, gpu, x, 8, bias=bias, score=score)


@pytest.mark.parametrize("experts", [8, 64, 255, 256, 257, 512, 1000, 1024])
def test_route_last_expert_far_below(experts, gpu, torch):  # noqa: F811
    """An expert that can be chosen is chosen, the last one and one of the lowest choice value
    among them: -1 stands only where none is left."""
    for last in (-5.0, -4.6, -1e9, -3e38):
        bias = np.zeros(experts, np.float32)
        bias[-1] = last
        x = logits(torch, 4, experts, "float32", experts)
        x[0, :-1] = -float("inf")
        x[1, 2:-1] = -float("inf")
        x[2, 1:] = -float("inf")
        x[2, -1] = 0.5
        for score in ("sigmoid", "softmax"):
            for k in (1, 4, 8):
                got = check_route(torch, gpu, x, k, bias=bias, score=score)
                assert got[0][0, 0] == experts - 1
                check_route(torch, gpu, x, k, bias=np.full(experts, last, np.float32), score=score)


# ---- plan: places near 2^31 -------------------------------------------------------------------------

def test_plan_padding_up_to_the_last_place(gpu, torch):  # noqa: F811
    """Segments that end at place 2^31 - 1 or next to it: the padding is -1 to its end, in one
    block's plan (a single pair) and in a large one (2^30 pairs)."""
    for pairs, align in ((1, 2 ** 31 - 1), (2 ** 30, 2 ** 30 - 1)):
        capacity = pairs + align - 1
        ids = torch.zeros(pairs, dtype=torch.int32, device="cuda")
        offsets = torch.empty(2, dtype=torch.int32, device="cuda")
        order = torch.full((capacity,), 7, dtype=torch.int32, device="cuda")
        position = torch.empty_like(ids)
        gpu.route_plan(ids, 1, offsets, order, position, align=align, stream=0)
        end = -(-pairs // align) * align
        assert end == capacity and offsets.tolist() == [0, end]
        assert torch.equal(order[:pairs], torch.arange(pairs, dtype=torch.int32, device="cuda"))
        assert torch.equal(position, order[:pairs])
        assert (order[pairs:] == -1).all()
        del ids, order, position
        torch.cuda.empty_cache()


# ---- gradient: what is not finite ------------------------------------------------------------------

@pytest.mark.parametrize("experts", [24, 64, 100, 256, 1000])
def test_gradient_of_masked_stays_zero(experts, gpu, torch):  # noqa: F811
    """A gradient that overflowed (inf or NaN at an expert that takes part) leaves masked experts
    at 0: they have no part in the scores."""
    for dtype in TYPES:
        x = logits(torch, 9, experts, dtype, experts)
        x[:, 1::4] = -float("inf")
        x[:, 2::4] = float("nan")
        masked = ~(x > -float("inf")).cpu().numpy()
        xs = x.double().cpu().numpy()
        for score in ("softmax", "sigmoid"):
            for renormalize in (True, False):
                ids = ref.route(xs, 4, score=score)[0]
                for bad in (np.inf, -np.inf, np.nan):
                    for where in ("weights", "scores"):
                        dw = np.ones((9, 4), np.float32)
                        ds = np.ones((9, experts), np.float32)
                        if where == "weights":
                            dw[:, 1] = bad
                        else:
                            ds[:, 0] = bad
                        for dense in (True, False):
                            got = run_backward(torch, gpu, x, ids, dw, ds if dense else None,
                                               score=score, renormalize=renormalize, scale=1.0)
                            assert (got[masked] == 0).all(), (score, renormalize, bad, where)


@pytest.mark.parametrize("experts", [24, 64, 100, 128, 256, 500, 1024])
def test_gradient_in_place_every_form(experts, gpu, torch):  # noqa: F811
    """Written over the logits, the gradient is the one that is written beside them, whether the
    call reads whole rows or the chosen experts only."""
    for dtype in TYPES:
        for tokens in (1, 77, 3001):
            x = logits(torch, tokens, experts, dtype, experts + tokens)
            rng = np.random.default_rng(tokens)
            ids = torch.topk(x.float(), 4).indices.int()
            dw = torch.from_numpy(rng.standard_normal((tokens, 4)).astype(np.float32)).cuda()
            ds = torch.from_numpy(rng.standard_normal((tokens, experts)).astype(np.float32)).cuda()
            for score in ("softmax", "sigmoid"):
                for renormalize in (True, False):
                    for dscores in (None, ds):
                        how = dict(score=score, renormalize=renormalize, dscores=dscores, stream=0)
                        want = torch.empty_like(x)
                        gpu.route_topk_backward(x, ids, dw, want, **how)
                        got = x.clone()
                        gpu.route_topk_backward(got, ids, dw, got, **how)
                        torch.cuda.synchronize()
                        assert torch.equal(got, want), (dtype, tokens, score, renormalize)
