"""Row operators on the GPU where a kernel's shortcut could show: biases of any size, ids at the
ends of a packed key, gradients that are not finite, weights and scores held to the accuracy that
is stated for them, places near 2^31."""

import numpy as np
import pytest

from tests import rows_reference as ref
from tests.test_gpu_rows import (  # noqa: F401
    TINY, TYPES, check_route, check_sample, logits, run_backward, run_sample, torch)

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of fp32


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


# ---- accuracy of scores, weights and gradients -----------------------------------------------------

def far_logits(torch, tokens, experts, seed):  # noqa: F811
    """fp32 logits on a grid of 1/64 within +-60: every difference of two is exact in fp32."""
    v = np.random.default_rng(seed).integers(-60 * 64, 60 * 64, (tokens, experts)) / 64.0
    return torch.from_numpy(v.astype(np.float32)).cuda()


@pytest.mark.parametrize("experts", [16, 64, 128, 256, 512, 1024])
def test_scores_far_from_the_largest(experts, gpu, torch):  # noqa: F811
    """A score's relative error does not grow with its logit. In units of 2^-24: an exponential of
    an exact argument 9 (the power of two 4, one rounding, and 0.05 a unit of the argument, up to 87
    of them), its sum over E experts E / 32 additions in a lane, 8 at least, and 5 between lanes, a
    reciprocal 2, each product, quotient or addition 1. A softmax score: 9 + (9 + E / 32 + 5) + 2 + 1;
    a sigmoid e / (1 + e): 9, half of them and 1 more below, 2, 1. A weight over the sum of the
    chosen: a relative score (an exponential of 9 and one of 4, their sum, a reciprocal: 12 at most),
    12 + 9 of the sum, a reciprocal 2, two products. (Exponentials of rounded arguments, x log2 e in
    fp32, are off by some 60 at the far end.)"""
    x = far_logits(torch, 200, experts, experts)
    xs = x.double().cpu().numpy()
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            ids = torch.empty(200, 6, dtype=torch.int32, device="cuda")
            w = torch.empty(200, 6, device="cuda")
            s = torch.empty(200, experts, device="cuda")
            gpu.route_topk(x, ids, w, score=score, renormalize=renormalize, scores=s, stream=0)
            want = ref.route(xs, 6, score=score, renormalize=renormalize)
            assert np.array_equal(ids.cpu().numpy(), want[0])
            per = 8 if experts <= 256 else experts / 32
            tol = (9 + 9 + per + 5 + 2 + 1 if score == "softmax" else 9 + 4.5 + 1 + 2 + 1) * U
            got = s.double().cpu().numpy()
            assert np.all(np.abs(got - want[2]) <= tol * want[2] + TINY), (score, "scores")
            if renormalize:
                tol = (12 + 12 + 9 + 2 + 2) * U
            got = w.double().cpu().numpy()
            assert np.all(np.abs(got - want[1]) <= (tol + U) * want[1] + TINY), (score, "weights")


def far_gradient(x, ids, dw, ds, score, renormalize):
    """(gradient, magnitudes added up for it) of rows without masks, 1 - s taken as 1 / (1 + e^x):
    from a logit of 37 on, 1 - s itself has no digit left in 64 bits."""
    s = np.stack([ref.scores_row(row, score) for row in x])
    rest = 1.0 / (1.0 + np.exp(x)) if score == "sigmoid" else np.ones_like(x)
    part = np.stack([ref.ratio_row(row, i, score) for row, i in zip(x, ids)])
    if not renormalize:
        part = np.take_along_axis(s, ids.astype(np.int64), 1)
    own, mag = part * dw, part * np.abs(dw)
    if renormalize:
        own, mag = part * (dw - own.sum(1, keepdims=True)), mag + part * mag.sum(1, keepdims=True)
    grad, size = s * ds * rest, s * np.abs(ds) * rest
    at = np.arange(len(x))[:, None]
    if score == "softmax":
        total, most = (s * ds).sum(1, keepdims=True), (s * np.abs(ds)).sum(1, keepdims=True)
        if not renormalize:
            total, most = total + own.sum(1, keepdims=True), most + mag.sum(1, keepdims=True)
        grad, size = grad - s * total, size + s * most
    grad[at, ids] += own * rest[at, ids]
    size[at, ids] += mag * rest[at, ids]
    return grad, size


@pytest.mark.parametrize("experts", [16, 64, 256, 1024])
def test_gradient_far_from_the_largest(experts, gpu, torch):  # noqa: F811
    """The same of the gradient's terms: a score (softmax 26 + E / 32, sigmoid 18) or a ratio of
    the chosen (37), 1 - s (18), a sum of products over the experts (E / 32 + 5 additions, a
    product and a score each), three more products and sums, in units of 2^-24 of the magnitudes
    added up."""
    x = far_logits(torch, 60, experts, experts + 1)
    xs = x.double().cpu().numpy()
    rng = np.random.default_rng(experts)
    dw = rng.standard_normal((60, 5)).astype(np.float32)
    ds = rng.standard_normal((60, experts)).astype(np.float32)
    per = 8 if experts <= 256 else experts / 32
    for score in ("softmax", "sigmoid"):
        ids = ref.route(xs, 5, score=score)[0]
        for renormalize in (True, False):
            for dense in (True, False):
                d = ds if dense else None
                how = dict(score=score, renormalize=renormalize, scale=1.0)
                got = run_backward(torch, gpu, x, ids, dw, d, **how)
                want, size = far_gradient(xs, ids, dw.astype(np.float64), ds.astype(np.float64)
                                          * dense, score, renormalize)
                one = max(26 + per, 37)
                tol = (one + 18 + (per + 5 + 1 + one) + 6) * U
                assert np.all(np.abs(got - want) <= tol * size + TINY), (score, renormalize, dense)


# ---- accuracy of a draw's weights ------------------------------------------------------------------

def borders(lowest, highest, count=1 << 23):
    """Scores x (fp32, beside a score of 0) and uniforms u = j / 2^24 whose distance from
    w / (w + 1), w = exp(x), lies between the two powers of two; and which side u is on. In 80-bit
    arithmetic, whose 2^-63 is far below the distances."""
    x = (-3 * np.random.default_rng(9).random(count, dtype=np.float32)).astype(np.float32)
    w = np.exp(x.astype(np.longdouble))
    f = w / (w + 1)
    j = np.rint(f * 2 ** 24)
    off = np.abs(f - j / np.longdouble(2 ** 24))
    at = np.flatnonzero((off > 2.0 ** lowest) & (off < 2.0 ** highest))
    return x[at], (j[at] / 2 ** 24).astype(np.float32), (f[at] <= j[at] / 2 ** 24).astype(np.int64)


def test_draws_next_to_a_border(gpu, torch):  # noqa: F811
    """Weights are exact to their grid: 2^-50 of the largest up to 4,096 columns, and a draw's
    border is off by no more. Two columns' w / (w + 1) is off by what w is off, so a border 2^-48
    away has to be seen from its right side. (A weight good to 2^-38 sees most of them from
    either.)"""
    assert np.finfo(np.longdouble).nmant >= 63
    x, u, want = borders(-48, -41)
    assert len(x) > 30 and 5 < want.sum() < len(x) - 5
    rows = torch.zeros(len(x), 2, device="cuda")
    rows[:, 0] = torch.from_numpy(x)
    ids = run_sample(torch, gpu, rows, u[:, None])[0][:, 0]
    assert np.array_equal(ids, want)
    # the same two columns far apart in a long row of nothing else: a cluster of blocks, and a grid
    # of 2^-47 of the largest
    x, u, want = borders(-45, -39)
    assert len(x) > 100
    rows = torch.full((len(x), 30000), -float("inf"), device="cuda")
    rows[:, 77] = torch.from_numpy(x)
    rows[:, 29000] = 0.0
    for part in range(0, len(x), 40):  # not a batch that one block a row takes
        ids = run_sample(torch, gpu, rows[part:part + 40], u[part:part + 40, None])[0][:, 0]
        assert np.array_equal(ids, np.where(want[part:part + 40] == 0, 77, 29000))


def test_top_p_over_blocks_of_equal_scores(gpu, torch):  # noqa: F811
    """A long row whose first part is one score, so often that its parts in the histogram that
    brackets the edge come near 2^32: the edge, among the different scores behind, is right, and
    is found by its bracket. That shows in the time alone: by the long way a row takes twice as
    long, so that the least of several times is compared with that of a row 1 % shorter whose parts
    stay clear of 2^32 however they are rounded."""
    how = dict(top_p=[0.999, 0.99997])
    times = {}
    for cols in (540000, 544001, 584011, 592013):
        x = logits(torch, 2, cols, "float32", cols, 1.0)
        x[:, :cols // 8 + 8] = 6.0
        u = np.array([[0.01, 0.5, 0.93, 0.99999]] * 2, np.float32)
        check_sample(torch, gpu, x, u, **how)
        top_p = torch.tensor(how["top_p"], device="cuda")
        ud, ids = torch.from_numpy(u).cuda(), torch.empty(2, 4, dtype=torch.int64, device="cuda")
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        least = []
        for _ in range(10):
            a.record()
            gpu.sample_rows(x, ud, ids, top_p=top_p, stream=0)
            b.record()
            torch.cuda.synchronize()
            least.append(a.elapsed_time(b))
        times[cols] = min(least)
    assert all(t < 1.5 * times[540000] for t in times.values()), times


# ---- outputs over inputs ---------------------------------------------------------------------------

def test_outputs_over_inputs_are_refused(ovvs, gpu, torch):  # noqa: F811
    x = logits(torch, 6, 64, "float32", 1)
    u = torch.rand(6, 2, device="cuda")
    i64 = torch.empty(6, 2, dtype=torch.int64, device="cuda")
    kept = torch.full((6,), 3, dtype=torch.int32, device="cuda")
    ids = torch.topk(x, 4).indices.int()
    w = torch.rand(6, 4, device="cuda")
    before = [t.clone() for t in (x, u, ids, w)]
    cut = [t.flatten()[:n].view(s) for t, n, s in ((x, 12, (6, 2)), (x, 24, (6, 4)))]
    plan = torch.empty(65, dtype=torch.int32, device="cuda")
    order = torch.empty(24, dtype=torch.int32, device="cuda")
    calls = [
        lambda: gpu.sample_rows(x, u, i64, probs=u, stream=0),
        lambda: gpu.sample_rows(x, u, i64, probs=cut[0], stream=0),
        lambda: gpu.sample_rows(x, u, i64, kept=kept, top_k=kept, stream=0),
        lambda: gpu.route_topk(x, ids, w, scores=x, stream=0),
        lambda: gpu.route_topk(x, ids, ids.view(torch.float32), stream=0),
        lambda: gpu.route_topk(x, ids, cut[1], stream=0),
        lambda: gpu.route_topk_backward(x[:5], ids[:5], w[:5], x[1:], stream=0),
        lambda: gpu.route_topk_backward(x, ids, w, x.flatten()[:192].view(6, 32)
                                        .as_strided((6, 64), (64, 1), 0), dscores=x, stream=0),
        lambda: gpu.route_plan(ids, 64, plan, order, ids, stream=0),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(ovvs.OvvsError, match="invalid argument"):
            call()
            pytest.fail(f"call {i} was not refused")
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, (x, u, ids, w)))


def test_column_ranges_of_one_buffer_are_taken(gpu, torch):  # noqa: F811
    """Logits and their gradient side by side in one buffer share no byte."""
    buf = logits(torch, 9, 150, "bfloat16", 2)
    x, out = buf[:, :64], buf[:, 70:134]
    ids = torch.topk(x.float(), 4).indices.int()
    dw = torch.rand(9, 4, device="cuda")
    want = torch.empty_like(x, memory_format=torch.contiguous_format)
    gpu.route_topk_backward(x, ids, dw, want, stream=0)
    gpu.route_topk_backward(x, ids, dw, out, stream=0)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
