"""Row operators on the GPU against their plain 64-bit implementations: draws, routing, its
gradient and the grouping plan.

Whole numbers (ids, kept counts, plans) have to be equal. Tolerances of the rest:
- a drawn probability is the quotient of two integers, rounded once to fp32 (2^-24), of weights
  held to 2^-44 of the row's largest (64-bit integers, frac >= 42 bits at the sizes here, and an
  exponential good to some 2^-43): 2^-23 relative + 2^-40 absolute;
- fp32 exponentials of arguments up to D have a relative error of at most (2 D + 8) 2^-24, and a
  sum over E of them adds (E / 32 + 5) 2^-24: scores, weights and the terms of a gradient are held
  to (4 D + E / 16 + 64) 2^-24 of their own size, a gradient to that times the sum of the
  magnitudes added up for it, plus half a step of the type that it is rounded to.
"""

import numpy as np
import pytest

from tests import rows_reference as ref

pytestmark = pytest.mark.gpu

TYPES = ["float32", "float16", "bfloat16"]
TINY = 1e-37  # below it fp32 results may be subnormal


@pytest.fixture(scope="module")
def torch():
    import torch

    return torch


def guarded(torch, shape, dtype, fill):
    """A tensor inside a larger one, and a check that nothing beside it was written."""
    n = int(np.prod(shape))
    buf = torch.full((n + 128,), fill, dtype=dtype, device="cuda")
    view = buf[64:64 + n].view(shape)

    def untouched():
        torch.cuda.synchronize()
        assert (buf[:64] == fill).all() and (buf[64 + n:] == fill).all(), "written out of range"

    return view, untouched


def run_sample(torch, gpu, x, u, temperature=None, top_k=None, top_p=None, min_p=None, stream=0):
    rows = x.shape[0]
    ids, ok1 = guarded(torch, u.shape, torch.int64, -77)
    probs, ok2 = guarded(torch, u.shape, torch.float32, -77.0)
    kept, ok3 = guarded(torch, (rows,), torch.int32, -77)
    put = lambda a, t: None if a is None else torch.tensor(np.asarray(a), dtype=t, device="cuda")  # noqa: E731
    gpu.sample_rows(x, torch.from_numpy(u).cuda(), ids, probs=probs, kept=kept,
                    temperature=put(temperature, torch.float32),
                    top_k=put(top_k, torch.int32), top_p=put(top_p, torch.float32),
                    min_p=put(min_p, torch.float32), stream=stream)
    for ok in (ok1, ok2, ok3):
        ok()
    return ids.cpu().numpy(), probs.cpu().numpy(), kept.cpu().numpy()


def f32(a):
    return None if a is None else np.asarray(a, np.float32)


def check_sample(torch, gpu, x, u, **how):
    got = run_sample(torch, gpu, x, u, **how)
    how = {k: (v if k == "top_k" else f32(v)) for k, v in how.items() if k != "stream"}
    want = ref.sample(x.double().cpu().numpy(), u.reshape(len(u), -1), **how)
    assert np.array_equal(got[2], want[2]), ("kept", got[2], want[2])
    assert np.array_equal(got[0].reshape(len(u), -1), want[0]), "ids"
    p = got[1].reshape(len(u), -1)
    assert np.all(np.abs(p - want[1]) <= 2.0 ** -23 * want[1] + 2.0 ** -40), "probabilities"


def logits(torch, rows, cols, dtype, seed, spread=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(rows, cols, generator=g, device="cuda") * spread).to(getattr(torch, dtype))


def uniforms(seed, *shape):
    return np.random.default_rng(seed).random(shape, dtype=np.float32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [1, 2, 7, 31, 32, 33, 257, 1000, 4099, 20011, 65537])
def test_sample_settings(dtype, cols, gpu, torch):
    """Every setting alone and together, per row, at odd sizes."""
    x = logits(torch, 24, cols, dtype, cols)
    u = uniforms(cols, 24, 3)
    rng = np.random.default_rng(cols)
    t = rng.uniform(0.3, 2.0, 24)
    k = np.array([0, 1, 2, 5, 40, cols, cols + 1, max(1, cols // 2)] * 3)
    p = np.repeat([1.0, 0.9, 0.4], 8)
    q = np.array([0.0, 0.05, 0.0] * 8)
    check_sample(torch, gpu, x, u)
    check_sample(torch, gpu, x, u, temperature=t)
    check_sample(torch, gpu, x, u, top_k=k)
    check_sample(torch, gpu, x, u, top_p=p)
    check_sample(torch, gpu, x, u, min_p=q)
    check_sample(torch, gpu, x, u, temperature=t, top_k=k, top_p=p, min_p=q)


@pytest.mark.parametrize("dtype", TYPES)
def test_sample_long_rows(dtype, gpu, torch):
    """Rows beyond what a group of blocks can hold on chip, and one near the usual vocabularies."""
    for cols, rows in ((131072, 3), (1_000_003, 2), (3_000_017, 1)):
        x = logits(torch, rows, cols, dtype, 11)
        u = uniforms(12, rows, 5)
        check_sample(torch, gpu, x, u)
        check_sample(torch, gpu, x, u, temperature=[0.7] * rows, top_k=[300] * rows,
                     top_p=[0.9] * rows)
        check_sample(torch, gpu, x, u, top_p=[0.95] * rows, min_p=[1e-4] * rows)


@pytest.mark.parametrize("rows", [1, 2, 3, 17, 37, 150, 400])
def test_sample_row_counts(rows, gpu, torch):
    x = logits(torch, rows, 9001, "bfloat16", rows)
    check_sample(torch, gpu, x, uniforms(rows, rows), top_p=[0.8] * rows)
    check_sample(torch, gpu, x, uniforms(rows, rows), top_k=[30] * rows, top_p=[0.9] * rows)


def test_sample_ties(gpu, torch):
    """Few distinct scores: the edge falls among equal ones, of which the lower columns stay."""
    for cols in (40, 1000, 30000):
        x = (logits(torch, 16, cols, "float32", 3, 1.0)).round()
        u = uniforms(4, 16, 9)
        k = np.arange(1, 17) * max(1, cols // 20)
        check_sample(torch, gpu, x, u, top_k=k)
        check_sample(torch, gpu, x, u, top_p=np.linspace(0.02, 0.999, 16))
        check_sample(torch, gpu, x, u, top_k=k, top_p=np.linspace(0.3, 0.999, 16))
        check_sample(torch, gpu, torch.zeros_like(x), u, top_p=[0.5] * 16)
        check_sample(torch, gpu, torch.zeros_like(x), u, top_k=k, top_p=[0.25] * 16)
        flat = torch.zeros_like(x)
        flat[:, ::2] = -0.0  # equal to +0
        check_sample(torch, gpu, flat, u, top_k=k)


def test_sample_near_equal_scores(gpu, torch):
    """Scores that differ in their last bits only: one narrow range holds the whole row."""
    cols = 20000
    steps = torch.randint(0, 5000, (4, cols), generator=torch.Generator().manual_seed(1))
    x = (torch.full((4, cols), 8.0).view(torch.int32) + steps.int()).view(torch.float32).cuda()
    u = uniforms(5, 4, 6)
    check_sample(torch, gpu, x, u, top_k=[1, 10, 777, 15000])
    check_sample(torch, gpu, x, u, top_p=[0.1, 0.5, 0.77, 0.999])
    check_sample(torch, gpu, x, u, top_p=[0.1, 0.5, 0.77, 0.999], temperature=[1e-6] * 4)
    check_sample(torch, gpu, x, u, top_k=[1, 10, 777, 15000], temperature=[1e-3] * 4)


@pytest.mark.parametrize("dtype", TYPES)
def test_sample_masked(dtype, gpu, torch):
    lowest = torch.finfo(getattr(torch, dtype)).min
    for cols in (5, 300, 40000):
        x = logits(torch, 10, cols, dtype, 21)
        x[0] = -float("inf")
        x[1] = float("nan")
        x[2, 1:] = -float("inf")
        x[3, ::2] = -float("inf")
        x[4, ::2] = float("nan")
        x[4, 1::4] = -float("inf")
        x[5, ::2] = lowest
        x[6] = lowest
        x[7, 3] = float("inf")
        x[8, 1:4] = float("inf")
        x[9, :] = -float("inf")
        x[9, -1] = lowest
        u = uniforms(22, 10, 4)
        check_sample(torch, gpu, x, u)
        check_sample(torch, gpu, x, u, top_k=[4] * 10)
        check_sample(torch, gpu, x, u, top_p=[0.7] * 10)
        check_sample(torch, gpu, x, u, top_k=[cols // 2 + 1] * 10, top_p=[0.9] * 10,
                     min_p=[0.01] * 10)
        check_sample(torch, gpu, x, u, temperature=[0.0] * 10)


@pytest.mark.parametrize("dtype", TYPES)
def test_sample_masked_stretches(dtype, gpu, torch):
    """Long stretches of NaN and of -inf, in batches of each size class; what stands between them
    is little, or together in one place, or in order."""
    for rows, cols in ((300, 9001), (5, 40003)):
        x = logits(torch, rows, cols, dtype, 23)
        x[::2, 100:cols - 3000] = float("nan")
        x[1::2, :cols - 50] = -float("inf")
        x[2::5] = x[2::5].sort(1).values
        x[3::5] = x[3::5].sort(1, descending=True).values
        u = uniforms(24, rows, 2)
        check_sample(torch, gpu, x, u, top_k=[40] * rows)
        check_sample(torch, gpu, x, u, top_k=[40] * rows, top_p=[0.8] * rows)
        check_sample(torch, gpu, x, u, top_p=[0.95] * rows)


def test_sample_batch_of_many_kinds(gpu, torch):
    """One large batch whose rows take every way: greedy, small and large top-k, top-p alone,
    nothing, ties, all masked."""
    rows, cols = 320, 7001
    x = logits(torch, rows, cols, "float32", 25)
    x[5::16] = x[5::16].round()
    x[6::16] = 0.0
    x[7::16] = -float("inf")
    i = np.arange(rows)
    check_sample(torch, gpu, x, uniforms(26, rows, 3),
                 temperature=np.where(i % 8 == 0, 0.0, 0.5 + i % 5 * 0.4),
                 top_k=np.array([0, 1, 50, 447, 448, 449, 2500, cols])[i // 2 % 8],
                 top_p=np.array([1.0, 0.9, 0.3, 1.0, 0.99])[i % 5],
                 min_p=np.array([0.0, 0.0, 0.02])[i % 3])


def test_sample_odd_settings(gpu, torch):
    """Settings outside their ranges mean what the header says."""
    inf, nan = float("inf"), float("nan")
    x = logits(torch, 12, 3001, "float32", 31)
    u = uniforms(32, 12, 4)
    u[:, 0] = 0.0
    u[:, 1] = np.float32(1 - 2.0 ** -24)
    u[:6, 2] = [1.0, nan, -3.0, inf, -inf, 2.0]
    check_sample(torch, gpu, x, u, temperature=[0.0, -1.0, nan, inf, 1e-30, 1e30, 1e-3, 100.0,
                                                1.0, 1.0, 1e-45, 3e38])
    check_sample(torch, gpu, x, u, top_k=[0, -1, -2 ** 31, 2 ** 31 - 1, 1, 2, 3000, 3001, 3002,
                                          1500, 7, 100])
    check_sample(torch, gpu, x, u, top_p=[0.0, -1.0, nan, inf, -inf, 1.0, 2.0, 1e-30, 1e-6,
                                          0.9999, 0.99999994, 0.5])
    check_sample(torch, gpu, x, u, min_p=[0.0, -1.0, nan, inf, -inf, 1.0, 2.0, 1e-30, 1e-6,
                                          0.9999, 0.99999994, 0.5])
    check_sample(torch, gpu, x, u, temperature=[inf] * 12, top_k=[9] * 12,
                 top_p=np.linspace(0.05, 1.0, 12), min_p=[1.0] * 12)
    check_sample(torch, gpu, x, u, temperature=[1e-4] * 12, top_k=[50] * 12,
                 top_p=np.linspace(0.05, 1.0, 12))


def test_sample_many_draws(gpu, torch):
    for cols in (100, 50000):
        x = logits(torch, 5, cols, "float32", 41)
        check_sample(torch, gpu, x, uniforms(42, 5, 1000))
        check_sample(torch, gpu, x, uniforms(42, 5, 1000), top_k=[1, 20, 99, 3000, 0])
        check_sample(torch, gpu, x, uniforms(42, 5, 513), top_p=[0.999] * 5)


@pytest.mark.parametrize("dtype", TYPES)
def test_sample_strides_and_alignment(dtype, gpu, torch):
    base = logits(torch, 7, 5003, dtype, 51)
    u = uniforms(52, 7, 2)
    for first, cols in ((0, 5003), (1, 5000), (3, 4097), (5, 33), (2, 1)):
        x = base[:, first:first + cols]  # rows start anywhere, stride 5003
        check_sample(torch, gpu, x, u)
        check_sample(torch, gpu, x, u, top_k=[12] * 7, top_p=[0.9] * 7)
    check_sample(torch, gpu, base[::3], u[::3], top_k=[12] * 3)


def test_sample_large_offsets(gpu, torch):
    """Rows whose elements lie beyond 2^31 elements from the base."""
    ld = (1 << 30) + 8
    x = torch.empty(4 * ld, dtype=torch.bfloat16, device="cuda").as_strided((4, 1000), (ld, 1))
    x.copy_(logits(torch, 4, 1000, "bfloat16", 61))
    check_sample(torch, gpu, x, uniforms(62, 4, 3), top_p=[0.9] * 4)


def test_sample_repeats_bit_for_bit(gpu, torch):
    x = logits(torch, 64, 30011, "bfloat16", 71)
    u = uniforms(72, 64, 8)
    first = run_sample(torch, gpu, x, u, top_p=[0.93] * 64)
    for _ in range(5):
        again = run_sample(torch, gpu, x, u, top_p=[0.93] * 64)
        assert all(np.array_equal(a, b) for a, b in zip(first, again))


def test_sample_frequencies(gpu, torch):
    """Draws follow the kept probabilities: 200,000 uniforms spread evenly over [0, 1) hit each
    column within one draw at each of its two edges."""
    x = logits(torch, 1, 50, "float32", 81, 1.0)
    n = 200_000
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)[None]
    ids = run_sample(torch, gpu, x, u, top_k=[20])[0][0]
    w = np.exp(x[0].double().cpu().numpy())
    keep = ref.in_order(x[0].double().cpu().numpy())[:20]
    p = np.zeros(50)
    p[keep] = w[keep] / w[keep].sum()
    assert np.all(np.abs(np.bincount(ids, minlength=50) - n * p) <= 2)


# ---- routing -------------------------------------------------------------------------------------

def spread_of(x, score):
    v = np.where(np.isfinite(x), x, 0.0)
    if score == "sigmoid":
        return np.abs(v).max(1, keepdims=True)
    return v.max(1, keepdims=True) - v.min(1, keepdims=True)


def tolerance(x, score):
    return (4 * np.minimum(spread_of(x, score), 256.0) + x.shape[1] / 16 + 64) * 2.0 ** -24


def run_route(torch, gpu, x, k, bias=None, scores=True, stream=0, **how):
    t, n = x.shape
    ids, ok1 = guarded(torch, (t, k), torch.int32, -77)
    w, ok2 = guarded(torch, (t, k), torch.float32, -77.0)
    s, ok3 = guarded(torch, (t, n), torch.float32, -77.0)
    gpu.route_topk(x, ids, w, bias=None if bias is None else torch.from_numpy(bias).cuda(),
                   scores=s if scores else None, stream=stream, **how)
    for ok in (ok1, ok2, ok3):
        ok()
    return ids.cpu().numpy(), w.cpu().numpy(), s.cpu().numpy()


def check_route(torch, gpu, x, k, bias=None, scores=True, **how):
    got = run_route(torch, gpu, x, k, bias=bias, scores=scores, **how)
    xs = x.double().cpu().numpy()
    want = ref.route(xs, k, bias=None if bias is None else bias.astype(np.float64), **how)
    assert np.array_equal(got[0], want[0]), "ids"
    tol = tolerance(xs, how.get("score", "softmax"))
    assert np.all(np.abs(got[1] - want[1]) <= tol * np.abs(want[1]) + TINY), "weights"
    if scores:
        assert np.all(np.abs(got[2] - want[2]) <= tol * want[2] + TINY), "scores"
    return got


ROUTES = [
    dict(),
    dict(renormalize=False),
    dict(score="sigmoid", scale=2.5),
    dict(score="sigmoid", renormalize=False),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("experts", [1, 2, 8, 31, 32, 33, 60, 64, 128, 160, 256, 257, 512, 1000,
                                     1024])
def test_route_plain(dtype, experts, gpu, torch):
    for tokens in (1, 5, 129):
        x = logits(torch, tokens, experts, dtype, experts + tokens, 1.5)
        for i, how in enumerate(ROUTES):
            for k in sorted({1, min(6, experts), min(32, experts)}):
                check_route(torch, gpu, x, k, scores=i % 2 == 0, **how)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("experts,groups,topk_groups,k", [
    (256, 8, 4, 8), (64, 8, 3, 6), (160, 8, 3, 6), (60, 4, 2, 4), (32, 32, 5, 5), (8, 4, 1, 2),
    (1024, 32, 7, 32), (512, 16, 16, 9), (7, 7, 3, 2), (96, 3, 2, 12), (256, 1, 1, 8)])
def test_route_groups_and_bias(dtype, experts, groups, topk_groups, k, gpu, torch):
    x = logits(torch, 200, experts, dtype, experts, 1.5)
    bias = np.random.default_rng(experts).normal(0, 0.1, experts).astype(np.float32)
    for score in ("softmax", "sigmoid"):
        for rule in ("max", "top2"):
            for b in (None, bias):
                check_route(torch, gpu, x, k, bias=b, score=score, groups=groups,
                            topk_groups=topk_groups, group_rule=rule, scale=2.5,
                            renormalize=rule == "top2")


def test_route_near_ties(gpu, torch):
    """Biases that bring many experts within a few 2^-24 of one another, and exact ties: the
    choice is the one of 64 bits, equal ones by lower id."""
    rng = np.random.default_rng(7)
    for score in ("sigmoid", "softmax"):
        for experts in (64, 256):
            row = rng.standard_normal(experts).astype(np.float32)
            s = ref.scores_row(row.astype(np.float64), score)
            bias = (0.5 - s).astype(np.float32)  # s + bias is 0.5 to within one rounding
            x = torch.from_numpy(np.tile(row, (64, 1))).cuda()
            check_route(torch, gpu, x, 8, bias=bias, score=score)
            check_route(torch, gpu, x, 8, bias=bias, score=score, groups=8, topk_groups=3,
                        group_rule="top2")
            x[1:] += torch.randn(63, experts, device="cuda",
                                 generator=torch.Generator(device="cuda").manual_seed(1)) * 2e-7
            check_route(torch, gpu, x, 8, bias=bias, score=score)
            check_route(torch, gpu, x, 8, bias=bias, score=score, groups=8, topk_groups=3)
    level = torch.randint(0, 3, (100, 64), device="cuda").float()
    for bias in (None, np.zeros(64, np.float32)):
        for how in (dict(), dict(groups=8, topk_groups=3, group_rule="top2"),
                    dict(groups=8, topk_groups=3)):
            check_route(torch, gpu, level, 9, bias=bias, score="sigmoid", **how)
            check_route(torch, gpu, level, 9, bias=bias, **how)
    check_route(torch, gpu, torch.zeros(3, 256, device="cuda"), 32)


@pytest.mark.parametrize("dtype", TYPES)
def test_route_masked(dtype, gpu, torch):
    lowest = torch.finfo(getattr(torch, dtype)).min
    bias = np.random.default_rng(9).normal(0, 0.1, 64).astype(np.float32)
    blocked = bias.copy()
    blocked[::3] = -np.inf
    blocked[1] = np.nan
    x = logits(torch, 9, 64, dtype, 91)
    x[0] = -float("inf")
    x[1] = float("nan")
    x[2, 3:] = -float("inf")
    x[3, ::2] = float("nan")
    x[4, ::2] = lowest
    x[5] = lowest
    x[6, 3] = float("inf")
    x[7, 1:4] = float("inf")
    x[8, 8:] = -float("inf")  # one group of eight is left
    for score in ("softmax", "sigmoid"):
        for b in (None, bias, blocked):
            for renormalize in (True, False):
                how = dict(score=score, renormalize=renormalize)
                check_route(torch, gpu, x, 6, bias=b, **how)
                check_route(torch, gpu, x, 10, bias=b, groups=8, topk_groups=2, **how)
                check_route(torch, gpu, x, 10, bias=b, groups=8, topk_groups=2,
                            group_rule="top2", **how)


def test_route_far_logits(gpu, torch):
    """Scores that vanish, or saturate, in 32 bits: the renormalised weights stay ratios."""
    x = logits(torch, 6, 32, "float32", 95, 1.0)
    x[0] -= 200.0
    x[1] -= 90.0
    x[2] += 200.0
    x[3] *= 40.0
    x[4, :16] -= 120.0
    x[4, 16:] = -float("inf")
    for score in ("softmax", "sigmoid"):
        got = run_route(torch, gpu, x, 4, score=score)
        want = ref.route(x.double().cpu().numpy(), 4, score=score)
        assert np.array_equal(got[0], want[0])
        tol = tolerance(x.double().cpu().numpy(), score)
        assert np.all(np.abs(got[1] - want[1]) <= tol * want[1] + TINY)


@pytest.mark.parametrize("dtype", TYPES)
def test_route_strides(dtype, gpu, torch):
    base = logits(torch, 40, 131, dtype, 97)
    for first, n in ((0, 131), (1, 128), (3, 64), (2, 8), (5, 1)):
        x = base[:, first:first + n]
        check_route(torch, gpu, x, min(3, n))
        check_backward(torch, gpu, x, min(3, n), "sigmoid", True, True, pad=3)
    check_route(torch, gpu, base[::7], 5)


# ---- gradient ------------------------------------------------------------------------------------

def run_backward(torch, gpu, x, ids, dw, ds, pad=0, stream=0, **how):
    t, n = x.shape
    wide, ok = guarded(torch, (t, n + pad), x.dtype, -77.0)
    out = wide[:, :n]
    gpu.route_topk_backward(x, torch.from_numpy(ids).cuda(), torch.from_numpy(dw).cuda(), out,
                            dscores=None if ds is None else torch.from_numpy(ds).cuda(),
                            stream=stream, **how)
    ok()
    if pad:
        assert (wide[:, n:] == -77.0).all(), "columns behind the row were written"
    return out.double().cpu().numpy()


def check_backward(torch, gpu, x, k, score, renormalize, dense, pad=0, ids=None, seed=0,
                   spoil=False):
    t, n = x.shape
    rng = np.random.default_rng(seed + 17 * n + k)
    xs = x.double().cpu().numpy()
    how = dict(score=score, renormalize=renormalize, scale=1.5)
    if ids is None:
        ids = ref.route(xs, k, **how)[0]
    dw = rng.standard_normal((t, k)).astype(np.float32)
    ds = (rng.standard_normal((t, n)) * 0.3).astype(np.float32) if dense else None
    if spoil:  # what stands at masked places is not looked at
        dw[ids < 0] = np.nan
        if dense:
            ds[~(xs > -np.inf)] = np.inf
    got = run_backward(torch, gpu, x, ids, dw, ds, pad=pad, **how)
    want, size = ref.route_backward(xs, ids, dw, dscores=ds, **how)
    half = {4: 2.0 ** -24, 2: 2.0 ** -11 if x.dtype == torch.float16 else 2.0 ** -8}[
        x.element_size()]
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else TINY  # half of fp16's smallest step
    tol = tolerance(xs, score) * size
    bad = np.abs(got - want) > tol + half * (np.abs(want) + tol) + tiny
    assert not bad.any(), (score, renormalize, dense, np.argwhere(bad)[:5], got[bad][:5],
                           want[bad][:5])
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("experts", [1, 2, 8, 33, 60, 64, 128, 256, 257, 1000, 1024])
def test_backward(dtype, experts, gpu, torch):
    for tokens in (1, 131):
        x = logits(torch, tokens, experts, dtype, experts, 1.5)
        for score in ("softmax", "sigmoid"):
            for renormalize in (True, False):
                for dense in (True, False):
                    for k in sorted({1, min(6, experts), min(32, experts)}):
                        check_backward(torch, gpu, x, k, score, renormalize, dense)


@pytest.mark.parametrize("dtype", TYPES)
def test_backward_masked(dtype, gpu, torch):
    lowest = torch.finfo(getattr(torch, dtype)).min
    x = logits(torch, 8, 64, dtype, 191)
    x[0] = -float("inf")
    x[1] = float("nan")
    x[2, 3:] = -float("inf")
    x[3, ::2] = float("nan")
    x[4, ::2] = lowest
    x[5] = lowest
    x[6, 3] = float("inf")
    x[7, 1:4] = float("inf")
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            for dense in (True, False):
                check_backward(torch, gpu, x, 6, score, renormalize, dense, spoil=True)


def test_backward_ids_outside_and_twice(gpu, torch):
    x = logits(torch, 50, 24, "float32", 193)
    rng = np.random.default_rng(3)
    ids = rng.integers(-3, 30, (50, 5)).astype(np.int32)
    ids[7] = 4
    ids[8] = -1
    ids[9] = 2 ** 31 - 1
    ids[10] = -2 ** 31
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            for dense in (True, False):
                check_backward(torch, gpu, x, 5, score, renormalize, dense, ids=ids)


def test_backward_against_differences(gpu, torch):
    """The kernel's fp32 gradient against central differences of the forward formula in 64 bits
    (h = 1e-5: an error of some 1e-9 from the third derivative and the rounding)."""
    rng = np.random.default_rng(23)
    x = logits(torch, 3, 10, "float32", 195, 1.0)
    xs = x.double().cpu().numpy()
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            ids = ref.route(xs, 3, score=score)[0]
            dw = rng.standard_normal((3, 3)).astype(np.float32)
            ds = rng.standard_normal((3, 10)).astype(np.float32)
            got = run_backward(torch, gpu, x, ids, dw, ds, score=score, renormalize=renormalize,
                               scale=1.5)
            for t in range(3):
                def loss(v):
                    s = ref.scores_row(v, score)
                    w = ref.ratio_row(v, ids[t], score) if renormalize else s[ids[t]]
                    return (dw[t] * w * 1.5).sum() + (ds[t] * s).sum()

                size = ref.route_backward_row(xs[t], ids[t], dw[t].astype(float), score=score,
                                              renormalize=renormalize, scale=1.5,
                                              dscores=ds[t].astype(float))[1]
                tol = tolerance(xs, score)[t, 0] * size + 1e-8
                for e in range(10):
                    step = np.zeros(10)
                    step[e] = 1e-5
                    slope = (loss(xs[t] + step) - loss(xs[t] - step)) / 2e-5
                    assert abs(got[t, e] - slope) <= tol[e], (score, renormalize, t, e)


def test_backward_in_place(gpu, torch):
    for dtype in TYPES:
        x = logits(torch, 77, 100, dtype, 197)
        ids = ref.route(x.double().cpu().numpy(), 4)[0]
        dw = np.random.default_rng(1).standard_normal((77, 4)).astype(np.float32)
        want = run_backward(torch, gpu, x, ids, dw, None)
        gpu.route_topk_backward(x, torch.from_numpy(ids).cuda(), torch.from_numpy(dw).cuda(), x,
                                stream=0)
        torch.cuda.synchronize()
        assert np.array_equal(x.double().cpu().numpy(), want)


# ---- plan ----------------------------------------------------------------------------------------

def run_plan(torch, gpu, ids, experts, align, extra=0, stream=0):
    pairs = ids.size
    capacity = pairs + min(experts, pairs) * (align - 1) + extra
    offsets, ok1 = guarded(torch, (experts + 1,), torch.int32, -77)
    order, ok2 = guarded(torch, (capacity,), torch.int32, -77)
    position, ok3 = guarded(torch, ids.shape, torch.int32, -77)
    gpu.route_plan(torch.from_numpy(ids).cuda(), experts, offsets, order, position, align=align,
                   stream=stream)
    for ok in (ok1, ok2, ok3):
        ok()
    got = [a.cpu().numpy() for a in (offsets, order, position.view(-1))]
    want = ref.plan(ids, experts, align, capacity)
    for name, g, w in zip(("offsets", "order", "position"), got, want):
        assert np.array_equal(g, w), name
    return got


@pytest.mark.parametrize("experts", [1, 2, 8, 60, 64, 256, 1000, 1024])
@pytest.mark.parametrize("align", [1, 16, 128])
def test_plan(experts, align, gpu, torch):
    rng = np.random.default_rng(experts + align)
    for tokens, k in ((1, 1), (1, 8), (3, 2), (64, 8), (333, 6), (4099, 4), (20000, 8)):
        ids = rng.integers(0, experts, (tokens, k)).astype(np.int32)
        run_plan(torch, gpu, ids, experts, align, extra=int(rng.integers(0, 70)))
        ids[rng.random(ids.shape) < 0.2] = -1
        run_plan(torch, gpu, ids, experts, align)


def test_plan_skewed(gpu, torch):
    for n in (5, 1000, 100_000, 1_000_003):
        run_plan(torch, gpu, np.zeros((n, 1), np.int32), 64, 128)
        run_plan(torch, gpu, np.full((n, 1), 63, np.int32), 64, 7)
        run_plan(torch, gpu, np.full((n, 1), -1, np.int32), 64, 16, extra=5)
    wild = np.array([[5, -1, 64, 63, 2 ** 31 - 1, -2 ** 31, 0, 5]], np.int32)
    run_plan(torch, gpu, wild, 64, 4, extra=9)


# ---- together, on streams, in graphs ---------------------------------------------------------------

def test_route_plan_products_and_gradient_together(gpu, torch):
    """A routed layer as it is used: route, group, one product per expert over the grouped rows,
    weighted sum, and back to the logits, against the dense layer in 64 bits."""
    tokens, experts, k, dim, align = 300, 16, 4, 24, 8
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(tokens, experts, generator=g, device="cuda")
    h = torch.randn(tokens, dim, generator=g, device="cuda", dtype=torch.float64)
    mats = torch.randn(experts, dim, dim, generator=g, device="cuda", dtype=torch.float64)
    ids = torch.empty(tokens, k, dtype=torch.int32, device="cuda")
    w = torch.empty(tokens, k, device="cuda")
    gpu.route_topk(x, ids, w, score="sigmoid", stream=0)
    cap = tokens * k + experts * (align - 1)
    offsets = torch.empty(experts + 1, dtype=torch.int32, device="cuda")
    order = torch.empty(cap, dtype=torch.int32, device="cuda")
    position = torch.empty_like(ids)
    gpu.route_plan(ids, experts, offsets, order, position, align=align, stream=0)
    rows = torch.where(order[:, None] >= 0, h[(order.clamp(min=0) // k).long()], 0.0)
    y = torch.zeros(cap, dim, dtype=torch.float64, device="cuda")
    at = offsets.tolist()
    for e in range(experts):
        y[at[e]:at[e + 1]] = rows[at[e]:at[e + 1]] @ mats[e]
    picked = y[position.long()]
    out = (picked * w[:, :, None].double()).sum(1)

    dense = torch.sigmoid(x.double()).requires_grad_(False)
    leaf = x.double().requires_grad_(True)
    s = torch.gather(torch.sigmoid(leaf), 1, ids.long())
    all_y = torch.einsum("td,edf->tef", h, mats)
    want = (torch.gather(all_y, 1, ids.long()[:, :, None].expand(-1, -1, dim))
            * (s / s.sum(1, keepdim=True))[:, :, None]).sum(1)
    assert torch.equal(ids.long(), torch.topk(dense, k).indices)
    # a weight's relative error times the sum of the magnitudes it is applied to
    err = 2.0 ** -18 * (picked.abs() * w[:, :, None]).sum(1)
    assert ((out - want).abs() <= err + 1e-9).all()
    dout = torch.randn(tokens, dim, generator=g, device="cuda", dtype=torch.float64)
    want.backward(dout)
    dw = (picked * dout[:, None]).sum(2).float()
    dx = torch.empty_like(x)
    gpu.route_topk_backward(x, ids, dw, dx, score="sigmoid", stream=0)
    err = 2.0 ** -18 * (w.double() * dw.abs().double()).sum(1, keepdim=True) * 4
    assert ((dx - leaf.grad).abs() <= err + 1e-9).all()


def test_draws_from_a_search(ovvs, gpu, torch):
    """Negatives drawn from a search's scores: the distances of the index's own device search are
    the logits, the drawn columns index its neighbours."""
    rng = np.random.default_rng(4)
    data = rng.standard_normal((5000, 32)).astype(np.float32)
    q = rng.standard_normal((20, 32)).astype(np.float32)
    ix = ovvs.BruteIndex.build(data, metric="inner_product", resources=gpu)
    nb = torch.empty(20, 10, dtype=torch.int64, device="cuda")
    sc = torch.empty(20, 10, dtype=torch.float32, device="cuda")
    dq = torch.from_numpy(q).cuda()
    u = torch.from_numpy(uniforms(6, 20, 4)).cuda()
    ids = torch.empty(20, 4, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    ix.search_device(dq, 10, nb, sc)
    gpu.sample_rows(sc, u, ids)  # the same stream: after the search
    gpu.synchronize()
    want = ref.sample(sc.double().cpu().numpy(), u.cpu().numpy())[0]
    assert np.array_equal(ids.cpu().numpy(), want)
    drawn = torch.gather(nb, 1, ids).cpu().numpy()
    assert ((drawn >= 0) & (drawn < 5000)).all()
    ix.close()


def everything(torch, gpu, x, u, out, stream):
    """One pass through all four operators into preallocated outputs."""
    gpu.sample_rows(x, u, out["draw"], probs=out["p"], top_k=out["k"], stream=stream)
    gpu.route_topk(x, out["ids"], out["w"], groups=4, topk_groups=2, stream=stream)
    gpu.route_plan(out["ids"], x.shape[1], out["offsets"], out["order"], out["position"],
                   align=4, stream=stream)
    gpu.route_topk_backward(x, out["ids"], out["w"], out["dx"], stream=stream)


def outputs(torch, t, n):
    z = lambda *s, d=torch.int32: torch.full(s, -9, dtype=d, device="cuda")  # noqa: E731
    return {"draw": z(t, 2, d=torch.int64), "p": z(t, 2, d=torch.float32),
            "k": torch.full((t,), 5, dtype=torch.int32, device="cuda"),
            "ids": z(t, 4), "w": z(t, 4, d=torch.float32), "offsets": z(n + 1),
            "order": z(t * 4 + n * 3), "position": z(t, 4), "dx": z(t, n, d=torch.float32)}


def test_streams_and_graphs(gpu, torch):
    """The same results on another stream, on two streams at once, and from two captured graphs
    replayed at once with new inputs."""
    t, n = 300, 64
    xs = [logits(torch, t, n, "float32", 300 + i) for i in range(4)]
    us = [torch.from_numpy(uniforms(310 + i, t, 2)).cuda() for i in range(4)]
    want = []
    for x, u in zip(xs, us):
        out = outputs(torch, t, n)
        everything(torch, gpu, x, u, out, 0)
        torch.cuda.synchronize()
        want.append({k: v.clone() for k, v in out.items()})
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [outputs(torch, t, n) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for i in (0, 1):
            everything(torch, gpu, xs[i], us[i], got[i], side[i].cuda_stream)
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(got[i][k], want[i][k]) for k in got[i])
    graphs, ins = [], []
    for i in (0, 1):
        x, u, out = xs[i].clone(), us[i].clone(), outputs(torch, t, n)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side[i]):
            everything(torch, gpu, x, u, out, side[i].cuda_stream)
        graphs.append(graph)
        ins.append((x, u, out))
    for shift in (0, 2):
        for i in (0, 1):
            ins[i][0].copy_(xs[i + shift])
            ins[i][1].copy_(us[i + shift])
        torch.cuda.synchronize()
        for _ in range(10):
            for i in (0, 1):
                with torch.cuda.stream(side[i]):
                    graphs[i].replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            assert all(torch.equal(ins[i][2][k], want[i + shift][k]) for k in ins[i][2])


def test_threads_at_once(gpu, torch):
    import threading

    t, n = 200, 64
    x, u = logits(torch, t, n, "float32", 400), torch.from_numpy(uniforms(401, t, 2)).cuda()
    want = outputs(torch, t, n)
    everything(torch, gpu, x, u, want, 0)
    torch.cuda.synchronize()
    outs = [outputs(torch, t, n) for _ in range(4)]
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            for _ in range(50):
                everything(torch, gpu, x, u, outs[i], streams[i].cuda_stream)
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    torch.cuda.synchronize()
    assert not failed
    for out in outs:
        assert all(torch.equal(out[k], want[k]) for k in out)


def test_default_stream_is_the_resources_own(gpu, torch):
    x = logits(torch, 4, 32, "float32", 500)
    ids = torch.empty(4, 3, dtype=torch.int32, device="cuda")
    w = torch.empty(4, 3, device="cuda")
    torch.cuda.synchronize()
    gpu.route_topk(x, ids, w)
    gpu.synchronize()
    assert np.array_equal(ids.cpu().numpy(), ref.route(x.double().cpu().numpy(), 3)[0])
    assert gpu.last_device() == 3


def test_outputs_that_are_left_out(gpu, torch):
    """Without probabilities, kept counts and scores, the rest is the same."""
    for rows, cols in ((3, 20001), (310, 3001)):
        x = logits(torch, rows, cols, "bfloat16", 600)
        u = torch.from_numpy(uniforms(601, rows, 2)).cuda()
        for how in (dict(), dict(k=30), dict(p=0.9), dict(k=600, p=0.9), dict(t=0.0), dict(q=0.02),
                    dict(p=0.9, q=0.02)):
            put = lambda n, d: (torch.full((rows,), how[n], dtype=d, device="cuda")  # noqa: E731
                                if n in how else None)
            kw = dict(temperature=put("t", torch.float32), top_k=put("k", torch.int32),
                      top_p=put("p", torch.float32), min_p=put("q", torch.float32), stream=0)
            a = torch.empty(rows, 2, dtype=torch.int64, device="cuda")
            b = torch.empty_like(a)
            gpu.sample_rows(x, u, a, probs=torch.empty(rows, 2, device="cuda"),
                            kept=torch.empty(rows, dtype=torch.int32, device="cuda"), **kw)
            gpu.sample_rows(x, u, b, **kw)
            assert torch.equal(a, b), how
    x = logits(torch, 70, 256, "float32", 602)
    ids = [torch.empty(70, 8, dtype=torch.int32, device="cuda") for _ in range(2)]
    w = [torch.empty(70, 8, device="cuda") for _ in range(2)]
    s = torch.empty(70, 256, device="cuda")
    gpu.route_topk(x, ids[0], w[0], scores=s, stream=0)
    gpu.route_topk(x, ids[1], w[1], stream=0)
    assert torch.equal(ids[0], ids[1]) and torch.equal(w[0], w[1])


def test_binding_refusals(gpu, torch):
    x = torch.zeros(4, 8, device="cuda")
    u = torch.zeros(4, device="cuda")
    i64 = torch.zeros(4, dtype=torch.int64, device="cuda")
    i32 = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    w = torch.zeros(4, 2, device="cuda")
    with pytest.raises(ValueError):
        gpu.sample_rows(x, u[:3], i64)
    with pytest.raises(ValueError):
        gpu.sample_rows(x, u, i64.int())
    with pytest.raises(ValueError):
        gpu.sample_rows(x, u, i64, temperature=torch.zeros(4, dtype=torch.float64, device="cuda"))
    with pytest.raises(ValueError):
        gpu.sample_rows(x, u, i64, top_k=torch.zeros(4, device="cuda"))
    with pytest.raises(ValueError):
        gpu.sample_rows(x, u, i64, top_p=torch.zeros(5, device="cuda"))
    with pytest.raises(ValueError):
        gpu.sample_rows(x.cpu(), u, i64)
    with pytest.raises(ValueError):
        gpu.route_topk(x, i32, w[:, :1])
    with pytest.raises(ValueError):
        gpu.route_topk(x, i32, w, bias=torch.zeros(7, device="cuda"))
    with pytest.raises(KeyError):
        gpu.route_topk(x, i32, w, score="tanh")
    with pytest.raises(ValueError):
        gpu.route_topk_backward(x, i32, w, x.half())
    with pytest.raises(ValueError):
        gpu.route_plan(i32, 8, torch.zeros(8, dtype=torch.int32, device="cuda"), i32.view(-1), i32)
