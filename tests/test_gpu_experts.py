"""Routing, expert order and weighted sums of a mixture of experts against plain float64 restatements,
at the sizes, masks and orders where they can go wrong.

Tolerances.  u = 2^-24 (half a step of float32).  A share is exp(x - top) / sum: the argument carries
|x - top| u of relative error into the exponential (|x - top| <= 40 in these inputs, beyond that the share is
below 1e-17 of the largest), the exponential 4 u, the sum at most 37 additions, the quotient and the scale
u each: below 128 u = 2^-17, twice that with a softmax over all experts whose sum and quotient enter again.
Results in 16 bits add half a step of their type.
"""
import ctypes
import functools
import threading

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _order(keys):
    """Indices by descending key, NaN greatest, lowest index among equals."""
    k = np.where(np.isnan(keys), np.inf, keys)
    return sorted(range(len(k)), key=lambda e: (not np.isnan(keys[e]), -k[e], e))


def _scores(x, scoring):
    with np.errstate(all="ignore"):
        if scoring == "sigmoid":
            return 1 / (1 + np.exp(-x))
        top = x.max()
        e = np.exp(x - (0 if np.isneginf(top) else top))
        total = e.sum()
        return e / (1 if total == 0 else total)


def _shares(x, scoring):
    """What each of the chosen has of their sum, from the logarithms of the scores: float64 itself runs out
    of range for sigmoids of the lowest values."""
    with np.errstate(all="ignore"):
        log_s = -np.logaddexp(0, -x) if scoring == "sigmoid" else x
        log_s = np.where(x < -700, x, log_s)
        e = np.exp(log_s - log_s.max())
        return e / e.sum()


def ref_route(logits, k, bias=None, scoring="softmax", n_groups=1, topk_groups=None, group_best=1,
              renormalize=True, scale=1.0):
    n, e = logits.shape
    topk_groups = topk_groups or n_groups
    weights, experts = np.zeros((n, k)), np.full((n, k), -1, np.int32)
    for i in range(n):
        x = logits[i]
        s = _scores(x, scoring)
        key = s + bias if bias is not None else s
        choose = key if bias is not None else x.copy()
        choose = np.where(np.isneginf(x), -np.inf, choose)
        if n_groups > 1:
            size = e // n_groups
            gkey = choose if group_best == 1 else np.where(np.isneginf(x), -np.inf, key)
            score = []
            for g in range(n_groups):
                part = gkey[g * size:(g + 1) * size]
                o = _order(part)[:group_best]
                with np.errstate(all="ignore"):
                    score.append(part[o].sum())
            kept = _order(np.array(score))[:topk_groups]
            for g in range(n_groups):
                if g not in kept:
                    choose[g * size:(g + 1) * size] = -np.inf
        o = [j for j in _order(choose)[:k] if not np.isneginf(choose[j])]
        w = s[o]
        if renormalize and len(o):
            w = _shares(x[o], scoring) if not np.isnan(s).all() else w
        experts[i, :len(o)] = o
        weights[i, :len(o)] = w * scale
    return weights, experts


def ref_route_grad(logits, experts, grad, scoring, renormalize, scale):
    """By the chain rule through the scores: d weights / d scores, then d scores / d logits.  Renormalised
    weights depend on the logarithms of the chosen scores alone, whose slopes are 1 or 1 - s."""
    out = np.zeros_like(logits)
    for i in range(logits.shape[0]):
        s = _scores(logits[i], scoring)
        there = experts[i] >= 0
        idx, g = experts[i][there], grad[i][there].astype(np.float64) * scale
        ds = np.zeros_like(s)
        if renormalize and len(idx):
            p = _shares(logits[i][idx], scoring)
            out[i][idx] = p * (g - (p * g).sum()) * (1 - s[idx] if scoring == "sigmoid" else 1)
            continue
        ds[idx] = g
        out[i] = s * (1 - s) * ds if scoring == "sigmoid" else s * (ds - (s * ds).sum())
    return out


def _logits(n, e, dtype, seed, masked=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, e, generator=g) * 1.5
    if masked and e > 1 and n > 4:
        x[torch.rand(n, e, generator=g) < 0.15] = float("-inf")
        x[1] = float("-inf")                 # a padding token
        x[2] = 0.25                          # all equal
        x[3] = torch.finfo(dtype).min        # masked by the type's lowest value: still numbers
    return x.to(dtype).cuda()


def _same_route(x, k, **kw):
    from sklearn_numba_dpex_b200.common import route_topk

    weights, experts = route_topk(x, k, **kw)
    if kw.get("bias") is not None:
        kw = {**kw, "bias": kw["bias"].double().cpu().numpy()}
    want_w, want_e = ref_route(x.double().cpu().numpy(), k, **kw)
    assert weights.dtype == torch.float32 and experts.dtype == torch.int32
    np.testing.assert_array_equal(experts.cpu().numpy(), want_e)
    np.testing.assert_allclose(weights.cpu().double().numpy(), want_w, rtol=256 * U, atol=0)
    return weights, experts


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,e,k", [(1, 1, 1), (5, 2, 2), (7, 31, 3), (33, 32, 1), (9, 33, 8), (6, 64, 6), (17, 100, 9),
                                   (13, 128, 8), (7, 257, 16), (5, 600, 32), (6, 1024, 4), (3, 1023, 32)])
@pytest.mark.parametrize("scoring,renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True),
                                                 ("sigmoid", False)])
def test_route_sizes(dtype, n, e, k, scoring, renormalize):
    _same_route(_logits(n, e, TYPES[dtype], 1), k, scoring=scoring, renormalize=renormalize, scale=2.5)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("e,groups,topk_groups,best,k", [(256, 8, 4, 2, 8), (256, 8, 4, 1, 8), (64, 32, 3, 2, 6),
                                                         (96, 3, 1, 2, 5), (105, 7, 7, 1, 9), (40, 8, 8, 2, 4),
                                                         (1024, 16, 2, 2, 32), (6, 6, 2, 1, 2)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_route_groups_and_bias(scoring, e, groups, topk_groups, best, k, with_bias):
    g = torch.Generator().manual_seed(3)
    bias = (torch.randn(e, generator=g) * 0.1).cuda() if with_bias else None
    for dtype in TYPES.values():
        _same_route(_logits(23, e, dtype, 4), k, bias=bias, scoring=scoring, n_groups=groups, topk_groups=topk_groups,
                    group_best=best, scale=1.5)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_near_ties_are_ordered_as_64_bits_order_them(scoring):
    """Keys that differ by less than 32 bits resolve: the bias undoes the difference of the scores up to its
    own rounding, so that every pair of experts lies within a few 2^-25 of each other."""
    g = torch.Generator().manual_seed(9)
    x = torch.randn(64, generator=g)
    s = torch.from_numpy(_scores(x.double().numpy(), scoring))
    bias = (0.7 - s).float().cuda()
    _same_route(x[None].repeat(5, 1).cuda(), 16, bias=bias, scoring=scoring)
    # and a bias of zeros leaves equal logits equal: lowest index
    xs = torch.randint(0, 3, (50, 64), generator=g).float().cuda()
    _same_route(xs, 20, bias=torch.zeros(64, device="cuda"), scoring=scoring)
    _same_route(xs, 20, bias=torch.zeros(64, device="cuda"), scoring=scoring, n_groups=8, topk_groups=3, group_best=2)


@pytest.mark.parametrize("e", [30, 64, 128, 200, 1000])
@pytest.mark.parametrize("base", [1.0, -1.0, 0.0, 37.5])
def test_route_orders_logits_that_differ_in_their_last_bits(e, base):
    """Neighbouring float32 numbers in random order, some of them equal: every token lies in the low bits of its
    logits, or one does among ordinary ones."""
    g = torch.Generator().manual_seed(e)
    ulps = torch.randint(0, 2 * e, (9, e), generator=g)
    x = (torch.full((9, e), base).view(torch.int32) + ulps.to(torch.int32)).view(torch.float32)
    if base == 0.0:
        x = x * (torch.randint(0, 2, (9, e), generator=g) * 2 - 1)         # subnormals, -0 among them
    _same_route(x.cuda(), min(9, e))
    y = torch.randn(9, e, generator=g)
    y[4] = x[4]
    _same_route(y.cuda(), min(9, e), scoring="sigmoid")


# experts and greatest k, in every layout of the routing kernel (lanes of a token, experts of a lane)
LAYOUTS = [(32, 8), (30, 12), (64, 8), (128, 16), (100, 20), (256, 8), (500, 8), (1000, 32)]


@pytest.mark.parametrize("e,most", LAYOUTS)
@pytest.mark.parametrize("base", [0.25, 1.0, -3.0])
def test_route_finds_a_greater_logit_behind_a_tie(e, most, base):
    """Equal logits on both sides of the last place, and among or behind them one that differs in its last bits."""
    g = torch.Generator().manual_seed(e)
    up, down = (float(np.nextafter(np.float32(base), np.float32(to))) for to in (9, -9))
    for k in sorted({1, 4, 8, most}):
        if k > most:
            continue
        rows = []
        for place in sorted({0, k - 1, k, min(k + 1, e - 1), e // 2, e - 1}):
            for value in (up, down, base * 1.00005):
                x = torch.full((e,), base)
                x[place] = value
                rows.append(x)
        some = torch.full((20, e), base)
        some[torch.rand(20, e, generator=g) < 0.02] = up
        some[torch.rand(20, e, generator=g) < 0.3] = down
        some[:10][torch.rand(10, e, generator=g) < 0.5] = -9.0
        _same_route(torch.cat([torch.stack(rows), some]).cuda(), k)
    x = torch.full((3, e), -3.0)
    x[:, :2] = 1.0
    x[0, 2] = x[1, e - 1] = float(np.nextafter(np.float32(1), np.float32(2)))
    _same_route(x.cuda(), 1)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("e,most", LAYOUTS)
def test_route_finds_a_greater_key_behind_equal_ones(scoring, e, most):
    """Few kinds of experts with equal logits and biases, whose keys differ by less than 32 bits from kind to
    kind: the last place falls among equals while a greater key may lie behind them."""
    for seed in range(12):
        g = torch.Generator().manual_seed(seed)
        kinds = torch.randn(max(2, e // 16), generator=g)
        x = kinds[torch.randint(0, len(kinds), (e,), generator=g)]
        bias = (0.7 - torch.from_numpy(_scores(x.double().numpy(), scoring))).float()
        for k in sorted({1, 4, 8, most}):
            if k <= most:
                _same_route(x[None].repeat(3, 1).cuda(), k, scoring=scoring, bias=bias.cuda())


@pytest.mark.parametrize("e,most", LAYOUTS)
def test_route_equal_keys_of_a_bias_step(e, most):
    """Two equal experts and one behind them, greater by 1.7e-8 where 32 bits see three equal keys."""
    x = torch.full((2, e), -9.0)
    x[0, :2], x[0, e - 1] = 0.22753906, 0.19921875
    x[1, 1:3], x[1, 3] = 0.22753906, 0.19921875
    bias = torch.zeros(2, e)
    bias[0, :2], bias[0, e - 1] = -0.002, 0.005
    bias[1, 1:3], bias[1, 3] = -0.002, 0.005
    for dtype in (torch.float32, torch.bfloat16):
        for i in range(2):
            _same_route(x[i:i + 1].to(dtype).cuda(), 1, scoring="sigmoid", bias=bias[i].cuda())


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_nan_and_infinity(scoring, renormalize):
    x = torch.randn(6, 40, generator=torch.Generator().manual_seed(2))
    x[0, 7] = float("nan")
    x[1, 3] = float("inf")
    x[2, 3], x[2, 30] = float("nan"), float("-inf")
    x[3, :] = float("nan")
    _same_route(x.cuda(), 5, scoring=scoring, renormalize=renormalize)
    b = torch.zeros(40, device="cuda")
    b[4], b[5] = float("-inf"), float("nan")      # an expert that is switched off, and one that is broken
    _same_route(x[4:].cuda(), 5, scoring=scoring, renormalize=renormalize, bias=b)


def test_route_extreme_scores_stay_finite():
    x = torch.tensor([[-200.0, -150.0, -151.0, -300.0], [90.0, 88.0, 1.0, -90.0], [-62.0, -59.0, -61.0, -1e30]])
    for scoring in ("softmax", "sigmoid"):
        w, e = _same_route(x.cuda(), 3, scoring=scoring)
        assert torch.isfinite(w).all() and torch.allclose(w.sum(1), torch.ones(3, device="cuda"))
    _same_route(x[1:2].cuda(), 4, scoring="sigmoid", renormalize=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,e,k", [(1, 1, 1), (7, 31, 3), (6, 64, 6), (13, 130, 8), (5, 600, 32), (6, 1024, 4)])
@pytest.mark.parametrize("scoring,renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True),
                                                 ("sigmoid", False)])
def test_route_gradient_is_the_formula(dtype, n, e, k, scoring, renormalize):
    from sklearn_numba_dpex_b200.common import route_topk, route_topk_grad

    x = _logits(n, e, TYPES[dtype], 5)
    grad = torch.randn(n, k, generator=torch.Generator().manual_seed(6)).cuda()
    leaf = x.clone().requires_grad_(True)
    weights, experts = route_topk(leaf, k, scoring=scoring, renormalize=renormalize, scale=2.5)
    assert not experts.requires_grad
    weights.backward(grad)
    explicit = route_topk_grad(x, experts, grad, scoring=scoring, renormalize=renormalize, scale=2.5)
    assert leaf.grad.dtype == x.dtype and torch.equal(leaf.grad, explicit)
    x64, e64 = x.double().cpu().numpy(), experts.cpu().numpy()
    want = ref_route_grad(x64, e64, grad.cpu().numpy(), scoring, renormalize, 2.5)
    # the formulas are a share or score (at most one) times a difference of terms of at most |g|
    s = np.stack([_scores(r, scoring) for r in x64])
    size = np.where(want != 0, 1.0, 0.0) if renormalize else s
    bound = 256 * U * 2 * 2.5 * np.abs(grad.cpu().numpy()).max() * size
    bound = bound + torch.finfo(x.dtype).eps / 2 * np.abs(want) + torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    assert (np.abs(explicit.double().cpu().numpy() - want) <= bound).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_gradient_of_saturated_sigmoids(dtype, renormalize):
    """1 - s keeps its digits: relative to it the two sigmoids are off by 6 u each (exponential 4, sum, quotient),
    their product with the gradient and the scale by 4 more; shares and what they sum to as ever."""
    from sklearn_numba_dpex_b200.common import route_topk, route_topk_grad

    t, k = TYPES[dtype], 32
    x = torch.stack([torch.linspace(low, low + 36, k) for low in (-40.0, -10.0, 0.0, 8.0)]).to(t)
    grad = torch.randn(4, k, generator=torch.Generator().manual_seed(3))
    _, experts = route_topk(x.cuda(), k, scoring="sigmoid", renormalize=renormalize, scale=2.5)
    got = route_topk_grad(x.cuda(), experts, grad.cuda(), scoring="sigmoid", renormalize=renormalize, scale=2.5)
    x64, at = x.double().numpy(), experts.cpu().numpy().astype(np.int64)
    assert (np.sort(at, 1) == np.arange(k)).all()
    g = np.zeros((4, k))
    np.put_along_axis(g, at, grad.double().numpy() * 2.5, 1)
    rest = 1 / (1 + np.exp(x64))
    if renormalize:
        share = np.stack([_shares(r, "sigmoid") for r in x64])
        want = share * (g - (share * g).sum(1, keepdims=True)) * rest
        bound = 256 * U * 2 * np.abs(g).max() * share * rest
    else:
        want = g / (1 + np.exp(-x64)) * rest
        bound = 16 * U * np.abs(want)
    info = torch.finfo(t)
    bound = bound * (1 + info.eps) + info.eps / 2 * np.abs(want) + info.smallest_normal * info.eps
    assert (np.abs(got.double().cpu().numpy() - want) <= bound).all()


@pytest.mark.parametrize("scoring,renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True),
                                                 ("sigmoid", False)])
def test_route_gradient_is_the_slope(scoring, renormalize):
    """Central differences of the forward pass with step h = 2^-6.  Third derivatives of a share in one
    logit are below 1, so the difference is off by h^2 / 6 = 4.1e-5 per unit of sum |g|; its rounding is
    256 u / (2 h) = 4.9e-4 of the weights."""
    from sklearn_numba_dpex_b200.common import route_topk, route_topk_grad

    h, k = 2.0 ** -6, 3
    x = torch.linspace(-1, 1, 12)[torch.randperm(12, generator=torch.Generator().manual_seed(1))][None].cuda()
    grad = torch.tensor([[0.7, -1.1, 0.4]], device="cuda")
    kw = dict(scoring=scoring, renormalize=renormalize, scale=1.0)
    _, experts = route_topk(x, k, **kw)
    got = route_topk_grad(x, experts, grad, **kw)
    steps = torch.cat([x + h * torch.eye(12, device="cuda"), x - h * torch.eye(12, device="cuda")])
    w, e = route_topk(steps, k, **kw)
    assert (e == experts).all()          # gaps of the logits are 2 / 11, far above h
    slope = ((w[:12] - w[12:]).double() * grad.double()).sum(1) / (2 * h)
    bound = (h * h / 6 + 256 * U / (2 * h)) * float(grad.abs().sum())
    assert float((slope - got[0].double()).abs().max()) <= bound


def test_route_gradient_of_a_broadcast_and_of_a_view():
    """The gradient that arrives may have strides of 0 (a sum's), the logits may be a slice."""
    from sklearn_numba_dpex_b200.common import route_topk, route_topk_grad

    base = torch.randn(20, 48, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    leaf = base.clone().requires_grad_(True)
    w, e = route_topk(leaf[::2, 3:43], 4, scoring="sigmoid", renormalize=False)
    w.sum().backward()
    want = torch.zeros_like(base)
    want[::2, 3:43] = route_topk_grad(base[::2, 3:43], e, torch.ones(10, 4, device="cuda"), "sigmoid", False)
    assert torch.equal(leaf.grad, want)


# --------------------------------------------------------------------------- expert order
def ref_slots(experts, n_experts):
    flat = experts.reshape(-1)
    key = np.where((flat >= 0) & (flat < n_experts), flat, n_experts)
    order = np.argsort(key, kind="stable")
    valid = int((key < n_experts).sum())
    slots, rows = np.full(flat.size, -1), np.full(flat.size, -1)
    slots[order[:valid]] = np.arange(valid)
    rows[:valid] = order[:valid] // experts.shape[1]
    return slots.reshape(experts.shape), rows, np.concatenate([[0], np.cumsum(np.bincount(key, minlength=n_experts + 1)[:n_experts])])


@pytest.mark.parametrize("n,k,e", [(0, 3, 4), (1, 1, 1), (1, 8, 256), (64, 8, 256), (511, 8, 7), (512, 8, 1024), (513, 8, 64),
                                   (4097, 1, 3), (5000, 6, 1024), (30011, 9, 129)])
@pytest.mark.parametrize("kind", ["all", "some", "none", "one", "repeated"])
def test_expert_slots(n, k, e, kind):
    from sklearn_numba_dpex_b200.common import expert_slots

    rng = np.random.default_rng(n + k + e)
    x = rng.integers(0, e, (n, k))
    if kind == "some":
        x[rng.random((n, k)) < 0.3] = -1
        x[rng.random((n, k)) < 0.05] = e + 3        # not an expert either
    elif kind == "none":
        x[:] = -1
    elif kind == "one":
        x[:] = e - 1
    elif kind == "repeated" and n:
        x[:] = x[:, :1]                             # a token names the same expert k times
    x = x.astype(np.int32)
    got = expert_slots(torch.from_numpy(x).cuda(), e)
    for a, b in zip(got, ref_slots(x, e)):
        assert a.dtype == torch.int32
        np.testing.assert_array_equal(a.cpu().numpy(), b)


@pytest.mark.parametrize("n,k,e", [(131073, 8, 33), (300007, 8, 129), (1200000, 2, 1024)])
def test_expert_slots_of_many_chunks(n, k, e):
    """More chunks of 4096 choices than the scan takes at a time (256): what it carries on."""
    from sklearn_numba_dpex_b200.common import expert_slots

    x = np.random.default_rng(n).integers(-1, e, (n, k)).astype(np.int32)
    for a, b in zip(expert_slots(torch.from_numpy(x).cuda(), e), ref_slots(x, e)):
        np.testing.assert_array_equal(a.cpu().numpy(), b)


@pytest.mark.parametrize("n,k", [(0, 1 << 20), (1, 600000), (3, 700001)])
def test_expert_slots_of_many_choices_a_token(n, k):
    from sklearn_numba_dpex_b200.common import combine_experts_grad, expert_slots

    x = np.random.default_rng(k).integers(-1, 7, (n, k)).astype(np.int32)
    slots, rows, offsets = expert_slots(torch.from_numpy(x).cuda(), 7)
    for a, b in zip((slots, rows, offsets), ref_slots(x, 7)):
        np.testing.assert_array_equal(a.cpu().numpy(), b)
    values, weights, grad = torch.ones(n * k, 1, device="cuda"), torch.full((n, k), 0.5, device="cuda"), torch.full((n, 1), 4.0, device="cuda")
    got_v, got_w = combine_experts_grad(values, slots, weights, grad)
    assert (got_v[: int(offsets[-1])] == 2).all() and (got_v[int(offsets[-1]):] == 0).all()
    assert torch.equal(got_w, torch.where(slots >= 0, 4.0, 0.0))


def test_expert_order_from_several_threads():
    """Through the C interface, which runs without the interpreter's lock: calls that need much shared memory
    beside calls that need little."""
    from sklearn_numba_dpex_b200 import _cabi

    n, k, counts, failed = 500, 8, (1024, 256, 1000, 210), []
    together = threading.Barrier(len(counts))

    def calls(e):
        x = np.random.default_rng(e).integers(0, e, (n, k)).astype(np.int32)
        xd = torch.from_numpy(x).cuda()
        out = [torch.empty(size, dtype=torch.int32, device="cuda") for size in ((n, k), (n * k,), (e + 1,))]
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        at = [_cabi.ptr(t) for t in (xd, *out)]
        run = functools.partial(_cabi.lib.kmb_expert_slots, at[0], n, k, e, *at[1:], None, 0, ctypes.c_void_p(stream.cuda_stream))
        together.wait()
        for _ in range(20000):
            if run() != _cabi.KMB_OK:
                failed.append((e, _cabi.last_error()))
                break
        stream.synchronize()
        if not all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(out, ref_slots(x, e))):
            failed.append((e, "another order"))

    threads = [threading.Thread(target=calls, args=(e,)) for e in counts]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


# --------------------------------------------------------------------------- weighted sums
def _combine_inputs(n, k, d, m, dtype, seed, repeated=False):
    g = torch.Generator().manual_seed(seed)
    values = torch.randn(m, d, generator=g).to(dtype)
    if repeated:
        slots = torch.randint(-1, m + 2, (n, k), generator=g)
    else:
        slots = torch.randperm(max(m, n * k), generator=g)[: n * k].view(n, k)
        slots[torch.rand(n, k, generator=g) < 0.2] = -1
    weights = torch.randn(n, k, generator=g)
    weights[(slots < 0) | (slots >= m)] = float("nan")       # what a missing row weighs counts nowhere
    return values, slots.to(torch.int32), weights, torch.randn(n, d, generator=g).to(dtype)


def ref_combine(values, slots, weights, grad):
    v, w, g = values.double(), weights.double(), grad.double()
    out, gv, gw = torch.zeros(grad.shape, dtype=torch.float64), torch.zeros(v.shape, dtype=torch.float64), torch.zeros(w.shape, dtype=torch.float64)
    big_o, big_v = torch.zeros_like(out), torch.zeros_like(gv)
    for t in range(slots.shape[0]):
        for j in range(slots.shape[1]):
            r = int(slots[t, j])
            if 0 <= r < v.shape[0]:
                out[t] += w[t, j] * v[r]
                big_o[t] += (w[t, j] * v[r]).abs()
                gv[r] += w[t, j] * g[t]
                big_v[r] += (w[t, j] * g[t]).abs()
                gw[t, j] = (v[r] * g[t]).sum()
    return out, gv, gw, big_o, big_v


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,d,m", [(1, 1, 1, 1), (1, 8, 4096, 8), (3, 2, 7, 9), (5, 8, 1031, 40), (17, 9, 64, 153), (33, 20, 129, 700),
                                     (9, 3, 8200, 27), (4, 2, 16, 0), (0, 2, 16, 5), (40, 3, 100, 130),
                                     (40, 2, 12, 90), (6, 2, 1028, 13)])
@pytest.mark.parametrize("repeated", [False, True])
def test_combine(dtype, n, k, d, m, repeated):
    """Every sum of N products is off by N u of the sum of their magnitudes at most."""
    from sklearn_numba_dpex_b200.common import combine_experts, combine_experts_grad

    t = TYPES[dtype]
    values, slots, weights, grad = _combine_inputs(n, k, d, m, t, 7, repeated)
    out, gv, gw, big_o, big_v = ref_combine(values, slots, weights, grad)
    dev = [x.cuda() for x in (values, slots, weights, grad)]
    half = torch.finfo(t).eps / 2
    tiny = torch.finfo(t).smallest_normal * torch.finfo(t).eps
    got = combine_experts(*dev[:3])
    assert got.dtype == t
    assert ((got.double().cpu() - out).abs() <= (k + 1) * U * big_o + half * out.abs() + tiny).all()
    got_v, got_w = combine_experts_grad(*dev)
    users = max(1, int(torch.bincount(slots[(slots >= 0) & (slots < m)].long(), minlength=1).max())) if n else 1
    assert ((got_v.double().cpu() - gv).abs() <= (users + 1) * U * big_v + half * gv.abs() + tiny).all()
    size = torch.zeros(n, k, dtype=torch.float64)
    for a in range(n):
        for b in range(k):
            if 0 <= slots[a, b] < m:
                size[a, b] = (values[int(slots[a, b])].double() * grad[a].double()).abs().sum()
    assert ((got_w.double().cpu() - gw).abs() <= (d + 1) * U * size).all()
    again = combine_experts_grad(*dev)
    assert torch.equal(again[0], got_v) and torch.equal(again[1], got_w)       # no order left to chance
    if n and m:
        a, b = dev[0].clone().requires_grad_(True), dev[2].clone().requires_grad_(True)
        combine_experts(a, dev[1], b).backward(dev[3])
        assert torch.equal(a.grad, got_v) and torch.equal(b.grad, got_w)


@pytest.mark.parametrize("dtype,d", [("fp32", 1024), ("fp32", 1031), ("fp32", 7), ("fp32", 2049), ("fp32", 4), ("bf16", 2048), ("bf16", 50), ("bf16", 51),
                                     ("fp16", 4104), ("bf16", 2064), ("fp16", 2050)])
@pytest.mark.parametrize("k", [1, 2, 3, 4, 5, 8])
def test_combine_many_tokens(dtype, d, k):
    """Tokens enough for the rows to be copied ahead: every warp walks several, and the last ones fewer."""
    from sklearn_numba_dpex_b200.common import combine_experts, combine_experts_grad

    t, n = TYPES[dtype], 5003
    g = torch.Generator("cuda").manual_seed(d + k)
    values = torch.randn(n * k + 3, d, device="cuda", generator=g).to(t)
    slots = torch.randperm(n * k + 3, device="cuda", generator=g)[: n * k].view(n, k).to(torch.int32)
    slots[torch.rand(n, k, device="cuda", generator=g) < 0.1] = -1
    if k > 2:
        slots[100:110, 1] = slots[200, 0]                # rows with several users
    weights, grad = torch.randn(n, k, device="cuda", generator=g), torch.randn(n, d, device="cuda", generator=g).to(t)
    there = (slots >= 0)[..., None]
    at = slots.long().clamp_min(0)
    weights[~there[..., 0]] = float("nan")
    w64 = torch.where(there, weights.double()[..., None], torch.zeros((), dtype=torch.float64, device="cuda"))
    v64 = values.double()[at] * there
    half, tiny = torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps
    out = (v64 * w64).sum(1)
    got = combine_experts(values, slots, weights)
    assert ((got.double() - out).abs() <= (k + 1) * U * (v64 * w64).abs().sum(1) + half * out.abs() + tiny).all()
    rows = (w64 * grad.double()[:, None]).reshape(-1, d)
    gv, big = torch.zeros_like(values, dtype=torch.float64), torch.zeros_like(values, dtype=torch.float64)
    gv.index_add_(0, at.reshape(-1), rows)
    big.index_add_(0, at.reshape(-1), rows.abs())
    got_v, got_w = combine_experts_grad(values, slots, weights, grad)
    assert ((got_v.double() - gv).abs() <= 13 * U * big + half * gv.abs() + tiny).all()
    gw, size = (v64 * grad.double()[:, None]).sum(2), (v64 * grad.double()[:, None]).abs().sum(2)
    assert ((got_w.double() - gw).abs() <= (d + 1) * U * size).all()


def test_combine_many_choices_of_many_tokens():
    from sklearn_numba_dpex_b200.common import combine_experts

    n, k, d = 3000, 70, 24
    values, slots = torch.randn(500, d, device="cuda"), torch.randint(-1, 500, (n, k), device="cuda", dtype=torch.int32)
    weights = torch.randn(n, k, device="cuda")
    v64 = values.double()[slots.long().clamp_min(0)] * (slots >= 0)[..., None] * weights.double()[..., None]
    err = (combine_experts(values, slots, weights).double() - v64.sum(1)).abs()
    assert (err <= (k + 1) * U * v64.abs().sum(1)).all()


def test_combine_many_users_of_one_row():
    from sklearn_numba_dpex_b200.common import combine_experts_grad

    n, k, d = 700, 3, 40
    values, grad = torch.randn(5, d), torch.randn(n, d)
    slots = torch.full((n, k), 2, dtype=torch.int32)
    slots[::3, 1] = 4
    weights = torch.rand(n, k)
    out, gv, gw, _, big_v = ref_combine(values, slots, weights, grad)
    got_v, _ = combine_experts_grad(values.cuda(), slots.cuda(), weights.cuda(), grad.cuda())
    assert ((got_v.double().cpu() - gv).abs() <= (n * k + 1) * U * big_v).all()


def _shared_slots(kind, n, k, m, gen):
    """(n, k) rows of m: every row named by some; all the choices on one; rows of 2, 31 to 33, 64 and 65, 127 to 129 and more
    users among rows of one and none."""
    if kind == "random":
        return torch.randint(-1, m, (n, k), generator=gen)
    if kind == "one":
        return torch.full((n, k), m // 2)
    users = torch.ones(m, dtype=torch.int64)
    users[::5] = 0
    for i, c in enumerate((2, 3, 31, 32, 33, 64, 65, 127, 128, 129, 500, n * k // 8)):
        users[i * (m // 13)] = c
    flat = torch.repeat_interleave(torch.arange(m), users)[: n * k]
    flat = torch.cat([flat, torch.full((n * k - flat.numel(),), -1)])
    return flat[torch.randperm(n * k, generator=gen)].view(n, k)


def _grad_of_values(slots, weights, grad, m):
    """In 64 bits, with the sum of the magnitudes and the number of users of each row."""
    there = slots >= 0
    at = slots.long()[there]
    rows = (weights.double()[..., None] * grad.double()[:, None])[there]
    out, big = (torch.zeros(m, grad.shape[1], dtype=torch.float64, device=rows.device) for _ in range(2))
    return out.index_add_(0, at, rows), big.index_add_(0, at, rows.abs()), torch.bincount(at, minlength=m)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,m,d", [(50, 3, 40, 5), (1000, 8, 700, 24), (1024, 8, 8192, 16), (1025, 8, 900, 130), (5003, 7, 9001, 33),
                                     (9000, 8, 40000, 8), (3000, 6, 30, 1100)])
@pytest.mark.parametrize("kind", ["random", "one", "mixed"])
def test_combine_gradient_of_shared_rows(dtype, n, k, m, d, kind):
    """Sums over the users of a row, however they are found: one chain after the other, or by a walk over the choices.
    The order of the sum is that of the choices: the same bits every time, with either workspace."""
    from sklearn_numba_dpex_b200 import _cabi
    from sklearn_numba_dpex_b200.common import combine_experts_grad

    t, gen = TYPES[dtype], torch.Generator().manual_seed(n + m)
    slots = _shared_slots(kind, n, k, m, gen).to(torch.int32).cuda()
    values, grad = torch.randn(m, d, generator=gen).to(t).cuda(), torch.randn(n, d, generator=gen).to(t).cuda()
    weights = torch.randn(n, k, generator=gen).cuda()
    got, got_w = combine_experts_grad(values, slots, weights, grad)
    want, big, users = _grad_of_values(slots, weights, grad, m)
    info = torch.finfo(t)
    bound = (users[:, None] + 1) * U * big + info.eps / 2 * want.abs() * (1 + 2.0 ** -9) + info.smallest_normal * info.eps
    assert ((got.double() - want).abs() <= bound).all()
    for _ in range(3):
        again = combine_experts_grad(values, slots, weights, grad)
        assert torch.equal(again[0], got) and torch.equal(again[1], got_w)
    lib, small = _cabi.lib, torch.empty_like(got).fill_(7)
    size = lib.kmb_combine_experts_grad_workspace_bytes(m)
    assert size < lib.kmb_combine_experts_grad_workspace_bytes_for(m, n, k)
    ws, small_w = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.empty_like(got_w)
    code = {"fp32": _cabi.KMB_F32, "fp16": _cabi.KMB_F16, "bf16": _cabi.KMB_BF16}[dtype]
    p = _cabi.ptr
    _cabi.check(lib.kmb_combine_experts_grad(code, p(values), m, p(slots), p(weights), p(grad), n, k, d, p(small), p(small_w),
                                             p(ws), size, _cabi.stream_ptr()), "kmb_combine_experts_grad")
    assert torch.equal(small, got) and torch.equal(small_w, got_w)


def test_combine_gradient_of_the_longest_chains():
    """A million choices, rows of 2047, 2048 and 2049 users among rows of few and one of half a million."""
    from sklearn_numba_dpex_b200.common import combine_experts_grad

    n, k, d, gen = 1 << 17, 8, 8, torch.Generator().manual_seed(5)
    users = torch.cat([torch.tensor([2047, 2048, 2049, 0, 1, 4095, 500000]), torch.full((100000,), 2), torch.full((3000,), 60)])
    flat = torch.repeat_interleave(torch.arange(users.numel()), users)
    assert flat.numel() <= n * k
    flat = torch.cat([flat, torch.full((n * k - flat.numel(),), -1)])[torch.randperm(n * k, generator=gen)]
    slots, m = flat.view(n, k).to(torch.int32).cuda(), users.numel()
    weights, grad = torch.randn(n, k, generator=gen).cuda(), torch.randn(n, d, generator=gen).cuda()
    got, _ = combine_experts_grad(torch.zeros(m, d, device="cuda"), slots, weights, grad)
    want, big, _ = _grad_of_values(slots, weights, grad, m)
    assert ((got.double() - want).abs() <= (users.cuda()[:, None] + 1) * U * big + 2.0 ** -24 * want.abs()).all()


def test_combine_gradient_costs_what_its_users_cost():
    """4096 rows of 64 users, which took 189 ms where each row meant a walk over all choices; read, their gradients
    are 67 MB."""
    from sklearn_numba_dpex_b200.common import combine_experts_grad

    n, k, d, m = 32768, 8, 64, 4096
    slots = torch.arange(n * k, device="cuda")[torch.randperm(n * k, device="cuda")].view(n, k).remainder(m).to(torch.int32)
    values, weights, grad = torch.randn(m, d, device="cuda"), torch.randn(n, k, device="cuda"), torch.randn(n, d, device="cuda")
    times = []
    for _ in range(3):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        combine_experts_grad(values, slots, weights, grad)
        end.record()
        torch.cuda.synchronize()
        times.append(start.elapsed_time(end))
    assert min(times) < 10, times


# --------------------------------------------------------------------------- used together
def _layer(x, logits, w, w_scales, k, n_experts):
    from sklearn_numba_dpex_b200 import common

    weights, experts = common.route_topk(logits, k)
    slots, rows, offsets = common.expert_slots(experts, n_experts)
    q, scales = common.quantize_rows(x, rows=rows)
    y = common.int8_matmul(q, scales, w, w_scales, offsets=offsets, out_dtype=torch.float32)
    return weights, experts, slots, y, common.combine_experts(y, slots, weights)


def _layer_inputs(n, e, dim, out, seed):
    g = torch.Generator().manual_seed(seed)
    x, logits = torch.randn(n, dim, generator=g), torch.randn(n, e, generator=g)
    logits[n // 2] = float("-inf")                # a padding token in the middle of the batch
    w = torch.randint(-127, 128, (e, out, dim), generator=g, dtype=torch.int8)
    return x.cuda(), logits.cuda(), w.cuda(), (torch.rand(e, out, generator=g) * 0.01).cuda()


def _ref_layer(x, logits, w, w_scales, k):
    """float64, each token by itself; returns the result and what its sums add up to in magnitude."""
    x, logits, w, ws = x.cpu().double().numpy(), logits.cpu().double().numpy(), w.cpu().numpy().astype(np.float64), w_scales.cpu().double().numpy()
    weights, experts = ref_route(logits, k)
    out = np.zeros((x.shape[0], w.shape[1]))
    size = np.zeros_like(out)
    for t in range(x.shape[0]):
        top = np.abs(x[t]).max()
        q = np.rint(x[t] * 127 / top)
        for j in range(k):
            if experts[t, j] >= 0:
                y = (w[experts[t, j]] @ q) * (top / 127) * ws[experts[t, j]]
                out[t] += weights[t, j] * y
                size[t] += weights[t, j] * np.abs(y)
    return out, size


@pytest.mark.parametrize("n,e,dim,out,k", [(1, 8, 64, 96, 2), (37, 16, 200, 130, 4), (300, 5, 129, 257, 3)])
def test_layer_of_experts(n, e, dim, out, k):
    x, logits, w, ws = _layer_inputs(n, e, dim, out, 11)
    weights, experts, slots, y, got = _layer(x, logits, w, ws, k, e)
    want, size = _ref_layer(x, logits, w, ws, k)
    # a share is off by 256 u, a product by 4 u (scales, their product), the sum by k + 1 roundings
    assert (np.abs(got.cpu().double().numpy() - want) <= (256 + 4 + k + 1) * U * size).all()
    # gradients through the sum and the routing, against float64 autograd of the same choice
    leaf, values = logits.clone().requires_grad_(True), y.clone().requires_grad_(True)
    from sklearn_numba_dpex_b200.common import combine_experts, route_topk

    wts, _ = route_topk(leaf, k)
    g = torch.randn(n, out, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    combine_experts(values, slots, wts).backward(g)
    l64, v64 = logits.double().requires_grad_(True), y.double().requires_grad_(True)
    there = experts >= 0
    picked = torch.where(there, l64.gather(1, experts.long().clamp_min(0)), torch.tensor(-1e300, dtype=torch.float64, device="cuda"))
    share = torch.softmax(picked, 1) * there
    rows = torch.where(there[..., None], v64[slots.long().clamp_min(0)], torch.zeros((), dtype=torch.float64, device="cuda"))
    (rows * share[..., None]).sum(1).backward(g.double())
    gw = (rows.detach() * g.double()[:, None]).sum(2).abs().max()
    dots = (rows.detach() * g.double()[:, None]).abs().sum(2).max()
    grad = torch.nan_to_num(l64.grad)
    assert float((leaf.grad.double() - grad).abs().max()) <= 512 * U * float(gw) + 2 * (out + 1) * U * float(dots)
    assert float((values.grad.double() - v64.grad).abs().max()) <= 257 * U * float(g.abs().max())


def test_layer_on_another_stream_and_in_a_graph():
    """The run of operators on a stream of its own, captured, and replayed on new inputs."""
    n, e, dim, out, k = 65, 16, 144, 100, 3
    first, second = _layer_inputs(n, e, dim, out, 21), _layer_inputs(n, e, dim, out, 22)
    want = [_layer(*a, k, e) for a in (first, second)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _layer(*first, k, e)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want[0]):
        assert torch.equal(a, b)
    inputs = [t.clone() for t in first]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _layer(*inputs, k, e)
    for source, expected in ((second, want[1]), (first, want[0])):
        for t, s in zip(inputs, source):
            t.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, expected):
            assert torch.equal(a, b)


def test_layers_in_a_graph_that_forks_and_joins():
    """Calls whose kernels may start early, behind a join of two streams, captured and replayed; and two
    graphs replayed at the same time."""
    n, e, dim, out, k = 300, 8, 256, 192, 2
    args = [_layer_inputs(n, e, dim, out, s) for s in (31, 32)]
    want = [_layer(*a, k, e) for a in args]
    from sklearn_numba_dpex_b200.common import combine_experts

    def forked(a, b):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        first = _layer(*a, k, e)
        with torch.cuda.stream(side):
            second = _layer(*b, k, e)
        torch.cuda.current_stream().wait_stream(side)
        return first, second, combine_experts(first[3], second[2], second[0])

    joined = forked(*args)
    torch.cuda.synchronize()
    graphs, held = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(forked(*args))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for got in (joined, *held):
        for i in (0, 1):
            for x, y in zip(got[i], want[i]):
                assert torch.equal(x, y)
        assert torch.equal(got[2], joined[2])


def test_gradients_in_a_graph():
    from sklearn_numba_dpex_b200.common import combine_experts_grad, route_topk_grad

    x = torch.randn(50, 32, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    from sklearn_numba_dpex_b200.common import route_topk

    w, e = route_topk(x, 4)
    values, grad = torch.randn(200, 24, device="cuda"), torch.randn(50, 24, device="cuda")
    slots = torch.randperm(200, device="cuda").to(torch.int32).view(50, 4)

    def back():
        gv, gw = combine_experts_grad(values, slots, w, grad)
        return gv, route_topk_grad(x, e, gw)

    want = back()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = back()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held[0], want[0]) and torch.equal(held[1], want[1])


def test_refusals_on_the_gpu():
    from sklearn_numba_dpex_b200.common import combine_experts, expert_slots, route_topk, route_topk_grad

    x = torch.randn(4, 8, device="cuda")
    for bad in (dict(k=0), dict(k=9), dict(k=2, scoring="relu"), dict(k=2, n_groups=3), dict(k=2, n_groups=0),
                dict(k=5, n_groups=2, topk_groups=1), dict(k=2, n_groups=2, topk_groups=3), dict(k=2, n_groups=2, group_best=3),
                dict(k=1, n_groups=8, topk_groups=2, group_best=2), dict(k=2, bias=torch.zeros(7, device="cuda")),
                dict(k=2, bias=torch.zeros(8)), dict(k=2, bias=torch.zeros(8, device="cuda", dtype=torch.float64))):
        with pytest.raises(ValueError):
            route_topk(x, **bad)
    with pytest.raises(ValueError):
        route_topk(x.double(), 2)
    with pytest.raises(ValueError):
        route_topk(torch.randn(4, 1025, device="cuda"), 2)
    with pytest.raises(ValueError):
        route_topk(torch.randn(4, 64, device="cuda"), 33)
    w, e = route_topk(x, 2)
    with pytest.raises(ValueError):
        route_topk_grad(x, e.long(), w)
    with pytest.raises(ValueError):
        route_topk_grad(x, e[:3], w[:3])
    with pytest.raises(ValueError):
        expert_slots(e, 1025)
    with pytest.raises(ValueError):
        expert_slots(e, 0)
    with pytest.raises(ValueError):
        expert_slots(e.float(), 8)
    with pytest.raises(ValueError):
        combine_experts(x, e, w[:, :1])
    with pytest.raises(ValueError):
        combine_experts(x.double(), e, w)
    assert torch.isfinite(route_topk(x, 2)[0]).all()


def test_transforms_are_refused():
    """Nothing that carries a tangent, or stands for other tensors, loses it in silence."""
    import torch.autograd.forward_ad as forward

    from sklearn_numba_dpex_b200 import common

    x, slots, w = torch.randn(4, 8, device="cuda"), torch.zeros(3, 2, dtype=torch.int32, device="cuda"), torch.ones(3, 2, device="cuda")
    q, s = common.quantize_rows(x)
    calls = [lambda t: common.route_topk(t, 2)[0], lambda t: common.route_topk(x, 2, bias=t[0])[0],
             lambda t: common.route_topk_grad(x, slots[:1].repeat(4, 1), t[:, :2]), lambda t: common.quantize_rows(t)[1],
             lambda t: common.combine_experts(t, slots, w), lambda t: common.combine_experts(x, slots, t[:3, :2].contiguous()),
             lambda t: common.combine_experts_grad(x, slots, w, t[:3])[0], lambda t: common.int8_matmul(q, t[:, 0].contiguous(), q, s),
             lambda t: common.int8_matmul(q, s, q, s, bias=t[:, 0].contiguous())]
    for call in calls:
        with forward.dual_level():
            dual = forward.make_dual(x, torch.ones_like(x))
            with pytest.raises((NotImplementedError, RuntimeError)):
                call(dual)
        with pytest.raises((NotImplementedError, RuntimeError)):
            torch.func.jvp(call, (x,), (x,))
        with pytest.raises((NotImplementedError, RuntimeError)):
            torch.vmap(call)(x[None].repeat(3, 1, 1))
        call(x)
    leaf = x.clone().requires_grad_(True)
    with forward.dual_level(), pytest.raises((NotImplementedError, RuntimeError)):
        common.route_topk(forward.make_dual(leaf, torch.ones_like(x)), 2)


def test_views_that_stand_for_negated_values():
    """The imaginary part of a conjugate is a view of memory with the other sign: of one column it is contiguous too."""
    from sklearn_numba_dpex_b200 import common

    z = torch.randn(6, 1, dtype=torch.complex64, device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    q, _ = common.quantize_rows(torch.ones(6, 1, device="cuda"))
    slots, w = torch.arange(6, dtype=torch.int32, device="cuda")[:, None], torch.ones(6, 1, device="cuda")
    for view in (z[:1].conj().imag, z.conj().imag, torch._neg_view(z.real.contiguous())):
        assert view.is_neg()
        plain, n = view.resolve_neg().clone(), view.shape[0]
        for call in (lambda t: common.route_topk(t, 1, scoring="sigmoid", renormalize=False)[0], lambda t: common.quantize_rows(t)[0],
                     lambda t: common.combine_experts(t, slots[:n], w[:n]), lambda t: common.combine_experts(w[:n], slots[:n], t)):
            assert torch.equal(call(view), call(plain))
        with pytest.raises(ValueError, match="contiguous"):
            common.int8_matmul(q[:n], view[:, 0], q, w[:, 0])
    eights = torch.full((4, 16), 8, dtype=torch.int8, device="cuda")
    one = torch.ones(4, device="cuda")
    assert (common.int8_matmul(torch._neg_view(eights), one, eights, one) == -1024).all()
