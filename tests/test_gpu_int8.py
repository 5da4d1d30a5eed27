"""Products in 8-bit integers and the quantisation of rows against exact arithmetic.

Tolerance of a product: the sum is an exact whole number; its conversion to 32 bits, the product of the
scales, their product with the sum and the bias's addition round once each (4 u, u = 2^-24, of the
magnitudes), and results in 16 bits once more (half a step of their type).
"""
import os
import subprocess
import sys
import textwrap
from fractions import Fraction

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


# --------------------------------------------------------------------------- quantisation
def ref_quantize(x):
    x = x.double().numpy()
    top = np.abs(x).max(1, keepdims=True)
    return np.rint(x * 127 / np.where(top == 0, 1, top)).astype(np.int8), top[:, 0] / 127


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d", [(1, 1), (3, 7), (5, 16), (4, 255), (9, 512), (3, 513), (7, 2048), (2, 2049), (3, 4100), (2, 8192),
                                 (2, 20000)])
def test_quantize_rows(dtype, n, d):
    from sklearn_numba_dpex_b200.common import quantize_rows

    x = (torch.randn(n, d, generator=torch.Generator().manual_seed(d)) * 3).to(TYPES[dtype])
    if n > 2:
        x[1] = 0
    q, s = quantize_rows(x.cuda())
    assert q.dtype == torch.int8 and s.dtype == torch.float32 and q.shape == x.shape and q.stride(0) % 16 == 0
    want_q, want_s = ref_quantize(x)
    np.testing.assert_array_equal(q.cpu().numpy(), want_q)
    np.testing.assert_allclose(s.cpu().numpy(), want_s, rtol=U, atol=0)


def test_quantize_rounds_the_exact_quotient():
    """Values on and one step beside the borders of the rounding, for maxima of every size."""
    from sklearn_numba_dpex_b200.common import quantize_rows

    rows = []
    for top in (127.0, 1.0, 0.3, 3.1e-5, 1e-38, 1e-44, 3.4e38, 254.0, 1.9921875):
        top = np.float32(top)
        half = (np.arange(1, 254, 2) * np.float64(top) / 254).astype(np.float32)
        row = np.concatenate([[top], half, np.nextafter(half, np.float32(0)), np.nextafter(half, top), -half])
        rows.append(np.clip(row, -top, top))
    x = np.stack(rows).astype(np.float32)
    q, _ = quantize_rows(torch.from_numpy(x).cuda())
    want = [[round(Fraction(float(v)) * 127 / Fraction(float(np.abs(r).max()))) for v in r] for r in x]   # half to even
    np.testing.assert_array_equal(q.cpu().numpy(), np.array(want))


def test_quantize_takes_rows_and_marks_broken_ones():
    from sklearn_numba_dpex_b200.common import int8_matmul, quantize_rows

    x = torch.randn(6, 40)
    x[2, 3], x[4, 39] = float("nan"), float("-inf")
    rows = torch.tensor([5, -1, 2, 0, 0, 6, 4, 1], dtype=torch.int32)
    q, s = quantize_rows(x.cuda(), rows=rows.cuda())
    want_q, want_s = ref_quantize(x[[5, 0, 0, 1]])
    np.testing.assert_array_equal(q.cpu().numpy()[[0, 3, 4, 7]], want_q)
    np.testing.assert_allclose(s.cpu().numpy()[[0, 3, 4, 7]], want_s, rtol=U)
    assert (q[[1, 2, 5, 6]] == 0).all() and (s[[1, 5]] == 0).all() and torch.isnan(s[[2, 6]]).all()
    w, ws = quantize_rows(torch.randn(9, 40).cuda())
    y = int8_matmul(q, s, w, ws)
    assert torch.isnan(y[[2, 6]]).all() and torch.isfinite(y[[0, 1, 3, 4, 5, 7]]).all() and (y[1] == 0).all()
    empty, es = quantize_rows(x.cuda()[:0])
    assert empty.shape == (0, 40) and es.shape == (0,)


# --------------------------------------------------------------------------- product
def _operands(m, n, d, g=None, seed=0, bias=False):
    gen = torch.Generator().manual_seed(seed)
    lead = (g, n) if g else (n,)
    a = torch.randint(-128, 128, (m, d), generator=gen, dtype=torch.int8)
    b = torch.randint(-128, 128, (*lead, d), generator=gen, dtype=torch.int8)
    sa, sb = torch.rand(m, generator=gen) + 0.1, (torch.rand(lead, generator=gen) + 0.1) * 1e-4
    return a, sa, b, sb, torch.randn(lead, generator=gen) if bias else None


def ref_product(a, sa, b, sb, bias):
    acc = torch.from_numpy(a.numpy().astype(np.int64) @ b.numpy().astype(np.int64).T).double() if a.shape[1] < 4000 else \
        (a.double() @ b.double().T)                       # exact: below 2^53
    prod = acc * sa.double()[:, None] * sb.double()
    return (prod if bias is None else prod + bias.double()), prod.abs() + (0 if bias is None else bias.double().abs())


def _check(out, want, size):
    t = out.dtype
    err = (out.double().cpu() - want).abs()
    assert (err <= 4 * U * size + torch.finfo(t).eps / 2 * want.abs() * (1 + 4 * U) + torch.finfo(t).smallest_normal
            * torch.finfo(t).eps).all(), float(err.max())


@pytest.mark.parametrize("m,n,d", [(1, 1, 1), (1, 128, 16), (2, 300, 31), (15, 7, 32), (16, 129, 33), (17, 128, 127), (33, 200, 128),
                                   (64, 127, 129), (65, 256, 255), (128, 130, 1000), (130, 64, 96), (257, 300, 160), (300, 512, 64),
                                   (513, 129, 2049), (1, 4096, 4096), (2000, 1500, 272), (300, 200, 3000),
                                   (100, 256, 2100), (33, 128, 5000), (20, 1000, 600),
                                   (5000, 1000, 400), (4000, 2700, 136), (100, 19000, 130), (2561, 1921, 1300)])
@pytest.mark.parametrize("out", TYPES)
def test_product_sizes(m, n, d, out):
    from sklearn_numba_dpex_b200.common import int8_matmul

    for bias in (False, True):
        ops = _operands(m, n, d, seed=m + n + d, bias=bias)
        want, size = ref_product(*ops)
        a, sa, b, sb, c = [None if t is None else t.cuda() for t in ops]
        got = int8_matmul(a, sa, b, sb, bias=c, out_dtype=TYPES[out])
        assert got.dtype == TYPES[out] and got.shape == (m, n)
        _check(got, want, size)


# a tile to a CTA, clusters that share one, pairs of CTAs, groups
@pytest.mark.parametrize("m,n,d,g", [(3, 8, 32, None), (300, 512, 64, None), (1, 4096, 4096, None), (2, 4096, 4096, None), (40, 300, 3000, None), (4000, 2700, 136, None),
                                     (700, 130, 48, 5)])
@pytest.mark.parametrize("out", TYPES)
def test_product_of_scales_far_from_one(m, n, d, g, out):
    """Scales whose product leaves the range of 32 bits, or its full precision, where the result does not.  A result
    beyond the type's greatest value is an infinity; one below its normal numbers is off by half a step there."""
    from sklearn_numba_dpex_b200.common import int8_matmul

    a, sa, b, sb, c = _operands(m, n, d, g=g, seed=d, bias=True)
    gen = torch.Generator().manual_seed(m)
    a[0] = 0                                  # a sum of zero stays the bias alone
    sa = 10.0 ** (torch.rand(m, generator=gen, dtype=torch.float64) * 70 - 36)
    sb = 10.0 ** (torch.rand(sb.shape, generator=gen, dtype=torch.float64) * 70 - 36)
    sa, sb, c = sa.float(), sb.float(), torch.where(torch.rand(c.shape, generator=gen) < 0.5, torch.zeros(()), c * 1e-30)
    sa[0] = 1e30
    t = TYPES[out]
    off = None if g is None else torch.tensor([i * m // g for i in range(g + 1)], dtype=torch.int32)
    if g is None:
        want, size = ref_product(a, sa, b, sb, c)
    else:
        parts = [ref_product(a[off[i]:off[i + 1]], sa[off[i]:off[i + 1]], b[i], sb[i], c[i]) for i in range(g)]
        want, size = (torch.cat([p[j] for p in parts]) for j in (0, 1))
    got = int8_matmul(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), bias=c.cuda(), offsets=None if g is None else off.cuda(), out_dtype=t).double().cpu()
    info = torch.finfo(t)
    tiny = max(info.smallest_normal * info.eps, 2.0 ** -149)
    bound = 4 * U * size + info.eps / 2 * want.abs() * (1 + 4 * U) + tiny
    over = want.abs() + 4 * U * size > info.max        # may round to an infinity
    must = want.abs() - 4 * U * size > info.max * (1 + info.eps)
    assert not torch.isnan(got).any() and not torch.isinf(got[~over]).any() and torch.isinf(got[must]).all()
    assert ((got - want).abs() <= bound)[~over].all()
    assert (got[0].abs() <= 1e-20).all()


def test_product_of_the_longest_rows_does_not_overflow():
    from sklearn_numba_dpex_b200.common import int8_matmul

    d = 131071
    a = torch.full((3, d), -128, dtype=torch.int8, device="cuda")
    b = torch.full((2, d), -128, dtype=torch.int8, device="cuda")
    a[1], b[1] = 127, 127
    one = torch.ones(3, device="cuda")
    got = int8_matmul(a, one, b, one[:2], out_dtype=torch.float32).double().cpu()
    want = torch.tensor([[128 * 128, -128 * 127], [-128 * 127, 127 * 127], [128 * 128, -128 * 127]], dtype=torch.float64) * d
    assert ((got - want).abs() <= 4 * U * want.abs()).all()


@pytest.mark.parametrize("d", [48, 50])
def test_product_of_slices_and_odd_pitches(d):
    """Rows at a pitch, at an odd address, transposed: the same numbers as their contiguous copies."""
    from sklearn_numba_dpex_b200.common import int8_matmul

    a, sa, b, sb, _ = [None if t is None else t.cuda() for t in _operands(20, 40, d)]
    want = int8_matmul(a, sa, b, sb, out_dtype=torch.float32)
    wide = torch.zeros(20, 160, dtype=torch.int8, device="cuda")
    wide[:, 32:32 + d] = a
    odd = torch.zeros(40, 99, dtype=torch.int8, device="cuda")
    odd[:, 3:3 + d] = b
    for aa in (wide[:, 32:32 + d], a.t().contiguous().t()):
        for bb in (odd[:, 3:3 + d], b.t().contiguous().t()):
            assert torch.equal(int8_matmul(aa, sa, bb, sb, out_dtype=torch.float32), want)


def _group_offsets(kind, g, m, rng):
    cuts = np.sort(rng.integers(0, m + 1, g + 1))
    if kind == "whole":
        cuts[0], cuts[-1] = 0, m
    elif kind == "tail":
        cuts = cuts * 2 // 3
        cuts[0] = 0
    elif kind == "empty":
        cuts[:] = 0
    elif kind == "one":
        cuts[:] = 0
        cuts[g // 2 + 1:] = m
    elif kind == "late":
        cuts = m - (m - cuts) // 2          # the first rows belong to nobody
        cuts[-1] = m
    return cuts.astype(np.int32)


@pytest.mark.parametrize("g,m,n,d", [(1, 5, 20, 40), (3, 50, 129, 64), (8, 333, 200, 100), (64, 300, 70, 144), (40, 3000, 130, 48),
                                     (255, 700, 16, 32), (1024, 2048, 9, 16), (1023, 10, 9, 17), (4, 4000, 64, 272),
                                     (4, 40, 130, 2048), (2, 300, 256, 4096), (3, 200, 100, 1500), (5, 5000, 700, 400),
                                     (20, 2500, 1100, 150)])
@pytest.mark.parametrize("kind", ["whole", "tail", "empty", "one"])
def test_product_by_group(g, m, n, d, kind):
    from sklearn_numba_dpex_b200.common import int8_matmul

    off = _group_offsets(kind, g, m, np.random.default_rng(g + m))
    ops = _operands(m, n, d, g=g, seed=g, bias=g % 2 == 0)
    a, sa, b, sb, c = [None if t is None else t.cuda() for t in ops]
    got = int8_matmul(a, sa, b, sb, bias=c, offsets=torch.from_numpy(off).cuda(), out_dtype=torch.float32)
    want, size = torch.zeros(m, n, dtype=torch.float64), torch.zeros(m, n, dtype=torch.float64)
    for e in range(g):
        r = slice(off[e], off[e + 1])
        if off[e + 1] > off[e]:
            want[r], size[r] = ref_product(ops[0][r], ops[1][r], ops[2][e], ops[3][e], None if c is None else ops[4][e])
    _check(got, want, size)
    assert (got[off[-1]:] == 0).all()


@pytest.mark.parametrize("d", [50, 130, 2056])
def test_weights_as_quantize_rows_lays_them_out(d):
    """Rows at quantize_rows' pitch, seen as a matrix for each group, are read in place."""
    from sklearn_numba_dpex_b200.common import int8_matmul, quantize_rows

    g, n, m = 3, 37, 90
    gen = torch.Generator("cuda").manual_seed(d)
    w, ws = quantize_rows(torch.randn(g * n, d, device="cuda", generator=gen))
    x, xs = quantize_rows(torch.randn(m, d, device="cuda", generator=gen))
    assert w.stride(0) % 16 == 0 and w.stride(0) - d <= max(15, d // 8)
    off = torch.tensor([0, 10, 60, m], dtype=torch.int32, device="cuda")
    got = int8_matmul(x, xs, w.view(g, n, d), ws.view(g, n), offsets=off, out_dtype=torch.float32)
    for e in range(g):
        r = slice(int(off[e]), int(off[e + 1]))
        want, size = ref_product(x.cpu()[r], xs.cpu()[r], w.cpu().view(g, n, d)[e], ws.cpu().view(g, n)[e], None)
        _check(got[r], want, size)


def test_product_by_group_that_begins_late():
    """The rows ahead of the first group become zeros, as those behind the last do."""
    from sklearn_numba_dpex_b200.common import int8_matmul

    off = _group_offsets("late", 5, 200, np.random.default_rng(0))
    ops = _operands(200, 30, 64, g=5)
    a, sa, b, sb, _ = [None if t is None else t.cuda() for t in ops]
    got = int8_matmul(a, sa, b, sb, offsets=torch.from_numpy(off).cuda(), out_dtype=torch.float32)
    for e in range(5):
        r = slice(off[e], off[e + 1])
        if off[e + 1] > off[e]:
            want, size = ref_product(ops[0][r], ops[1][r], ops[2][e], ops[3][e], None)
            _check(got[r], want, size)
    assert off[0] > 0 and (got[: off[0]] == 0).all()


@pytest.mark.parametrize("g,m,n,d", [(3, 50, 129, 64), (64, 300, 70, 144), (1024, 700, 9, 16), (20, 2500, 1100, 150)])
def test_product_of_wrong_offsets_stays_in_its_rows(g, m, n, d):
    """Offsets that go up and down, or lie outside the rows, give no right product, but touch nothing else: the memory
    around the result, and the next product."""
    from sklearn_numba_dpex_b200 import _cabi
    from sklearn_numba_dpex_b200.common import check_int8_waits, int8_matmul

    a, sa, b, sb, _ = [None if t is None else t.cuda() for t in _operands(m, n, d, g=g)]
    good = torch.from_numpy(_group_offsets("whole", g, m, np.random.default_rng(g))).cuda()
    want = int8_matmul(a, sa, b, sb, offsets=good, out_dtype=torch.float32)
    lda = (d + 15) // 16 * 16
    ap, bp = torch.zeros(m, lda, dtype=torch.int8, device="cuda"), torch.zeros(g, n, lda, dtype=torch.int8, device="cuda")
    ap[:, :d], bp[..., :d] = a, b
    for kind in range(4):
        off = torch.from_numpy(np.random.default_rng(kind).integers(-m, 2 * m + 1, g + 1).astype(np.int32))
        if kind == 0:
            off = torch.arange(g + 1, dtype=torch.int32).remainder(2) * m           # every row once for each second group
        elif kind == 1:
            off = torch.arange(g, -1, -1, dtype=torch.int32)
        off, held = off.cuda(), torch.full((m + 2, n), 7.0, device="cuda")
        p = _cabi.ptr
        _cabi.check(_cabi.lib.kmb_int8_matmul(_cabi.KMB_F32, p(ap), lda, p(sa), p(bp), lda, p(sb), None, p(off), g, p(held[1:]),
                                              m, n, d, _cabi.stream_ptr()), "kmb_int8_matmul")
        torch.cuda.synchronize()
        assert (held[0] == 7).all() and (held[-1] == 7).all()
        check_int8_waits()
    assert torch.equal(int8_matmul(a, sa, b, sb, offsets=good, out_dtype=torch.float32), want)


def test_product_whose_output_passes_32_bit_offsets():
    from sklearn_numba_dpex_b200.common import int8_matmul

    m, n, d = 70000, 40000, 16          # 2.8e9 values
    a, sa, b, sb, _ = [None if t is None else t.cuda() for t in _operands(m, n, d)]
    got = int8_matmul(a, sa, b, sb)
    rows, cols = torch.tensor([0, 1, 53687, 53688, 65535, 69999]), torch.tensor([0, 127, 128, 29999, 39999])
    want, size = ref_product(a.cpu()[rows], sa.cpu()[rows], b.cpu()[cols], sb.cpu()[cols], None)
    _check(got[rows.cuda()][:, cols.cuda()], want, size)


def test_two_products_at_once():
    from sklearn_numba_dpex_b200.common import int8_matmul

    sets = [[None if t is None else t.cuda() for t in _operands(400 + 100 * i, 700, 512, seed=i)][:4] for i in range(4)]
    want = [int8_matmul(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(5):
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(int8_matmul(*s))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % 4])


def test_refusals():
    from sklearn_numba_dpex_b200.common import int8_matmul, quantize_rows

    a, sa, b, sb, _ = [None if t is None else t.cuda() for t in _operands(4, 6, 32)]
    off = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    for args, kw in [((a.float(), sa, b, sb), {}), ((a, sa.double(), b, sb), {}), ((a, sa[:3], b, sb), {}), ((a, sa, b[:, :16], sb), {}),
                     ((a, sa, b, sb), dict(out_dtype=torch.float64)), ((a, sa, b, sb), dict(offsets=off)), ((a, sa, b[None], sb), {}),
                     ((a, sa, b.view(2, 3, 32), sb.view(2, 3)), dict(offsets=off.long())),
                     ((a, sa, b.view(2, 3, 32), sb.view(2, 3)), dict(offsets=off[:2])),
                     ((a, sa, b, sb), dict(bias=torch.zeros(5, device="cuda"))), ((a.cpu(), sa, b, sb), {}),
                     ((torch.zeros(1, 131072, dtype=torch.int8, device="cuda"), sa[:1],
                       torch.zeros(1, 131072, dtype=torch.int8, device="cuda"), sb[:1]), {})]:
        with pytest.raises(ValueError):
            int8_matmul(*args, **kw)
    for args, kw in [((a,), {}), ((sa,), {}), ((torch.zeros(3, 4, device="cuda").double(),), {}), ((torch.zeros(3, 4, device="cuda"),), dict(rows=off.long())),
                     ((torch.zeros(3, 4),), {})]:
        with pytest.raises(ValueError):
            quantize_rows(*args, **kw)
    assert int8_matmul(a[:0], sa[:0], b, sb).shape == (0, 6)


def test_operands_that_require_a_gradient_are_refused():
    from sklearn_numba_dpex_b200.common import int8_matmul, quantize_rows

    x, bias = torch.randn(4, 32, device="cuda", requires_grad=True), torch.zeros(4, device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="x requires a gradient"):
        quantize_rows(x)
    with torch.no_grad():
        q, s = quantize_rows(x)
    assert torch.equal(quantize_rows(x.detach())[0], q)
    t = s.clone().requires_grad_(True)
    for args, kw, name in (((q, t, q, s), {}, "a_scales"), ((q, s, q, t), {}, "b_scales"), ((q, s, q, s), dict(bias=bias), "bias")):
        with pytest.raises(ValueError, match=name + " requires a gradient"):
            int8_matmul(*args, **kw)
        with torch.no_grad():
            want = int8_matmul(*args, **kw)
        with torch.inference_mode():
            assert torch.equal(int8_matmul(*args, **kw), want)
    assert not int8_matmul(q, s, q, s).requires_grad


CHILD = textwrap.dedent("""
    import os, sys, time
    import torch
    sys.path.insert(0, os.getcwd())
    from sklearn_numba_dpex_b200._cabi import KmbError
    from sklearn_numba_dpex_b200.common import check_int8_waits, int8_matmul

    m, n, d = (int(v) for v in sys.argv[1:])
    g = torch.Generator(device="cuda").manual_seed(5)
    a = torch.randint(-128, 128, (m, d), device="cuda", generator=g, dtype=torch.int8)
    b = torch.randint(-128, 128, (n, d), device="cuda", generator=g, dtype=torch.int8)
    sa, sb = torch.ones(m, device="cuda"), torch.ones(b.shape[0], device="cuda")
    want = int8_matmul(a, sa, b, sb, out_dtype=torch.float32)
    check_int8_waits()
    os.environ["KMB_TC_TEST_STALL"], os.environ["KMB_TC_TIMEOUT_MS"] = "1", "200"
    t0 = time.time()
    y = int8_matmul(a, sa, b, sb, out_dtype=torch.float32)
    try:
        check_int8_waits()
    except KmbError as exc:
        assert "bounded wait" in str(exc), exc
    else:
        raise SystemExit("the stalled product did not report its wait")
    assert time.time() - t0 < 20.0
    bad = torch.isnan(y)
    assert bad.any() and torch.equal(y[~bad], want[~bad])        # what was not computed is NaN, not garbage
    os.environ["KMB_TC_TEST_STALL"], os.environ["KMB_TC_TIMEOUT_MS"] = "0", "0"
    check_int8_waits()                                           # reported once, then clear
    assert torch.equal(int8_matmul(a, sa, b, sb, out_dtype=torch.float32), want)
    check_int8_waits()
    print("stall-ok")
""")


# three tiles per CTA, and few tiles that clusters of CTAs share
@pytest.mark.parametrize("m,n,d", [(1, 56832, 256), (20, 56832, 256), (40, 56832, 256), (100, 56832, 256), (256, 56832, 256),
                                   (1, 4096, 4096), (100, 300, 3000), (256, 256, 2048), (700, 16000, 300), (128, 58000, 300),
                                   (16, 148 * 128 * 7, 128)])
def test_wait_that_runs_out_is_reported_and_the_context_survives(m, n, d):
    """No GPU fault is involved: the loading warp stops early, the others give up after 200 ms."""
    proc = subprocess.run([sys.executable, "-c", CHILD, str(m), str(n), str(d)], cwd=ROOT, capture_output=True, text=True, timeout=600)
    tail = (proc.stdout + proc.stderr)[-3000:]
    assert proc.returncode == 0, tail
    assert "stall-ok" in proc.stdout, tail
