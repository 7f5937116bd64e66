"""Grouped operators (affine maps, score blocks, float64 moments) and the 4-bit gallery against plain float64
implementations, group by group.

Tolerances, with u = 2^-24 (half a step of fp32, relative).  A product of two fp16 pairs differs from the
product of the numbers by at most 2^-22 of its size for each operand that is a pair and 2^-22 for the dropped
partial product; where the second fp16 is below its normal range an operand is off by at most 2^-25 of the
scaled unit, i.e. by 2^-33 of the largest magnitude that set the scale (rows of the affine map) or 2^-39 (all
others).  Every one of the three sums of d products rounds at most d times: 3 d u of the sum of magnitudes.  That
holds for every element; the root mean square of the errors is held to the size that independent roundings give,
sqrt(3 d) u + 2^-22 of the root of the summed squares, times four, which a lost half of a pair (2^-12) exceeds by
two orders of magnitude."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _torch():
    import torch

    return torch


def _rng(seed):
    return np.random.RandomState(seed)


def _offsets(sizes):
    return np.concatenate([[0], np.cumsum(sizes)]).astype(int)


def _product_bound(x, w, floor_x, floor_w=2.0 ** -39):
    """(bound of |x @ w - computed| per element, rms scale) for x [n, d], w [d, m] in float64."""
    d = x.shape[1]
    ax, aw = np.abs(x), np.abs(w)
    bound = (3 * 2.0 ** -22 + 3 * d * U) * (ax @ aw)
    bound += floor_x * ax.max(1, initial=0)[:, None] * aw.sum(0)[None, :]
    bound += floor_w * aw.max(0, initial=0)[None, :] * ax.sum(1)[:, None]
    rms = 4 * (math.sqrt(3 * d) * U + 2.0 ** -22) * np.sqrt((x * x) @ (w * w))
    return bound, rms


def _assert_close(got, want, bound, rms=None):
    got = got.double().cpu().numpy() if hasattr(got, "cpu") else got
    err = np.abs(got - want)
    bad = ~(err <= bound)
    assert not bad.any(), "worst %g of its bound at %s" % (np.nanmax(err[bad] / bound[bad]), np.argwhere(bad)[:5])
    if rms is not None and want.size > 64:
        ok = rms > 0
        assert np.sqrt(np.mean((err[ok] / rms[ok]) ** 2)) <= 1.0


# ---------------------------------------------------------------------------------------------- affine
def _affine_ref(x, W, b, sizes, order, lnorm, dims=None):
    n, m = x.shape[0], W.shape[2]
    y, bound, rms = np.zeros((n, m)), np.zeros((n, m)), np.zeros((n, m))
    off = _offsets(sizes)
    for e in range(len(sizes)):
        rows = np.arange(off[e], off[e + 1]) if order is None else order[off[e]:off[e + 1]]
        if len(rows) == 0:
            continue
        z = x[rows] @ W[e] + b[e]
        B, R = _product_bound(x[rows], W[e], 2.0 ** -33)
        B = B + 2 * U * (np.abs(z) + np.abs(b[e]))
        R = R + 2 * U * (np.abs(z) + np.abs(b[e]))
        if lnorm:
            norm = np.sqrt((z * z).sum(1, keepdims=True))
            f = math.sqrt(m if dims is None else dims[e]) / (norm + 1e-10)
            drift = np.sqrt((B * B).sum(1, keepdims=True)) / np.maximum(norm, 1e-300)
            # the sum of squares rounds m times, half of that reaches the norm; a few roundings of the factor
            z, B, R = z * f, B * f + np.abs(z * f) * (drift + (m / 2 + 8) * U), R * f + np.abs(z * f) * 8 * U
        y[rows], bound[rows], rms[rows] = z, B, R
    return y, bound, rms


AFFINE = [
    # sizes, d_in, d_out, lnorm, ordered
    ([1], 1, 1, False, False),
    ([3, 0, 1], 5, 3, True, False),
    ([2, 1, 1, 2, 1], 512, 200, True, True),
    ([16, 17, 0, 15, 1], 33, 16, False, True),
    ([64, 65, 63, 1, 0, 129], 96, 77, True, False),
    ([300, 0, 0, 41], 200, 150, True, True),
    ([1100, 1700], 130, 257, False, False),
    ([90, 20], 100, 300, True, True),
    ([1500, 1029], 515, 64, True, False),
    ([7, 9], 1024, 512, True, False),
    ([0, 0], 8, 8, True, False),
    # many rows a group: tiles of 128
    ([40000, 0, 3000], 64, 20, True, False),
    ([2500, 1, 2700], 67, 256, True, True),
    ([1001, 1500], 190, 270, True, False),
    ([36000], 129, 33, False, True),
    ([3000, 1300, 2500], 321, 130, True, False),
    # tiles of 64 over rows of several chunks
    ([60, 21, 100], 700, 100, True, True),
    ([30, 50, 1, 64], 300, 200, False, False),
]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("case", range(len(AFFINE)))
def test_affine(case, dtype):
    torch = _torch()
    from hyperion_amd import engine

    sizes, d, m, lnorm, ordered = AFFINE[case]
    r = _rng(case)
    n, E = sum(sizes), len(sizes)
    x = torch.from_numpy(r.randn(n, d) * np.exp(r.uniform(-2, 2, d))).to("cuda").to(getattr(torch, dtype))
    W = (r.randn(E, d, m) * np.exp(r.uniform(-2, 2, m))).astype(np.float32)
    b = r.randn(E, m).astype(np.float32)
    order = r.permutation(n) if ordered else None
    groups = engine.RowGroups(sizes, order=order)
    y = engine.grouped_affine(x, groups, engine.AffineBank(W, b), lnorm=lnorm)
    assert y.shape == (n, m) and y.dtype == torch.float32
    want, bound, rms = _affine_ref(x.double().cpu().numpy(), W.astype(float), b.astype(float), sizes, order, lnorm)
    _assert_close(y, want, bound, rms)


@pytest.mark.parametrize("sizes", [[50, 3, 200], [2, 1, 9], [1300, 1001, 1200]])
def test_affine_scales(sizes):
    """Rows and columns of very different magnitudes, zero rows, and rows that grow along their coordinates (the
    scale of a row is lowered while it is read)."""
    torch = _torch()
    from hyperion_amd import engine

    r = _rng(5)
    d, m = 700, 40
    n = sum(sizes)
    x = r.randn(n, d) * 10.0 ** r.randint(-25, 26, n)[:, None]
    x[::7] = 0
    x[1::7] *= np.exp(np.linspace(0, 30, d))  # a factor of 1e13 along the row
    x[2::7, :600] = 0
    x = x.astype(np.float32).astype(float)
    W = (r.randn(3, d, m) * 10.0 ** r.randint(-10, 11, (3, 1, m))).astype(np.float32).astype(float)
    y = engine.grouped_affine(torch.from_numpy(x).float().cuda(), engine.RowGroups(sizes), engine.AffineBank(W))
    want, bound, _ = _affine_ref(x, W, np.zeros((3, m)), sizes, None, False)
    bound += 2.0 ** -149
    top = float(np.finfo(np.float32).max)
    y = y.double().cpu().numpy()
    fits = np.abs(want) + bound <= top
    _assert_close(y[fits], want[fits], bound[fits])
    # what fp32 cannot hold comes out as an infinity (or, next to the border, as the largest number)
    over = ~fits & np.isfinite(want)
    assert fits.mean() > 0.8 and (np.abs(y[over]) >= top * (1 - 1e-3)).all()


@pytest.mark.parametrize("sizes", [[70, 30], [2000, 1200]])
def test_affine_non_finite_rows_stay_alone(sizes):
    torch = _torch()
    from hyperion_amd import engine

    r = _rng(6)
    n = sum(sizes)
    x = r.randn(n, 70).astype(np.float32)
    clean = torch.from_numpy(x).cuda()
    bad = clean.clone()
    bad[3, 5], bad[64, 0], bad[99, 69] = float("nan"), float("inf"), -float("inf")
    bank = engine.AffineBank(r.randn(2, 70, 30))
    groups = engine.RowGroups(sizes)
    for lnorm in (False, True):
        a, b = (engine.grouped_affine(t, groups, bank, lnorm=lnorm) for t in (clean, bad))
        rows = torch.ones(n, dtype=torch.bool)
        rows[[3, 64, 99]] = False
        assert torch.equal(a[rows.cuda()], b[rows.cuda()])
        assert torch.isnan(b[~rows.cuda()]).all()


def test_affine_strides_out_and_unlisted_rows():
    """Odd row pitch and start, rows outside every group, a caller's result with room around it."""
    torch = _torch()
    from hyperion_amd import engine

    r = _rng(7)
    d, m, sizes = 37, 21, [5, 0, 18]
    n = 40
    order = r.permutation(n)[:23]
    W, b = r.randn(3, d, m).astype(np.float32), r.randn(3, m).astype(np.float32)
    bank, groups = engine.AffineBank(W, b), engine.RowGroups(sizes, order=order)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        wide = torch.full((n, d + 4), float("nan"), dtype=dtype, device="cuda")
        wide[:, 3:3 + d] = torch.from_numpy(r.randn(n, d)).cuda().to(dtype)
        x = wide[:, 3:3 + d]
        want, bound, rms = _affine_ref(x.double().cpu().numpy(), W.astype(float), b.astype(float), sizes, order, True)
        y = engine.grouped_affine(x, groups, bank, lnorm=True)
        _assert_close(y, want, bound, rms)  # rows of no group are zero
        buf = torch.full((n, 32), 7.0, device="cuda")
        out = buf[:, 4:4 + m]
        res = engine.grouped_affine(x, groups, bank, lnorm=True, out=out)
        assert res is out
        listed = np.zeros(n, bool)
        listed[order] = True
        _assert_close(out[torch.from_numpy(listed).cuda()], want[listed], bound[listed])
        assert (out[torch.from_numpy(~listed).cuda()] == 7).all()
        assert (buf[:, :4] == 7).all() and (buf[:, 28:] == 7).all()
        assert (engine.grouped_affine(x.t().contiguous().t(), groups, bank, lnorm=True) == y).all()


@pytest.mark.parametrize("d_out", [1, 3, 77, 258])
def test_affine_out_leaves_what_lies_behind_a_row(d_out):
    torch = _torch()
    from hyperion_amd import engine

    r = _rng(17)
    sizes = [3, 0, 150]
    n, ld = sum(sizes), (d_out + 3) // 4 * 4 + 4
    x = r.standard_normal((n, 9)).astype(np.float32)
    groups = engine.RowGroups(sizes)
    bank = engine.AffineBank(r.standard_normal((3, 9, d_out)), r.standard_normal((3, d_out)))
    flat = torch.full(((n - 1) * ld + d_out,), 7.0, device="cuda")  # ends with the last row
    out = flat.as_strided((n, d_out), (ld, 1))
    for lnorm in (False, True):
        want = engine.grouped_affine(torch.from_numpy(x).cuda(), groups, bank, lnorm=lnorm)
        got = engine.grouped_affine(torch.from_numpy(x).cuda(), groups, bank, lnorm=lnorm, out=out)
        assert got is out and torch.equal(got, want)
    behind = torch.as_strided(flat[:-d_out], (n - 1, ld - d_out), (ld, 1), d_out)
    assert torch.all(behind == 7.0)


@pytest.mark.parametrize("d_out", [30, 300])
@pytest.mark.parametrize("scale", [1e-24, 1e25])
def test_affine_lnorm_of_rows_whose_squares_leave_fp32(scale, d_out):
    """A product is off by less than 2^-20 of the sum of the magnitudes of its 20 terms, so a row's norm by 2^-20 of
    their norm, which is some sqrt(20 * 2 / pi) < 4 times its own; the three roundings after that are below it."""
    torch = _torch()
    from hyperion_amd import engine

    r = _rng(23)
    x = r.standard_normal((5, 20))
    W, sizes = r.standard_normal((2, 20, d_out)), [2, 3]
    x32 = (x * scale).astype(np.float32)
    y = np.concatenate([x32[:2].astype(np.float64) @ W[0].astype(np.float32), x32[2:].astype(np.float64) @ W[1].astype(np.float32)])
    want = y * np.sqrt(d_out) / (np.linalg.norm(y, axis=1, keepdims=True) + 1e-10)
    mags = np.concatenate([np.abs(x32[:2].astype(np.float64)) @ np.abs(W[0]), np.abs(x32[2:].astype(np.float64)) @ np.abs(W[1])])
    bound = 2.0 ** -20 * mags * np.sqrt(d_out) / (np.linalg.norm(y, axis=1, keepdims=True) + 1e-10) + 2.0 ** -18 * np.abs(want)
    got = engine.grouped_affine(torch.from_numpy(x32).cuda(), engine.RowGroups(sizes), engine.AffineBank(W), lnorm=True)
    assert np.all(np.abs(got.double().cpu().numpy() - want) <= bound)


def test_no_groups():
    torch = _torch()
    from hyperion_amd import engine

    none = engine.RowGroups([])
    x = torch.zeros(0, 12, device="cuda")
    assert engine.grouped_affine(x, none, engine.AffineBank(np.zeros((0, 12, 5))), lnorm=True).shape == (0, 5)
    C, F = engine.grouped_gram64(x, none)
    assert C.shape == (0, 12, 12) and F.shape == (0, 12)
    G = torch.zeros(0, 40, device="cuda")
    pairs = engine.GroupPairs(none, none)
    assert engine.grouped_score(G, G, pairs).numel() == 0 and pairs.blocks(engine.grouped_score(G, G, pairs)) == []
    assert engine.q4_score(engine.q4_rows(G, 30, none), G, pairs).numel() == 0
    assert engine.grouped_pack(x, none, np.zeros((0, 4, 12)), np.zeros(0))[0].shape[0] == 0
    assert engine.RowGroups.from_ids([], 3).sizes.tolist() == [0, 0, 0]


def test_groups_keep_their_own_order():
    torch = _torch()
    from hyperion_amd import engine

    r = _rng(29)
    x = torch.from_numpy(r.standard_normal((6, 8)).astype(np.float32)).cuda()
    order = torch.tensor([5, 0, 3, 1], dtype=torch.int32, device="cuda")
    groups = engine.RowGroups([1, 3], order=order)
    bank = engine.AffineBank(r.standard_normal((2, 8, 4)))
    want = engine.grouped_affine(x, groups, bank)
    order.fill_(2)
    assert torch.equal(engine.grouped_affine(x, groups, bank), want)


def test_affine_dims_of_each_group():
    torch = _torch()
    from hyperion_amd import engine

    r = _rng(8)
    for m in (30, 300):
        dims = np.array([m, 1, 17])
        W = r.randn(3, 50, m)
        b = r.randn(3, m)
        for e, k in enumerate(dims):
            W[e, :, k:] = 0
            b[e, k:] = 0
        W, b = W.astype(np.float32), b.astype(np.float32)
        x = torch.from_numpy(r.randn(60, 50)).float().cuda()
        y = engine.grouped_affine(x, engine.RowGroups([20, 21, 19]), engine.AffineBank(W, b, dims=dims), lnorm=True)
        want, bound, rms = _affine_ref(x.double().cpu().numpy(), W.astype(float), b.astype(float), [20, 21, 19], None,
                                       True, dims)
        _assert_close(y, want, bound, rms)
        assert (y[20:41, 1:] == 0).all()


def test_groups_by_id():
    torch = _torch()
    from hyperion_amd import engine

    ids = np.array([4, 0, 0, 2, 4, 4])
    g = engine.RowGroups.from_ids(ids, 6)
    assert g.sizes.tolist() == [2, 0, 1, 0, 3, 0] and g.order.tolist() == [1, 2, 3, 0, 4, 5]
    x = torch.arange(18.0, device="cuda").view(6, 3)
    W = np.stack([np.eye(3) * (e + 1) for e in range(6)])
    y = engine.grouped_affine(x, g, engine.AffineBank(W))
    assert torch.equal(y, x * torch.from_numpy(ids + 1.0).float().cuda()[:, None])


# ---------------------------------------------------------------------------------------------- score
def _packed(r, n, k, kp, enrol, spread=True):
    G = np.zeros((n, kp))
    G[:, :k] = r.randn(n, k) * (np.exp(r.uniform(-2, 2, k)) if spread else 1)
    G[:, k + (0 if enrol else 1)] = r.randn(n) * 10
    G[:, k + (1 if enrol else 0)] = 1
    return G.astype(np.float32)


SCORE = [
    ([1], [1], 8),
    ([2, 0, 5, 1], [3, 4, 0, 1], 32),
    ([31, 33, 64, 1], [33, 31, 65, 400], 152),
    ([129, 0, 255], [129, 9, 1030], 152),
    ([70, 130], [513, 3], 200),
    ([65, 20], [64, 70], 232),
    ([40, 100], [100, 37], 320),
    ([66], [35], 376),
    ([20, 90], [90, 33], 512),
    ([1, 1], [2000, 1], 40),
    ([200, 17], [40, 600], 72),
    ([70], [90], 128),
    ([130, 5], [70, 33], 176),
    ([33], [40], 264),
    ([18, 65], [33, 1], 392),
]


@pytest.mark.parametrize("case", range(len(SCORE)))
def test_score(case):
    torch = _torch()
    from hyperion_amd import engine

    n1, n2, kp = SCORE[case]
    r = _rng(20 + case)
    k = kp - 2
    G1, G2 = _packed(r, sum(n1), k, kp, True), _packed(r, sum(n2), k, kp, False)
    pairs = engine.GroupPairs(engine.RowGroups(n1), engine.RowGroups(n2))
    flat = engine.grouped_score(torch.from_numpy(G1).cuda(), torch.from_numpy(G2).cuda(), pairs)
    assert flat.shape == (sum(a * b for a, b in zip(n1, n2)),)
    o1, o2 = _offsets(n1), _offsets(n2)
    for e, blk in enumerate(pairs.blocks(flat)):
        a, b = G1[o1[e]:o1[e + 1]].astype(float), G2[o2[e]:o2[e + 1]].astype(float)
        if a.size and b.size:
            bound, rms = _product_bound(a, b.T, 2.0 ** -39)
            _assert_close(blk, a @ b.T, bound + U * np.abs(a @ b.T), rms)
        else:
            assert blk.numel() == 0


def test_score_scales_and_non_finite():
    torch = _torch()
    from hyperion_amd import engine

    r = _rng(40)
    G1 = _packed(r, 90, 38, 40, True) * (10.0 ** r.randint(-15, 16, 90))[:, None].astype(np.float32)
    G2 = _packed(r, 80, 38, 40, False) * (10.0 ** r.randint(-15, 16, 80))[:, None].astype(np.float32)
    G1[4] = 0
    pairs = engine.GroupPairs(engine.RowGroups([90]), engine.RowGroups([80]))
    d1, d2 = torch.from_numpy(G1).cuda(), torch.from_numpy(G2).cuda()
    blk = pairs.block(engine.grouped_score(d1, d2, pairs), 0)
    a, b = G1.astype(float), G2.astype(float)
    bound, _ = _product_bound(a, b.T, 2.0 ** -39)
    _assert_close(blk, a @ b.T, bound + U * np.abs(a @ b.T))
    d1[3, 7], d2[70, 1] = float("nan"), float("inf")
    bad = pairs.block(engine.grouped_score(d1, d2, pairs), 0)
    keep = torch.ones(90, 80, dtype=torch.bool, device="cuda")
    keep[3], keep[:, 70] = False, False
    assert torch.equal(bad[keep], blk[keep]) and not torch.isfinite(bad[~keep]).any()


def test_score_matches_the_ungrouped_product():
    """One group: the scores of engine.score on the same packed rows, to both products' bounds."""
    torch = _torch()
    from hyperion_amd import engine

    r = _rng(41)
    G1, G2 = _packed(r, 200, 150, 152, True), _packed(r, 333, 150, 152, False)
    d1, d2 = torch.from_numpy(G1).cuda(), torch.from_numpy(G2).cuda()
    pairs = engine.GroupPairs(engine.RowGroups([200]), engine.RowGroups([333]))
    bound, _ = _product_bound(G1.astype(float), G2.astype(float).T, 2.0 ** -39)
    _assert_close(pairs.block(engine.grouped_score(d1, d2, pairs), 0), engine.score(d1, d2).double().cpu().numpy(),
                  2 * bound)


# ---------------------------------------------------------------------------------------------- moments
GRAM = [
    ([1], 1),
    ([0, 3, 1], 5),
    ([17, 64, 0, 2, 5], 32),
    ([30, 200], 33),
    ([1024, 1025, 10], 40),
    ([3000, 0, 1, 2049], 77),
    ([100, 41], 200),
    ([64], 520),
    ([0, 0], 9),
    ([192, 193, 256, 4095], 50),
    ([4096, 4097, 4289, 0, 8192], 20),
    ([2048, 2049, 2112, 0, 6145], 20),
    ([59521, 1], 6),  # thirty chunks, the last of 129 rows
]


@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("case", range(len(GRAM)))
def test_gram(case, dtype, weighted):
    """A sum of n float64 products rounds at most n + 2 times (a weight adds one rounding): 2^-53 each."""
    torch = _torch()
    from hyperion_amd import engine

    sizes, d = GRAM[case]
    r = _rng(60 + case)
    n = sum(sizes)
    order = r.permutation(n) if case % 2 else None
    wide = torch.from_numpy(r.randn(n, d + 3) * np.exp(r.uniform(-3, 3, d + 3)) + 0.5).cuda().to(getattr(torch, dtype))
    x = wide[:, 1:1 + d] if case % 3 else wide[:, :d].contiguous()
    w = r.uniform(0.1, 2, n) if weighted else None
    groups = engine.RowGroups(sizes, order=order)
    wd = None if w is None else torch.from_numpy(w).cuda()
    C, F = engine.grouped_gram64(x, groups, wd)
    assert C.dtype == F.dtype == torch.float64 and C.shape == (len(sizes), d, d) and F.shape == (len(sizes), d)
    assert torch.equal(C, C.transpose(1, 2))
    X, off = x.double().cpu().numpy().astype(np.longdouble), _offsets(sizes)
    for e in range(len(sizes)):
        rows = np.arange(off[e], off[e + 1]) if order is None else order[off[e]:off[e + 1]]
        xe = X[rows]
        we = np.ones(len(rows), np.longdouble) if w is None else w[rows].astype(np.longdouble)
        eps = (len(rows) + 3) * 2.0 ** -53
        _assert_close(C[e], (xe.T @ (xe * we[:, None])).astype(float),
                      (eps * (np.abs(xe).T @ np.abs(xe * we[:, None]))).astype(float))
        _assert_close(F[e], (xe * we[:, None]).sum(0).astype(float), (eps * np.abs(xe * we[:, None]).sum(0)).astype(float))
    C2, F2 = engine.grouped_gram64(x, groups, wd)
    assert torch.equal(C, C2) and torch.equal(F, F2)


def test_gram_non_finite_groups_stay_alone():
    torch = _torch()
    from hyperion_amd import engine

    x = torch.from_numpy(_rng(80).randn(50, 20)).cuda()
    bad = x.clone()
    bad[19, 3] = float("nan")  # the last row of the first group: rows past a group's end are copies of it
    bad[49, 0] = float("inf")
    groups = engine.RowGroups([20, 10, 20])
    C, F = engine.grouped_gram64(x, groups)
    Cb, Fb = engine.grouped_gram64(bad, groups)
    assert torch.equal(C[1], Cb[1]) and torch.equal(F[1], Fb[1])
    assert torch.isnan(Cb[0, 3]).all() and torch.isnan(Fb[0, 3]) and torch.equal(Fb[0, :3], F[0, :3])
    assert torch.equal(Cb[0][:3, :3], C[0][:3, :3]) and torch.isinf(Cb[2, 0, 0])


# ---------------------------------------------------------------------------------------------- 4 bits
def _q4_definition(g):
    """Codes and scales of rows [n, k] by the definition, in exact arithmetic on integers."""
    from fractions import Fraction

    n, k = g.shape
    values = np.zeros((n, k))
    steps = np.zeros((n, k))
    for i in range(n):
        for c0 in range(0, k, 32):
            x = [Fraction(float(v)) for v in g[i, c0:c0 + 32]]
            top = max(abs(v) for v in x)
            if top == 0:
                continue
            e = math.frexp(float(top) / 7)[1] - 8  # eight significant bits: step 2^e, mantissa 128 .. 256
            e = max(e, -133)
            step = Fraction(2) ** e
            mant = -((-top / 7) // step)  # ceil
            s = mant * step
            for j, v in enumerate(x):
                values[i, c0 + j] = float(round(v / s) * s)  # round() of a Fraction takes halves to even
                steps[i, c0 + j] = float(s)
    return values, steps


def test_q4_codes_follow_the_definition():
    """Every value that the codes stand for, over rows with halves and quotients next to halves, zeros,
    sub-normal and huge magnitudes, and partitions that end inside a block."""
    torch = _torch()
    from hyperion_amd import engine

    r = _rng(90)
    for k in (1, 31, 32, 33, 70):
        n = 130
        g = r.randn(n, k).astype(np.float32)
        g[:40] = (r.randint(-14, 15, (40, k)) * 0.5).astype(np.float32)  # halves of a scale of one
        g[:40, 0] = 7.0
        g[40:60] = np.nextafter(g[:20], np.float32(np.inf))
        g[60:80] = np.nextafter(g[:20], np.float32(-np.inf))
        g[80:90] *= np.float32(1e-41)
        g[90:95] *= np.float32(3e37)
        g[95] = 0
        g[96:110] *= (10.0 ** r.randint(-20, 20, (14, 1))).astype(np.float32)
        G = np.concatenate([g, r.randn(n, 2).astype(np.float32)], 1)
        sizes = [1, 0, 63, 64, 2]
        gallery = engine.q4_rows(torch.from_numpy(G).cuda(), k, engine.RowGroups(sizes))
        want, _ = _q4_definition(g)
        assert np.array_equal(gallery.values().double().cpu().numpy(), want)
        assert gallery.nbytes == gallery.codes.shape[0] * (1152 * gallery.codes.shape[1] + 256)


Q4 = [
    # tests per group, gallery rows per group, coordinates
    ([1], [1], 1),
    ([1], [5000], 150),
    ([16], [1024], 40),
    ([17, 0, 3], [100, 50, 0], 64),
    ([2, 31, 5, 1], [1, 64, 65, 1100], 150),
    ([70, 1], [300, 2000], 96),
    ([3, 33], [90, 130], 200),
    ([5, 100], [1025, 70], 310),
    ([64, 2], [65, 64], 512),
    ([0, 0], [5, 6], 30),
    # hundreds of tests: tiles of 64
    ([300, 0, 9], [130, 5, 1], 150),
    ([210], [70], 310),
    ([257], [1100], 33),
    ([250, 190], [65, 64], 512),
]


@pytest.mark.parametrize("case", range(len(Q4)))
def test_q4_score(case):
    """Against the product with the values that the codes stand for.  Test rows are pairs (2^-22 of a product,
    2^-39 of the row's largest magnitude per coordinate), codes are exact and at most 7; a scale group takes 64
    roundings, the groups and the two additive terms one each."""
    torch = _torch()
    from hyperion_amd import engine

    tests, rows, k = Q4[case]
    r = _rng(100 + case)
    G1, G2 = _packed(r, sum(rows), k, k + 2, True), _packed(r, sum(tests), k, k + 2, False)
    gallery = engine.q4_rows(torch.from_numpy(G1).cuda(), k, engine.RowGroups(rows))
    pairs = engine.GroupPairs(engine.RowGroups(tests), gallery.groups)
    flat = engine.q4_score(gallery, torch.from_numpy(G2).cuda(), pairs)
    V = gallery.values().double().cpu().numpy()
    ng = (k + 31) // 32
    o1, o2 = _offsets(rows), _offsets(tests)
    for e, blk in enumerate(pairs.blocks(flat)):
        v, t = V[o1[e]:o1[e + 1]], G2[o2[e]:o2[e + 1]].astype(float)
        if not (len(v) and len(t)):
            assert blk.numel() == 0
            continue
        g = np.abs(t[:, :k])
        q, add = G1[o1[e]:o1[e + 1], k].astype(float), t[:, k + 1]
        want = t[:, :k] @ v.T + q[None, :] + add[:, None]
        bound = 2.0 ** -22 * (g @ np.abs(v).T) + (64 + ng) * U * (g @ np.abs(v).T)
        bound += 2.0 ** -39 * g.max(1)[:, None] * np.abs(v).sum(1)[None, :]
        bound += 3 * U * (np.abs(want) + np.abs(q)[None, :] + np.abs(add)[:, None])
        _assert_close(blk, want, bound)


def test_q4_non_finite_rows_stay_alone():
    torch = _torch()
    from hyperion_amd import engine

    r = _rng(120)
    G1, G2 = (torch.from_numpy(_packed(r, n, 70, 72, e)).cuda() for n, e in ((200, True), (5, False)))
    pairs = engine.GroupPairs(engine.RowGroups([5]), engine.RowGroups([200]))
    ok = pairs.block(engine.q4_score(engine.q4_rows(G1, 70), G2, pairs), 0)
    G1[7, 69], G1[130, 0], G2[2, 33] = float("nan"), float("inf"), float("nan")
    bad = pairs.block(engine.q4_score(engine.q4_rows(G1, 70), G2, pairs), 0)
    keep = torch.ones(5, 200, dtype=torch.bool, device="cuda")
    keep[2], keep[:, [7, 130]] = False, False
    assert torch.equal(bad[keep], ok[keep]) and torch.isnan(bad[~keep]).all()


# ---------------------------------------------------------------------------------------------- together
def _chain_inputs(seed=3):
    torch = _torch()
    from hyperion_amd import engine

    r = _rng(seed)
    sizes = [40, 0, 1, 300, 77, 1500]
    n, d, m = sum(sizes), 60, 30
    x = torch.from_numpy(r.randn(n, d)).float().cuda()
    bank = engine.AffineBank(r.randn(len(sizes), d, m) / 8, r.randn(len(sizes), m))
    groups = engine.RowGroups(sizes)
    return x, bank, groups, engine.GroupPairs(groups, groups)


def _chain(x, bank, groups, pairs):
    """Moments, projection and self-scores of a batch, and the same rows as a 4-bit gallery."""
    torch = _torch()
    from hyperion_amd import engine

    C, F = engine.grouped_gram64(x, groups)
    y = engine.grouped_affine(x, groups, bank, lnorm=True)
    G = torch.zeros(y.shape[0], 32, device=y.device)
    G[:, :30] = y
    G[:, 31] = 1
    S = engine.grouped_score(G, G, pairs)
    q = engine.q4_score(engine.q4_rows(G, 30, groups), G, pairs)
    return C, F, y, S, q


def test_graph_capture_and_replay():
    """The operators in one captured graph, replayed with other inputs between eager calls; a second graph of the
    same plans in between."""
    torch = _torch()

    x, bank, groups, pairs = _chain_inputs()
    static, other = x.clone(), x.clone()
    _chain(static, bank, groups, pairs)  # kernel attributes are set on first use
    torch.cuda.synchronize()
    graphs = []
    for buf in (static, other):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = _chain(buf, bank, groups, pairs)
        graphs.append((g, buf, res))
    for i in range(4):
        for j, (g, buf, res) in enumerate(graphs):
            new = x * (1 + i) - j
            buf.copy_(new)
            want = _chain(new, bank, groups, pairs)
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip(res, want):
                assert torch.equal(a, b)


def test_streams():
    """Calls on two other streams at once, with plans made on the default one and dropped right after."""
    torch = _torch()

    want = [t.clone() for t in _chain(*_chain_inputs())]
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream() for _ in range(2)], []
    for rep in range(3):
        for s in streams:
            args = _chain_inputs()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                args[0].record_stream(s)
                results.append(_chain(*args))
            del args
            torch.empty(1 << 20, device="cuda").fill_(float("nan"))
    torch.cuda.synchronize()
    for res in results:
        for a, b in zip(res, want):
            assert torch.equal(a, b)


# ---------------------------------------------------------------------------------------------- refusals
def test_refusals():
    torch = _torch()
    from hyperion_amd import engine

    def refuses(match, fn, *a, **k):
        with pytest.raises(ValueError, match=match):
            fn(*a, **k)

    x = torch.zeros(6, 4, device="cuda")
    g = engine.RowGroups([2, 4])
    bank = engine.AffineBank(np.ones((2, 4, 3)))
    refuses("more than once", engine.RowGroups, [2, 1], order=[0, 3, 3])
    refuses("lists 2 rows", engine.RowGroups, [2, 1], order=[0, 3])
    refuses("row numbers", engine.RowGroups, [2, 1], order=[0, -1, 3])
    refuses("1-D sequence", engine.RowGroups, [1], order=[0.5])
    refuses("lie in", engine.RowGroups.from_ids, [0, 5], 3)
    refuses("lie in", engine.RowGroups.from_ids, [0, -1])
    refuses("expected 4-dim", engine.grouped_affine, torch.zeros(6, 5, device="cuda"), g, bank)
    refuses("has 5 rows", engine.grouped_affine, x[:5], g, bank)
    refuses("names row 5", engine.grouped_affine, x[:5], engine.RowGroups([2, 4], order=np.arange(6)), bank)
    refuses("device tensor", engine.grouped_affine, x.cpu(), g, bank)
    refuses("expected one of", engine.grouped_affine, x.double(), g, bank)
    refuses("2-D", engine.grouped_affine, x[0], g, bank)
    refuses("3 maps for 2", engine.grouped_affine, x, g, engine.AffineBank(np.ones((3, 4, 3))))
    for out in (torch.zeros(6, 3, device="cuda"), torch.zeros(5, 4, device="cuda")[:, :3],
                torch.zeros(6, 8, device="cuda")[:, 1:4], torch.zeros(6, 4, device="cuda").double()[:, :3]):
        refuses("out must be", engine.grouped_affine, x, g, bank, out=out)
    flat = torch.zeros(48, device="cuda")
    refuses("share memory", engine.grouped_affine, flat.view(6, 8)[:, :4], g, bank, out=flat.view(6, 8)[:, 4:7])
    refuses(r"W must be", engine.AffineBank, np.ones((2, 4)))
    refuses(r"b must be", engine.AffineBank, np.ones((2, 4, 3)), np.ones((2, 4)))
    refuses("dims must be", engine.AffineBank, np.ones((2, 4, 3)), dims=[1, 4])
    refuses("floating-point", engine.AffineBank, np.ones((2, 4, 3), int))
    refuses("2 and 1 groups", engine.GroupPairs, g, engine.RowGroups([6]))
    refuses("group order", engine.GroupPairs, g, engine.RowGroups([2, 4], order=np.arange(6)))
    pairs = engine.GroupPairs(g, g)
    G = torch.zeros(6, 40, device="cuda")
    refuses("widths differ", engine.grouped_score, G, torch.zeros(6, 48, device="cuda"), pairs)
    refuses("no grouped kernel", engine.grouped_score, G[:, :36], G[:, :36], pairs)
    refuses("16-byte", engine.grouped_score, G[:, 1:33], G[:, 1:33], pairs)
    refuses("has 5 rows", engine.grouped_score, G[:5], G, pairs)
    refuses("out must be", engine.grouped_score, G, G, pairs, out=torch.zeros(21, device="cuda"))
    refuses("share memory", engine.grouped_score, G, G, pairs, out=G.view(-1)[200:220])
    refuses("rows", engine.RowGroups, [1 << 62, 1 << 62])
    refuses("scores", engine.GroupPairs, *[engine.RowGroups([1 << 32])] * 2)
    refuses("expected one of", engine.grouped_gram64, x.half(), g)
    refuses("w must be", engine.grouped_gram64, x, g, torch.zeros(6, device="cuda"))
    refuses("no columns", engine.grouped_gram64, x[:, :0], g)
    refuses("0 coordinates", engine.q4_rows, G, 0)
    refuses("513 coordinates", engine.q4_rows, torch.zeros(2, 600, device="cuda"), 513)
    refuses("40 coordinates", engine.q4_rows, G, 40)
    refuses("group order", engine.q4_rows, G, 30, engine.RowGroups([6], order=np.arange(6)))
    gallery = engine.q4_rows(G, 38)
    one = engine.GroupPairs(engine.RowGroups([6]), gallery.groups)
    refuses("not the groups", engine.q4_score, gallery, G, pairs)
    refuses("packed rows of 39", engine.q4_score, gallery, G[:, :39], one)
    refuses("out must be", engine.q4_score, gallery, G, one, out=torch.zeros(36, device="cuda", dtype=torch.float64))
    refuses("share memory", engine.q4_score, gallery, G, one, out=G.view(-1)[:36])
