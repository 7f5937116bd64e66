"""Grouped affine maps over rows and columns whose magnitudes span many decades, against float64.

Operands are pairs of fp16 numbers, the second scaled by 2^11.  A row's largest magnitude lies above 2^8 of the scaled
unit, a column's above 2^14.  Per coordinate of a row:
  2^-22 of it where both numbers are normal, otherwise half a step of the second, 2^-25 2^-11 of the scaled unit, plus the
  dropped product of the second numbers, at most 2^-25 2^-11 of the weight where the first is below its normal range
  (half a step of it, times 2^-11), plus what aligning a product with such a number may cost, 2^-24 of 2^-14: together less
  than 2^-34 of the scaled unit, 2^-42 of the row's largest magnitude.  Weights: the same with 2^14 in place of 2^8, 2^-48.
The products of order 2^-22 that are rounded or dropped where all numbers are normal: 3 2^-22 of each product.  Three sums
of d products and d / 32 additions of the second two: fewer than 4 d roundings of 2^-24 of the sum of magnitudes."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _bound(x, w):
    """Bound per element and the size that independent errors give, times four."""
    d = x.shape[1]
    ax, aw = np.abs(x), np.abs(w)
    top_x, top_w = ax.max(1, initial=0)[:, None], aw.max(0, initial=0)[None, :]
    bound = (3 * 2.0 ** -22 + 4 * d * U) * (ax @ aw)
    bound += 2.0 ** -42 * top_x * aw.sum(0)[None, :] + 2.0 ** -48 * top_w * ax.sum(1)[:, None]
    rms = (math.sqrt(4 * d) * U + 2.0 ** -22) * np.sqrt((x * x) @ (w * w))
    rms += 2.0 ** -42 * top_x * np.sqrt((w * w).sum(0))[None, :] + 2.0 ** -48 * top_w * np.sqrt((x * x).sum(1))[:, None]
    return bound, 4 * rms


SIZES = {16: [3, 0, 9], 64: [70, 1, 100], 128: [1500, 1100, 1300]}  # by the tile that the mean size selects


@pytest.mark.parametrize("dtype,decades", [(t, k) for t in ("float32", "bfloat16", "float16") for k in (4, 5, 6, 8)
                                           if (t, k) != ("float16", 8)])  # fp16 holds no wider range
@pytest.mark.parametrize("d", [40, 200, 520])
@pytest.mark.parametrize("tile", [16, 64, 128])
def test_maps_that_undo_the_scales_of_their_coordinates(tile, dtype, d, decades):
    """What centring and whitening are for: coordinates whose deviations span many decades, maps that bring all of
    them to the same size, so that the smallest coordinate weighs as much as the largest."""
    import torch

    from hyperion_amd import engine

    r = np.random.RandomState(tile + d + decades)
    sizes, m = SIZES[tile], 30
    n = sum(sizes)
    s = 10.0 ** np.linspace(-decades / 2, decades / 2, d)[r.permutation(d)]
    x = torch.from_numpy(r.randn(n, d) * s).to("cuda").to(getattr(torch, dtype))
    W = (r.randn(3, d, m) / s[:, None]).astype(np.float32)
    y = engine.grouped_affine(x, engine.RowGroups(sizes), engine.AffineBank(W)).double().cpu().numpy()
    x, W, at = x.double().cpu().numpy(), W.astype(float), 0
    for e, k in enumerate(sizes):
        if k:
            rows = x[at:at + k]
            bound, rms = _bound(rows, W[e])
            err = np.abs(y[at:at + k] - rows @ W[e])
            assert (err <= bound + U * np.abs(rows @ W[e])).all()
            assert np.sqrt(np.mean((err / (rms + U * np.abs(rows @ W[e]))) ** 2)) <= 1
            if decades <= 6 and d <= 200:
                # the size of the errors of a plain fp32 product, sqrt(d) 2^-24 of the terms, and 2^-22 for the pairs
                size = np.sqrt(np.mean((rows @ W[e]) ** 2))
                assert np.sqrt(np.mean(err ** 2)) <= 4 * (math.sqrt(d) * U + 2.0 ** -22) * size
        at += k


@pytest.mark.parametrize("tile", [16, 64, 128])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_every_coordinate_of_a_row_of_wide_range(dtype, tile):
    """Maps that pick single coordinates (weights 1, -2 and 2^-20): each comes out as it went in, the largest and the
    smallest numbers of the type in one row.  fp16 rows are exact: their products with a power of two are, and nothing is
    added to them but zeros."""
    import torch

    from hyperion_amd import engine

    r = np.random.RandomState(7)
    sizes, d = SIZES[tile], 96
    n = sum(sizes)
    if dtype == "float16":
        x = r.randn(n, d) * 2.0 ** r.randint(-24, 15, (n, d))
        x[:, 5] = 65504 * r.choice([-1, 1], n)
        x[:, 70] = 2.0 ** -24
    else:
        x = r.randn(n, d) * 2.0 ** r.randint(-45, 1, (n, d))
        x[:, 5], x[:, 70] = 1.7, 2.0 ** -36
    x[1] = 0
    x = torch.from_numpy(x).to("cuda").to(getattr(torch, dtype))
    w = np.array([1, -2, 2.0 ** -20])
    W = np.eye(d)[None] * w[:, None, None]
    y = engine.grouped_affine(x, engine.RowGroups(sizes), engine.AffineBank(W)).double().cpu().numpy()
    want = x.double().cpu().numpy() * np.repeat(w, sizes)[:, None]
    if dtype == "float16":
        ok = np.isfinite(want).all(1)  # a draw beyond the type's range is an infinity: its row has no finite values
        assert np.array_equal(y[ok], want[ok]) and not np.isfinite(y[~ok]).any() and ok.mean() > 0.9
    else:
        top = np.abs(want).max(1, keepdims=True)
        assert (np.abs(y - want) <= 2.0 ** -22 * np.abs(want) + 2.0 ** -42 * top).all()


def test_rows_that_grow_and_shrink_from_chunk_to_chunk():
    """Coordinates in blocks of 32 and 64 whose magnitudes go up and down by up to 2^30, small weights against the large
    ones: the scale of a row is set, kept and lowered, with all three tiles and types."""
    import torch

    from hyperion_amd import engine

    r = np.random.RandomState(11)
    d, m = 320, 50
    for tile, sizes in SIZES.items():
        n = sum(sizes)
        e = np.repeat(r.randint(-6, 7, (n, d // 32)), 32, axis=1)
        for dtype, spread in (("float32", 5.0), ("bfloat16", 5.0), ("float16", 2.0)):
            x = torch.from_numpy(r.randn(n, d) * 2.0 ** (e * spread / 2)).to("cuda").to(getattr(torch, dtype))
            W = (r.randn(3, d, m) * 2.0 ** r.uniform(-8, 8, (3, d, 1))).astype(np.float32)
            b = r.randn(3, m).astype(np.float32)
            y = engine.grouped_affine(x, engine.RowGroups(sizes), engine.AffineBank(W, b)).double().cpu().numpy()
            xs, at = x.double().cpu().numpy(), 0
            assert np.isfinite(xs).all()
            for g, k in enumerate(sizes):
                if k:
                    want = xs[at:at + k] @ W[g].astype(float) + b[g]
                    bound, _ = _bound(xs[at:at + k], W[g].astype(float))
                    assert (np.abs(y[at:at + k] - want) <= bound + 2 * U * (np.abs(want) + np.abs(b[g]))).all()
                at += k


def test_columns_behind_the_dimension_of_a_map_are_refused():
    """They would enter the length normalisation and be written where zeros are promised."""
    from hyperion_amd import engine

    W, b = np.ones((3, 5, 8)), np.ones((3, 8))
    dims = [8, 2, 5]
    for e, k in enumerate(dims):
        W[e, :, k:], b[e, k:] = 0, 0
    engine.AffineBank(W, b, dims=dims)
    engine.AffineBank(W, dims=dims)
    for bad in (1e-30, np.nan, np.inf):
        for array, at in ((W, (1, 4, 2)), (W, (2, 0, 7)), (b, (1, 7))):
            array[at] = bad
            with pytest.raises(ValueError, match="behind dims"):
                engine.AffineBank(W, b, dims=dims)
            array[at] = 0
    engine.AffineBank(W, b, dims=dims)


def test_more_rows_than_waves_of_a_launch():
    """The length normalisation of wide rows and the packing take rows in turn: 32 768 are one round."""
    import torch

    from hyperion_amd import engine

    n, d, m = 70001, 4, 258
    r = np.random.RandomState(5)
    sizes = [32767, 0, 2, 37232]
    x = torch.from_numpy(r.randn(n, d)).float().cuda()
    W = r.randn(4, d, m).astype(np.float32)
    groups = engine.RowGroups(sizes)
    y = engine.grouped_affine(x, groups, engine.AffineBank(W), lnorm=True)
    plain = engine.grouped_affine(x, groups, engine.AffineBank(W)).double()
    want = plain * math.sqrt(m) / plain.norm(dim=1, keepdim=True)
    assert ((y.double() - want).abs() <= 8 * U * want.abs()).all()  # the factor and the product, both rounded
    s = torch.from_numpy(r.randn(n, 6)).float().cuda()
    maps, c = r.randn(4, 4, 6).astype(np.float32), r.randn(4).astype(np.float32)
    G1, G2 = engine.grouped_pack(s, groups, maps, c)
    at = np.cumsum([0] + sizes)
    for e in (0, 2, 3):
        one = engine.RowGroups([sizes[e]])
        for part in range(at[e], at[e + 1], 20000):  # no more than one round at a time
            end = min(part + 20000, int(at[e + 1]))
            one = engine.RowGroups([end - part])
            for got, want in zip((G1, G2), engine.grouped_pack(s[part:end], one, maps[e:e + 1], c[e:e + 1])):
                assert torch.equal(got[part:end], want)


def test_an_empty_order():
    import torch

    from hyperion_amd import engine

    x = torch.ones(3, 4, device="cuda")
    for order in ([], np.zeros(0, int), torch.zeros(0, dtype=torch.int32)):
        groups = engine.RowGroups([0, 0], order=order)
        assert (engine.grouped_affine(x, groups, engine.AffineBank(np.ones((2, 4, 5)))) == 0).all()
        C, F = engine.grouped_gram64(x, groups)
        assert (C == 0).all() and (F == 0).all()
    with pytest.raises(ValueError, match="lists 0 rows"):
        engine.RowGroups([1], order=[])
    with pytest.raises(ValueError, match="1-D"):
        engine.RowGroups([0], order=[[]])
