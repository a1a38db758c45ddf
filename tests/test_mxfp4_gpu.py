"""MXFP4 on a B200: rows to codes and back bit for bit, the dense and routed
products within bounds derived from how their sums are held, against the
definition in binary64."""

import numpy as np
import pytest

from oracle import oracle as O
from tests import mxfp4_check as X

pytestmark = pytest.mark.gpu

SUFFIX = {"f32": "", "bf16": "_xbf16", "f16": "_xf16"}
TYPES = ["f32", "bf16", "f16"]
MARK = 77.0


@pytest.fixture(scope="module")
def ctx():
    from furykernel_b200 import _native as N

    c = N.Context(0)
    yield c
    c.close()


def strided(t, x, ld):
    """x [rows, k] as rows ld apart of type t, a mark between them."""
    wide = np.full((x.shape[0], ld), MARK, np.float32)
    wide[:, :x.shape[1]] = x
    return X.narrow(t, wide)


def quant(ctx, x, t="f32", ldx=None):
    rows, k = x.shape
    xd = ctx.to_device(strided(t, x, ldx or k))
    cd, sd = ctx.zeros((rows, k // 2), np.uint8), ctx.zeros((rows, k // 32), np.uint8)
    ctx.launch("quant_mxfp4" + SUFFIX[t], {"rows": rows, "k": k, "ldx": ldx or k}, [xd, cd, sd])
    got = cd.download(), sd.download()
    for b in (xd, cd, sd):
        b.free()
    return got


# --------------------------------------------------------------------------
# Quantisation


@pytest.mark.parametrize("rows,k,ldx", [(1, 32, 32), (3, 96, 99), (33, 1056, 1056), (130, 2880, 2884), (2000, 64, 64)])
@pytest.mark.parametrize("t", TYPES)
def test_quant(ctx, rows, k, ldx, t):
    x = 0.02 * O.normal(311, rows * k).reshape(rows, k) * np.exp2(np.arange(rows) % 9 - 4.0)[:, None]
    held = X.widen_type(t, X.narrow(t, x))
    codes, scales = X.quantise(held)
    got = quant(ctx, x, t, ldx)
    assert np.array_equal(got[1], scales)
    assert np.array_equal(got[0], codes)


def test_quant_edges(ctx):
    """Every tie and its neighbours, zeros of both signs, the ends of the
    range, subnormals, infinities and NaNs."""
    rows = []
    for scale in (1.0, 2.0 ** -126, 2.0 ** -149 * 64, 2.0 ** 120, 2.0 ** -40):
        v = np.concatenate([[4.0], X.MIDDLE, np.nextafter(X.MIDDLE.astype(np.float32), np.float32(9)),
                            np.nextafter(X.MIDDLE.astype(np.float32), np.float32(0)), [6.0, 7.0, 7.999, 0.0, -0.0]])
        b = np.zeros(32)
        b[:len(v)] = v
        rows += [b * scale, -b * scale]
    rows += [np.zeros(32), -np.zeros(32), np.full(32, 2.0 ** -149), np.full(32, np.finfo(np.float32).max)]
    for odd in (np.inf, -np.inf, np.nan):
        b = np.linspace(-1, 1, 32)
        b[11] = odd
        rows.append(b)
    x = np.stack(rows).astype(np.float32)
    codes, scales = X.quantise(x)
    got = quant(ctx, x)
    assert np.array_equal(got[1], scales)
    assert np.array_equal(got[0], codes)
    assert (scales[-3:] == 255).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("k,ldy", [(32, 32), (96, 101), (1056, 1056)])
def test_widen(ctx, t, k, ldy):
    rows = 256  # every scale byte, every code
    codes = O.ints(312, rows * k // 2, 256).astype(np.uint8).reshape(rows, k // 2)
    scales = np.repeat(np.arange(rows, dtype=np.uint8)[:, None], k // 32, 1)
    cd, sd = ctx.to_device(codes), ctx.to_device(scales)
    yd = ctx.to_device(strided(t, np.full((rows, k), MARK, np.float32), ldy))
    name = "widen_mxfp4" + ("" if t == "f32" else "_y" + t)
    ctx.launch(name, {"rows": rows, "k": k, "ldy": ldy}, [cd, sd, yd])
    y = yd.download()
    with np.errstate(over="ignore"):
        want = X.widen(codes, scales).astype(np.float32)
    assert np.array_equal(X.widen_type(t, y[:, :k]), X.widen_type(t, X.narrow(t, want)), equal_nan=True)
    assert (X.widen_type(t, y[:, k:]) == MARK).all()
    for b in (cd, sd, yd):
        b.free()


# --------------------------------------------------------------------------
# The dense product


def weights(seed, *shape, spread=0):
    """Quantised N(0, 0.02) weights, each row's scales spread over `spread` binades."""
    w = O.normal(seed, int(np.prod(shape)), 0.0, 0.02).reshape(shape)
    if spread:
        blocks = O.ints(seed + 1, w.size // 32, spread).reshape(shape[:-1] + (-1,))
        w = w * np.repeat(np.exp2(blocks.astype(np.float64) - spread // 2), 32, -1)
    return X.quantise(w)


def linear(ctx, codes, scales, x, t, ldx=None, ldy=None):
    from furykernel_b200 import _native as N

    n, k = codes.shape[0], codes.shape[1] * 2
    m = x.shape[0]
    ldx, ldy = ldx or k, ldy or n
    wd, sd, xd = ctx.to_device(codes), ctx.to_device(scales), ctx.to_device(strided(t, x, ldx))
    yd = ctx.to_device(strided(t, np.full((m, n), MARK, np.float32), ldy))
    work = ctx.alloc(N.linear_mxfp4_work(n, k, m), np.uint8)
    work.upload(np.full(work.nbytes, 0xFF, np.uint8))
    ctx.launch("linear_mxfp4" + SUFFIX[t], {"n": n, "k": k, "m": m, "ldx": ldx, "ldy": ldy}, [wd, sd, xd, yd, work])
    y = X.widen_type(t, yd.download())
    assert ctx.status() == 0
    assert (y[:, n:] == MARK).all()
    for b in (wd, sd, xd, yd, work):
        b.free()
    return y[:, :n].astype(np.float64)


def held(t, x):
    return X.widen_type(t, X.narrow(t, x)).astype(np.float64)


SHAPES = [(1, 1, 32), (1, 7, 96), (2, 40, 2880), (3, 130, 160), (5, 257, 1056), (8, 64, 8192), (9, 128, 544), (16, 300, 4096), (17, 129, 512),
          (33, 96, 2048), (64, 300, 1056), (129, 640, 1536), (300, 1000, 544)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("t", TYPES)
def test_linear(ctx, m, n, k, t):
    codes, scales = weights(321, n, k)
    w = X.widen(codes, scales)
    x = O.normal(322, m * k).reshape(m, k) * np.exp(O.normal(323, k))[None]
    y = linear(ctx, codes, scales, x, t)
    xh = held(t, x)
    want = xh @ w.T
    assert (np.abs(y - want) <= X.linear_bound(w, xh, t)).all()
    # By norm: truncated sums of at most 64 steps lose at most 2^-24 a step of what they hold on
    # average; inputs and the runs' sums 2^-23 more; 16-bit outputs their own rounding.
    far = np.linalg.norm(y - want) / np.linalg.norm(want)
    assert far <= {"f32": 66 * 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[t]


# Inputs that fill a block's shared memory, and past it; single rows' and short
# runs of the tiles; two passes over few weights and tiles over many.
@pytest.mark.parametrize("m,n,k", [(1, 40, 16384), (2, 40, 12288), (3, 48, 5120), (4, 64, 4608), (4, 40, 11008),
                                   (7, 100, 4352), (8, 33, 1024), (10, 40, 32), (20, 140, 96), (40, 200, 288),
                                   (70, 260, 800), (150, 129, 1312), (11, 5, 64),
                                   (66, 40, 32), (100, 140, 96), (90, 200, 288), (65, 15, 1056)])
@pytest.mark.parametrize("t", TYPES)
def test_linear_ends(ctx, m, n, k, t):
    codes, scales = weights(324, n, k)
    w = X.widen(codes, scales)
    x = O.normal(325, m * k).reshape(m, k)
    y = linear(ctx, codes, scales, x, t)
    xh = held(t, x)
    assert (np.abs(y - xh @ w.T) <= X.linear_bound(w, xh, t)).all()


@pytest.mark.parametrize("m", [6, 8])
@pytest.mark.parametrize("t", TYPES)
def test_linear_few_rows_many_weights(ctx, m, t):
    """Held at some of the columns."""
    n, k = 16500, 4096
    codes = O.ints(326, n * k // 2, 256).astype(np.uint8).reshape(n, k // 2)
    scales = (120 + O.ints(327, n * k // 32, 5)).astype(np.uint8).reshape(n, k // 32)
    x = O.normal(328, m * k).reshape(m, k)
    y = linear(ctx, codes, scales, x, t)
    at = np.unique(np.concatenate([[0, 127, 128, n - 1], O.ints(329, 40, n)]))
    w, xh = X.widen(codes[at], scales[at]), held(t, x)
    assert (np.abs(y[:, at] - xh @ w.T) <= X.linear_bound(w, xh, t)).all()


@pytest.mark.parametrize("m", [1, 6, 40])
@pytest.mark.parametrize("t", TYPES)
def test_linear_strides(ctx, m, t):
    n, k = 77, 352
    codes, scales = weights(324, n, k)
    x = O.normal(325, m * k).reshape(m, k)
    a = linear(ctx, codes, scales, x, t)
    for ldx, ldy in ((k + 1, n), (k + 8, n + 3), (k + 5, n + 1)):
        assert np.array_equal(linear(ctx, codes, scales, x, t, ldx, ldy), a)


@pytest.mark.parametrize("m", [1, 12, 70])
def test_linear_spread_scales(ctx, m):
    """Scales over 30 binades within a row, inputs over 20 within a run."""
    n, k = 96, 1056
    codes, scales = weights(326, n, k, spread=30)
    w = X.widen(codes, scales)
    x = O.normal(328, m * k).reshape(m, k) * np.exp2(O.ints(329, m * k, 20).reshape(m, k) - 10.0)
    y = linear(ctx, codes, scales, x, "f32")
    xh = held("f32", x)
    assert (np.abs(y - xh @ w.T) <= X.linear_bound(w, xh, "f32")).all()


@pytest.mark.parametrize("m", [1, 12, 70])
@pytest.mark.parametrize("t", TYPES)
def test_linear_odd_values(ctx, m, t):
    """A NaN scale spoils its row's outputs, an infinite or NaN input its
    row of outputs where a weight meets it, and nothing else; zero rows give
    zeros."""
    n, k = 64, 1088
    codes, scales = weights(331, n, k)
    scales[5, 3] = 255
    codes[6] = 0
    x = O.normal(332, m * k).reshape(m, k)
    xh = held(t, x)
    w = X.widen(codes, scales)
    y = linear(ctx, codes, scales, x, t)
    assert np.isnan(y[:, 5]).all() and (y[:, 6] == 0).all()
    fine = np.arange(n) != 5
    assert (np.abs(y - xh @ w.T) <= X.linear_bound(w, xh, t))[:, fine].all()
    x[0, 700] = np.inf
    x[m - 1, 40] = np.nan if m > 1 else x[0, 40]
    got = linear(ctx, codes, scales, x, t)
    with np.errstate(invalid="ignore"):
        met = w[:, 700]
        assert np.array_equal(got[0, fine & (met > 0)], np.full((fine & (met > 0)).sum(), np.inf))
        assert np.array_equal(got[0, fine & (met < 0)], np.full((fine & (met < 0)).sum(), -np.inf))
        assert np.isnan(got[0, met == 0]).all()
    if m > 1:
        assert np.isnan(got[m - 1]).all()
        assert np.array_equal(got[1:m - 1], y[1:m - 1], equal_nan=True)


@pytest.mark.parametrize("m", [1, 40])
def test_linear_tiny_and_large_inputs(ctx, m):
    n, k = 48, 640
    codes, scales = weights(333, n, k)
    w = X.widen(codes, scales)
    for size in (2.0 ** -120, 2.0 ** 100):
        x = O.normal(334, m * k).reshape(m, k) * size
        xh = held("f32", x)
        y = linear(ctx, codes, scales, x, "f32")
        assert (np.abs(y - xh @ w.T) <= X.linear_bound(w, xh, "f32")).all()


# A scale byte of all weights and the inputs' binade: results at either end of
# the range, and well inside it where only one of the factors is not.
RANGE_ENDS = [(0, 30), (2, 0), (20, -10), (60, -60), (116, -113), (10, 100), (140, 80), (236, -3), (247, -60),
              (254, -100)]


@pytest.mark.parametrize("m", [70, 200])
@pytest.mark.parametrize("byte,binade", RANGE_ENDS)
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_linear_range_ends_in_tiles(ctx, m, byte, binade, t):
    n, k = 40, 640
    assert tokens(ctx, n, k, m, t) > 0
    codes = O.ints(341, n * k // 2, 256).astype(np.uint8).reshape(n, k // 2)
    scales = np.full((n, k // 32), byte, np.uint8)
    w = X.widen(codes, scales)
    x = O.normal(342, m * k).reshape(m, k).astype(np.float64) * 2.0 ** binade
    xh = held(t, x)
    y = linear(ctx, codes, scales, x, t)
    assert (np.abs(y - xh @ w.T) <= X.linear_bound(w, xh, t)).all()


@pytest.mark.parametrize("m", [1, 2, 4])
@pytest.mark.parametrize("byte,binade", RANGE_ENDS)
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_linear_range_ends_streamed(ctx, m, byte, binade, t):
    n, k = 40, 736
    assert tokens(ctx, n, k, m, t) == 0
    codes = O.ints(346, n * k // 2, 256).astype(np.uint8).reshape(n, k // 2)
    scales = np.full((n, k // 32), byte, np.uint8)
    w = X.widen(codes, scales)
    x = O.normal(347, m * k).reshape(m, k).astype(np.float64) * 2.0 ** binade
    xh = held(t, x)
    y = linear(ctx, codes, scales, x, t)
    assert (np.abs(y - xh @ w.T) <= X.linear_bound(w, xh, t)).all()


def test_linear_large_scales_beside_small_ones_streamed(ctx):
    """Blocks at both ends of a row and beside other rows, NaN scales among them."""
    m, n, k = 3, 48, 1120
    assert tokens(ctx, n, k, m, "f32") == 0
    codes = O.ints(348, n * k // 2, 256).astype(np.uint8).reshape(n, k // 2)
    scales = np.full((n, k // 32), 118, np.uint8)
    scales[5, 2], scales[5, 9] = 230, 20
    scales[17, 34], scales[18, 34], scales[40] = 191, 192, 3
    x = O.normal(349, m * k).reshape(m, k).astype(np.float64) * np.array([1.0, 2.0 ** -60, 2.0 ** -100])[:, None]
    w, xh = X.widen(codes, scales), held("f32", x)
    y = linear(ctx, codes, scales, x, "f32")
    assert (np.abs(y - xh @ w.T) <= X.linear_bound(w, xh, "f32")).all()
    scales[7, 34] = 255
    got = linear(ctx, codes, scales, x, "f32")
    fine = np.arange(n) != 7
    assert np.isnan(got[:, 7]).all() and np.array_equal(got[:, fine], y[:, fine])


def test_linear_zero_codes_of_the_largest_scale_in_tiles(ctx):
    m, n, k = 70, 20, 128
    assert tokens(ctx, n, k, m, "f32") > 0
    x = O.normal(343, m * k).reshape(m, k).astype(np.float64) * 2.0 ** 120
    codes, scales = np.zeros((n, k // 2), np.uint8), np.full((n, k // 32), 254, np.uint8)
    assert (linear(ctx, codes, scales, x, "f32") == 0).all()


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_linear_rows_at_both_ends_in_tiles(ctx, t):
    """Rows of weights and of inputs over the whole range in one call, held
    where the sums of magnitudes stay inside it."""
    m, n, k = 130, 150, 1056
    assert tokens(ctx, n, k, m, t) > 0
    codes = O.ints(344, n * k // 2, 256).astype(np.uint8).reshape(n, k // 2)
    scales = np.repeat(np.linspace(0, 254, n).astype(np.uint8)[:, None], k // 32, 1)
    x = O.normal(345, m * k).reshape(m, k).astype(np.float64) * np.exp2(np.linspace(-120, 120, m).round())[:, None]
    w, xh = X.widen(codes, scales), held(t, x)
    inside = np.abs(xh) @ np.abs(w).T < 2.0 ** 126
    assert inside.sum() > m * n / 2
    # bf16's subnormals are 2^-133 apart: half of that for a result below its normal numbers, which
    # the bound does not have (the exact result, rounded once, is past it at 421 of these places).
    bound = X.linear_bound(w, xh, t) + {"f32": 0.0, "bf16": 2.0 ** -134}[t]
    y = linear(ctx, codes, scales, x, t)
    assert (np.abs(y - xh @ w.T) <= bound)[inside].all()


@pytest.mark.parametrize("changed,says", [
    ({"k": 48}, "the dimension k is 48, outside its range 32..65536 multiple of 32"),
    ({"ldx": 63}, "ldx 63 is less than a row's 64 inputs"), ({"ldy": 9}, "ldy 9 is less than a row's 10 outputs"),
    ({"m": 0}, "the dimension m is 0, outside its range 1..65535")])
def test_linear_refusals(ctx, changed, says):
    from furykernel_b200 import _native as N

    b = [ctx.zeros(1 << 18, np.uint8) for _ in range(5)]
    p = {"n": 10, "k": 64, "m": 2, "ldx": 64, "ldy": 10} | changed
    with pytest.raises(N.Refused, match=says):
        ctx.launch("linear_mxfp4", p, b)
    with pytest.raises(N.Refused, match="buffer w is not aligned to 16 bytes"):
        ctx.launch("linear_mxfp4", {"n": 10, "k": 64, "m": 2, "ldx": 64, "ldy": 10}, [b[0].ptr + 8] + b[1:])
    for v in b:
        v.free()


# --------------------------------------------------------------------------
# The routed product


def routed(ctx, codes, scales, ids, x, t, per_rank, ldx=None, ldy=None):
    from furykernel_b200 import _native as N

    entries, n, kk = codes.shape[0], codes.shape[1], codes.shape[2] * 2
    m, k = ids.shape
    ldx, ldy = ldx or x.shape[1], ldy or k * n
    wd, sd, idd = ctx.to_device(codes), ctx.to_device(scales), ctx.to_device(ids.astype(np.uint32))
    xd = ctx.to_device(strided(t, x, ldx))
    yd = ctx.to_device(strided(t, np.full((m, k * n), MARK, np.float32), ldy))
    work = ctx.alloc(N.linear_mxfp4_work(n, kk, m, entries, k), np.uint8)
    work.upload(np.full(work.nbytes, 0xFF, np.uint8))
    ctx.launch("linear_routed_mxfp4" + SUFFIX[t],
               {"entries": entries, "n": n, "kk": kk, "m": m, "k": k, "ldx": ldx, "ldy": ldy,
                "per_rank": int(per_rank)}, [wd, sd, idd, xd, yd, work])
    y = X.widen_type(t, yd.download())
    assert ctx.status() == 0
    assert (y[:, k * n:] == MARK).all()
    for b in (wd, sd, idd, xd, yd, work):
        b.free()
    return y[:, :k * n].reshape(m, k, n).astype(np.float64)


def held_to_experts(y, codes, scales, ids, x, t, per_rank):
    """Every (row, rank) against its expert's weights; 0 where there is none."""
    m, k = ids.shape
    kk = codes.shape[2] * 2
    xh = held(t, x).reshape(m, -1, kk)
    pairs = [(r, j) for r in range(m) for j in range(k)]
    for e in np.unique(ids):
        mine = [(r, j) for r, j in pairs if ids[r, j] == e]
        got = np.stack([y[p] for p in mine])
        if e >= codes.shape[0]:
            assert (got == 0).all()
            continue
        w = X.widen(codes[e], scales[e])
        xe = np.stack([xh[r, j if per_rank else 0] for r, j in mine])
        assert (np.abs(got - xe @ w.T) <= X.linear_bound(w, xe, t)).all()


@pytest.mark.parametrize("entries,n,kk,m,k", [(1, 40, 64, 1, 1), (8, 130, 96, 1, 2), (64, 72, 352, 16, 4),
                                              (8, 200, 1056, 33, 2), (40, 1500, 512, 60, 4), (16, 129, 544, 100, 8), (4, 260, 512, 300, 3)])
@pytest.mark.parametrize("per_rank", [False, True])
@pytest.mark.parametrize("t", TYPES)
def test_routed(ctx, entries, n, kk, m, k, per_rank, t):
    codes, scales = weights(341, entries, n, kk)
    ids = O.ints(342, m * k, entries).reshape(m, k)
    x = O.normal(343, m * kk * (k if per_rank else 1)).reshape(m, -1)
    y = routed(ctx, codes, scales, ids, x, t, per_rank, ldx=x.shape[1] + 4, ldy=k * n + 2)
    held_to_experts(y, codes, scales, ids, x, t, per_rank)


@pytest.mark.parametrize("m", [1, 9, 150])
def test_routed_uneven(ctx, m):
    """All rows on one expert; experts without rows; ids past the table;
    one expert for all ranks of a row."""
    entries, n, kk, k = 6, 140, 608, 3
    codes, scales = weights(351, entries, n, kk)
    x = O.normal(352, m * kk).reshape(m, kk)
    for ids in (np.full((m, k), 5), np.stack([np.arange(m) % 2, np.full(m, 4), np.full(m, 6)], 1),
                np.full((m, k), 0xFFFFFFFF, np.uint32), np.stack([np.full(m, 2), np.full(m, 7), np.full(m, 2)], 1)):
        y = routed(ctx, codes, scales, ids, x, "f32", False)
        held_to_experts(y, codes, scales, ids, x, "f32", False)


@pytest.mark.parametrize("entries,n,kk,m,k", [(16, 1300, 2080, 400, 8), (16, 2600, 4096, 600, 8)])
@pytest.mark.parametrize("t", TYPES)
def test_routed_many_tiles(ctx, entries, n, kk, m, k, t):
    """Several tiles a block, several runs a tile, uneven experts, one without
    rows; held at some of the columns."""
    codes = O.ints(381, entries * n * kk // 2, 256).astype(np.uint8).reshape(entries, n, kk // 2)
    scales = (120 + O.ints(382, entries * n * kk // 32, 5)).astype(np.uint8).reshape(entries, n, kk // 32)
    ids = np.minimum(O.ints(383, m * k, entries), O.ints(384, m * k, entries)).reshape(m, k)
    ids[ids == 2] = 9
    x = O.normal(385, m * kk).reshape(m, kk)
    y = routed(ctx, codes, scales, ids, x, t, False)
    at = np.unique(np.concatenate([[0, 127, 128, n - 1], O.ints(386, 24, n)]))
    held_to_experts(y[:, :, at], codes[:, at], scales[:, at], ids, x, t, False)


@pytest.mark.parametrize("m", [4, 120])
def test_routed_same_every_time(ctx, m):
    entries, n, kk, k = 8, 256, 1024, 4
    codes, scales = weights(361, entries, n, kk)
    ids = O.ints(362, m * k, entries).reshape(m, k)
    x = O.normal(363, m * kk).reshape(m, kk)
    a = routed(ctx, codes, scales, ids, x, "f32", False)
    for _ in range(3):
        assert np.array_equal(routed(ctx, codes, scales, ids, x, "f32", False), a)


@pytest.mark.parametrize("t,entries,n,kk,m,k", [("f32", 8, 256, 2048, 300, 4), ("f32", 3, 520, 2720, 500, 3),
                                                ("bf16", 8, 700, 2048, 900, 6)])
def test_routed_same_every_time_over_cut_tiles(ctx, t, entries, n, kk, m, k):
    """Several token tiles an expert and three and more runs a tile, cut at other
    runs from tile to tile: where a pair's sums are cut has to be the same."""
    assert tokens(ctx, n, kk, m, t, entries, k, True) * entries < m * k
    codes, scales = weights(364, entries, n, kk)
    ids = O.ints(365, m * k, entries).reshape(m, k)
    x = O.normal(366, m * kk).reshape(m, kk)
    a = routed(ctx, codes, scales, ids, x, t, False)
    for _ in range(8):
        assert np.array_equal(routed(ctx, codes, scales, ids, x, t, False), a)


@pytest.mark.parametrize("entries,m,k", [(1, 700, 1), (31, 513, 2), (1162, 2100, 3), (1163, 2100, 3), (4096, 2111, 8)])
def test_routed_grouping(ctx, entries, m, k):
    """Every pair meets its expert, with many experts and few, some of them past the table."""
    n, kk = 20, 64
    codes = O.ints(367, entries * n * kk // 2, 256).astype(np.uint8).reshape(entries, n, kk // 2)
    scales = (120 + O.ints(368, entries * n * kk // 32, 5)).astype(np.uint8).reshape(entries, n, kk // 32)
    ids = O.ints(369, m * k, entries + entries // 8).reshape(m, k)
    x = O.normal(370, m * kk).reshape(m, kk)
    y = routed(ctx, codes, scales, ids, x, "f32", False)
    w, xh = X.widen(codes, scales), held("f32", x)
    kept = np.where(ids < entries, ids, 0)
    want = np.einsum("rjnc,rc->rjn", w[kept], xh) * (ids < entries)[..., None]
    sums = np.einsum("rjnc,rc->rjn", np.abs(w[kept]), np.abs(xh)) * (ids < entries)[..., None]
    # One run: at most 4 truncated sums of 2^-23, the inputs' parts 2^-22 (or 2^-38 of the row's largest).
    top = np.abs(xh).max(-1)[:, None, None] * np.abs(w[kept]).sum(-1)
    assert (np.abs(y - want) <= sums * 2.0 ** -20 + top * 2.0 ** -38).all()


@pytest.mark.parametrize("m", [1, 64])
def test_routed_past_4_gib(ctx, m):
    """A table whose last expert starts past 2^32 bytes."""
    from furykernel_b200 import _native as N

    entries, n, kk = 1100, 1024, 8192
    codes, scales = weights(371, 1, n, kk)
    size = n * kk // 2
    wd, sd = ctx.alloc(entries * size, np.uint8), ctx.alloc(entries * size // 16, np.uint8)
    N.check(N.lib().fkc_buf_zero(ctx.handle, wd.ptr, wd.nbytes))
    N.check(N.lib().fkc_buf_zero(ctx.handle, sd.ptr, sd.nbytes))
    last = entries - 1
    N.check(N.lib().fkc_buf_upload(ctx.handle, wd.ptr + last * size, codes.ctypes.data, codes.nbytes))
    N.check(N.lib().fkc_buf_upload(ctx.handle, sd.ptr + last * size // 16, scales.ctypes.data, scales.nbytes))
    assert last * size > 2 ** 32
    x = O.normal(372, m * kk).reshape(m, kk)
    ids = np.full((m, 2), last, np.uint32)
    ids[:, 1] = 3
    idd, xd, yd = ctx.to_device(ids), ctx.to_device(x.astype(np.float32)), ctx.zeros((m, 2 * n))
    work = ctx.alloc(N.linear_mxfp4_work(n, kk, m, entries, 2), np.uint8)
    ctx.launch("linear_routed_mxfp4", {"entries": entries, "n": n, "kk": kk, "m": m, "k": 2, "ldx": kk,
                                       "ldy": 2 * n, "per_rank": 0}, [wd, sd, idd, xd, yd, work])
    y = yd.download().astype(np.float64)
    assert ctx.status() == 0
    w = X.widen(codes[0], scales[0])
    xh = held("f32", x)
    assert (np.abs(y[:, :n] - xh @ w.T) <= X.linear_bound(w, xh, "f32")).all()
    assert (y[:, n:] == 0).all()
    for b in (wd, sd, idd, xd, yd, work):
        b.free()


# --------------------------------------------------------------------------
# Each kernel by name: the sizes state which one they reach, and a change of the
# rule that sends them elsewhere fails here.


def tokens(ctx, n, k, m, t, entries=1, ranks=1, routed=False):
    from furykernel_b200 import _native as N

    return N.linear_mxfp4_tokens(ctx.sms, n, k, m, entries, ranks, routed, 4 if t == "f32" else 2)


def any_weights(seed, *shape):
    """Codes of every kind, scales over 5 binades."""
    size = int(np.prod(shape))
    codes = O.ints(seed, size // 2, 256).astype(np.uint8).reshape(shape[:-1] + (-1,))
    return codes, (116 + O.ints(seed + 1, size // 32, 5)).astype(np.uint8).reshape(shape[:-1] + (-1,))


def some_columns(seed, n):
    return np.unique(np.concatenate([[0, min(127, n - 1), min(128, n - 1), n - 1], O.ints(seed, 40, n)]))


# By norm, as test_linear: 66 steps of 2^-24, 16-bit outputs their own rounding.
NORM = {"f32": 66 * 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
# (rows, n, k, tokens a tile: f32, 16-bit)
DENSE_TILES = [(70, 300, 1120, 16, 16), (65, 2100, 4128, 32, 32), (128, 4500, 4128, 64, 64), (500, 8900, 4128, 128, 160)]


@pytest.mark.parametrize("m,n,k,wide,narrow", DENSE_TILES)
@pytest.mark.parametrize("t", TYPES)
def test_linear_tiles(ctx, m, n, k, wide, narrow, t):
    """Every width of tile, tiles cut over the blocks, rows and columns off the
    tiles' ends, rows off 16 bytes."""
    assert tokens(ctx, n, k, m, t) == (wide if t == "f32" else narrow)
    codes, scales = any_weights(401, n, k)
    x = O.normal(403, m * k).reshape(m, k) * np.exp(O.normal(404, k))[None]
    y = linear(ctx, codes, scales, x, t)
    assert np.array_equal(linear(ctx, codes, scales, x, t, k + 1, n + 3), y)
    at = some_columns(405, n)
    w, xh = X.widen(codes[at], scales[at]), held(t, x)
    want = xh @ w.T
    assert (np.abs(y[:, at] - want) <= X.linear_bound(w, xh, t)).all()
    assert np.linalg.norm(y[:, at] - want) / np.linalg.norm(want) <= NORM[t]


@pytest.mark.parametrize("m,n,k,wide,narrow", DENSE_TILES)
@pytest.mark.parametrize("t", TYPES)
def test_linear_tiles_tiny_and_large_inputs(ctx, m, n, k, wide, narrow, t):
    """Rows of inputs over the type's range, zeros, an infinity and a NaN among them."""
    assert tokens(ctx, n, k, m, t) == (wide if t == "f32" else narrow)
    codes, scales = any_weights(406, n, k)
    ends = 8 if t == "f16" else 100
    x = O.normal(408, m * k).reshape(m, k) * np.exp2(np.linspace(-ends, ends, m).round())[:, None]
    x[7] = 0
    x[20, 600], x[m - 1, 0] = np.inf, np.nan
    y = linear(ctx, codes, scales, x, t)
    at = some_columns(409, n)
    w, xh = X.widen(codes[at], scales[at]), held(t, x)
    fine = np.isfinite(xh).all(-1)
    assert fine.sum() == m - 2
    assert (np.abs(y[fine][:, at] - xh[fine] @ w.T) <= X.linear_bound(w, xh[fine], t)).all()
    assert (y[7] == 0).all() and np.isnan(y[m - 1]).all()
    with np.errstate(invalid="ignore"):
        assert np.array_equal(y[20, at], np.inf * w[:, 600], equal_nan=True)


@pytest.mark.parametrize("m,n,k", [(1, 300, 1120), (2, 2100, 608), (3, 130, 4128), (40, 48, 640), (40, 77, 352)])
@pytest.mark.parametrize("t", TYPES)
def test_linear_streamed(ctx, m, n, k, t):
    assert tokens(ctx, n, k, m, t) == 0
    codes, scales = any_weights(411, n, k)
    x = O.normal(413, m * k).reshape(m, k) * np.exp(O.normal(414, k))[None]
    y = linear(ctx, codes, scales, x, t)
    assert np.array_equal(linear(ctx, codes, scales, x, t, k + 1, n + 3), y)
    w, xh = X.widen(codes, scales), held(t, x)
    want = xh @ w.T
    assert (np.abs(y - want) <= X.linear_bound(w, xh, t)).all()
    assert np.linalg.norm(y - want) / np.linalg.norm(want) <= NORM[t]


@pytest.mark.parametrize("entries,n,kk,m,k,wide,narrow", [
    (8, 300, 1120, 2, 3, 0, 0), (4, 260, 544, 300, 3, 16, 16), (8, 900, 2080, 200, 4, 32, 32),
    (8, 900, 2080, 300, 8, 64, 64), (2, 7000, 4128, 900, 2, 128, 160)])
@pytest.mark.parametrize("per_rank", [False, True])
@pytest.mark.parametrize("t", TYPES)
def test_routed_kernels(ctx, entries, n, kk, m, k, wide, narrow, per_rank, t):
    """As test_linear_tiles, with some ids past the table; held at some of the columns."""
    assert tokens(ctx, n, kk, m, t, entries, k, True) == (wide if t == "f32" else narrow)
    codes, scales = any_weights(421, entries, n, kk)
    ids = O.ints(423, m * k, entries).reshape(m, k)
    ids[m - 1, 0] = entries
    width = kk * (k if per_rank else 1)
    x = O.normal(424, m * width).reshape(m, width)
    y = routed(ctx, codes, scales, ids, x, t, per_rank, width + 1, k * n + 3)
    at = some_columns(425, n)
    held_to_experts(y[:, :, at], codes[:, at], scales[:, at], ids, x, t, per_rank)
    w, xh = X.widen(codes[:, at], scales[:, at]), held(t, x).reshape(m, -1, kk)
    off = total = 0.0
    for r, j in np.argwhere(ids < entries):
        want = w[ids[r, j]] @ xh[r, j if per_rank else 0]
        off += ((y[r, j, at] - want) ** 2).sum()
        total += (want ** 2).sum()
    assert np.sqrt(off / total) <= NORM[t]


def test_routed_refusals(ctx):
    from furykernel_b200 import _native as N

    b = [ctx.zeros(1 << 18, np.uint8) for _ in range(6)]
    p = {"entries": 4, "n": 10, "kk": 64, "m": 2, "k": 2, "ldx": 64, "ldy": 20, "per_rank": 0}
    for changed, says in (({"per_rank": 1}, "ldx 64 is less than a row's 128 inputs"),
                          ({"ldy": 19}, "ldy 19 is less than a row's 20 outputs"),
                          ({"kk": 80}, "the dimension kk is 80, outside its range 32..65536 multiple of 32"),
                          ({"k": 9}, "the dimension k is 9, outside its range 1..8"),
                          ({"entries": 4097}, "the dimension entries is 4097, outside its range 1..4096")):
        with pytest.raises(N.Refused, match=says):
            ctx.launch("linear_routed_mxfp4", p | changed, b)
    with pytest.raises(N.Refused, match="5 buffers bound, not 6"):
        ctx.launch("linear_routed_mxfp4", p, b[:5])
    for v in b:
        v.free()
