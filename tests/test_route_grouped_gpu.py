"""The grouped router on a B200: the experts exactly, the weights within the
rounding of their last operations, against the definition in numpy."""

import numpy as np
import pytest

from oracle import oracle as O
from tests import mxfp4_check as X

pytestmark = pytest.mark.gpu

SUFFIX = {"f32": "", "bf16": "_xbf16", "f16": "_xf16"}


@pytest.fixture(scope="module")
def ctx():
    from furykernel_b200 import _native as N

    c = N.Context(0)
    yield c
    c.close()


def run(ctx, x, k, t="f32", bias=None, ldx=None, **o):
    m, n = x.shape
    ldx = ldx or n
    wide = np.full((m, ldx), np.nan, np.float32)  # what lies between the rows is not read
    wide[:, :n] = x
    xd = ctx.to_device(X.narrow(t, wide))
    ids, ws = ctx.to_device(np.full((m, k), 77, np.uint32)), ctx.to_device(np.full((m, k), 77, np.float32))
    params = {"m": m, "n": n, "k": k, "groups": o.get("groups", 1), "top_groups": o.get("top_groups", 1),
              "group_by": o.get("group_by", 1), "sigmoid": int(o.get("sigmoid", False)),
              "renorm": int(o.get("renorm", False)), "ldx": ldx, "factor": o.get("factor", 1.0)}
    held = [xd, ids, ws]
    if bias is None:
        ctx.launch("route_grouped" + SUFFIX[t], params, [xd, ids, ws])
    else:
        bd = ctx.to_device(np.asarray(bias, np.float32))
        held.append(bd)
        ctx.launch("route_grouped_bias" + SUFFIX[t], params, [xd, bd, ids, ws])
    got = ids.download(), ws.download()
    for b in held:
        b.free()
    return got


def held_to(got, x, k, t="f32", **o):
    ids, ws, _ = X.route_grouped(X.widen_type(t, X.narrow(t, x)), k, **o)
    assert np.array_equal(got[0], ids)
    assert np.array_equal(np.isnan(got[1]), np.isnan(ws))
    # A score, k - 1 sums, a quotient and a product, each within 2^-24: (k + 3) of them.
    far = np.abs(got[1].astype(np.float64) - ws)
    assert (far[~np.isnan(ws)] <= ((k + 3) * 2.0 ** -24 * np.abs(ws) + 2.0 ** -149)[~np.isnan(ws)]).all()


@pytest.mark.parametrize("m,n,k,groups,top_groups,group_by", [
    (1, 1, 1, 1, 1, 1), (1, 64, 4, 1, 1, 1), (5, 33, 8, 1, 1, 1), (3, 160, 6, 8, 3, 1), (130, 256, 8, 8, 4, 2),
    (7, 96, 8, 32, 8, 2), (9, 32, 4, 32, 8, 2), (4, 1000, 8, 4, 1, 2), (2, 1024, 8, 1, 1, 1), (6, 8, 8, 4, 4, 1)])
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
def test_route(ctx, m, n, k, groups, top_groups, group_by, sigmoid, t):
    x = 2 * O.normal(301, m * n).reshape(m, n)
    o = dict(groups=groups, top_groups=top_groups, group_by=group_by, sigmoid=sigmoid)
    held_to(run(ctx, x, k, t, **o), x, k, t, **o)
    bias = 0.3 * O.normal(302, n)
    o |= dict(renorm=True, factor=2.5, bias=bias)
    held_to(run(ctx, x, k, t, ldx=n + 3, **o), x, k, t, **o)


@pytest.mark.parametrize("sigmoid", [False, True])
def test_ties_and_masked_logits(ctx, sigmoid):
    n, k = 40, 6
    x = O.normal(303, 9 * n).reshape(9, n).astype(np.float32)
    x[0] = 0.25  # all equal: the lowest indices, the lowest groups
    x[1, 10:30] = 3.0  # a tie over two groups
    x[2, :35] = -np.inf  # all but 5 experts masked
    x[3] = -np.inf  # all of them: weights 0
    x[4, 7] = np.nan
    x[5] = np.finfo(np.float32).min
    x[6] = np.finfo(np.float32).min
    x[6, 33] = 1.0
    x[7] = -200.0  # sigmoid underflows to 0, softmax does not
    x[8, ::2] = -np.inf
    for o in (dict(), dict(groups=4, top_groups=2, group_by=2), dict(groups=8, top_groups=3, group_by=1)):
        o |= dict(sigmoid=sigmoid, renorm=True)
        got = run(ctx, x, k, **o)
        held_to(got, x, k, **o)
        assert (got[1][3] == 0).all()


def test_infinite_logits(ctx):
    x = O.normal(304, 2 * 16).reshape(2, 16).astype(np.float32)
    x[0, 5] = np.inf
    got = run(ctx, x, 3, sigmoid=True)
    held_to(got, x, 3, sigmoid=True)
    assert got[0][0, 0] == 5 and got[1][0, 0] == 1.0


def test_same_every_time(ctx):
    x = O.normal(305, 64 * 200).reshape(64, 200)
    o = dict(groups=8, top_groups=4, group_by=2, renorm=True)
    a, b = run(ctx, x, 8, **o), run(ctx, x, 8, **o)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1].view(np.uint32), b[1].view(np.uint32))


@pytest.mark.parametrize("changed,says", [
    ({"groups": 3}, "64 experts do not form 3 groups"), ({"top_groups": 5}, "top_groups 5 is more than the 4 groups"),
    ({"k": 8, "groups": 32, "top_groups": 2}, "k 8 is more than the 4 experts of 2 groups"),
    ({"ldx": 63}, "ldx 63 is less than n 64"), ({"k": 9}, "the dimension k is 9, outside its range 1..8"),
    ({"group_by": 3}, "the dimension group_by is 3, outside its range 1..2"),
    ({"n": 1025}, "the dimension n is 1025, outside its range 1..1024")])
def test_refusals(ctx, changed, says):
    from furykernel_b200 import _native as N

    x, ids, ws = ctx.zeros((2, 64)), ctx.zeros((2, 8), np.uint32), ctx.zeros((2, 8))
    p = {"m": 2, "n": 64, "k": 4, "groups": 4, "top_groups": 2, "group_by": 1, "sigmoid": 0, "renorm": 0, "ldx": 64,
         "factor": 1.0} | changed
    with pytest.raises(N.Refused, match=says):
        ctx.launch("route_grouped", p, [x, ids, ws])
    for b in (x, ids, ws):
        b.free()
