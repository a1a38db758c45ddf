"""The routed FFN of MXFP4 experts on a B200: route, products, gate and
combine together, against the same steps in binary64."""

import math

import numpy as np
import pytest

from oracle import oracle as O
from tests import mxfp4_check as X

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from furykernel_b200 import _native as N

    c = N.Context(0)
    yield c
    c.close()


def gelu(v):
    return 0.5 * v * (1 + np.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))


E, D, F, K = 16, 192, 96, 4


def block(ctx, rows, bias):
    from furykernel_b200.experts import RoutedExperts

    router = O.normal(501, E * D, 0.0, 0.1).reshape(E, D)
    gate_up = O.normal(502, E * 2 * F * D, 0.0, 0.05).reshape(E, 2 * F, D).astype(np.float32)
    down = O.normal(503, E * D * F, 0.0, 0.05).reshape(E, D, F).astype(np.float32)
    opts = dict(groups=4, top_groups=2, group_by=2, sigmoid=True, renorm=True, factor=2.5,
                bias=O.normal(504, E, 0.0, 0.2).astype(np.float32) if bias else None)
    return RoutedExperts(ctx, router, gate_up, down, F, K, rows, **opts), router, gate_up, down, opts


def expected(router, gate_up, down, opts, x, ids):
    """The block in binary64 with the device's picks."""
    wgu, wdn = X.widen(*X.quantise(gate_up)), X.widen(*X.quantise(down))
    s = 1 / (1 + np.exp(-(x.astype(np.float64) @ router.astype(np.float32).astype(np.float64).T)))
    y = x.astype(np.float64).copy()
    for r in range(x.shape[0]):
        w = s[r, ids[r]]
        w = w / w.sum() * opts["factor"]
        for j, e in enumerate(ids[r]):
            gu = wgu[e] @ x[r].astype(np.float64)
            y[r] += w[j] * (wdn[e] @ (gelu(gu[:F]) * gu[F:]))
    return y


@pytest.mark.parametrize("m", [1, 5, 70, 300])
@pytest.mark.parametrize("bias", [False, True])
def test_experts_block(ctx, m, bias):
    b, router, gate_up, down, opts = block(ctx, 300, bias)
    x = O.normal(505, m * D).reshape(m, D).astype(np.float32)
    xd, yd = ctx.to_device(x), ctx.zeros((m, D))
    b.launch(xd, yd, m)
    y, ids, logits = yd.download().astype(np.float64), b.ids.download()[:m], b.logits.download()[:m]
    assert ctx.status() == 0
    # The picks are the route's of the device's own logits.
    want_ids, _, _ = X.route_grouped(logits, K, 4, 2, 2, True, True, 2.5, opts["bias"])
    assert np.array_equal(ids, want_ids)
    want = expected(router, gate_up, down, opts, x, ids)
    # Two products, each within 2^-17 of the sums of magnitudes (64 truncated steps of 2^-23), the
    # gate and the weights a few 2^-23; those sums are under 16 times the result's own norm here.
    assert np.linalg.norm(y - want) <= 2.0 ** -12 * np.linalg.norm(want - x)
    # The same from a graph, over other values.
    ctx.capture_begin()
    b.launch(xd, yd, m)
    g = ctx.capture_end()
    yd.upload(np.zeros((m, D), np.float32))
    g.launch()
    ctx.sync()
    assert np.array_equal(yd.download().astype(np.float64), y)
    g.destroy()
    b.free()
    xd.free()
    yd.free()


@pytest.mark.parametrize("m", [5, 70])
def test_experts_block_captured(ctx, m):
    """A graph of the block computes all of it from the rows that it finds: every buffer
    between the rows and the result is marked before each replay, and the rows change."""
    b = block(ctx, 300, True)[0]
    xd, yd = ctx.zeros((m, D)), ctx.zeros((m, D))
    rows = [O.normal(506 + i, m * D).reshape(m, D).astype(np.float32) for i in range(3)]
    xd.upload(rows[0])
    ctx.capture_begin()
    b.launch(xd, yd, m)
    g = ctx.capture_end()
    eager = []
    for x in rows:
        xd.upload(x)
        b.launch(xd, yd, m)
        eager.append((yd.download(), b.ids.download()[:m]))
    assert not np.array_equal(eager[0][1], eager[1][1])
    for x, (y, ids) in zip(rows, eager):
        xd.upload(x)
        for between in (b.logits, b.ids, b.ws, b.gu, b.act, b.out, b.work, b.parts, yd):
            between.upload(np.full(between.shape, 0x7F, between.dtype))
        g.launch()
        ctx.sync()
        assert np.array_equal(yd.download(), y)
        assert np.array_equal(b.ids.download()[:m], ids)
    assert ctx.status() == 0
    g.destroy()
    b.free()
    xd.free()
    yd.free()


def test_refusals(ctx):
    from furykernel_b200 import _native as N
    from furykernel_b200.experts import Mxfp4Table

    b = block(ctx, 4, False)[0]
    xd = ctx.zeros((5, D))
    for m in (0, 5):
        with pytest.raises(N.Refused, match="outside 1..4"):
            b.launch(xd, xd, m)
    with pytest.raises(N.Refused, match="not 2 x 8 x 32"):
        Mxfp4Table(ctx, np.zeros((2, 8, 64), np.float32), 2, 8, 32)
    b.free()
    xd.free()
