"""MXFP4 and the grouped route without a GPU: known answers of the numpy
restatement that the kernels are held to, and the entries' interfaces."""

import numpy as np

from furykernel_b200 import _native as N
from tests import mxfp4_check as X


def test_quantise_known_answers():
    x = np.zeros((1, 32), np.float32)
    x[0, :8] = [6, -3, 0.25, 0.75, 2.5, 5, -0.0, 1.25]  # ties: 0, 1, 2, 4 and 1 are the even ones
    codes, scales = X.quantise(x)
    assert scales[0, 0] == 127
    assert list(X.widen(codes, scales)[0, :8]) == [6, -3, 0, 1, 2, 4, 0, 1]
    assert np.signbit(X.widen(codes, scales)[0, 6])
    x[0, 9] = 7.9  # still the same scale: past 6 to 6
    codes, scales = X.quantise(x)
    assert scales[0, 0] == 127 and X.widen(codes, scales)[0, 9] == 6
    x[0, 9] = 8.0
    assert X.quantise(x)[1][0, 0] == 128
    x[0, 9] = np.nan
    codes, scales = X.quantise(x)
    assert scales[0, 0] == 255 and np.isnan(X.widen(codes, scales)).all() and not codes.any()


def test_quantise_is_its_own_inverse():
    rng = np.random.default_rng(5)
    codes = rng.integers(0, 256, (64, 32), np.uint8)
    codes[:, ::16] |= 0x07  # a 6 in every block of 32, so that the scale is the block's own
    scales = rng.integers(3, 250, (64, 2)).astype(np.uint8)
    again = X.quantise(X.widen(codes, scales).astype(np.float32))
    assert np.array_equal(again[0], codes) and np.array_equal(again[1], scales)


def test_route_known_answers():
    x = np.log(np.array([[1, 2, 3, 4, 4, 3, 2, 1]], np.float32))
    ids, ws, _ = X.route_grouped(x, 3)
    assert list(ids[0]) == [3, 4, 2] and np.allclose(ws, [[0.2, 0.2, 0.15]])
    ids, ws, _ = X.route_grouped(x, 2, groups=4, top_groups=1, group_by=2, renorm=True, factor=2.0)
    assert list(ids[0]) == [3, 2] and np.allclose(ws, [[8 / 7, 6 / 7]])
    bias = np.zeros(8, np.float32)
    bias[7] = 1.0
    ids, ws, _ = X.route_grouped(x, 2, sigmoid=True, bias=bias)
    assert list(ids[0]) == [7, 3] and np.allclose(ws, [[0.5, 0.8]])  # the bias chooses, the score weighs


def test_work_bytes():
    assert N.linear_mxfp4_work(100, 64, 3) == 5 * 3 * 64 + 16 * 3 * 100 + 16 * 3 + 64 + 65536
    assert (N.linear_mxfp4_work(1 << 20, 65536, 65535, 4096, 8)
            == 5 * 65535 * 8 * 65536 + 16 * 512 * (1 << 20) + 16 * 65535 * 8 + 64 * 4096 + 65536)


def test_forms_retype_the_activations():
    table = N.table()
    for base, typed in (("route_grouped", {"x"}), ("route_grouped_bias", {"x"}), ("quant_mxfp4", {"x"}),
                        ("linear_mxfp4", {"x", "y"}), ("linear_routed_mxfp4", {"x", "y"})):
        for t in ("bf16", "f16"):
            for a, b in zip(table[base].buffers, table[f"{base}_x{t}"].buffers):
                assert b.type == (t if a.name in typed else a.type)


def test_routed_experts_refuse_buffers_that_are_too_short():
    """Before anything is allocated or launched: what is read past its end would be another's memory."""
    import pytest

    from furykernel_b200.experts import RoutedExperts

    e, d, ffn = 8, 64, 32
    arrays = np.zeros((e, d)), np.zeros((e, 2 * ffn, d)), np.zeros((e, d, ffn))
    for short in (e - 1, e + 1, 1):
        with pytest.raises(N.Refused, match=f"routed experts: the bias has {short} values, not 8"):
            RoutedExperts(None, *arrays, ffn, 2, 4, bias=np.zeros(short))
    block = object.__new__(RoutedExperts)
    block.rows, block.d = 4, d
    rows = [N.DeviceBuffer(None, 256, 4 * n * d) for n in (2, 3)]
    with pytest.raises(N.Refused, match="routed experts: x holds fewer than 3 rows of 64"):
        block.launch(rows[0], rows[1], 3)
    with pytest.raises(N.Refused, match="routed experts: y holds fewer than 3 rows of 64"):
        block.launch(rows[1], rows[0], 3)


def test_packing_words_a_wrong_name():
    import pytest

    e = N.table()["linear_mxfp4"]
    with pytest.raises(N.Refused, match="linear_mxfp4 has no parameter kk"):
        e.pack({"n": 1, "kk": 32, "m": 1, "ldx": 32, "ldy": 1})
    with pytest.raises(N.Refused, match="linear_mxfp4: no value for the parameter ldy"):
        e.pack({"n": 1, "k": 32, "m": 1, "ldx": 32})
    assert e.pack({"ldy": 5, "ldx": 4, "m": 3, "k": 32, "n": 1}) == b"".join(
        v.to_bytes(4, "little") for v in (1, 32, 3, 4, 5))


def test_which_kernel():
    """One row streams, a prompt goes to the widest tiles; the tests of each kernel state their own sizes."""
    import pytest

    assert N.linear_mxfp4_tokens(148, 11008, 4096, 1) == 0
    assert [N.linear_mxfp4_tokens(148, 22016, 4096, 511, elem_bytes=b) for b in (4, 2)] == [128, 160]
    assert N.linear_mxfp4_tokens(148, 1408, 2048, 1, 64, 4, True) == 0
    for bad in ((0, 64, 64, 1), (148, 64, 48, 1), (148, 64, 64, 0), (148, 64, 64, 1, 1, 1, False, 1)):
        with pytest.raises(N.Refused, match="fkc_linear_mxfp4_tokens: bad argument"):
            N.linear_mxfp4_tokens(*bad)
