"""The int8 lane where f32 ends and where sizes do: squares past the largest f32, an epsilon of 0, rows of no values, very long rows, single rows of any
stride, more workgroups than one launch may have, and large products cell by cell.

Tolerances are those of the lane's other tests: 4e-6 on scales and normalised values, whatever a row's length; bits elsewhere.
"""
import numpy as np
import pytest

from camelid_amd import binding as B
from camelid_amd.binding import check, lib
from tests import gpu_util as G
from tests.test_gpu_int8_lane import check_norm, f32, norm, operands, product, want_product
from tests.typed_rows import BITS, TYPES, Rows, from_bits, to_bits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [4, 600, 5000, 40001])
def test_squares_past_the_largest_f32_say_so(t, cols):
    """No quants, a scale and normalised values that are not finite, and nothing of it in the rows beside."""
    rng = np.random.default_rng(cols)
    x = rng.standard_normal((7, cols)).astype(np.float32)
    x[1, :4] = [1e20, -5e19, 1e18, 3]  # one square alone
    x[3] = 0
    x[3, :4] = 1.2e19                  # each square is finite, their sum is not
    x[5] = 3e38 * np.sign(x[5])
    w = (0.5 + rng.random(cols)).astype(np.float32)
    bits = to_bits(x, t)
    for residual in (None, np.zeros_like(bits)):
        s, y, q, d = norm(t, bits, residual, w, 1e-5)
        bad, good = [1, 3, 5], [0, 2, 4, 6]
        assert not np.any(np.isfinite(d[bad])) and np.all(q[bad] == 0), (d, q[bad][:, :4])
        assert np.all(np.isnan(y[bad]))
        assert np.array_equal(s, bits)
        check_norm(t, bits[good], None, w, 1e-5, (s[good], y[good], q[good], d[good]))


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cols", [1, 600, 5000, 40001])
def test_an_epsilon_of_zero(t, cols):
    rng = np.random.default_rng(cols)
    x = rng.standard_normal((5, cols)).astype(np.float32)
    x[1] = 0
    x[3] = -0.0
    r = np.zeros_like(x)
    r[4] = -from_bits(to_bits(x[4], t), t)  # the residual takes it all away
    w = (0.5 + rng.random(cols)).astype(np.float32)
    s, y, q, d = norm(t, to_bits(x, t), to_bits(r, t), w, 0.0)
    zero = [1, 3, 4]
    assert np.all(d[zero] == 0) and np.all(q[zero] == 0) and np.all(y[zero] == 0), d
    check_norm(t, to_bits(x[[0, 2]], t), None, w, 0.0, (s[[0, 2]], y[[0, 2]], q[[0, 2]], d[[0, 2]]))
    if t != "f16":  # squares that all vanish: not a row of zeros, and no scale that could be given
        tiny = np.full((1, cols), 1e-30, np.float32)
        _, y, q, d = norm(t, to_bits(tiny, t), None, w, 0.0)
        assert not np.isfinite(d[0]) and np.all(q == 0)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_rows_of_no_values_have_scale_zero(t):
    B.init(0)
    n = 700
    x, q, w, D = Rows.empty(1, 8, BITS[t]), Rows.empty(1, 8, np.int8), f32(np.ones(1)), Rows.empty(1, n, np.float32)
    G.say(f"quantize_i8 / add_rms_norm_i8 {t} {n}x0")
    check(lib().cml_quantize_i8(TYPES[t], x.ptr, 0, n, 0, q.ptr, 0, D.ptr, None))
    check(lib().cml_stream_sync(None))
    assert np.all(D.get() == 0)
    D = Rows.empty(1, n, np.float32)
    check(lib().cml_add_rms_norm_i8(TYPES[t], x.ptr, 0, x.ptr, 0, w.ptr, 0.0, n, 0, x.ptr, 0, None, q.ptr, 0, D.ptr, None))
    check(lib().cml_stream_sync(None))
    assert np.all(D.get() == 0)
    assert np.all(x.get().view(np.uint8) == 0xA5) and np.all(q.get().view(np.uint8) == 0xA5)  # (nothing else was written)
    assert lib().cml_quantize_i8(TYPES[t], x.ptr, 0, n, 0, q.ptr, 0, None, None) == 2
    assert lib().cml_quantize_i8(TYPES[t], None, 0, n, 0, None, 0, D.ptr, None) == 0  # (nothing to read, nothing else to write)
    check(lib().cml_stream_sync(None))


@pytest.mark.parametrize("t,cols", [("f32", 1 << 22), ("bf16", (1 << 22) + 3), ("f32", 1 << 24)])
@pytest.mark.parametrize("value", [0.7, 1.1, 2.7])
def test_very_long_rows_of_values_alike(t, cols, value):
    """Roundings of a running sum all go one way here."""
    rng = np.random.default_rng(1)
    x = (value * (1 + 1e-6 * rng.standard_normal((1, cols)))).astype(np.float32)
    w = np.ones(cols, np.float32)
    bits = to_bits(x, t)
    check_norm(t, bits, None, w, 1e-5, norm(t, bits, None, w, 1e-5))


def strided_product(q, w, s, ws, bias, q_stride, w_stride):
    B.init(0)
    n, rows, cols = q.shape[0], w.shape[0], q.shape[1]
    Q, W, O, S, WS, BI = Rows(q), Rows(w), Rows.empty(n, rows, np.uint32), f32(s), f32(ws), f32(bias)
    G.say(f"matmul_i8 tokens={n} rows={rows} cols={cols} strides {q_stride} {w_stride}")
    check(lib().cml_matmul_i8(Q.ptr, q_stride, S.ptr, n, W.ptr, w_stride, WS.ptr, rows, cols, BI.ptr, 0, O.ptr, rows, None))
    check(lib().cml_stream_sync(None))
    return O.get()


@pytest.mark.parametrize("stride", [0, 1, 1025, -16, -1, (1 << 26) + 1, 1 << 40])
def test_the_stride_of_a_single_row_says_nothing(stride):
    q, w, s, ws, bias = operands(1, 1, 200, 1024)
    with G.engaged("^i8.matmul.slim$", none=["any", "staged"]):
        assert np.array_equal(strided_product(q, w, s, ws, bias, stride, 1024), want_product("f32", q, w, s, ws, bias))
    q, w, s, ws, bias = operands(2, 40, 1, 1024)
    with G.engaged("^i8.matmul.slim$", none=["any", "staged"]):
        assert np.array_equal(strided_product(q, w, s, ws, bias, 1024, stride), want_product("f32", q, w, s, ws, bias))
    q, w, s, ws, bias = operands(3, 1, 1, 1024)
    with G.engaged("^i8.matmul.slim$", none=["any", "staged"]):
        assert np.array_equal(strided_product(q, w, s, ws, bias, stride, stride), want_product("f32", q, w, s, ws, bias))


@pytest.mark.parametrize("t,n,rows,out_pad", [("bf16", 3100, 16512, 0), ("bf16", 3100, 16513, 0), ("f32", 1700, 16384, 32), ("f32", 1700, 16384, 1)])
def test_large_outputs_cell_by_cell(t, n, rows, out_pad):
    q, w, s, ws, bias = operands(n, n, rows, 144)
    with G.engaged("^i8.matmul.walk$"):
        got = product(t, q, w, s, ws, bias, out_pad=out_pad)
    for r in range(0, rows, 2048):
        at = slice(r, r + 2048)
        assert np.array_equal(got[:, at], want_product(t, q, w[at], s, ws[at], bias[at])), r


def launched(call, name):
    before = G.launch_counts().get(name, 0)
    out = call()
    return out, G.launch_counts().get(name, 0) - before


def test_more_rows_than_one_launch_has_workgroups():
    """A launch has fewer than 2^32 work items: 2^24 workgroups of 256 are one too many."""
    B.init(0)
    n, cols = (1 << 24) + 5, 3
    rng = np.random.default_rng(0)
    q, d = rng.integers(-127, 128, (n, cols)).astype(np.int8), rng.random(n).astype(np.float32)
    Q, D, O = Rows(q), Rows(d.reshape(1, -1)), Rows.empty(n, cols, np.uint32)
    G.say(f"dequantize_i8 {n}x{cols}")
    check(lib().cml_dequantize_i8(Q.ptr, cols, D.ptr, n, cols, 0, O.ptr, cols, None))
    check(lib().cml_stream_sync(None))
    assert np.array_equal(O.get(), to_bits(q.astype(np.float32) * d[:, None], "f32"))


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("n,cols", [(300, 40), (37, 700), (29, 3000), (21, 6000), (11, 17000), (9, 20001), (7, 33000)])
def test_rows_in_several_launches(t, n, cols):
    """With a limit of four workgroups of 1024: the same bits, in as many launches as that makes."""
    rng = np.random.default_rng(n)
    x, r = to_bits(rng.standard_normal((n, cols)), t), to_bits(rng.standard_normal((n, cols)), t)
    w = (0.5 + rng.random(cols)).astype(np.float32)
    want = norm(t, x, r, w, 1e-5, pad=1)
    with G.env(CAMELID_HIP_LAUNCH_ITEMS=4096):
        got, launches = launched(lambda: norm(t, x, r, w, 1e-5, pad=1), "i8.add_rms_norm")
    for a, b in zip(got, want):
        assert np.array_equal(a, b)
    assert launches > 1
    q, d = want[2], want[3]
    Q, D, O, P = Rows(q, cols + 1), Rows(d.reshape(1, -1)), Rows.empty(n, cols, BITS[t], cols + 2), Rows.empty(n, cols, np.int8)
    with G.env(CAMELID_HIP_LAUNCH_ITEMS=4096):
        _, launches = launched(lambda: check(lib().cml_dequantize_i8(Q.ptr, cols + 1, D.ptr, n, cols, TYPES[t], O.ptr, cols + 2, None)), "i8.dequantize")
        check(lib().cml_quantize_i8(TYPES[t], O.ptr, cols + 2, n, cols, P.ptr, cols, D.ptr, None))
    check(lib().cml_stream_sync(None))
    assert np.array_equal(O.get(), to_bits(q.astype(np.float32) * d[:, None], t)) and launches > 1
    assert np.all(np.abs(P.get().astype(int)).max(axis=1) == 127)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("n,rows,cols,pad", [(1100, 200, 256, 0), (1100, 200, 256, 1), (300, 3000, 130, 0), (300, 3000, 130, 14), (2100, 33, 1040, 0)])
def test_tokens_in_several_launches(t, n, rows, cols, pad):
    q, w, s, ws, bias = operands(n, n, rows, cols)
    for tile in (0, 2, 4, 6, 11, 15, 16, 19):  # (a variant that does not serve the call is not taken)
        with G.env(CAMELID_HIP_I8_TILE=tile, CAMELID_HIP_LAUNCH_ITEMS=1 << 13):
            got, launches = launched(lambda: product(t, q, w, s, ws, bias, q_pad=pad, w_pad=pad, out_pad=3), "i8.matmul.staged")
        assert np.array_equal(got, want_product(t, q, w, s, ws, bias)), tile
        if tile == 16:
            assert launches > 1
