"""The int8 lane through the C ABI against plain numpy: residual + RMS norm + quantizer, the quantizer alone, its inverse, and the product.

Tolerances.  A row's sum of squares is a chain of at most 64 fused multiply-adds and 26 additions: 90 roundings of 2^-24, half of
that (2.7e-6) on the inverse root, and five more roundings behind it: 4e-6 on scale and normalised values.  A quant is the rounding of a quotient
that four roundings have moved by at most 127 * 4 * 2^-24 = 3.1e-5.  The residual stream, the dequantized values and the product are
defined operation by operation: their bits are compared.
"""
import numpy as np
import pytest

from camelid_amd import binding as B
from camelid_amd.binding import check, lib
from tests import gpu_util as G
from tests.typed_rows import BITS, TYPES, Rows, from_bits, to_bits

pytestmark = pytest.mark.gpu
REL = 4e-6


def f32(a):
    return Rows(np.ascontiguousarray(a, np.float32).reshape(1, -1))


def norm(t, x, residual, weight, eps, *, pad=0, offset=0, in_place=False, want_sum=True, want_normed=True, stream=None):
    """(sum bits, normed, q, scales) of one call on bit patterns x, residual."""
    B.init(0)
    n, cols = x.shape
    X = Rows(x, cols + pad, offset)
    R = Rows(residual, cols + pad, offset) if residual is not None else None
    S = (R if R else X) if in_place else Rows.empty(n, cols, BITS[t], cols + pad, offset) if want_sum else None
    N = Rows.empty(n, cols, np.float32) if want_normed else None
    Q, D, W = Rows.empty(n, cols, np.int8, cols + pad, offset), Rows.empty(1, n, np.float32), f32(weight)
    G.say(f"add_rms_norm_i8 {t} {n}x{cols} pad={pad} offset={offset} residual={R is not None}")
    check(lib().cml_add_rms_norm_i8(TYPES[t], X.ptr, X.stride, R.ptr if R else None, R.stride if R else 0, W.ptr, eps, n, cols, S.ptr if S else None, S.stride if S else 0,
                                    N.ptr if N else None, Q.ptr, Q.stride, D.ptr, stream))
    check(lib().cml_stream_sync(stream))
    return S.get() if S else None, N.get() if N else None, Q.get(), D.get()[0]


def check_norm(t, x, residual, weight, eps, got):
    sum_bits, normed, q, scales = got
    h = from_bits(x, t)
    if residual is not None:
        h = from_bits(to_bits(h + from_bits(residual, t), t), t)
    if sum_bits is not None:
        assert np.array_equal(sum_bits, to_bits(h, t))
    h = h.astype(np.float64)
    y = h / np.sqrt(np.mean(h * h, axis=1, keepdims=True) + eps) * weight.astype(np.float64)
    step = np.abs(y).max(axis=1) / 127
    if normed is not None:
        assert np.all(np.abs(normed - y) <= REL * np.abs(y))
    assert np.all(np.abs(scales - step) <= REL * step)
    live = step > 0
    assert np.all(q[~live] == 0)
    assert np.all(np.abs(q[live] - y[live] / step[live, None]) <= 0.5 + 3.1e-5)
    assert np.all(np.abs(q[live].astype(int)).max(axis=1) == 127)


# one value; odd; the last of one wave; either side of every number of values a thread holds; the longest
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,cols,pad,offset", [(1, 1, 0, 0), (5, 7, 3, 1), (9, 512, 0, 0), (3, 513, 0, 0), (4, 2048, 8, 8), (2, 2049, 1, 3), (3, 4096, 0, 0), (2, 4100, 0, 0),
                                               (2, 8193, 0, 1), (1, 16384, 0, 0), (1, 16391, 0, 0), (1, 40000, 0, 0), (1, 65536, 0, 0), (2, 32768, 0, 0), (3, 32770, 3, 0), (2100, 96, 0, 0)])
def test_norm_sizes(t, n, cols, pad, offset):
    rng = np.random.default_rng(cols + n)
    channel = np.exp(0.5 * rng.standard_normal(cols))
    x, r = to_bits(rng.standard_normal((n, cols)) * channel, t), to_bits(2 * rng.standard_normal((n, cols)) * channel, t)
    w = (0.5 + rng.random(cols)).astype(np.float32)
    check_norm(t, x, r, w, 1e-5, norm(t, x, r, w, 1e-5, pad=pad, offset=offset))


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [1000, 40001])
def test_norm_without_residual_in_place_and_without_the_optional_outputs(t, cols):
    rng = np.random.default_rng(3)
    x, r = to_bits(rng.standard_normal((6, cols)), t), to_bits(rng.standard_normal((6, cols)), t)
    w = (0.5 + rng.random(cols)).astype(np.float32)
    w[5] = -2.0
    full = norm(t, x, r, w, 1e-6)
    check_norm(t, x, None, w, 1e-6, norm(t, x, None, w, 1e-6))
    for got in (norm(t, x, r, w, 1e-6, in_place=True), norm(t, x, r, w, 1e-6, want_sum=False, want_normed=False)):
        for a, b in zip(got, full):
            assert a is None or np.array_equal(a, b)


def test_norm_rows_of_zeros_tiny_values_infinities_and_nan():
    cols = 600
    rng = np.random.default_rng(4)
    x = rng.standard_normal((7, cols)).astype(np.float32)
    x[1] = 0.0
    x[2] *= 1e-38       # (squares vanish; eps alone is left)
    x[3, 17] = np.inf
    x[4, 599] = np.nan
    x[5] = 0.0
    x[5, 0] = 1e-41     # subnormal
    w = np.ones(cols, np.float32)
    s, y, q, d = norm("f32", x.view(np.uint32), None, w, 1e-5)
    keep = [0, 1, 2, 6]
    check_norm("f32", x[keep].view(np.uint32), None, w, 1e-5, (s[keep], None, q[keep], d[keep]))
    assert np.all(q[1] == 0) and d[1] == 0
    assert not np.isfinite(d[3]) and not np.isfinite(d[4]) and np.all(q[3:5] == 0)
    assert q[5, 0] == 127 and np.all(q[5, 1:] == 0)
    w[9] = np.nan
    s, y, q, d = norm("f32", x.view(np.uint32), None, w, 1e-5)
    assert np.isnan(d[0]) and np.all(q[0] == 0)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,cols,pad", [(1, 1, 0), (6, 33, 2), (300, 512, 0), (3, 5000, 0), (2, 20001, 5)])
def test_quantizer_alone_and_back(t, n, cols, pad):
    B.init(0)
    rng = np.random.default_rng(n)
    x = to_bits(rng.standard_normal((n, cols)) * 3, t)
    X, Q, D = Rows(x, cols + pad), Rows.empty(n, cols, np.int8, cols + pad), Rows.empty(1, n, np.float32)
    O = Rows.empty(n, cols, BITS[t], cols + pad)
    G.say(f"quantize_i8 / dequantize_i8 {t} {n}x{cols}")
    check(lib().cml_quantize_i8(TYPES[t], X.ptr, X.stride, n, cols, Q.ptr, Q.stride, D.ptr, None))
    check(lib().cml_dequantize_i8(Q.ptr, Q.stride, D.ptr, n, cols, TYPES[t], O.ptr, O.stride, None))
    check(lib().cml_stream_sync(None))
    v, q, d = from_bits(x, t).astype(np.float64), Q.get(), D.get()[0]
    step = np.abs(v).max(axis=1) / 127
    assert np.all(np.abs(d - step) <= 2.0 ** -23 * step)
    assert np.all(np.abs(q - v / step[:, None]) <= 0.5 + 3.1e-5)
    assert np.array_equal(O.get(), to_bits(q.astype(np.float32) * d[:, None], t))


def product(t, q, w, s, ws, bias, *, q_pad=0, w_pad=0, out_pad=0, offset=0):
    B.init(0)
    n, rows, cols = q.shape[0], w.shape[0], q.shape[1]
    Q, W, O = Rows(q, cols + q_pad, offset), Rows(w, cols + w_pad, offset), Rows.empty(n, rows, BITS[t], rows + out_pad)
    S, WS, BI = f32(s), f32(ws), f32(bias) if bias is not None else None
    G.say(f"matmul_i8 {t} tokens={n} rows={rows} cols={cols} pads={q_pad},{w_pad},{out_pad} offset={offset}")
    check(lib().cml_matmul_i8(Q.ptr, Q.stride, S.ptr, n, W.ptr, W.stride, WS.ptr, rows, cols, BI.ptr if BI else None, TYPES[t], O.ptr, O.stride, None))
    check(lib().cml_stream_sync(None))
    return O.get()


def want_product(t, q, w, s, ws, bias):
    total = (q.astype(np.float64) @ w.astype(np.float64).T).astype(np.int64)  # exact: below 2^53
    out = total.astype(np.float32) * s[:, None] * ws[None, :]
    return to_bits(out if bias is None else out + bias[None, :], t)


def operands(seed, n, rows, cols):
    rng = np.random.default_rng(seed)
    q, w = rng.integers(-128, 128, (n, cols)).astype(np.int8), rng.integers(-128, 128, (rows, cols)).astype(np.int8)
    return q, w, (0.01 + rng.random(n)).astype(np.float32), (rng.random(rows) * 1e-3).astype(np.float32), rng.standard_normal(rows).astype(np.float32)


# tokens: one, odd, either side of 16 / 32 / 64 / 128 / 256; rows and columns inside, at and past whole tiles
@pytest.mark.parametrize("n,rows,cols", [(1, 1, 1), (1, 64, 16), (1, 4096, 4096), (2, 130, 48), (3, 1000, 2816), (8, 257, 528), (16, 4096, 512), (17, 96, 80), (33, 704, 2816), (37, 1003, 2048),
                                         (64, 512, 4096), (65, 63, 1040), (100, 333, 14336), (128, 256, 256), (129, 257, 272), (200, 1000, 1024), (256, 512, 128), (300, 2050, 4096), (513, 769, 384),
                                         (1024, 1024, 144), (1100, 1300, 2048)])
def test_product_sizes(n, rows, cols):
    q, w, s, ws, bias = operands(n + rows + cols, n, rows, cols)
    t = ["f32", "f16", "bf16"][(n + rows) % 3]
    assert np.array_equal(product(t, q, w, s, ws, bias), want_product(t, q, w, s, ws, bias))


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,rows,cols,q_pad,w_pad,out_pad,offset", [(5, 70, 1, 0, 0, 0, 0), (5, 70, 77, 0, 0, 1, 0), (40, 100, 129, 0, 15, 0, 0), (70, 90, 256, 16, 32, 3, 0), (70, 90, 256, 1, 0, 0, 0),
                                                                    (70, 90, 256, 0, 0, 0, 4), (3, 200, 100, 12, 12, 0, 16), (300, 300, 500, 12, 12, 5, 0), (260, 520, 1000, 8, 8, 0, 0)])
def test_product_strides_alignments_and_no_bias(t, n, rows, cols, q_pad, w_pad, out_pad, offset):
    q, w, s, ws, _ = operands(cols, n, rows, cols)
    assert np.array_equal(product(t, q, w, s, ws, None, q_pad=q_pad, w_pad=w_pad, out_pad=out_pad, offset=offset), want_product(t, q, w, s, ws, None))


# every kernel that can serve a call gives the same bits: whole and cut tiles, one step and many, rows that end inside a step and inside 16 bytes
@pytest.mark.parametrize("n,rows,cols", [(256, 256, 64), (300, 700, 128), (257, 2400, 272), (640, 5000, 400), (2500, 2300, 130), (16, 300, 1100), (2, 5000, 127), (1030, 4100, 512), (1, 17, 5000), (33, 100, 128), (70, 33, 2057)])
def test_product_by_every_kernel(n, rows, cols):
    q, w, s, ws, bias = operands(n * rows, n, rows, cols)
    pad = -cols % 16
    t = ["f32", "f16", "bf16"][rows % 3]
    want = want_product(t, q, w, s, ws, bias)
    for tile, kernel in [(1, "walk"), (2, "tile"), (3, "tile"), (4, "tile"), (5, "tile"), (6, "tile"), (7, "tile.once"), (8, "tile.once"), (9, "slim"), (10, "slim"), (11, "slim"), (12, "slim"),
                         (13, "slim"), (14, "slim"), (15, "staged"), (16, "staged"), (17, "slim.any"), (18, "slim.any"), (19, "slim.any")]:
        if tile == 1 and n < 256:
            continue
        with G.env(CAMELID_HIP_I8_TILE=tile), G.engaged(f"^i8.matmul.{kernel}$"):
            assert np.array_equal(product(t, q, w, s, ws, bias, q_pad=pad, w_pad=pad), want), tile


@pytest.mark.parametrize("n,rows,cols", [(1, 17, 5001), (33, 100, 128), (70, 33, 2057), (300, 700, 131), (16, 300, 1100), (513, 600, 1025)])
def test_product_of_rows_that_start_anywhere_by_every_kernel(n, rows, cols):
    q, w, s, ws, bias = operands(n * rows, n, rows, cols)
    want = want_product("f32", q, w, s, ws, bias)
    for tile, kernel in [(15, "staged"), (16, "staged"), (17, "slim.any"), (18, "slim.any"), (19, "slim.any")]:
        for pad, offset in ((0, 0), (3, 1), (-cols % 16, 5)):
            with G.env(CAMELID_HIP_I8_TILE=tile), G.engaged(f"^i8.matmul.{kernel}$"):
                assert np.array_equal(product("f32", q, w, s, ws, bias, q_pad=pad, w_pad=pad, offset=offset), want), (tile, pad, offset)


@pytest.mark.parametrize("stride", [(1 << 27) + 5, 1 << 27, (1 << 24) + 16, (1 << 24) + 1])
def test_rows_far_apart(stride):
    """Offsets past 32 bits."""
    n, rows, cols = 3, 40, 200
    q, w, s, ws, _ = operands(5, n, rows, cols)
    B.init(0)
    W = B.DeviceBuffer(stride * (rows - 1) + cols)
    for r in range(rows):
        check(lib().cml_memcpy_h2d(W.ptr + r * stride, np.ascontiguousarray(w[r]).ctypes.data, cols, None))
    Q, O, S, WS = Rows(q), Rows.empty(n, rows, BITS["f32"]), f32(s), f32(ws)
    G.say(f"matmul_i8 rows {stride} bytes apart")
    check(lib().cml_matmul_i8(Q.ptr, cols, S.ptr, n, W.ptr, stride, WS.ptr, rows, cols, None, TYPES["f32"], O.ptr, rows, None))
    check(lib().cml_stream_sync(None))
    assert np.array_equal(O.get(), want_product("f32", q, w, s, ws, None))


def test_kernels_by_size():
    for n, rows, cols, pad, kernel in [(1, 512, 1024, 0, "slim"), (1, 512, 1024, 1, "slim.any"), (40, 512, 1024, 0, "slim"), (400, 4096, 512, 0, "tile"), (40, 512, 1024, 1, "slim.any"), (2000, 2000, 1024, 1, "staged"), (40, 98304, 1024, 0, "tile.once"), (2048, 8192, 512, 0, "walk")]:
        q, w, s, ws, _ = operands(n, n, rows, cols)
        with G.engaged(f"^i8.matmul.{kernel}$"):
            assert np.array_equal(product("f32", q, w, s, ws, None, q_pad=pad, w_pad=pad), want_product("f32", q, w, s, ws, None))


@pytest.mark.parametrize("t,n,rows,out_pad", [("bf16", 3100, 16512, 0), ("bf16", 3100, 16513, 0), ("f32", 1700, 16384, 32), ("f32", 1700, 16384, 1)])
def test_large_outputs(t, n, rows, out_pad):
    """On either side of whole lines; columns at random against the formula, all of them against the sum over rows."""
    cols = 144
    q, w, s, ws, bias = operands(n, n, rows, cols)
    with G.engaged("^i8.matmul.walk$"):
        got = product(t, q, w, s, ws, bias, out_pad=out_pad)
    pick = np.unique(np.concatenate([np.random.default_rng(1).integers(rows, size=600), [0, 255, 256, rows - 257, rows - 1]]))
    assert np.array_equal(got[:, pick], want_product(t, q, w[pick], s, ws[pick], bias[pick]))
    total = (q.astype(np.int64) @ w.astype(np.int64).sum(axis=0)).astype(np.float64)
    exact = (from_bits(got, t).astype(np.float64) - bias.astype(np.float64)) / (s.astype(np.float64)[:, None] * ws.astype(np.float64))
    # every cell is off by its roundings alone: 2^-7 of itself at most and of the bias, in a sum of signs at random; a cell that was not written would be off by its whole value
    size = np.abs(from_bits(got, t).astype(np.float64)) + np.abs(bias)
    bound = (size * 2.0 ** -7 / (s.astype(np.float64)[:, None] * ws.astype(np.float64))).sum(axis=1)
    assert np.all(np.abs(exact.sum(axis=1) - total) <= bound)


@pytest.mark.parametrize("n", [1, 20, 300])
def test_product_extremes_stay_exact(n):
    cols, rows = 131071 // 16 * 16, 33
    q, w = np.full((n, cols), -128, np.int8), np.full((rows, cols), -128, np.int8)
    w[1::2] = 127
    q[::3, ::2] = 127
    one, rows_one = np.ones(n, np.float32), np.ones(rows, np.float32)
    assert np.array_equal(product("f32", q, w, one, rows_one, None), want_product("f32", q, w, one, rows_one, None))


def test_product_of_a_token_does_not_depend_on_the_batch():
    q, w, s, ws, bias = operands(11, 700, 600, 2048)
    full = product("f32", q, w, s, ws, bias)
    for n in (1, 2, 16, 17, 40, 64, 130, 257):
        assert np.array_equal(product("f32", q[:n], w, s[:n], ws, bias), full[:n])


def test_scales_that_are_not_finite_reach_their_cells_alone():
    q, w, s, ws, _ = operands(12, 20, 50, 64)
    s[3], ws[7] = np.nan, np.inf
    got = from_bits(product("f32", q, w, s, ws, None), "f32")
    assert np.all(np.isnan(got[3])) and not np.any(np.isfinite(got[:, 7]))
    rest = np.delete(np.delete(got, 3, 0), 7, 1)
    assert np.all(np.isfinite(rest))


@pytest.mark.parametrize("tile,n,rows,cols", [(0, 5, 300, 512), (0, 300, 700, 512), (1, 600, 1000, 272), (16, 70, 90, 272), (17, 7, 90, 272)])
def test_the_lane_on_a_stream_and_replayed_from_a_graph(tile, n, rows, cols):
    """Norm and product captured together; every replay on other inputs against the eager calls."""
    import ctypes as C
    B.init(0)
    L, rng = lib(), np.random.default_rng(n)
    st, graph = C.c_void_p(), C.c_void_p()
    check(L.cml_stream_create(C.byref(st)))
    _, w, _, ws, bias = operands(n, 1, rows, cols)
    sets = [to_bits(rng.standard_normal((n, cols)), "bf16") for _ in range(3)]
    X, Q, D, O, back = Rows(sets[0]), Rows.empty(n, cols, np.int8), Rows.empty(1, n, np.float32), Rows.empty(n, rows, np.float32), Rows.empty(n, cols, np.uint16)
    N, W, WS, BI = f32(1 + rng.random(cols)), Rows(w), f32(ws), f32(bias)

    def calls():
        check(L.cml_add_rms_norm_i8(TYPES["bf16"], X.ptr, cols, None, 0, N.ptr, 1e-6, n, cols, None, 0, None, Q.ptr, cols, D.ptr, st))
        check(L.cml_matmul_i8(Q.ptr, cols, D.ptr, n, W.ptr, cols, WS.ptr, rows, cols, BI.ptr, 0, O.ptr, rows, st))
        check(L.cml_dequantize_i8(Q.ptr, cols, D.ptr, n, cols, TYPES["bf16"], back.ptr, cols, st))

    def load(k):
        check(L.cml_memcpy_h2d(X.ptr, sets[k].ctypes.data, sets[k].nbytes, st))

    def results():
        check(L.cml_stream_sync(st))
        return [r.get() for r in (Q, D, O, back)]

    with G.env(CAMELID_HIP_I8_TILE=tile):
        want = []
        for k in range(3):
            load(k)
            G.say(f"int8 lane {n}x{rows}x{cols} eager {k}")
            calls()
            want.append(results())
        check(L.cml_graph_begin_capture(st))
        calls()
        check(L.cml_graph_end_capture(st, C.byref(graph)))
    for k in (2, 0, 1, 1, 2):
        load(k)
        G.say(f"int8 lane {n}x{rows}x{cols} replay {k}")
        check(L.cml_graph_launch(graph, st))
        for got, w in zip(results(), want[k]):
            assert np.array_equal(got, w)
    check(L.cml_graph_destroy(graph))
    check(L.cml_stream_destroy(st))


def test_refusals():
    B.init(0)
    L = lib()
    x, q, d, o = Rows.empty(4, 64, np.float32), Rows.empty(4, 64, np.int8), Rows.empty(1, 4, np.float32), Rows.empty(4, 64, np.float32)
    wt = f32(np.ones(64))
    ok_norm = dict(dtype=0, x=x.ptr, xs=64, r=None, rs=0, w=wt.ptr, eps=1e-5, n=4, cols=64, s=None, ss=0, y=None, q=q.ptr, qs=64, d=d.ptr)

    def norm_status(**kw):
        a = {**ok_norm, **kw}
        return L.cml_add_rms_norm_i8(a["dtype"], a["x"], a["xs"], a["r"], a["rs"], a["w"], a["eps"], a["n"], a["cols"], a["s"], a["ss"], a["y"], a["q"], a["qs"], a["d"], None)

    assert norm_status() == 0 and norm_status(n=0) == 0 and norm_status(cols=0) == 0 and norm_status(n=1, xs=0, qs=0) == 0
    for kw in (dict(dtype=2), dict(x=None), dict(w=None), dict(q=None), dict(d=None), dict(x=x.ptr + 2), dict(w=wt.ptr + 1), dict(y=x.ptr + 2), dict(r=x.ptr + 1, rs=64)):
        assert norm_status(**kw) == 2, kw
        assert L.cml_last_error()
    for kw in (dict(n=-1), dict(cols=-1), dict(xs=63), dict(qs=63), dict(r=x.ptr, rs=8), dict(s=o.ptr, ss=63), dict(n=(1 << 30) + 1)):
        assert norm_status(**kw) == 3, kw
    assert norm_status(cols=(1 << 24) + 1, xs=(1 << 24) + 1, qs=(1 << 24) + 1, n=1) == 6

    assert L.cml_quantize_i8(0, x.ptr, 64, 4, 64, q.ptr, 64, d.ptr, None) == 0
    assert L.cml_quantize_i8(7, x.ptr, 64, 4, 64, q.ptr, 64, d.ptr, None) == 2
    assert L.cml_quantize_i8(0, x.ptr, 63, 4, 64, q.ptr, 64, d.ptr, None) == 3
    assert L.cml_quantize_i8(0, x.ptr, 1 << 25, 1, 1 << 25, q.ptr, 1 << 25, d.ptr, None) == 6
    assert L.cml_dequantize_i8(q.ptr, 64, d.ptr, 4, 64, 0, o.ptr, 64, None) == 0
    assert L.cml_dequantize_i8(q.ptr, 64, None, 4, 64, 0, o.ptr, 64, None) == 2
    assert L.cml_dequantize_i8(q.ptr, 64, d.ptr, 4, 64, 3, o.ptr, 64, None) == 2
    assert L.cml_dequantize_i8(q.ptr, 64, d.ptr, 4, 64, 0, o.ptr, 60, None) == 3
    assert L.cml_dequantize_i8(q.ptr, 64, d.ptr, -4, 64, 0, o.ptr, 64, None) == 3

    w, ws = Rows.empty(8, 64, np.int8), f32(np.ones(8))
    ok = dict(q=q.ptr, qs=64, s=d.ptr, n=4, w=w.ptr, wst=64, ws=ws.ptr, rows=8, cols=64, b=None, dtype=0, o=o.ptr, os=64)

    def status(**kw):
        a = {**ok, **kw}
        return L.cml_matmul_i8(a["q"], a["qs"], a["s"], a["n"], a["w"], a["wst"], a["ws"], a["rows"], a["cols"], a["b"], a["dtype"], a["o"], a["os"], None)

    assert status() == 0 and status(n=0) == 0 and status(rows=0) == 0
    for kw in (dict(q=None), dict(s=None), dict(w=None), dict(ws=None), dict(o=None), dict(dtype=24), dict(o=o.ptr + 2), dict(s=d.ptr + 1), dict(b=d.ptr + 2)):
        assert status(**kw) == 2, kw
    for kw in (dict(n=-1), dict(rows=-1), dict(cols=0), dict(cols=131072, qs=131072, wst=131072), dict(qs=63), dict(wst=1), dict(os=7)):
        assert status(**kw) == 3, kw
    assert status(n=(1 << 20) + 1) == 6
    check(L.cml_stream_sync(None))
