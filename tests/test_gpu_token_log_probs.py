"""cml_token_log_probs against the formulas in 64 bits: sizes, strides, ties, masks, empty rows, streams, refusals.

Tolerances.  An exponential's argument d is rounded twice (|d| 2^-23) and its result by one unit, so a term e^d is off by at most (|d| + 2) 2^-23 of itself and
|d| e^d stays below 0.37: the sum is off by less than 2 e-6 of itself with its additions (16 to 2048 per lane of 2^-24 each, mostly cancelling: 1e-5 at
the very most).  A log probability then is off by 1e-5 + 2^-23 |it|, the entropy by 1e-5 (1 + it).  Ids and ranks are exact.
"""
import numpy as np
import pytest

from camelid_amd import binding as B
from camelid_amd.binding import DeviceBuffer, check, lib
from tests import gpu_util as G
from tests.typed_rows import TYPES, Rows, from_bits, to_bits

pytestmark = pytest.mark.gpu
LOWEST = np.float32(-3.4028235e38)


def score(t, logits, target, top, pad=0, offset=0, stream=None):
    B.init(0)
    n, vocab = logits.shape
    X, T = Rows(logits, vocab + pad, offset), Rows(np.ascontiguousarray(target, np.int32).reshape(1, -1))
    P, R, H = Rows.empty(1, n, np.float32), Rows.empty(1, n, np.int32), Rows.empty(1, n, np.float32)
    I, A = (Rows.empty(n, top, np.int32), Rows.empty(n, top, np.float32)) if top else (None, None)
    need = lib().cml_token_log_probs_workspace_bytes(n, vocab, top)
    ws = DeviceBuffer(need + 16)
    ws.fill(0xFF)
    G.say(f"token_log_probs {t} {n}x{vocab} top={top} pad={pad} offset={offset} workspace={need}")
    check(lib().cml_token_log_probs(TYPES[t], X.ptr, X.stride, n, vocab, T.ptr, top, P.ptr, R.ptr, H.ptr, I.ptr if I else None, A.ptr if A else None, ws.ptr, need, stream))
    check(lib().cml_stream_sync(stream))
    assert np.all(ws.to_numpy(np.uint8, need + 16)[need:] == 0xFF)
    return P.get()[0], R.get()[0], H.get()[0], I.get() if I else np.empty((n, 0), np.int32), A.get() if A else np.empty((n, 0), np.float32)


def compare(t, logits, target, top, **kw):
    got = score(t, logits, target, top, **kw)
    values = from_bits(logits, t).astype(np.float64)
    for r, v in enumerate(values):
        p, rank, h, ids, lps = (g[r] for g in got)
        live = v > -np.inf
        if live.any():
            m = v[live].max()
            e = np.exp(np.where(live, v - m, -np.inf))
            lp = np.where(live, v - m, -np.inf) - np.log(e.sum())
            entropy = -np.sum(np.where(e > 0, e / e.sum() * np.where(e > 0, lp, 0), 0))
        else:
            lp, entropy = np.full(len(v), -np.inf), 0.0
        order = [i for i in np.lexsort((np.arange(len(v)), -v))[:top] if live[i]]
        assert ids.tolist() == order + [-1] * (top - len(order)), r
        want = np.concatenate([lp[order], np.full(top - len(order), -np.inf)])
        for a, b in [(p, lp[target[r]])] + list(zip(lps, want)):
            with np.errstate(over="ignore"):
                b = np.float64(np.float32(b))  # (the difference of both ends of a type is past f32)
            assert a == b if np.isinf(b) else abs(a - b) <= 1e-5 + 2.0 ** -23 * abs(b), (r, a, b)
        assert abs(h - entropy) <= 1e-5 * (1 + entropy), (r, h, entropy)
        ahead = np.sum(v > v[target[r]]) + np.sum(v[:target[r]] == v[target[r]])
        assert rank == ahead + 1, r


# one token; inside, at and past a batch; rows that start off a 16-byte boundary; one row over many parts, many rows of one part
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,vocab,top,pad,offset", [(1, 1, 1, 0, 0), (3, 2, 5, 0, 0), (2, 63, 64, 1, 0), (5, 1000, 20, 0, 3), (2, 1024, 1, 0, 0), (4, 1025, 20, 0, 0), (1, 2047, 0, 0, 1), (3, 5001, 33, 4, 0),
                                                    (61, 32003, 5, 1, 0), (1, 128256, 20, 0, 0), (1, 151937, 64, 0, 5), (5000, 300, 3, 1, 0), (4200, 2100, 8, 0, 0), (1100, 5001, 4, 1, 0), (700, 9001, 6, 0, 0)])
def test_sizes(t, n, vocab, top, pad, offset):
    rng = np.random.default_rng(vocab + n)
    v = (2 * rng.standard_normal((n, vocab))).astype(np.float32)
    v[np.arange(n), rng.integers(vocab, size=n)] += 10
    compare(t, to_bits(v, t), rng.integers(vocab, size=n), top, pad=pad, offset=offset)


# parts as long as they can be, a row of one part, and a part a batch
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("waves,vocab", [(1, 60000), (1, 65536), (1, 65537), (1, 200000), (9, 131072), (4096, 30000), (15, 30000), (16, 70000), (36, 70000), (48, 9000), (45, 100000)])
def test_rows_cut_otherwise(t, waves, vocab):
    rng = np.random.default_rng(vocab)
    v = (2 * rng.standard_normal((3, vocab))).astype(np.float32)
    v[1] = np.sort(v[1])
    with G.env(CAMELID_HIP_SCORE_WAVES=waves):
        compare(t, to_bits(v, t), np.array([vocab - 1, vocab // 2, 65535 % vocab]), 20)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["alike", "ascending", "descending", "few_values", "one_high_last", "grid"])
def test_orders_and_ties(t, kind):
    vocab, top = 9000, 20
    rng = np.random.default_rng(1)
    v = {"alike": np.zeros(vocab), "ascending": np.linspace(-20, 20, vocab), "descending": np.linspace(20, -20, vocab), "few_values": rng.integers(0, 3, vocab),
         "one_high_last": np.where(np.arange(vocab) == vocab - 1, 30.0, 0.0), "grid": rng.integers(-40, 40, vocab) / 4}[kind]
    rows = to_bits(np.stack([v, v, v, np.roll(v, 1234)]), t)
    compare(t, rows, np.array([0, vocab - 1, 4321, 1024]), top)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_logits_of_any_size(t):
    """Large ones beside ordinary ones, in either order, of both signs; some of them masked later on."""
    vocab, rng = 9000, np.random.default_rng(9)
    small, up = rng.standard_normal(vocab), np.linspace(-30, 12000, vocab)
    v = np.stack([up, up[::-1], 4090 + 4 * small, -5000 + 4 * small, 60 + small, np.where(np.arange(vocab) % 4097 == 0, 20000.0, small), 1000 + small, 4096 * np.sign(small), small * 1e-6])
    v[6, 5000:8000] = -np.inf
    v[4, 8191] = -np.inf
    v[8, 100:300] = -np.inf
    compare(t, to_bits(v.astype(np.float32), t), rng.integers(vocab, size=len(v)), 20)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("top", [20, 33, 64])
def test_the_best_side_by_side(t, top):
    """All of them in the last part, in the first one, and in a few parts; alike in value."""
    vocab = 150000
    up = np.linspace(-20, 20, vocab)
    few = np.where(np.arange(vocab) % 30000 < 40, 9.0, 0.0) + np.arange(vocab) % 7 / 8
    compare(t, to_bits(np.stack([up, up[::-1], few, np.zeros(vocab)]).astype(np.float32), t), np.array([0, 149999, 70000, 5]), top)


@pytest.mark.parametrize("vocab", [1025, 1200, 1280, 2303])
@pytest.mark.parametrize("top", [24, 40, 64])
def test_lists_longer_than_a_short_last_batch(vocab, top):
    v = np.random.default_rng(vocab).standard_normal((70, vocab)).astype(np.float32)
    compare("f32", v.view(np.uint32), np.zeros(70, int), top)


def test_signed_zeros_tie():
    v = np.zeros((1, 3000), np.float32)
    v[0, ::2] = -0.0
    compare("f32", v.view(np.uint32), np.array([2999]), 10)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_masks(t):
    vocab = 5000
    rng = np.random.default_rng(2)
    v = (2 * rng.standard_normal((9, vocab))).astype(np.float32)
    low = {"f32": LOWEST, "f16": np.float32(-65504), "bf16": np.float32(-3.3895314e38)}[t]
    target = np.full(9, 4242)
    v[0] = -np.inf                         # nothing is left
    v[1] = -np.inf
    v[1, 4242] = 3.0                       # one token
    v[2, :4990] = -np.inf                  # ten, in the last batch
    v[3, 10:] = -np.inf                    # ten, in the first; the given token is masked
    v[4] = low                             # a uniform row
    v[5, 1000:] = low                      # masked by the lowest value, behind ordinary ones
    v[6, :4000] = low                      # and before them
    v[7, ::2] = -np.inf
    v[8] = low
    v[8, 17] = -low                        # both ends of the type
    compare(t, to_bits(v, t), target, 20)


def test_rows_with_nan_or_infinity_say_so_and_targets_outside():
    v = np.random.default_rng(3).standard_normal((5, 3000)).astype(np.float32)
    v[0, 2999] = np.nan
    v[1, 0] = np.nan
    v[1, 2000] = 500.0     # (what came before it no longer counts in the sum)
    v[2, 100] = np.inf
    p, rank, h, ids, lps = score("f32", v.view(np.uint32), np.array([5, 5, 5, -1, 3000]), 4)
    assert np.all(np.isnan(p)) and np.all(np.isnan(h[:3])) and np.all(np.isfinite(h[3:]))
    assert rank[3] == 0 and rank[4] == 0
    assert ids[1, 0] == 2000 and ids[2, 0] == 100 and ids[0, 0] == np.nanargmax(v[0])


def test_on_another_stream_and_replayed_from_a_graph():
    import ctypes as C
    B.init(0)
    L = lib()
    n, vocab, top = 3, 20000, 7
    rng = np.random.default_rng(6)
    st = C.c_void_p()
    check(L.cml_stream_create(C.byref(st)))
    a, b = (to_bits(3 * rng.standard_normal((n, vocab)), "bf16") for _ in range(2))
    target = np.array([1, 2, 3])
    want = [score("bf16", v, target, top, stream=st) for v in (a, b)]
    X, T = Rows(a), Rows(np.int32(target).reshape(1, -1))
    P, R, H, I, A = Rows.empty(1, n, np.float32), Rows.empty(1, n, np.int32), Rows.empty(1, n, np.float32), Rows.empty(n, top, np.int32), Rows.empty(n, top, np.float32)
    need = L.cml_token_log_probs_workspace_bytes(n, vocab, top)
    ws, graph = DeviceBuffer(max(16, need)), C.c_void_p()
    check(L.cml_graph_begin_capture(st))
    check(L.cml_token_log_probs(TYPES["bf16"], X.ptr, X.stride, n, vocab, T.ptr, top, P.ptr, R.ptr, H.ptr, I.ptr, A.ptr, ws.ptr, need, st))
    check(L.cml_graph_end_capture(st, C.byref(graph)))
    for k in range(4):
        v = (a, b)[k % 2]
        check(L.cml_memcpy_h2d(X.ptr, np.ascontiguousarray(v).ctypes.data, v.nbytes, st))
        G.say(f"token_log_probs replay {k}")
        check(L.cml_graph_launch(graph, st))
        check(L.cml_stream_sync(st))
        for got, w in zip((P.get()[0], R.get()[0], H.get()[0], I.get(), A.get()), want[k % 2]):
            assert np.array_equal(got, w)
    check(L.cml_graph_destroy(graph))
    check(L.cml_stream_destroy(st))


def test_refusals():
    B.init(0)
    L = lib()
    n, vocab, top = 2, 40000, 4
    x, tg = Rows.empty(n, vocab, np.float32), Rows(np.zeros((1, n), np.int32))
    p, r, h, i, a = Rows.empty(1, n, np.float32), Rows.empty(1, n, np.int32), Rows.empty(1, n, np.float32), Rows.empty(n, top, np.int32), Rows.empty(n, top, np.float32)
    need = L.cml_token_log_probs_workspace_bytes(n, vocab, top)
    assert need > 0
    ws = DeviceBuffer(need + 16)
    ok = dict(dtype=0, x=x.ptr, st=vocab, n=n, v=vocab, t=tg.ptr, top=top, p=p.ptr, r=r.ptr, h=h.ptr, i=i.ptr, a=a.ptr, ws=ws.ptr, nb=need)

    def status(**kw):
        c = {**ok, **kw}
        return L.cml_token_log_probs(c["dtype"], c["x"], c["st"], c["n"], c["v"], c["t"], c["top"], c["p"], c["r"], c["h"], c["i"], c["a"], c["ws"], c["nb"], None)

    assert status() == 0 and status(n=0) == 0 and status(r=None, h=None) == 0 and status(top=0, i=None, a=None) == 0
    for kw in (dict(dtype=1 << 8), dict(x=None), dict(t=None), dict(p=None), dict(i=None), dict(a=None), dict(ws=None), dict(x=x.ptr + 2), dict(ws=ws.ptr + 4), dict(h=h.ptr + 1)):
        assert status(**kw) == 2, kw
        assert L.cml_last_error()
    for kw in (dict(n=-1), dict(v=0), dict(v=(1 << 30) + 1, st=(1 << 30) + 1), dict(top=-1), dict(top=65), dict(st=vocab - 1), dict(nb=need - 1)):
        assert status(**kw) == 3, kw
    assert L.cml_token_log_probs_workspace_bytes(-1, 5, 1) == 0
    check(L.cml_stream_sync(None))
