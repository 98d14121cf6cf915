"""cml_moe_route_scored against the formula in 64 bits: scores, bias, groups, ties, masked experts, refusals.

Keys come from coarse grids, so that two of them are either equal (and the lower index has to win) or apart by far more than f32 rounds; rows where a
64-bit gap at a decision lies between 0 and 1e-5 are left out of the comparison, and counted.  A weight is an exponential, an addition and a division
(3 roundings and 2 units of expf), a sum of at most 64 terms in 8 steps and two more roundings: 2e-6.
"""
import numpy as np
import pytest

from camelid_amd import binding as B
from camelid_amd.binding import check, lib
from tests import gpu_util as G
from tests.typed_rows import TYPES, Rows, from_bits, to_bits

pytestmark = pytest.mark.gpu
SOFTMAX, SIGMOID = B.CML_ROUTE_SOFTMAX, B.CML_ROUTE_SIGMOID


def route(score, t, logits, bias, groups, kept, group_top, k, renormalise=1, scale=1.0, pad=0):
    B.init(0)
    n, experts = logits.shape
    X, I, W = Rows(logits, experts + pad), Rows.empty(n, k, np.int32), Rows.empty(n, k, np.float32)
    BI = Rows(np.ascontiguousarray(bias, np.float32).reshape(1, -1)) if bias is not None else None
    G.say(f"moe_route_scored score={score} {t} {n}x{experts} groups={groups}/{kept}/{group_top} k={k} bias={bias is not None}")
    check(lib().cml_moe_route_scored(score, TYPES[t], X.ptr, X.stride, BI.ptr if BI else None, n, experts, groups, kept, group_top, k, renormalise, scale, I.ptr, W.ptr, None))
    check(lib().cml_stream_sync(None))
    return I.get(), W.get()


def formula(score, logits, bias, groups, kept, group_top, k, renormalise=1, scale=1.0):
    """One row in 64 bits: (ids, weights, the smallest non-zero gap at a decision)."""
    v = np.minimum(logits.astype(np.float64), 3.4028234663852886e38)
    live = v > -np.inf
    s = np.zeros(len(v))
    if score == SIGMOID:
        with np.errstate(over="ignore"):
            s[live] = 1 / (1 + np.exp(-v[live]))
    elif live.any():
        s[live] = np.exp(v[live] - v[live].max())
        s /= s.sum()
    key = s + bias.astype(np.float64) if bias is not None else v
    live &= key > -np.inf
    gap = [np.inf]

    def best(values, ids, count):
        order = sorted(ids, key=lambda i: (-values[i], i))
        if len(order) > count:
            d = abs(values[order[count - 1]] - values[order[count]])
            gap.append(d if d > 0 else np.inf)
        for a, b in zip(order[:count], order[1:count]):
            d = abs(values[a] - values[b])
            gap.append(d if d > 0 else np.inf)
        return order[:count]

    ids = [e for e in range(len(v)) if live[e]]
    if groups > 1:
        size, worth = len(v) // groups, {}
        for g in range(groups):
            mine = [e for e in ids if e // size == g]
            if mine:
                top = sorted(mine, key=lambda e: (-key[e], e))[:group_top]
                worth[g] = sum((key if bias is not None or group_top == 1 else s)[e] for e in top)
        stay = best(worth, list(worth), kept)
        ids = [e for e in ids if e // size in stay]
    chosen = best(key, ids, k)
    w = np.array([s[e] for e in chosen])
    if renormalise and len(w):
        w = w / w.sum() if w.sum() > 0 else np.full(len(w), 1 / len(w))
    return np.array(chosen + [-1] * (k - len(chosen))), np.concatenate([w * scale, np.zeros(k - len(chosen))]), min(gap)


def compare(score, t, logits, bias, groups, kept, group_top, k, renormalise=1, scale=1.0, pad=0, least=0.9):
    ids, w = route(score, t, logits, bias, groups, kept, group_top, k, renormalise, scale, pad)
    values, seen = from_bits(logits, t), 0
    for r in range(len(values)):
        want, ww, gap = formula(score, values[r], bias, groups, kept, group_top, k, renormalise, scale)
        if gap < 1e-5:
            continue
        seen += 1
        assert np.array_equal(ids[r], want), (r, ids[r], want)
        assert np.all(np.abs(w[r] - ww) <= 2e-6 * np.abs(ww) + 1e-37), (r, w[r], ww)
    assert seen >= least * len(values)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,experts,k", [(1, 1, 1), (1, 8, 2), (3, 128, 8), (5, 60, 60), (130, 64, 6), (9, 65, 4), (7, 200, 64), (6, 256, 8), (3, 257, 10), (2, 512, 9), (2, 1000, 64), (1, 1024, 1)])
def test_softmax_without_groups(t, n, experts, k):
    rng = np.random.default_rng(experts)
    compare(SOFTMAX, t, to_bits(rng.integers(-64, 64, (n, experts)) / 16.0, t), None, 1, 1, 1, k, pad=experts % 3)


@pytest.mark.parametrize("score", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("experts,groups,kept,group_top,k", [(256, 8, 4, 2, 8), (160, 8, 3, 1, 6), (64, 16, 3, 2, 5), (60, 5, 2, 2, 7), (48, 48, 6, 2, 6), (64, 64, 64, 1, 64), (1024, 64, 9, 2, 20), (12, 1, 1, 2, 3), (320, 4, 4, 2, 16)])
def test_groups_and_bias(score, bias, experts, groups, kept, group_top, k):
    rng = np.random.default_rng(experts + groups)
    logits = to_bits(rng.integers(-32, 32, (24, experts)) / 8.0, "f32")
    b = (rng.integers(-8, 8, experts) / 64.0).astype(np.float32) if bias else None
    # (softmax scores with a bias come within 1e-5 of each other by themselves)
    compare(score, "f32", logits, b, groups, kept, group_top, k, scale=2.5, least=0.9 if score == SIGMOID or not bias else 0.0)


@pytest.mark.parametrize("renormalise", [0, 1])
def test_masked_experts_leave_slots_empty(renormalise):
    rng = np.random.default_rng(5)
    v = (rng.integers(-32, 32, (8, 64)) / 8.0).astype(np.float32)
    v[0] = -np.inf              # nobody
    v[1, 3:] = -np.inf          # three
    v[2, ::2] = np.nan          # half
    v[3, 16:] = -np.inf         # one group
    v[4, 7] = np.inf
    v[5] = -3.4028235e38        # the lowest value is an ordinary logit
    v[6] = -200.0               # sigmoids that vanish in f32
    v[7] = 0.0                  # all alike
    bits = v.view(np.uint32)
    for score in (SOFTMAX, SIGMOID):
        for groups, kept, top in ((1, 1, 1), (4, 2, 2), (4, 2, 1)):
            rows = np.array([0, 1, 2, 3, 4, 5, 7] + ([6] if score == SOFTMAX else []))
            compare(score, "f32", bits[rows], None, groups, kept, top, 8, renormalise, least=0.8)
    ids, w = route(SIGMOID, "f32", bits, None, 1, 1, 1, 8)
    assert np.all(ids[0] == -1) and np.all(w[0] == 0)
    assert np.array_equal(ids[6], np.arange(8)) and np.array_equal(w[6], np.full(8, 0.125, np.float32))
    bias = np.zeros(64, np.float32)
    bias[:4] = -np.inf
    bias[4] = np.nan
    ids, w = route(SIGMOID, "f32", bits[7:], bias, 1, 1, 1, 8)
    assert np.array_equal(ids[0], np.arange(5, 13))


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,experts,groups,kept,group_top,k,pad", [(1, 1, 1, 1, 1, 1, 0), (5, 7, 1, 1, 1, 7, 0), (18, 64, 1, 1, 1, 6, 3), (33, 64, 4, 2, 2, 8, 0), (16, 64, 16, 5, 2, 8, 1), (17, 65, 1, 1, 1, 8, 0), (9, 128, 8, 3, 1, 4, 0), (50, 128, 1, 1, 1, 8, 5), (31, 200, 1, 1, 1, 8, 0), (34, 256, 8, 4, 2, 8, 0), (7, 256, 16, 1, 2, 8, 1), (15, 256, 2, 1, 2, 3, 0), (21, 160, 8, 3, 2, 6, 0), (10, 60, 5, 2, 2, 7, 0), (11, 39, 3, 2, 1, 5, 2), (13, 208, 16, 4, 2, 8, 0), (12, 512, 16, 4, 2, 8, 0), (9, 500, 4, 2, 2, 16, 1), (10, 240, 8, 4, 1, 15, 0), (6, 100, 1, 1, 1, 9, 0), (8, 33, 3, 2, 2, 12, 0)])
def test_four_tokens_a_wave(t, n, experts, groups, kept, group_top, k, pad):
    """The form that long prompts take, at lengths that leave its last wave part empty."""
    rng = np.random.default_rng(experts + n)
    logits = to_bits(rng.integers(-32, 32, (n, experts)) / 8.0, t)
    bias = (rng.integers(-8, 8, experts) / 64.0).astype(np.float32)
    with G.env(CAMELID_HIP_ROUTE_QUARTER=1):
        compare(SIGMOID, t, logits, bias, groups, kept, group_top, k, scale=2.5, pad=pad)
        compare(SIGMOID, t, logits, -1 - bias, groups, kept, group_top, k, renormalise=0, pad=pad)  # (keys below 0)
        compare(SOFTMAX, t, logits, None, groups, kept, group_top, k, pad=pad)


def test_four_tokens_a_wave_with_masked_experts():
    with G.env(CAMELID_HIP_ROUTE_QUARTER=1):
        test_masked_experts_leave_slots_empty(0)
        test_masked_experts_leave_slots_empty(1)


@pytest.mark.parametrize("experts,groups,kept,group_top,k", [(1000, 8, 3, 2, 9), (992, 62, 30, 2, 64), (1023, 33, 5, 2, 8), (1023, 3, 2, 1, 8), (1020, 17, 4, 2, 12), (1024, 2, 1, 2, 8), (39, 13, 4, 1, 5), (77, 7, 3, 2, 3)])
def test_groups_of_any_size(experts, groups, kept, group_top, k):
    rng = np.random.default_rng(experts + groups)
    logits = to_bits(rng.integers(-32, 32, (9, experts)) / 8.0, "f16")
    compare(SIGMOID, "f16", logits, (rng.integers(-8, 8, experts) / 64.0).astype(np.float32), groups, kept, group_top, k, pad=1)


@pytest.mark.parametrize("experts,groups,kept,group_top,k", [(64, 1, 1, 1, 6), (100, 1, 1, 1, 8), (128, 2, 1, 2, 8), (160, 8, 3, 2, 6), (192, 16, 4, 1, 16), (256, 8, 4, 2, 8), (300, 3, 2, 2, 9), (512, 1, 1, 1, 10)])
def test_a_token_does_not_depend_on_the_batch(experts, groups, kept, group_top, k):
    rng = np.random.default_rng(experts)
    logits = to_bits(2 * rng.standard_normal((40, experts)), "f32")
    bias = (0.1 * rng.standard_normal(experts)).astype(np.float32)
    for score in (SOFTMAX, SIGMOID):
        for b in (None, bias):
            few = route(score, "f32", logits, b, groups, kept, group_top, k)
            with G.env(CAMELID_HIP_ROUTE_QUARTER=1), G.engaged("^moe.route.scored.quarter$"):
                many = route(score, "f32", logits, b, groups, kept, group_top, k)
            assert np.array_equal(few[0], many[0]) and np.array_equal(few[1].view(np.uint32), many[1].view(np.uint32))


@pytest.mark.parametrize("n", [4095, 4096, 4098])
def test_long_prompts(n):
    rng = np.random.default_rng(n)
    logits = to_bits(rng.integers(-32, 32, (n, 48)) / 8.0, "bf16")
    compare(SIGMOID, "bf16", logits, (rng.integers(-8, 8, 48) / 64.0).astype(np.float32), 4, 2, 2, 6)


def test_on_a_stream_and_replayed_from_a_graph():
    import ctypes as C
    B.init(0)
    L, rng = lib(), np.random.default_rng(3)
    st = C.c_void_p()
    check(L.cml_stream_create(C.byref(st)))
    for n in (3, 5000):
        graph = C.c_void_p()
        sets = [to_bits(rng.standard_normal((n, 64)), "bf16") for _ in range(2)]
        want = [route(SIGMOID, "bf16", v, None, 4, 2, 2, 6) for v in sets]
        X, I, W = Rows(sets[0]), Rows.empty(n, 6, np.int32), Rows.empty(n, 6, np.float32)
        check(L.cml_graph_begin_capture(st))
        check(L.cml_moe_route_scored(SIGMOID, TYPES["bf16"], X.ptr, 64, None, n, 64, 4, 2, 2, 6, 1, 1.0, I.ptr, W.ptr, st))
        check(L.cml_graph_end_capture(st, C.byref(graph)))
        for k in (1, 0, 1, 1):
            check(L.cml_memcpy_h2d(X.ptr, sets[k].ctypes.data, sets[k].nbytes, st))
            G.say(f"moe_route_scored {n} replay {k}")
            check(L.cml_graph_launch(graph, st))
            check(L.cml_stream_sync(st))
            assert np.array_equal(I.get(), want[k][0]) and np.array_equal(W.get(), want[k][1])
        check(L.cml_graph_destroy(graph))
    check(L.cml_stream_destroy(st))


def test_results_feed_the_plan():
    """Slots without an expert are dropped by the grouping."""
    v = np.full((3, 16), -np.inf, np.float32)
    v[0, :4] = [1, 2, 3, 4]
    v[2, 9] = 0.5
    X, I, W = Rows(v.view(np.uint32)), Rows.empty(3, 2, np.int32), Rows.empty(3, 2, np.float32)
    O, T, S, U = Rows.empty(1, 17, np.int32), Rows.empty(1, 6, np.int32), Rows.empty(1, 6, np.int32), Rows.empty(1, 16, np.int32)
    B.init(0)
    G.say("moe_route_scored into moe_plan")
    check(lib().cml_moe_route_scored(SIGMOID, 0, X.ptr, 16, None, 3, 16, 1, 1, 1, 2, 1, 1.0, I.ptr, W.ptr, None))
    check(lib().cml_moe_plan(I.ptr, 3, 2, 16, O.ptr, T.ptr, S.ptr, U.ptr, None))
    check(lib().cml_stream_sync(None))
    assert I.get().tolist() == [[3, 2], [-1, -1], [9, -1]]
    assert S.get()[0].tolist() == [1, 0, -1, -1, 2, -1]
    assert U.get()[0][:4].tolist() == [2, 3, 9, -1]


def test_refusals():
    B.init(0)
    L = lib()
    x, i, w = Rows.empty(2, 64, np.float32), Rows.empty(2, 8, np.int32), Rows.empty(2, 8, np.float32)
    ok = dict(score=1, dtype=0, x=x.ptr, st=64, b=None, n=2, e=64, g=8, kept=4, top=2, k=8, i=i.ptr, w=w.ptr)

    def status(**kw):
        a = {**ok, **kw}
        return L.cml_moe_route_scored(a["score"], a["dtype"], a["x"], a["st"], a["b"], a["n"], a["e"], a["g"], a["kept"], a["top"], a["k"], 1, 1.0, a["i"], a["w"], None)

    assert status() == 0 and status(n=0) == 0
    for kw in (dict(score=2), dict(dtype=5), dict(x=None), dict(i=None), dict(w=None), dict(x=x.ptr + 1), dict(b=x.ptr + 2)):
        assert status(**kw) == 2, kw
    for kw in (dict(n=-1), dict(e=0), dict(e=1025, st=1025), dict(g=0), dict(g=7), dict(g=65, e=65, st=65), dict(kept=0), dict(kept=9), dict(top=0), dict(top=3), dict(k=0), dict(k=65), dict(k=33, kept=4), dict(st=63)):
        assert status(**kw) == 3, kw
        assert L.cml_last_error()
    check(L.cml_stream_sync(None))
