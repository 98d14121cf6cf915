"""The example that scores tokens on the int8 lane: against the same model in 64 bits (with the quantized weights it uses), on a stream, and replayed from a graph.

What separates the two is the 8-bit rounding of two activations, which is part of the model: the comparison follows it with the quants' scale as its measure.  A quant is off by half a step,
1 / 254 of the row's largest value; a logit is a sum of 512 such errors times weights of 0.1, with the largest value near 4: 0.1 * sqrt(512 / 12) * 4 / 127 = 0.02 in the mean, and a
few times that at most: 0.15.
"""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest

import oracle
from camelid_amd import binding as B
from camelid_amd.binding import check, lib
from examples import score_int8 as E
from tests import gpu_util as G

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def q8_0(w):
    rows, cols = w.shape
    return oracle.dequant(B.CML_Q8_0, B.quantize_weights(B.CML_Q8_0, w)).reshape(rows, cols).astype(np.float64)


def rows_i8(w):
    s = np.abs(w).max(axis=1, keepdims=True).astype(np.float64) / 127
    return np.rint(w / s) * s


def reference(s, attention, stream, experts):
    """The model in 64 bits on the experts that were chosen: (router scores, stream, logits)."""
    h = s.host
    norm = lambda v, w: v / np.sqrt(np.mean(v * v, axis=1, keepdims=True) + E.EPS) * w  # noqa: E731
    stream = np.float32(np.float32(attention) + np.float32(stream)).astype(np.float64)
    y = norm(stream, h["norm1"])
    score = 1 / (1 + np.exp(-(y @ rows_i8(h["router"]).T)))
    gate, up, down = (q8_0(h[k]).reshape(E.EXPERTS, -1, h[k].shape[1]) for k in ("gate", "up", "down"))
    out = np.zeros_like(y)
    for t in range(len(y)):
        w = score[t, experts[t]]
        for e, we in zip(experts[t], w / w.sum()):
            g, u = gate[e] @ y[t], up[e] @ y[t]
            out[t] += we * (down[e] @ (g / (1 + np.exp(-g)) * u))
    stream = stream + out
    return score, stream, norm(stream, h["norm2"]) @ rows_i8(h["head"]).T


@pytest.mark.parametrize("n", [1, 12, 70])
def test_scores_of_the_example(n):
    s = E.Scorer(n)
    attention, stream, target = E.inputs(n, 7)
    s.load(attention, stream, target)
    G.say(f"example: {n} tokens")
    s.enqueue()
    r = s.results()
    score, want_stream, logits = reference(s, attention, stream, r["experts"])
    # routing: the chosen experts' keys are not below those left out of the groups kept by more than what the router's activation rounding moves them
    key = score + s.host["bias"]
    size = E.EXPERTS // E.GROUPS
    for t in range(n):
        groups = set(r["experts"][t] // size)
        assert len(groups) <= E.KEPT and len(set(r["experts"][t])) == E.K
        rest = [e for e in range(E.EXPERTS) if e // size in groups and e not in r["experts"][t]]
        assert key[t, r["experts"][t]].min() >= key[t, rest].max() - 0.02
    assert np.abs(r["stream"] - want_stream).max() <= 0.05
    lp = logits - logits.max(axis=1, keepdims=True)
    lp = lp - np.log(np.exp(lp).sum(axis=1, keepdims=True))
    assert np.abs(r["log_prob"] - lp[np.arange(n), target]).max() <= 0.15
    assert np.abs(r["top_log_probs"] - np.take_along_axis(lp, r["top_ids"].astype(np.int64), 1)).max() <= 0.15
    assert np.all(np.diff(r["top_log_probs"], axis=1) <= 0)


def test_replays_give_the_eager_bits():
    L, n = lib(), 9
    s = E.Scorer(n)
    st, graph = C.c_void_p(), C.c_void_p()
    check(L.cml_stream_create(C.byref(st)))
    sets, want = [E.inputs(n, k) for k in range(3)], []
    for a in sets:
        s.load(*a)
        s.enqueue(st)
        want.append(s.results(st))
    check(L.cml_graph_begin_capture(st))
    s.enqueue(st)
    check(L.cml_graph_end_capture(st, C.byref(graph)))
    for k in (1, 0, 2, 2, 1):
        s.load(*sets[k])
        G.say(f"example: replay with inputs {k}")
        check(L.cml_graph_launch(graph, st))
        got = s.results(st)
        for name, v in want[k].items():
            assert np.array_equal(got[name], v), name
    check(L.cml_graph_destroy(graph))
    check(L.cml_stream_destroy(st))


def test_the_command():
    for args in ([], ["--tokens", "3", "--graph"]):
        r = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "score_int8.py"), *args], capture_output=True, text=True, timeout=100)
        assert r.returncode == 0, r.stderr
        assert "sum of log probabilities" in r.stdout and r.stdout.count("token ") == (3 if args else 12)
