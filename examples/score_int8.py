"""Scores given tokens with the tail of a small routed model on the int8 lane: everything between the last attention block and the
log probabilities, on the device, through the library's C ABI.

    python examples/score_int8.py [--tokens 12] [--graph]

  1. cml_add_rms_norm_i8    attention's output joins the residual stream; the norm leaves 8-bit quants for the router, f32 rows for the experts
  2. cml_matmul_i8          router logits
  3. cml_moe_route_scored   sigmoid scores, balance bias, experts in groups
  4. cml_moe_ffn            the routed experts (Q8_0 weights)
  5. cml_add_rms_norm_i8    the experts' output joins the stream; 8-bit quants for the vocabulary
  6. cml_matmul_i8          logits over the vocabulary
  7. cml_token_log_probs    the given tokens' log probabilities and ranks, entropy, alternatives

Weights are random; cml_quantize_i8 takes the int8 ones to 8 bits on the device.  Nothing is allocated between the calls, so --graph captures them.
"""
from __future__ import annotations

import argparse
import ctypes as C
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from camelid_amd import binding as B  # noqa: E402
from camelid_amd.binding import DeviceBuffer, Weight, check, lib  # noqa: E402

HIDDEN, FF, EXPERTS, GROUPS, KEPT, K, VOCAB, TOP, EPS = 512, 256, 32, 4, 2, 4, 3001, 5, 1e-6


class Int8Weight:
    """f32 rows quantized on the device: int8 values and one scale per row."""

    def __init__(self, values: np.ndarray):
        self.rows, self.cols = values.shape
        source = DeviceBuffer.from_numpy(np.ascontiguousarray(values, np.float32))
        self.values, self.scales = DeviceBuffer(values.size), DeviceBuffer(self.rows * 4)
        check(lib().cml_quantize_i8(B.CML_F32, source.ptr, self.cols, self.rows, self.cols, self.values.ptr, self.cols, self.scales.ptr, None), "cml_quantize_i8")
        check(lib().cml_stream_sync(None), "cml_stream_sync")


class Scorer:
    def __init__(self, n_tokens: int, seed: int = 0):
        B.init()
        rng = np.random.default_rng(seed)
        normal = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        self.n = n_tokens
        self.host = {"norm1": 0.5 + rng.random(HIDDEN, dtype=np.float32), "norm2": 0.5 + rng.random(HIDDEN, dtype=np.float32), "bias": 0.05 * normal(EXPERTS),
                     "router": normal(EXPERTS, HIDDEN) * 0.05, "head": normal(VOCAB, HIDDEN) * 0.1,
                     "gate": normal(EXPERTS * FF, HIDDEN) * 0.05, "up": normal(EXPERTS * FF, HIDDEN) * 0.05, "down": normal(EXPERTS * HIDDEN, FF) * 0.05}
        self.norm1, self.norm2, self.bias = (DeviceBuffer.from_numpy(self.host[k]) for k in ("norm1", "norm2", "bias"))
        self.router, self.head = Int8Weight(self.host["router"]), Int8Weight(self.host["head"])
        self.gate, self.up, self.down = (Weight.upload(B.CML_Q8_0, *self.host[k].shape, B.quantize_weights(B.CML_Q8_0, self.host[k])) for k in ("gate", "up", "down"))
        f32 = lambda *s: DeviceBuffer(int(np.prod(s)) * 4)  # noqa: E731
        n = n_tokens
        self.attention, self.stream, self.target = f32(n, HIDDEN), f32(n, HIDDEN), f32(n)
        self.normed, self.q, self.scales = f32(n, HIDDEN), DeviceBuffer(n * HIDDEN), f32(n)
        self.router_logits, self.idx, self.weight, self.experts = f32(n, EXPERTS), f32(n, K), f32(n, K), f32(n, HIDDEN)
        self.logits = f32(n, VOCAB)
        self.log_prob, self.rank, self.entropy, self.top_ids, self.top_log_probs = f32(n), f32(n), f32(n), f32(n, TOP), f32(n, TOP)
        self.moe_bytes = lib().cml_moe_workspace_bytes(B.CML_Q8_0, HIDDEN, FF, n, K, EXPERTS)
        self.score_bytes = lib().cml_token_log_probs_workspace_bytes(n, VOCAB, TOP)
        self.workspace = DeviceBuffer(max(16, self.moe_bytes, self.score_bytes))

    def load(self, attention: np.ndarray, stream: np.ndarray, target: np.ndarray) -> None:
        for buf, a in ((self.attention, np.float32(attention)), (self.stream, np.float32(stream)), (self.target, np.int32(target))):
            a = np.ascontiguousarray(a)
            check(lib().cml_memcpy_h2d(buf.ptr, a.ctypes.data, a.nbytes, None), "cml_memcpy_h2d")

    def enqueue(self, stream=None) -> None:
        """The seven calls.  The residual stream is updated in place by 1 and 5."""
        L, n, f32 = lib(), self.n, B.CML_F32
        check(L.cml_add_rms_norm_i8(f32, self.attention.ptr, HIDDEN, self.stream.ptr, HIDDEN, self.norm1.ptr, EPS, n, HIDDEN, self.stream.ptr, HIDDEN, self.normed.ptr,
                                    self.q.ptr, HIDDEN, self.scales.ptr, stream), "cml_add_rms_norm_i8")
        check(L.cml_matmul_i8(self.q.ptr, HIDDEN, self.scales.ptr, n, self.router.values.ptr, HIDDEN, self.router.scales.ptr, EXPERTS, HIDDEN, None, f32,
                              self.router_logits.ptr, EXPERTS, stream), "cml_matmul_i8")
        check(L.cml_moe_route_scored(B.CML_ROUTE_SIGMOID, f32, self.router_logits.ptr, EXPERTS, self.bias.ptr, n, EXPERTS, GROUPS, KEPT, 2, K, 1, 1.0, self.idx.ptr,
                                     self.weight.ptr, stream), "cml_moe_route_scored")
        check(L.cml_moe_ffn(self.gate.handle, self.up.handle, self.down.handle, EXPERTS, K, self.idx.ptr, self.weight.ptr, self.normed.ptr, n, self.experts.ptr,
                            self.workspace.ptr, self.moe_bytes, stream), "cml_moe_ffn")
        check(L.cml_add_rms_norm_i8(f32, self.experts.ptr, HIDDEN, self.stream.ptr, HIDDEN, self.norm2.ptr, EPS, n, HIDDEN, self.stream.ptr, HIDDEN, None, self.q.ptr,
                                    HIDDEN, self.scales.ptr, stream), "cml_add_rms_norm_i8")
        check(L.cml_matmul_i8(self.q.ptr, HIDDEN, self.scales.ptr, n, self.head.values.ptr, HIDDEN, self.head.scales.ptr, VOCAB, HIDDEN, None, f32, self.logits.ptr,
                              VOCAB, stream), "cml_matmul_i8")
        check(L.cml_token_log_probs(f32, self.logits.ptr, VOCAB, n, VOCAB, self.target.ptr, TOP, self.log_prob.ptr, self.rank.ptr, self.entropy.ptr, self.top_ids.ptr,
                                    self.top_log_probs.ptr, self.workspace.ptr, self.score_bytes, stream), "cml_token_log_probs")

    def results(self, stream=None) -> dict:
        check(lib().cml_stream_sync(stream), "cml_stream_sync")
        n = self.n
        return {"log_prob": self.log_prob.to_numpy(np.float32, n), "rank": self.rank.to_numpy(np.int32, n), "entropy": self.entropy.to_numpy(np.float32, n),
                "top_ids": self.top_ids.to_numpy(np.int32, (n, TOP)), "top_log_probs": self.top_log_probs.to_numpy(np.float32, (n, TOP)),
                "stream": self.stream.to_numpy(np.float32, (n, HIDDEN)), "experts": self.idx.to_numpy(np.int32, (n, K))}


def inputs(n: int, seed: int):
    rng = np.random.default_rng(seed)
    return rng.standard_normal((n, HIDDEN)), 2 * rng.standard_normal((n, HIDDEN)), rng.integers(0, VOCAB, n)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--tokens", type=int, default=12)
    ap.add_argument("--graph", action="store_true", help="capture the calls and replay them")
    a = ap.parse_args()
    s = Scorer(a.tokens)
    stream = C.c_void_p()
    check(lib().cml_stream_create(C.byref(stream)), "cml_stream_create")
    s.load(*inputs(a.tokens, 1))
    if a.graph:
        graph = C.c_void_p()
        check(lib().cml_graph_begin_capture(stream), "cml_graph_begin_capture")
        s.enqueue(stream)
        check(lib().cml_graph_end_capture(stream, C.byref(graph)), "cml_graph_end_capture")
        check(lib().cml_graph_launch(graph, stream), "cml_graph_launch")
    else:
        s.enqueue(stream)
    r = s.results(stream)
    for t in range(a.tokens):
        best = "  ".join("%d %.2f" % p for p in zip(r["top_ids"][t], r["top_log_probs"][t]))
        print("token %d: log probability %.3f, rank %d, entropy %.3f; experts %s; best: %s" % (t, r["log_prob"][t], r["rank"][t], r["entropy"][t], r["experts"][t].tolist(), best))
    print("sum of log probabilities: %.3f" % r["log_prob"].sum())
    if a.graph:
        check(lib().cml_graph_destroy(graph), "cml_graph_destroy")
    check(lib().cml_stream_destroy(stream), "cml_stream_destroy")


if __name__ == "__main__":
    main()
