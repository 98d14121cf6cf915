"""The operators of an int8 inference lane and of scoring, as cases that can be timed:

  norm     residual's addition and RMS norm of every token, with an int8 output and one scale per token
  matmul   int8 product with a scale for each token and each weight row
  route    choice of experts: softmax or sigmoid scores, balance bias, groups, top-k, renormalised weights
  score    log probability of a given token per row of logits, its rank, the row's entropy and best alternatives

A case is a dict of plain values; `op` names the operator.  With `own` set, run() calls this library; otherwise
it computes the same in elementary torch operations, in 32 bits.  exact() is the definition in 64 bits.
"""
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
IDS = {"f32": 0, "f16": 1, "bf16": 30}  # the GGUF type ids, as the library names types
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
SCORES = {"softmax": 0, "sigmoid": 1}
EPS = 1e-5


def listed():
    return [
        # one token of a decode loop, the norm in front of a projection: latency
        {"name": "norm_t1_4096_bf16", "op": "norm", "tokens": 1, "cols": 4096, "dtype": "bf16", "normed": False, "pad": 0},
        # a ragged batch in front of a routed layer: the router and the experts read the f32 row as well
        {"name": "norm_t333_2816_f32_normed", "op": "norm", "tokens": 333, "cols": 2816, "dtype": "f32", "normed": True, "pad": 0},
        # a long prompt's hidden states
        {"name": "norm_t8192_4096_bf16", "op": "norm", "tokens": 8192, "cols": 4096, "dtype": "bf16", "normed": False, "pad": 0},
        # one token of a decode loop through an attention projection: the weight's bytes
        {"name": "matmul_t1_4096x4096_bf16", "op": "matmul", "tokens": 1, "rows": 4096, "cols": 4096, "dtype": "bf16", "bias": False, "pad": 0},
        # a ragged batch through a vocabulary projection, logits in f32 for scoring
        {"name": "matmul_t37_128256x2048_f32", "op": "matmul", "tokens": 37, "rows": 128256, "cols": 2048, "dtype": "f32", "bias": True, "pad": 0},
        # a prompt chunk through a gate / up projection: arithmetic
        {"name": "matmul_t4096_14336x4096_bf16", "op": "matmul", "tokens": 4096, "rows": 14336, "cols": 4096, "dtype": "bf16", "bias": False, "pad": 0},
        # one token over many small experts
        {"name": "route_t1_128_softmax", "op": "route", "tokens": 1, "experts": 128, "k": 8, "score": "softmax", "bias": False, "groups": 1, "kept": 1, "group_top": 1, "dtype": "f32"},
        # a ragged batch, experts in groups (one group per device), balance bias
        {"name": "route_t517_256_sigmoid_groups", "op": "route", "tokens": 517, "experts": 256, "k": 8, "score": "sigmoid", "bias": True, "groups": 8, "kept": 4, "group_top": 2, "dtype": "f32"},
        # a long prompt's tokens
        {"name": "route_t8192_256_sigmoid_bf16", "op": "route", "tokens": 8192, "experts": 256, "k": 8, "score": "sigmoid", "bias": True, "groups": 8, "kept": 4, "group_top": 2, "dtype": "bf16"},
        # the token that a decode step picked, with the twenty best: one row over the whole chip
        {"name": "score_t1_128256_f32_top20", "op": "score", "tokens": 1, "vocab": 128256, "top": 20, "dtype": "f32", "allowed": 0, "pad": 0},
        # a batch of decode steps over a vocabulary of odd size in padded rows
        {"name": "score_t61_32003_f32_top5", "op": "score", "tokens": 61, "vocab": 32003, "top": 5, "dtype": "f32", "allowed": 0, "pad": 1},
        # scoring a prompt: the given tokens of 2048 positions
        {"name": "score_t2048_128256_bf16_top20", "op": "score", "tokens": 2048, "vocab": 128256, "top": 20, "dtype": "bf16", "allowed": 0, "pad": 0},
    ]


def _spread(rng, low, high):
    return min(high, max(low, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    op = rng.choice(["norm", "matmul", "route", "score"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "norm":
        cols = _spread(rng, 64, 16384)
        if rng.random() < 0.75:
            cols = (cols + 31) // 32 * 32
        tokens = _spread(rng, 1, min(8192, 8192 * 4096 // (2 * cols)))
        return {"op": op, "tokens": tokens, "cols": cols, "dtype": dtype, "normed": rng.random() < 0.3, "pad": rng.choice([0, 0, 8, 3])}
    if op == "matmul":
        cols = _spread(rng, 64, 16384)
        if rng.random() < 0.8:
            cols = (cols + 31) // 32 * 32
        rows = _spread(rng, 64, 65536)
        tokens = _spread(rng, 1, max(1, min(4096, 4096 * 14336 * 4096 // (rows * cols))))
        return {"op": op, "tokens": tokens, "rows": rows, "cols": cols, "dtype": dtype, "bias": rng.random() < 0.5, "pad": rng.choice([0, 0, 16])}
    if op == "route":
        tokens = _spread(rng, 1, 8192)
        if rng.random() < 0.5:
            experts = _spread(rng, 4, 512)
            return {"op": op, "tokens": tokens, "experts": experts, "k": rng.randint(1, min(16, experts)), "score": "softmax", "bias": False, "groups": 1, "kept": 1, "group_top": 1, "dtype": dtype}
        groups, size = rng.choice([1, 4, 8, 16]), rng.choice([4, 12, 16, 20, 32])
        kept = rng.randint(1, groups)
        return {"op": op, "tokens": tokens, "experts": groups * size, "k": rng.randint(1, min(16, kept * size)), "score": "sigmoid", "bias": rng.random() < 0.8,
                "groups": groups, "kept": kept, "group_top": rng.choice([1, 2]), "dtype": dtype}
    vocab = _spread(rng, 1000, 160000)
    tokens = _spread(rng, 1, min(2048, 2048 * 128256 // (2 * vocab)))
    return {"op": op, "tokens": tokens, "vocab": vocab, "top": rng.choice([0, 1, 5, 20, 32]), "dtype": dtype, "allowed": rng.choice([0, 0, 0, rng.randint(24, 500)]), "pad": rng.choice([0, 0, 1, 8])}


def _rows(values, pad):
    """The rows with `pad` unused elements behind each."""
    if not pad:
        return values.contiguous()
    wide = torch.zeros(values.shape[0], values.shape[1] + pad, dtype=values.dtype, device=values.device)
    wide[:, : values.shape[1]] = values
    return wide[:, : values.shape[1]]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    uniform = lambda *s: torch.rand(*s, generator=g, device="cuda")  # noqa: E731
    empty = lambda *s, dtype: torch.empty(*s, dtype=dtype, device="cuda")  # noqa: E731
    n, s = case["tokens"], {"case": case}
    if case["op"] == "norm":
        # hidden states: channels differ in scale, a few of them by much
        cols, t = case["cols"], TYPES[case["dtype"]]
        channel = torch.exp(0.5 * normal(cols)) * torch.where(uniform(cols) < 0.004, 20.0, 1.0)
        s["x"] = _rows((0.3 * normal(n, cols) * channel).to(t), case["pad"])
        s["residual"] = _rows((normal(n, cols) * channel).to(t), case["pad"])
        s["weight"] = 0.5 + uniform(cols)
        s["sum"] = empty(n, cols, dtype=t)
        s["normed"] = empty(n, cols, dtype=torch.float32) if case["normed"] else None
        s["q"] = empty(n, cols, dtype=torch.int8)
        s["scales"] = empty(n, dtype=torch.float32)
        s["values"] = empty(n, cols, dtype=torch.bfloat16)
    elif case["op"] == "matmul":
        # what a quantizer to 8 bits leaves: every row's largest value is 127
        rows, cols = case["rows"], case["cols"]
        s["q"] = _rows((normal(n, cols) * 30).round_().clamp_(-127, 127).to(torch.int8), case["pad"])
        s["w"] = _rows((normal(rows, cols) * 32).round_().clamp_(-127, 127).to(torch.int8), case["pad"])
        s["scales"] = 0.01 + 0.04 * uniform(n)
        s["w_scales"] = (0.5 + uniform(rows)) * 0.02 / 32
        s["bias"] = normal(rows) if case["bias"] else None
        s["out"] = empty(n, rows, dtype=TYPES[case["dtype"]])
    elif case["op"] == "route":
        experts = case["experts"]
        s["logits"] = (1.5 * normal(n, experts) + 0.5 * normal(experts)).to(TYPES[case["dtype"]])
        s["bias"] = 0.1 * normal(experts) if case["bias"] else None
        s["idx"] = empty(n, case["k"], dtype=torch.int32)
        s["weight"] = empty(n, case["k"], dtype=torch.float32)
    else:
        # many unlikely tokens, some likely ones; a grammar may leave `allowed` of them
        vocab, top = case["vocab"], case["top"]
        logits = 2.0 * normal(n, vocab)
        likely = torch.randint(vocab, (n, 20), generator=g, device="cuda")
        logits.scatter_(1, likely, 8.0 + 6.0 * uniform(n, 20))
        target = torch.where(uniform(n) < 0.7, likely[:, 0], torch.randint(vocab, (n,), generator=g, device="cuda"))
        if case["allowed"]:
            keep = torch.zeros(n, vocab, dtype=torch.bool, device="cuda")
            keep.scatter_(1, torch.randint(vocab, (n, case["allowed"]), generator=g, device="cuda"), True)
            keep.scatter_(1, target[:, None], True)
            logits.masked_fill_(~keep, float("-inf"))
        s["logits"] = _rows(logits.to(TYPES[case["dtype"]]), case["pad"])
        s["target"] = target.to(torch.int32)
        s["log_prob"], s["entropy"] = empty(n, dtype=torch.float32), empty(n, dtype=torch.float32)
        s["rank"] = empty(n, dtype=torch.int32)
        s["top_ids"], s["top_log_probs"] = empty(n, top, dtype=torch.int32), empty(n, top, dtype=torch.float32)
    return s


_library = None


def _lib():
    global _library
    if _library is None:
        from camelid_amd import binding
        binding.init()
        _library = binding
    return _library


def _own(s):
    case, B = s["case"], _lib()
    L, stream, dtype, n = B.lib(), torch.cuda.current_stream().cuda_stream, IDS[case["dtype"]], case["tokens"]
    if case["op"] == "norm":
        x, residual, total, normed, q, scales, values, cols = s["x"], s["residual"], s["sum"], s["normed"], s["q"], s["scales"], s["values"], case["cols"]
        B.check(L.cml_add_rms_norm_i8(dtype, x.data_ptr(), x.stride(0), residual.data_ptr(), residual.stride(0), s["weight"].data_ptr(), EPS, n, cols,
                                      total.data_ptr(), cols, normed.data_ptr() if normed is not None else None, q.data_ptr(), cols, scales.data_ptr(), stream))
        B.check(L.cml_dequantize_i8(q.data_ptr(), cols, scales.data_ptr(), n, cols, IDS["bf16"], values.data_ptr(), cols, stream))
        return {"sum": total, "values": values, "scales": scales, "normed": normed}
    if case["op"] == "matmul":
        q, w, out, bias = s["q"], s["w"], s["out"], s["bias"]
        B.check(L.cml_matmul_i8(q.data_ptr(), q.stride(0), s["scales"].data_ptr(), n, w.data_ptr(), w.stride(0), s["w_scales"].data_ptr(), case["rows"], case["cols"],
                                bias.data_ptr() if bias is not None else None, dtype, out.data_ptr(), case["rows"], stream))
        return {"out": out}
    if case["op"] == "route":
        logits, bias, idx, weight = s["logits"], s["bias"], s["idx"], s["weight"]
        B.check(L.cml_moe_route_scored(SCORES[case["score"]], dtype, logits.data_ptr(), case["experts"], bias.data_ptr() if bias is not None else None, n, case["experts"],
                                       case["groups"], case["kept"], case["group_top"], case["k"], 1, 2.5, idx.data_ptr(), weight.data_ptr(), stream))
        return {"idx": idx, "weight": weight}
    if "workspace" not in s:  # sized once, as a serving loop keeps it
        s["workspace_bytes"] = L.cml_token_log_probs_workspace_bytes(n, case["vocab"], case["top"])
        s["workspace"] = torch.empty(max(16, s["workspace_bytes"]), dtype=torch.uint8, device="cuda")
    logits, top = s["logits"], case["top"]
    B.check(L.cml_token_log_probs(dtype, logits.data_ptr(), logits.stride(0), n, case["vocab"], s["target"].data_ptr(), top, s["log_prob"].data_ptr(), s["rank"].data_ptr(),
                                  s["entropy"].data_ptr(), s["top_ids"].data_ptr() if top else None, s["top_log_probs"].data_ptr() if top else None,
                                  s["workspace"].data_ptr(), s["workspace_bytes"], stream))
    return {"log_prob": s["log_prob"], "rank": s["rank"], "entropy": s["entropy"], "top_ids": s["top_ids"], "top_log_probs": s["top_log_probs"]}


def _ordered(v):
    """f32 values as whole numbers that order like them, ties to the lower column (64 bits: value, then column)."""
    bits = (v + 0.0).view(torch.int32)
    bits = bits ^ ((bits >> 31) & 0x7FFFFFFF)
    column = torch.arange(v.shape[1], device=v.device)
    return (bits.to(torch.int64) << 32) | (0x7FFFFFFF - column)


def _norm(s):
    case = s["case"]
    total = (s["x"].float() + s["residual"].float()).to(s["sum"].dtype)
    h = total.float()
    y = h * torch.rsqrt((h * h).sum(1, keepdim=True) / case["cols"] + EPS) * s["weight"]
    largest = y.abs().amax(1, keepdim=True)
    q = torch.where(largest > 0, torch.round(y * (127.0 / largest)), 0.0).clamp(-127, 127).to(torch.int8)
    scales = largest / 127.0
    return {"sum": total, "values": (q * scales).to(torch.bfloat16), "scales": scales[:, 0], "normed": y if case["normed"] else None}


def _matmul(s):
    out = (s["q"].float() @ s["w"].float().t()) * s["scales"][:, None] * s["w_scales"]
    if s["bias"] is not None:
        out = out + s["bias"]
    return {"out": out.to(s["out"].dtype)}


def _route(s):
    case, logits = s["case"], s["logits"].float()
    n, experts = logits.shape
    if case["score"] == "softmax":
        e = torch.exp(logits - logits.amax(1, keepdim=True))
        score = e / e.sum(1, keepdim=True)
    else:
        score = 1.0 / (1.0 + torch.exp(-logits))
    key = score + s["bias"] if s["bias"] is not None else logits  # (without a bias the scores order as the logits do)
    if case["groups"] > 1:
        size = experts // case["groups"]
        rated = (key if s["bias"] is not None or case["group_top"] == 1 else score).view(n, case["groups"], size)
        best = rated.topk(min(case["group_top"], size), dim=2).values.sum(2)
        group = 0x7FFFFFFF - (_ordered(best).topk(case["kept"], dim=1).values & 0x7FFFFFFF)
        kept = torch.zeros(n, case["groups"], dtype=torch.bool, device=key.device).scatter_(1, group, True)
        key = key.masked_fill(~kept.repeat_interleave(size, 1), float("-inf"))
    idx = 0x7FFFFFFF - (_ordered(key).topk(case["k"], dim=1).values & 0x7FFFFFFF)
    weight = score.gather(1, idx)
    weight = weight / weight.sum(1, keepdim=True) * 2.5
    return {"idx": idx.to(torch.int32), "weight": weight}


def _score(s):
    case, v = s["case"], s["logits"].float()
    target = s["target"].long()[:, None]
    d = v - v.amax(1, keepdim=True)
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    entropy = log_total - torch.where(e > 0, e * d, 0.0).sum(1, keepdim=True) / total
    given = v.gather(1, target)
    column = torch.arange(case["vocab"], device=v.device)
    rank = 1 + ((v > given) | ((v == given) & (column < target))).sum(1)
    best = 0x7FFFFFFF - (_ordered(v).topk(case["top"], dim=1).values & 0x7FFFFFFF)
    log_probs = d.gather(1, best) - log_total
    out = torch.isinf(log_probs)
    return {"log_prob": (d.gather(1, target) - log_total)[:, 0], "rank": rank.to(torch.int32), "entropy": entropy[:, 0],
            "top_ids": best.masked_fill(out, -1).to(torch.int32), "top_log_probs": log_probs}


def run(state):
    if own:
        return _own(state)
    return {"norm": _norm, "matmul": _matmul, "route": _route, "score": _score}[state["case"]["op"]](state)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = (s["x"].double() + s["residual"].double()).to(s["sum"].dtype)  # (the sum is defined in the stream's type)
        y = h.double() / torch.sqrt(h.double().square().mean(1, keepdim=True) + EPS) * s["weight"].double()
        step = y.abs().max(1, keepdim=True).values / 127
        return {"sum": s["x"].double() + s["residual"].double(), "values": torch.round(y / step) * step, "scales": step[:, 0], "normed": y if case["normed"] else None}
    if case["op"] == "matmul":
        out = torch.mm(s["q"].double(), s["w"].double().t())
        out.mul_(s["scales"].double()[:, None]).mul_(s["w_scales"].double()[None, :])
        return {"out": out if s["bias"] is None else out.add_(s["bias"].double())}
    if case["op"] == "route":
        logits = s["logits"].double()
        n, experts = logits.shape
        p = torch.softmax(logits, 1) if case["score"] == "softmax" else torch.sigmoid(logits)
        key = p.clone() if s["bias"] is None else p + s["bias"].double()
        grouped = key.view(n, case["groups"], -1)
        worth = grouped.sort(dim=2, descending=True).values[:, :, : case["group_top"]].sum(2)
        order = worth.sort(dim=1, descending=True, stable=True).indices
        grouped.scatter_(1, order[:, case["kept"]:, None].expand(-1, -1, grouped.shape[2]), -1e9)
        idx = key.sort(dim=1, descending=True, stable=True).indices[:, : case["k"]]
        chosen = torch.take_along_dim(p, idx, 1)
        return {"idx": None, "weight": 2.5 * chosen / chosen.sum(1, keepdim=True)}
    v = s["logits"].double()
    lp = torch.log_softmax(v, 1)
    p = torch.exp(lp)
    entropy = -(p * lp.clamp(min=-1e9)).sum(1)
    return {"log_prob": torch.take_along_dim(lp, s["target"].long()[:, None], 1)[:, 0], "rank": None, "entropy": entropy, "top_ids": None,
            "top_log_probs": lp.topk(case["top"], dim=1).values}


def work(case):
    n, size = case["tokens"], BYTES[case["dtype"]]
    if case["op"] == "norm":  # x, residual and weight in; sum, 8-bit values and scales out, the f32 row where asked
        cols = case["cols"]
        return {"bytes": n * cols * (3 * size + 1 + (4 if case["normed"] else 0)) + 4 * cols + 4 * n, "flops": 8 * n * cols}
    if case["op"] == "matmul":
        rows, cols = case["rows"], case["cols"]
        return {"bytes": n * cols + rows * cols + n * rows * size + 4 * n + 4 * rows * (2 if case["bias"] else 1), "flops": 2 * n * rows * cols}
    if case["op"] == "route":
        return {"bytes": n * (case["experts"] * size + 8 * case["k"]) + (4 * case["experts"] if case["bias"] else 0), "flops": n * case["experts"] * (4 + case["k"])}
    return {"bytes": n * (case["vocab"] * size + 16 + 8 * case["top"]), "flops": 5 * n * case["vocab"]}
