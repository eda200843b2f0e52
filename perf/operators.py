"""The expert and integer matrix products of ``td_benchmark_b200.ops``: what is timed, and the same in plain torch.

Five operators, told apart by a case's ``"op"``:

* ``grouped``   ``ops.grouped_mm``: rows sorted by expert times that expert's weights, segments of any length
* ``backward``  ``ops.grouped_mm_dx`` and ``ops.grouped_mm_dw``: the gradients of the rows and of the weights
* ``quant``     ``ops.quant_int8``: 8-bit codes with one scale for each row
* ``int8``      ``ops.int8_mm``: 8-bit integer product with scales for each token and channel
* ``int8_grouped``  ``ops.int8_grouped_mm``: the same over expert segments

``own`` chooses the framework's kernels or the plain form; both take what ``prepare`` returns.
"""
import math

import torch

own = False

# zipf exponent of the skewed routings, as in the framework's DeepSeek-V3 workload
ZIPF = 1.2
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # One token of a decode step, top-8 of 128 experts, gate/up weights: eight segments of one row.
        dict(name="grouped_one_token", op="grouped", dtype="bf16", experts=128, rows=8, slack=0, n=1536, k=2048,
             skew="once"),
        # A decode batch of 32 tokens, top-8 of 128 experts, down weights: segments of zero to a few rows.
        dict(name="grouped_decode", op="grouped", dtype="fp16", experts=128, rows=256, slack=0, n=2048, k=768,
             skew="none"),
        # A prompt of 1031 tokens, top-2 of 8 experts: few long segments of odd lengths.
        dict(name="grouped_prompt", op="grouped", dtype="fp16", experts=8, rows=2062, slack=0, n=14336, k=4096,
             skew="none"),
        # One rank of an 8-way expert-parallel layer under skewed routing, with receive rows that no token filled.
        dict(name="grouped_prefill", op="grouped", dtype="bf16", experts=32, rows=8192, slack=37, n=4096, k=7168,
             skew="zipf"),
        # The gradients of a layer small enough that latency counts.
        dict(name="backward_small", op="backward", dtype="fp16", experts=8, rows=128, slack=0, n=1024, k=256,
             skew="none"),
        # A training step of one expert-parallel rank: skewed segments, the longest a third of all rows.
        dict(name="backward_large", op="backward", dtype="bf16", experts=32, rows=16384, slack=101, n=4096, k=7168,
             skew="zipf"),
        # The activations of one token ahead of an integer product.
        dict(name="quant_one_token", op="quant", dtype="bf16", rows=1, k=7168),
        # The activations of a whole prefill step.
        dict(name="quant_prefill", op="quant", dtype="bf16", rows=8192, k=7168),
        # A dense projection of one token.
        dict(name="int8_one_token", op="int8", out="bf16", rows=1, n=28672, k=4096),
        # The same projection over a prefill batch of odd length.
        dict(name="int8_prefill", op="int8", out="bf16", rows=4093, n=28672, k=4096),
        # A decode batch of 32 tokens, top-8 of 128 integer experts.
        dict(name="int8_grouped_decode", op="int8_grouped", out="fp16", experts=128, rows=256, slack=0, n=1536,
             k=2048, skew="none"),
        # Integer experts of one expert-parallel rank at prefill, skewed.
        dict(name="int8_grouped_prefill", op="int8_grouped", out="bf16", experts=32, rows=8192, slack=37, n=4096,
             k=7168, skew="zipf"),
    ]


def _log_int(rng, low, high, step=1):
    """A multiple of ``step`` in [low, high], spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high + step)))
    return min(max(int(v) // step * step, low), high)


def draw(rng):
    op = rng.choice(["grouped", "backward", "quant", "int8", "int8_grouped"])
    if op == "quant":
        return dict(op=op, dtype=rng.choice(["bf16", "fp16", "fp32"]), rows=_log_int(rng, 1, 8192),
                    k=_log_int(rng, 64, 7168))
    n_step = 8 if op == "backward" else rng.choice([1, 8, 128])   # the gradients read dy rows of n values
    k_step = rng.choice([16, 128])
    case = dict(op=op, rows=_log_int(rng, 1, 8192), n=_log_int(rng, 128, 14336, n_step),
                k=_log_int(rng, 128, 7168, k_step))
    case["rows"] = min(case["rows"], 16384 * 4096 * 7168 // (case["n"] * case["k"]))   # no dearer than the largest
    if op in ("int8", "int8_grouped"):
        case["out"] = rng.choice(["bf16", "fp16", "fp32"])
    else:
        case["dtype"] = rng.choice(["bf16", "fp16"])
    if op != "int8":
        room = 32 * 4096 * 7168 // (case["n"] * case["k"])         # weights within those of the largest listed case
        case.update(experts=_log_int(rng, 1, min(256, room)), slack=rng.choice([0, 0, 1, 57]),
                    skew=rng.choice(["none", "zipf"]))
    return case


def _segments(case, seed):
    """Rows of each expert (a list that sums to ``rows``): the routing of the case."""
    experts, rows = case["experts"], case["rows"]
    g = torch.Generator().manual_seed(seed + 1)
    if case["skew"] == "once":                                     # distinct experts, one row each
        ids = torch.randperm(experts, generator=g)[:rows]
    else:
        p = torch.ones(experts, dtype=torch.float64)
        if case["skew"] == "zipf":
            p = torch.arange(1, experts + 1, dtype=torch.float64) ** -ZIPF
            p = p[torch.randperm(experts, generator=g)]
        ids = torch.multinomial(p, rows, replacement=True, generator=g)
    return torch.bincount(ids, minlength=experts).tolist()


def _codes(x):
    """8-bit codes and row scales of a matrix in 32 bits: the plain form of the quantiser."""
    amax = x.abs().amax(-1)
    # divided by a tensor: torch divides by a number as a product with its rounded reciprocal
    scale = (amax / torch.full_like(amax, 127.0)).clamp(min=1e-12)
    return torch.round(x / scale[:, None]).clamp(-127, 127).to(torch.int8), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype).mul_(std)

    op = case["op"]
    if op == "quant":
        # activations: a common width and a few columns that are far larger, as after a norm
        x = normal(case["rows"], case["k"])
        x[:, :: max(1, case["k"] // 7)] *= 12.0
        return dict(op=op, x=x.to(TYPES[case["dtype"]]))
    rows, n, k = case["rows"], case["n"], case["k"]
    if op == "int8":
        a, a_scale = _codes(normal(rows, k))
        w, w_scale = _codes(normal(n, k, std=0.02))
        return dict(op=op, a=a, a_scale=a_scale, w=w, w_scale=w_scale, out=TYPES[case["out"]])
    counts = _segments(case, seed)
    ends = torch.tensor(counts).cumsum(0).to(torch.int32).cuda()
    experts, total = case["experts"], rows + case["slack"]
    state = dict(op=op, counts=counts, ends=ends)
    if op == "int8_grouped":
        a, a_scale = _codes(normal(total, k))
        w = torch.empty((experts, n, k), dtype=torch.int8, device="cuda")
        w_scale = torch.empty((experts, n), dtype=torch.float32, device="cuda")
        for e in range(experts):
            w[e], w_scale[e] = _codes(normal(n, k, std=0.02))
        return dict(state, a=a, a_scale=a_scale, w=w, w_scale=w_scale, out=TYPES[case["out"]])
    dtype = TYPES[case["dtype"]]
    state.update(x=normal(total, k, dtype=dtype), w=normal(experts, n, k, std=0.02, dtype=dtype))
    if op == "backward":
        state.update(dy=normal(total, n, dtype=dtype))
    return state


def _spans(counts):
    """(expert, first row, row behind the last) of the segments that have rows."""
    at, spans = 0, []
    for e, c in enumerate(counts):
        if c:
            spans.append((e, at, at + c))
        at += c
    return spans


# The plain forms go over the experts that have rows, one product each in 32 bits: the segments' lengths differ, and a
# batched product over the longest would do several times the work under a skewed routing.
def _rows_times(rows, spans, weight_of, width, dtype):
    """Each segment's rows times its expert's matrix; rows behind the last segment are zero."""
    parts = [(rows[a:b].float() @ weight_of(e)).to(dtype) for e, a, b in spans]
    behind = len(rows) - spans[-1][2]
    return torch.cat(parts + [torch.zeros((behind, width), dtype=dtype, device=rows.device)])


def _plain(s):
    op = s["op"]
    if op == "quant":
        return _codes(s["x"].float())
    if op == "int8":
        y = s["a"].float() @ s["w"].float().T
        return (y * s["a_scale"][:, None] * s["w_scale"]).to(s["out"])
    spans = _spans(s["counts"])
    if op == "int8_grouped":
        scaled = s["a"].float() * s["a_scale"][:, None]
        return _rows_times(scaled, spans, lambda e: (s["w"][e].float() * s["w_scale"][e][:, None]).T,
                           s["w"].shape[1], s["out"])
    x, w = s["x"], s["w"]
    if op == "grouped":
        return _rows_times(x, spans, lambda e: w[e].float().T, w.shape[1], x.dtype)
    dw = torch.zeros_like(w)
    for e, a, b in spans:
        dw[e] = s["dy"][a:b].float().T @ x[a:b].float()
    return _rows_times(s["dy"], spans, lambda e: w[e].float(), w.shape[2], x.dtype), dw


def _kernels(s):
    from td_benchmark_b200 import ops

    op = s["op"]
    if op == "quant":
        return ops.quant_int8(s["x"])
    if op == "int8":
        return ops.int8_mm(s["a"], s["a_scale"], s["w"], s["w_scale"], out_dtype=s["out"])
    if op == "int8_grouped":
        return ops.int8_grouped_mm(s["a"], s["a_scale"], s["w"], s["w_scale"], s["ends"], out_dtype=s["out"])
    if op == "grouped":
        return ops.grouped_mm(s["x"], s["w"], s["ends"])
    return ops.grouped_mm_dx(s["dy"], s["w"], s["ends"]), ops.grouped_mm_dw(s["dy"], s["x"], s["ends"])


def run(state):
    return _kernels(state) if own else _plain(state)


def _busy_experts(case):
    """Experts that have rows, on average over the routings of the case."""
    experts, rows = case["experts"], case["rows"]
    if case["skew"] == "once":
        return rows
    p = [1.0] * experts if case["skew"] == "none" else [(i + 1) ** -ZIPF for i in range(experts)]
    return sum(1.0 - (1.0 - v / sum(p)) ** rows for v in p)


def work(case):
    op, rows, k = case["op"], case["rows"], case["k"]
    if op == "quant":
        size = TYPES[case["dtype"]].itemsize
        return {"bytes": rows * k * (size + 1) + 4 * rows, "flops": 3 * rows * k}
    n = case["n"]
    flops = 2 * rows * n * k
    if op == "int8":
        return {"bytes": rows * k + n * k + 4 * (rows + n) + rows * n * TYPES[case["out"]].itemsize, "flops": flops}
    busy, total, experts = _busy_experts(case), rows + case["slack"], case["experts"]
    if op == "int8_grouped":
        size = TYPES[case["out"]].itemsize
        return {"bytes": int(rows * (k + 4) + busy * n * (k + 4) + 4 * experts + total * n * size), "flops": flops}
    if op == "grouped":
        return {"bytes": int(2 * (rows * k + busy * n * k + total * n) + 4 * experts), "flops": flops}
    # dy, x and the weights read once; the rows' gradient and every expert's weight gradient written once
    return {"bytes": int(2 * (rows * (n + k) + busy * n * k + total * k + experts * n * k) + 4 * experts),
            "flops": 2 * flops}


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "quant":
        # scale = fp32(max(amax / 127, 1e-12)), code = nearest even integer of the fp32 quotient, by definition. A
        # quotient in 64 bits rounded to 32 is the 32-bit quotient.
        x = s["x"].double()
        scale = torch.maximum(x.abs().max(dim=-1).values / 127, x.new_tensor(1e-12)).float()
        q = (x / scale.double().unsqueeze(-1)).float().double()
        return q.round().clip(-127, 127).to(torch.int8), scale.double()
    if op == "int8":
        sums = torch.einsum("mk,nk->mn", s["a"].double(), s["w"].double())
        return torch.einsum("mn,m,n->mn", sums, s["a_scale"].double(), s["w_scale"].double())
    start = torch.tensor([0] + s["counts"]).cumsum(0).tolist()
    if op == "int8_grouped":
        y = torch.zeros((len(s["a"]), case["n"]), dtype=torch.float64, device="cuda")
        for e in range(case["experts"]):
            at = slice(start[e], start[e + 1])
            y[at] = torch.einsum("mk,nk->mn", s["a"][at].double(), s["w"][e].double())
            y[at] *= s["a_scale"][at].double().outer(s["w_scale"][e].double())
        return y
    x, w = s["x"], s["w"]
    if op == "grouped":
        y = torch.zeros((len(x), case["n"]), dtype=torch.float64, device="cuda")
        for e in range(case["experts"]):
            at = slice(start[e], start[e + 1])
            y[at] = torch.einsum("mk,nk->mn", x[at].double(), w[e].double())
        return y
    dx = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    dw = torch.empty(w.shape, dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        at = slice(start[e], start[e + 1])
        dx[at] = torch.einsum("mn,nk->mk", s["dy"][at].double(), w[e].double())
        dw[e] = torch.einsum("mn,mk->nk", s["dy"][at].double(), x[at].double())
    return dx, dw
