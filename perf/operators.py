"""Cases of the grouped matrix products, their gradients, the 8-bit product and the row quantisation.

The rows of an activation matrix are sorted by the expert that they were routed to; ``offsets`` (int32, on the GPU)
says where each expert's rows begin.  Weights are [experts, out, in], as a linear layer keeps them.

  mm        y[r] = x[r] @ w[g]^T for the rows r of expert g
  grad_x    dx[r] = dy[r] @ w[g]
  grad_w    dw[g] = dy[rows of g]^T @ x[rows of g]
  int8      y[r, n] = xs[r] * ws[g, n] * sum_k xq[r, k] * wq[g, n, k], whole numbers inside the sum
  quantize  s[r] = max|x[r]| / 127, q[r] = x[r] / s[r] rounded to the nearest whole number, ties to even
"""
import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "int8": 1}


def _case(name, op, rows, experts, live, k, n, dtype):
    return {"name": name, "op": op, "rows": rows, "experts": experts, "live": live, "k": k, "n": n, "dtype": dtype}


def listed():
    return [
        # two tokens, two experts each: a small layer answering a single stream
        _case("mm, two tokens", "mm", 4, 8, 4, 1024, 1024, "bf16"),
        # a decoding step of a batch: every expert's weights are read for a handful of rows
        _case("mm, decoding batch", "mm", 128, 32, 32, 2048, 1024, "bf16"),
        # sizes that nothing divides, and an expert that got no rows
        _case("mm, odd sizes", "mm", 1003, 5, 4, 777, 1001, "fp16"),
        # a prompt of a few thousand tokens
        _case("mm, prompt", "mm", 8192, 16, 15, 2048, 4096, "fp16"),
        # a training batch through the wide product
        _case("mm, training batch", "mm", 32768, 16, 16, 4096, 4096, "bf16"),
        # the same layer's gradient with respect to its input
        _case("grad_x, training batch", "grad_x", 8192, 16, 16, 2048, 4096, "bf16"),
        # and with respect to its weights
        _case("grad_w, training batch", "grad_w", 8192, 16, 16, 2048, 4096, "bf16"),
        # many small experts, some without rows: short sums, and gradients that are zero
        _case("grad_w, many experts", "grad_w", 2000, 64, 50, 1024, 512, "fp16"),
        # one token through a dense layer in 8 bits
        _case("int8, one token", "int8", 1, 1, 1, 4096, 4096, "bf16"),
        # a prompt through experts in 8 bits
        _case("int8, prompt", "int8", 8192, 8, 8, 4096, 4096, "fp16"),
        # the activations of a decoding batch on their way to the 8-bit product
        _case("quantize, decoding batch", "quantize", 64, 1, 1, 4096, 0, "bf16"),
        # and of a long prompt
        _case("quantize, prompt", "quantize", 16384, 1, 1, 8192, 0, "bf16"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """A width: mostly a multiple of 16, as layers have them, now and then any whole number."""
    v = _spread(rng, low, high)
    return v if rng.random() < 0.2 else max(16, v // 16 * 16)


def draw(rng: random.Random):
    op = rng.choice(["mm", "mm", "grad_x", "grad_w", "int8", "int8", "quantize"])
    if op == "quantize":
        return {"op": op, "rows": _spread(rng, 1, 16384), "experts": 1, "live": 1, "k": _width(rng, 64, 8192), "n": 0,
                "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    rows = _spread(rng, 1, 16384)
    experts = rng.choice([1, _spread(rng, 2, 64)])
    live = min(rows, rng.randint(max(1, experts // 2), experts))
    return {"op": op, "rows": rows, "experts": experts, "live": live, "k": _width(rng, 256, 4096),
            "n": _width(rng, 256, 4096), "dtype": rng.choice(["bf16", "fp16"])}


def _group_sizes(case, seed):
    """Rows of each expert: some experts are more popular than others, the live ones get one row at least."""
    rng = random.Random(seed)
    live = rng.sample(range(case["experts"]), case["live"])
    sizes = [0] * case["experts"]
    for g in live:
        sizes[g] = 1
    popularity = [rng.uniform(0.5, 2.0) for _ in live]
    for g in rng.choices(live, popularity, k=case["rows"] - case["live"]):
        sizes[g] += 1
    return sizes


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, rows, experts, k, n = case["op"], case["rows"], case["experts"], case["k"], case["n"]
    dtype = _TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dtype):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    state = {"op": op, "dtype": dtype, "rows": rows, "experts": experts}
    if op == "quantize":
        # rows of very different size, as activations have them
        state["x"] = (torch.randn(rows, k, generator=gen, device="cuda")
                      * torch.exp(torch.randn(rows, 1, generator=gen, device="cuda"))).to(dtype)
    else:
        sizes = _group_sizes(case, seed)
        offsets = [0]
        for s in sizes:
            offsets.append(offsets[-1] + s)
        state["offsets"] = torch.tensor(offsets, dtype=torch.int32, device="cuda")
        state["most"] = max(sizes)
        if op in ("mm", "grad_w"):
            state["x"] = normal(rows, k)
        if op in ("grad_x", "grad_w"):
            state["dy"] = normal(rows, n)
        if op in ("mm", "grad_x"):
            state["w"] = torch.empty(experts, n, k, dtype=dtype, device="cuda")
            for g in range(experts):
                state["w"][g] = normal(n, k, scale=k ** -0.5)
        if op == "int8":
            state["xq"] = normal(rows, k, scale=36.0, dtype=torch.float32).round_().clamp_(-127, 127).to(torch.int8)
            state["wq"] = torch.empty(experts, n, k, dtype=torch.int8, device="cuda")
            for g in range(experts):
                state["wq"][g] = normal(n, k, scale=36.0, dtype=torch.float32).round_().clamp_(-127, 127)
            state["xs"] = torch.rand(rows, generator=gen, device="cuda") * 0.03 + 0.01
            state["ws"] = (torch.rand(experts, n, generator=gen, device="cuda") + 0.5) * (k ** -0.5 / 36.0)
    if own:
        _plan(state, case)
    return state


def _plan(state, case):
    """What a user's program keeps from call to call: handle, descriptors, results and the products' buffers."""
    from ops_sparse_b200 import _lib as L
    from ops_sparse_b200 import api

    op, rows, experts, k, n, dtype = (case["op"], case["rows"], case["experts"], case["k"], case["n"], state["dtype"])
    handle = api.Handle()
    if op == "quantize":
        state["out"] = (torch.empty(rows, k, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda"))
        state["call"] = api.QuantizeRows(handle, api.DnMat(rows, k, k, state["x"]),
                                         api.DnMat(rows, k, k, state["out"][0]), state["out"][1])
        return
    if op == "grad_w":
        state["out"] = torch.empty(experts, n, k, dtype=dtype, device="cuda")
        product = api.GroupedMMWeightGrad(handle, api.DnMat(rows, n, n, state["dy"]), api.DnMat(rows, k, k, state["x"]),
                                          api.DnMat(n, k, k, state["out"], batch_count=experts, batch_stride=n * k),
                                          state["offsets"])
    elif op == "grad_x":
        state["out"] = torch.empty(rows, k, dtype=dtype, device="cuda")
        product = api.GroupedMM(handle, api.DnMat(rows, n, n, state["dy"]),
                                api.DnMat(n, k, k, state["w"], batch_count=experts, batch_stride=n * k),
                                api.DnMat(rows, k, k, state["out"]), state["offsets"])
    else:
        state["out"] = torch.empty(rows, n, dtype=dtype, device="cuda")
        a, b = (state["xq"], state["wq"]) if op == "int8" else (state["x"], state["w"])
        product = api.GroupedMM(handle, api.DnMat(rows, k, k, a),
                                api.DnMat(n, k, k, b, batch_count=experts, batch_stride=n * k),
                                api.DnMat(rows, n, n, state["out"]), state["offsets"] if experts > 1 else None,
                                op_b=L.OP_T, row_scales=state.get("xs"), col_scales=state.get("ws"))
    product.preprocess()
    state["call"] = product


def _slots(state):
    """Each row's place when every expert has room for the largest group."""
    row = torch.arange(state["rows"], device="cuda")
    starts = state["offsets"].long()
    group = torch.searchsorted(starts[1:], row, right=True)
    return group * state["most"] + row - starts[group]


def _padded(state, rows, slots):
    out = torch.zeros(state["experts"] * state["most"], rows.shape[1], device="cuda")
    out[slots] = rows.float()
    return out.view(state["experts"], state["most"], -1)


def run(state):
    if own:
        state["call"]()
        return state["out"]
    op, dtype = state["op"], state["dtype"]
    if op == "quantize":
        x = state["x"].float()
        scale = x.abs().amax(dim=1) / 127
        # next to a tie 32 bits can land on the wrong side: the quotient is taken in 64
        ratio = x.double() / torch.where(scale == 0, torch.ones_like(scale), scale).double()[:, None]
        return torch.round(ratio).to(torch.int8), scale
    slots = _slots(state)
    if op == "grad_w":
        return torch.bmm(_padded(state, state["dy"], slots).transpose(1, 2), _padded(state, state["x"], slots)).to(dtype)
    if op == "grad_x":
        y = torch.bmm(_padded(state, state["dy"], slots), state["w"].float())
    else:
        x, w = (state["xq"], state["wq"]) if op == "int8" else (state["x"], state["w"])
        y = torch.bmm(_padded(state, x, slots), w.float().transpose(1, 2))
        if op == "int8":
            y = y * state["ws"][:, None, :]
    y = y.reshape(-1, y.shape[2])[slots]
    if op == "int8":
        y = y * state["xs"][:, None]
    return y.to(dtype)


def work(case):
    op, rows, experts, live, k, n = (case[x] for x in ("op", "rows", "experts", "live", "k", "n"))
    e = _BYTES[case["dtype"]]
    if op == "quantize":
        return {"bytes": rows * k * (e + 1) + 4 * rows, "flops": 3 * rows * k}
    flops = 2 * rows * k * n
    if op == "grad_w":
        return {"bytes": e * (rows * (k + n) + experts * k * n) + 4 * (experts + 1), "flops": flops}
    if op == "int8":
        return {"bytes": rows * k + live * k * n + e * rows * n + 4 * (rows + live * n + experts + 1), "flops": flops}
    return {"bytes": e * (rows * (k + n) + live * k * n) + 4 * (experts + 1), "flops": flops}


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        x = state["x"].double()
        scale = (x.abs().max(dim=1, keepdim=True).values / 127).float().double()
        return torch.where(scale > 0, x / scale, 0.0).round().to(torch.int8), scale[:, 0]
    bounds = state["offsets"].tolist()
    spans = [slice(bounds[g], bounds[g + 1]) for g in range(case["experts"])]
    if op == "grad_w":
        return torch.stack([state["dy"][s].double().T @ state["x"][s].double() for s in spans])
    if op == "grad_x":
        return torch.cat([state["dy"][s].double() @ state["w"][g].double() for g, s in enumerate(spans)])
    if op == "mm":
        return torch.cat([state["x"][s].double() @ state["w"][g].double().T for g, s in enumerate(spans)])
    return torch.cat([(state["xq"][s].double() @ state["wq"][g].double().T) * state["ws"][g].double()
                      * state["xs"][s].double()[:, None] for g, s in enumerate(spans)])
