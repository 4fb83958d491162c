"""Performance cases of the expert layers and of the INT8 product for serving.

A case names an operator ("op"), its sizes and its options:
  sort     moe.sort_tokens    x [T, H] and the expert ids [T, k] of its tokens -> the rows in the order of their experts,
                              each expert's rows padded to a multiple of `align`; with "grad" the gradient of x too
  combine  moe.combine        rows [R, H] back to tokens, y[t] = sum over j of weights[t, j] * rows[pos[t, j]]; with "grad"
                              the gradients of the rows and of the weights too
  experts  moe.expert_linear  rows [R, K] in the order of their experts x one int8 weight matrix an expert, a scale a row
                              and a scale an output channel
  linear   linear.linear_w8a8 the same product with one matrix, x [T, K]

Sizes are the library's own (4096 hidden, 11008 and 1408 wide MLPs, layers of 1024 and 2048) and odd ones between them, from
one token to 16384.  Data follow its other cases: activations ~ N(0,1) with 0.5 % of the channels x30, weights ~ N(0,0.02),
output gradients ~ N(0,1e-3), bias ~ N(0,0.01).  Experts are chosen by random logits with a bias per expert, so that some get
several times the rows of others.  "drop" is the share of choices that belong to no expert here (id -1): those of another
rank, or above a capacity.
"""
import math

import torch

own = False   # False: the plain forms below; True: the calls that a user makes

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # One token being generated: launches and latency are all there is.
        dict(name="sort 1x4096", op="sort", T=1, H=4096, k=2, E=8, align=1, dtype="bf16", ids="int64", drop=0.0, grad=False),
        # Training step of an expert layer whose experts are Int8Linear: segments of whole blocks of 128 rows.
        dict(name="sort train 16384x4096", op="sort", T=16384, H=4096, k=2, E=8, align=128, dtype="bf16", ids="int64", drop=0.0, grad=True),
        # One rank's share of many small experts, tokens that fill no block, rows that fill no 16 bytes.
        dict(name="sort train 4099x1405", op="sort", T=4099, H=1405, k=6, E=64, align=1, dtype="fp16", ids="int32", drop=0.5, grad=True),
        # The way back for one token.
        dict(name="combine 1x4096", op="combine", T=1, H=4096, k=2, E=8, align=1, dtype="bf16", wdtype="fp32", drop=0.0, grad=False),
        # The way back in the training step above.
        dict(name="combine train 16384x4096", op="combine", T=16384, H=4096, k=2, E=8, align=128, dtype="bf16", wdtype="fp32", drop=0.0, grad=True),
        # 32-bit rows with dropped choices at ragged sizes.
        dict(name="combine train 1037x2176", op="combine", T=1037, H=2176, k=4, E=60, align=1, dtype="fp32", wdtype="fp32", drop=0.25, grad=True),
        # One token through its two experts' up-projections: the weights of two matrices, nothing else.
        dict(name="experts 1x4096x11008", op="experts", T=1, k=2, E=8, K=4096, N=11008, bias=False, out="bf16", drop=0.0),
        # A batch of sequences generating together: every expert's weights for a few rows each.
        dict(name="experts 64x4096x1408", op="experts", T=64, k=6, E=64, K=4096, N=1408, bias=False, out="bf16", drop=0.0),
        # A short prompt through small experts at ragged sizes.
        dict(name="experts 1999x1408x2176", op="experts", T=1999, k=4, E=60, K=1408, N=2176, bias=True, out="bf16", drop=0.25),
        # Long prompts through large experts: the tensor cores' work, and the largest case.
        dict(name="experts 16384x4096x11008", op="experts", T=16384, k=2, E=8, K=4096, N=11008, bias=False, out="bf16", drop=0.0),
        # Five sequences generating together through a dense layer.
        dict(name="linear 5x4096x4096", op="linear", T=5, K=4096, N=4096, bias=True, out="bf16"),
        # A prompt of odd length through a dense layer.
        dict(name="linear 2047x2048x1000", op="linear", T=2047, K=2048, N=1000, bias=True, out="fp32"),
    ]


def _spread(rng, lo, hi, step=1):
    """A multiple of `step` between lo and hi, spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi // step * step, max(-(-lo // step) * step, int(round(v / step)) * step))


def draw(rng):
    top = {c["name"]: work(c) for c in listed()}
    most_bytes = max(w["bytes"] for w in top.values())
    most_flops = max(w["flops"] for w in top.values())
    while True:
        op = rng.choice(["sort", "sort", "combine", "combine", "experts", "experts", "experts", "linear", "linear"])
        T = _spread(rng, 1, 16384)
        case = dict(op=op, T=T)
        if op != "linear":
            case["E"] = rng.choice([2, 4, 8, 16, 32, 60, 64, 128])
            case["k"] = rng.randint(1, min(8, case["E"]))
            case["drop"] = rng.choice([0.0, 0.0, 0.25, 0.75])
        if op in ("sort", "combine"):
            case["H"] = _spread(rng, 64, 8192, rng.choice([1, 8, 8, 128]))
            case.update(align=rng.choice([1, 1, 16, 128]), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), grad=rng.random() < 0.6)
            if op == "sort":
                case["ids"] = rng.choice(["int32", "int64"])
            else:
                case["wdtype"] = rng.choice(["fp32", case["dtype"]])
        else:
            case.update(K=_spread(rng, 64, 11008, 16), N=_spread(rng, 64, 11008, 8), bias=rng.random() < 0.5, out=rng.choice(["bf16", "bf16", "fp32"]))
            if case.get("E", 1) * case["K"] * case["N"] > 8 * 4096 * 11008:
                continue
        w = work(case)
        if w["bytes"] <= most_bytes and w["flops"] <= most_flops:
            return case


# ------------------------------------------------------------------------------------------------ inputs
def _normal(g, shape, std, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=g)


def _activations(g, shape, dtype=torch.bfloat16):
    """~ N(0,1) with 0.5 % of the channels (last axis) x30."""
    x = _normal(g, shape, 1.0, dtype)
    n_out = -(-shape[-1] * 5 // 1000)
    x[..., torch.randperm(shape[-1], generator=g, device="cuda")[:n_out]] *= 30
    return x


def _choices(g, case):
    """The experts of each token, [T, k] int64, and their weights, fp32: the k largest of random logits, softmax over them."""
    T, k, E = case["T"], case["k"], case["E"]
    logits = _normal(g, (T, E), 1.0, torch.float32) + _normal(g, (E,), 0.5, torch.float32)
    top, ids = logits.topk(k, dim=-1)
    if case["drop"]:
        ids = ids.masked_fill(torch.rand((T, k), generator=g, device="cuda") < case["drop"], -1)
    return ids, top.softmax(-1)


def _rows_of(T, k, E, align):
    """Rows of the sorted tensor: enough for every choice and for the padding behind each expert."""
    return -(-(T * k + min(E, T * k) * (align - 1)) // align) * align


def _layout(ids, E, align):
    """offsets [E + 1], pos [T, k] and src [R], int32: see _plain_sort."""
    T, k = ids.shape
    flat = ids.reshape(-1).long()
    valid = (flat >= 0) & (flat < E)
    hot = (flat[:, None] == torch.arange(E, device=flat.device)) & valid[:, None]
    before = hot.cumsum(0)                                   # choices of the expert up to and with this one
    size = -(-before[-1] // align) * align
    offsets = torch.zeros(E + 1, dtype=torch.long, device=flat.device)
    offsets[1:] = size.cumsum(0)
    safe = flat.clamp(0, E - 1)
    pos = torch.where(valid, offsets[safe] + before.gather(1, safe[:, None])[:, 0] - 1, -1)
    rows = _rows_of(T, k, E, align)
    src = torch.full((rows + 1,), -1, dtype=torch.long, device=flat.device)
    src[torch.where(valid, pos, rows)] = torch.arange(T * k, device=flat.device)
    return offsets.int(), pos.view(T, k).int(), src[:rows].int()


def _quantized(w):
    """int8 w [..., N, K] with one scale a row, fp32."""
    amax = w.float().abs().amax(-1).clamp_min(1e-4)
    q = torch.floor(w.float() * (127.0 / amax)[..., None] + 0.5).clamp(-127, 127).to(torch.int8)
    return q, amax / 127.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    state = dict(case=case)
    if op == "linear":
        K, N = case["K"], case["N"]
        state["x"] = _activations(g, (case["T"], K))
        state["wq"], state["ws"] = _quantized(_normal(g, (N, K), 0.02))
        state["bias"] = _normal(g, (N,), 0.01) if case["bias"] else None
        return state
    ids, weights = _choices(g, case)
    T, k, E = case["T"], case["k"], case["E"]
    if op == "sort":
        state["ids"] = ids.to(getattr(torch, case["ids"]))
        state["x"] = _activations(g, (T, case["H"]), DTYPES[case["dtype"]]).requires_grad_(case["grad"])
        if case["grad"]:
            state["drows"] = _normal(g, (_rows_of(T, k, E, case["align"]), case["H"]), 1e-3, DTYPES[case["dtype"]])
        return state
    state["offsets"], state["pos"], state["src"] = _layout(ids, E, case.get("align", 1))
    rows = state["src"].numel()
    if op == "combine":
        dtype = DTYPES[case["dtype"]]
        state["rows"] = _activations(g, (rows, case["H"]), dtype).requires_grad_(case["grad"])
        state["weights"] = weights.to(DTYPES[case["wdtype"]]).requires_grad_(case["grad"])
        if case["grad"]:
            state["dy"] = _normal(g, (T, case["H"]), 1e-3, dtype)
        return state
    K, N = case["K"], case["N"]
    state["rows"] = _activations(g, (rows, K)) * (state["src"] >= 0)[:, None]
    state["wq"], state["ws"] = _quantized(_normal(g, (E, N, K), 0.02))
    state["bias"] = _normal(g, (E, N), 0.01) if case["bias"] else None
    return state


# ------------------------------------------------------------------------------------------------ plain forms
def _take(rows, pos):
    """rows[pos] in 32 bits, [T, k, H], zero where pos is -1."""
    return torch.where((pos >= 0)[..., None], rows[pos.clamp_min(0).long()].float(), 0.0)


def _plain_sort(s):
    """Rows of a token's choices in the order of (expert, token, choice); expert e has rows offsets[e] to offsets[e + 1], those
    behind its choices are zero, as are those behind offsets[E].  pos: the row of a choice, or -1; src: the choice of a
    row, t * k + j, or -1."""
    case, x, ids = s["case"], s["x"].detach(), s["ids"]
    offsets, pos, src = _layout(ids, case["E"], case["align"])
    rows = torch.where((src >= 0)[:, None], x[(src.clamp_min(0) // case["k"]).long()], 0)
    out = dict(rows=rows, offsets=offsets, pos=pos, src=src)
    if case["grad"]:
        out["dx"] = _take(s["drows"], pos).sum(1).to(x.dtype)
    return out


def _plain_combine(s):
    case, rows, weights, pos = s["case"], s["rows"].detach(), s["weights"].detach(), s["pos"]
    taken = _take(rows, pos)
    w = torch.where(pos >= 0, weights.float(), 0.0)
    out = dict(y=(w[..., None] * taken).sum(1).to(rows.dtype))
    if case["grad"]:
        dy, src = s["dy"].float(), s["src"]
        back = src.clamp_min(0).long()
        drows = w.view(-1)[back][:, None] * dy[back // case["k"]]
        out["drows"] = torch.where((src >= 0)[:, None], drows, 0.0).to(rows.dtype)
        out["dweights"] = (taken * dy[:, None]).sum(-1).to(weights.dtype)
    return out


def _plain_quant(x):
    """One scale a row, s = (1 / max |x|) * 127 in 32 bits; q = floor(x * s + 1/2)."""
    xf = x.float()
    amax = xf.abs().amax(-1, keepdim=True).clamp_min(1e-4)
    return torch.floor(xf * (torch.reciprocal(amax) * 127.0) + 0.5).clamp(-128, 127), amax / 127.0


def _plain_product(x, wq, ws, bias, out):
    """y = (q . wq^T) * scale of the row * scale of the channel + bias, x of one expert."""
    q, scale = _plain_quant(x)
    y = q @ wq.float().t() * scale * ws
    return (y if bias is None else y + bias.float()).to(out)


def _plain_experts(s):
    """An expert's rows are offsets[e] to offsets[e + 1]; those behind the last expert's come out zero."""
    out = DTYPES[s["case"]["out"]]
    ends = s["offsets"].tolist()
    parts = [_plain_product(s["rows"][a:b], s["wq"][e], s["ws"][e], None if s["bias"] is None else s["bias"][e], out)
             for e, (a, b) in enumerate(zip(ends, ends[1:])) if b > a]
    tail = torch.zeros((s["rows"].shape[0] - ends[-1], s["wq"].shape[1]), dtype=out, device=s["rows"].device)
    return torch.cat([*parts, tail])


def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        if op == "linear":
            return _plain_product(s["x"], s["wq"], s["ws"], s["bias"], DTYPES[s["case"]["out"]])
        return {"sort": _plain_sort, "combine": _plain_combine, "experts": _plain_experts}[op](s)
    from triton_int8_b200 import linear, moe
    case = s["case"]
    if op == "linear":
        return linear.linear_w8a8(s["x"], s["wq"], s["ws"], s["bias"], out_dtype=DTYPES[case["out"]])
    if op == "experts":
        return moe.expert_linear(s["rows"], s["wq"], s["ws"], s["offsets"], s["bias"], out_dtype=DTYPES[case["out"]])
    if op == "sort":
        rows, offsets, pos, src = moe.sort_tokens(s["x"], s["ids"], case["E"], align=case["align"])
        out = dict(rows=rows.detach(), offsets=offsets, pos=pos, src=src)
        if case["grad"]:
            rows.backward(s["drows"])
            out["dx"], s["x"].grad = s["x"].grad, None
        return out
    y = moe.combine(s["rows"], s["weights"], s["pos"], s["src"])
    out = dict(y=y.detach())
    if case["grad"]:
        y.backward(s["dy"])
        out["drows"], s["rows"].grad = s["rows"].grad, None
        out["dweights"], s["weights"].grad = s["weights"].grad, None
    return out


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_product(x, wq, ws, bias):
    """The int8 operand is defined by steps in 32 bits (the double_channel quantizer), each rounded here from 64; the rest is exact
    integers and 64 bits."""
    x = x.double()
    amax = x.abs().max(-1, keepdim=True).values.clamp_min(float(torch.tensor(1e-4)))
    s = ((1.0 / amax).float().double() * 127.0).float().double()
    q = torch.floor(((x * s).float().double() + 0.5).float()).double()
    y = (q @ wq.double().t()) * ((amax / 127.0).float().double() * ws.double())
    return y if bias is None else y + bias.double()


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "linear":
        return _exact_product(s["x"], s["wq"], s["ws"], s["bias"])
    k = case["k"]
    if op == "experts":
        y = torch.zeros((s["rows"].shape[0], case["N"]), dtype=torch.float64, device="cuda")
        offsets = s["offsets"].tolist()
        for e in range(case["E"]):
            part = slice(offsets[e], offsets[e + 1])
            y[part] = _exact_product(s["rows"][part], s["wq"][e], s["ws"][e], None if s["bias"] is None else s["bias"][e])
        return y
    if op == "sort":
        x, ids, E, align = s["x"].detach(), s["ids"].reshape(-1).long(), case["E"], case["align"]
        total = _rows_of(case["T"], k, E, align)
        order = torch.where((ids < 0) | (ids >= E), E, ids).sort(stable=True).indices.tolist()
        count = torch.bincount(ids[(ids >= 0) & (ids < E)], minlength=E).tolist()
        offsets, src, at = [0], [], 0
        for n in count:
            src += order[at:at + n] + [-1] * (-n % align)
            at += n
            offsets.append(len(src))
        src = torch.tensor(src + [-1] * (total - len(src)), device="cuda")
        live = src >= 0
        rows = torch.zeros((total, case["H"]), dtype=torch.float64, device="cuda")
        rows[live] = x.double()[src[live] // k]
        pos = torch.full((case["T"] * k,), -1, device="cuda")
        pos[src[live]] = live.nonzero()[:, 0]
        out = dict(rows=rows, offsets=torch.tensor(offsets, dtype=torch.int32, device="cuda"), pos=pos.view(-1, k).int(), src=src.int())
        if case["grad"]:
            out["dx"] = torch.zeros(x.shape, dtype=torch.float64, device="cuda").index_add_(0, src[live] // k, s["drows"].double()[live])
        return out
    rows, weights, src = s["rows"].detach().double(), s["weights"].detach().double().view(-1), s["src"].long()
    live = src >= 0
    at, token = src[live], src[live] // k
    y = torch.zeros((case["T"], case["H"]), dtype=torch.float64, device="cuda")
    out = dict(y=y.index_add_(0, token, weights[at][:, None] * rows[live]))
    if case["grad"]:
        dy = s["dy"].double()
        out["drows"] = torch.zeros_like(rows)
        out["drows"][live] = weights[at][:, None] * dy[token]
        out["dweights"] = torch.zeros_like(weights).index_add_(0, at, (rows[live] * dy[token]).sum(-1)).view(-1, k)
    return out


# ------------------------------------------------------------------------------------------------ work
def work(case):
    op, T = case["op"], case["T"]
    if op in ("experts", "linear"):
        K, N = case["K"], case["N"]
        if op == "linear":
            rows, matrices = T, 1
        else:   # of the rows there are, those that belong to an expert
            rows = max(1, round(T * case["k"] * (1 - case["drop"])))
            matrices = min(case["E"], rows)
        size = 4 if case["out"] == "fp32" else 2
        return {"bytes": 2 * rows * K + matrices * (N * K + 4 * N + (2 * N if case["bias"] else 0)) + size * rows * N, "flops": 2 * rows * K * N}
    k, H, E = case["k"], case["H"], case["E"]
    size = 4 if case["dtype"] == "fp32" else 2
    live = max(1, round(T * k * (1 - case["drop"])))
    if op == "sort":   # tokens read once, every row written; back: the rows that belong to a choice read, tokens written
        total = _rows_of(T, k, E, case["align"])
        moved = size * H * (T + total) + (8 if case["ids"] == "int64" else 4) * T * k + 4 * (E + 1 + T * k + total)
        return {"bytes": moved + (size * H * (live + T) if case["grad"] else 0), "flops": live * H if case["grad"] else 0}
    wsize = 4 if case["wdtype"] == "fp32" else 2
    moved = size * H * (live + T) + (wsize + 4) * T * k
    if not case["grad"]:
        return {"bytes": moved, "flops": 2 * live * H}
    total = _rows_of(T, k, E, case["align"])   # and dy, every row of the gradient, that of the weights
    return {"bytes": moved + size * H * (T + total) + wsize * T * k + 4 * total, "flops": 5 * live * H}
