"""Performance cases of the 8-bit integer layers and the routed experts: the
integer product with a scale per token and per channel, the linear layer that
quantizes its rows first, the same product over rows grouped by expert, and
tokens sorted by expert and back, with their gradients.

listed() names the fixed cases, draw(rng) gives one more of the same ranges,
prepare(case, seed) makes a case's inputs on the GPU, run(state) is one pass
(plain torch in 32 bits, or the library's operators where `own` is set),
work(case) the bytes and operations a pass cannot do without, and
exact(case, seed) the result in 64 bits.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"i32": torch.int32, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"i32": 4, "f32": 4, "f16": 2, "bf16": 2}

_lib = None


def library():
    """The front end's module and the process's context on GPU 0, which a program keeps."""
    global _lib
    if _lib is None:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, "cuda-zkml_amd"))
        import zkml_amd
        _lib = zkml_amd, zkml_amd.Context(0)
    return _lib


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one token through a square layer, weights and activations already in 8 bits: decoding
        {"name": "product 1x4096x4096", "kind": "product", "tokens": 1, "n_in": 4096, "n_out": 4096, "out": "bf16",
         "bias": False, "relu": False},
        # exact integer scores of a whole data set by the benchmark's 64 -> 32 layer
        {"name": "scores 100003x64x32", "kind": "product", "tokens": 100003, "n_in": 64, "n_out": 32, "out": "i32",
         "bias": False, "relu": False},
        # odd sizes in every direction, bias and ReLU applied
        {"name": "product 777x1001x1234", "kind": "product", "tokens": 777, "n_in": 1001, "n_out": 1234, "out": "f32",
         "bias": True, "relu": True},
        # the largest: a long prompt through a wide layer
        {"name": "product 8192x8192x8192", "kind": "product", "tokens": 8192, "n_in": 8192, "n_out": 8192,
         "out": "bf16", "bias": False, "relu": False},
        # one token, rows quantized within the call: latency
        {"name": "linear 1x8192x1024", "kind": "linear", "tokens": 1, "n_in": 8192, "n_out": 1024, "out": "f16",
         "bias": True, "relu": False},
        # an ordinary prompt, rows quantized within the call
        {"name": "linear 2048x4096x4096", "kind": "linear", "tokens": 2048, "n_in": 4096, "n_out": 4096,
         "out": "bf16", "bias": False, "relu": False},
        # five tokens in decoding, two experts each: almost every expert that runs has one row
        {"name": "experts 5x2 of 16", "kind": "experts", "tokens": 5, "slots": 2, "experts": 16, "n_in": 4096,
         "n_out": 2048, "out": "bf16", "bias": False, "relu": False, "dropped": 0.0},
        # a prompt over many small experts, bias and ReLU applied, unevenly filled
        {"name": "experts 4096x4 of 64", "kind": "experts", "tokens": 4096, "slots": 4, "experts": 64, "n_in": 2048,
         "n_out": 1024, "out": "f16", "bias": True, "relu": True, "dropped": 0.0},
        # a decoding batch sorted by expert: latency and launches
        {"name": "sort 33x2 of 8", "kind": "sort", "tokens": 33, "slots": 2, "experts": 8, "width": 1000,
         "type": "f32", "dropped": 0.0, "train": False},
        # a training batch with experts over capacity, the rows' gradient too
        {"name": "sort 16384x4 of 128", "kind": "sort", "tokens": 16384, "slots": 4, "experts": 128, "width": 2048,
         "type": "bf16", "dropped": 0.1, "train": True},
        # a decoding batch's answers put back
        {"name": "back 33x2", "kind": "back", "tokens": 33, "slots": 2, "experts": 8, "width": 1000, "type": "f32",
         "dropped": 0.0, "train": False},
        # a training batch put back, gradients of the rows and of the weights
        {"name": "back 16384x4", "kind": "back", "tokens": 16384, "slots": 4, "experts": 128, "width": 2048,
         "type": "bf16", "dropped": 0.1, "train": True},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["product", "product", "linear", "experts", "sort", "back"])
    if kind in ("product", "linear"):
        out = rng.choice(["f32", "f16", "bf16"] + (["i32"] if kind == "product" else []))
        layer = out != "i32"
        return {"kind": kind, "tokens": _log_uniform(rng, 1, 8192), "n_in": _log_uniform(rng, 16, 8192),
                "n_out": _log_uniform(rng, 16, 8192), "out": out, "bias": layer and rng.random() < 0.5,
                "relu": layer and rng.random() < 0.3}
    slots, experts = rng.choice([1, 2, 4, 8]), _log_uniform(rng, 8, 128)
    case = {"kind": kind, "slots": slots, "experts": experts, "dropped": rng.choice([0.0, 0.0, 0.1])}
    if kind == "experts":
        return dict(case, tokens=_log_uniform(rng, 1, 4096), n_in=_log_uniform(rng, 64, 4096),
                    n_out=_log_uniform(rng, 64, 4096), out=rng.choice(["f32", "f16", "bf16"]),
                    bias=rng.random() < 0.5, relu=rng.random() < 0.3)
    return dict(case, tokens=_log_uniform(rng, 1, 16384), width=_log_uniform(rng, 64, 4096),
                type=rng.choice(["f32", "f16", "bf16"]), train=rng.random() < 0.5)


# ------------------------------------------------------------------ inputs
def generator(case, seed):
    sizes = [case.get(k, 0) for k in ("tokens", "slots", "experts", "n_in", "n_out", "width")]
    h = seed
    for s in sizes:
        h = (h * 1000003 + s) % (1 << 61)
    return torch.Generator("cuda").manual_seed(h)


def normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def eight_bits(g, *shape):
    """What quantizing a normal row gives: up to 127, a third of them within 10."""
    return normal(g, *shape).mul_(32).round_().clamp_(-127, 127).to(torch.int8)


def scales(g, *shape):
    return torch.exp(normal(g, *shape) * 0.5 - 4)


def routes(case, g):
    """(expert, weight) of each token's slots: the largest of skewed gate
    scores, softmax weights, some pairs dropped (-1) for lack of room."""
    t, k, e = case["tokens"], case["slots"], case["experts"]
    gate = normal(g, t, e) + normal(g, e)
    top = torch.topk(gate, k, dim=1)
    expert = top.indices.to(torch.int32)
    if case["dropped"]:
        expert[torch.rand((t, k), generator=g, device="cuda") < case["dropped"]] = -1
    return expert.contiguous(), torch.softmax(top.values, dim=1).contiguous()


def sorted_pairs(expert, experts):
    """(offsets, order, place) of the pairs sorted by expert, as the sort defines them."""
    e = expert.reshape(-1).long()
    e = torch.where((e >= 0) & (e < experts), e, experts)
    order = torch.argsort(e, stable=True)
    counts = torch.bincount(e, minlength=experts + 1)[:experts]
    offsets = torch.zeros(experts + 1, dtype=torch.long, device=e.device)
    offsets[1:] = torch.cumsum(counts, 0)
    at = torch.arange(e.numel(), device=e.device)
    place = torch.empty_like(order)
    place[order] = at
    place = torch.where(e < experts, place, -1)
    order = torch.where(at < offsets[-1], order, -1)
    return offsets.to(torch.int32), order.to(torch.int32), place.to(torch.int32)


def prepare(case, seed):
    g, kind = generator(case, seed), case["kind"]
    st = {"case": case}
    if kind in ("product", "linear", "experts"):
        t, k, n = case["tokens"], case["n_in"], case["n_out"]
        lead = (case["experts"],) if kind == "experts" else ()
        st["w"], st["w_scale"] = eight_bits(g, *lead, n, k), scales(g, *lead, n)
        st["bias"] = normal(g, *lead, n) if case["bias"] else None
        if kind == "linear":
            st["x"] = (normal(g, t, k) * torch.exp(normal(g, t, 1))).to(TYPES[case["out"]])
        elif case["out"] == "i32":
            # pixels of 0 to 16, as the benchmark's quantized MLP takes them
            st["x"] = torch.randint(0, 17, (t, k), generator=g, device="cuda", dtype=torch.int8)
        else:
            st["x"], st["x_scale"] = eight_bits(g, t, k), scales(g, t)
        if kind == "experts":
            expert, _ = routes(case, g)
            st["offsets"], st["order"], _ = sorted_pairs(expert, case["experts"])
        return st
    t, s, h, dtype = case["tokens"], case["slots"], case["width"], TYPES[case["type"]]
    st["expert"], st["weight"] = routes(case, g)
    if kind == "sort":
        st["x"] = normal(g, t, h).to(dtype)
        st["grad"] = normal(g, t * s, h).to(dtype) if case["train"] else None
        return st
    st["offsets"], st["order"], st["place"] = sorted_pairs(st["expert"], case["experts"])
    st["y"] = normal(g, t * s, h).to(dtype)
    st["grad"] = normal(g, t, h).to(dtype) if case["train"] else None
    return st


# ------------------------------------------------------------------ plain form
def scaled(acc, case, x_scale, w_scale, bias):
    """The layer's epilogue on float sums."""
    y = acc * x_scale[:, None] * w_scale
    if bias is not None:
        y = y + bias
    return torch.clamp_min(y, 0) if case["relu"] else y


def plain_product(st):
    case, x, w = st["case"], st["x"], st["w"]
    if case["out"] == "i32":
        # exact in 32-bit floats: 4 bits of x at a time (15 * 127 * 8192 < 2^24)
        hi, wt = torch.div(x, 16, rounding_mode="floor"), w.float().t()
        return 16 * (hi.float() @ wt).to(torch.int32) + ((x - 16 * hi).float() @ wt).to(torch.int32)
    return scaled(x.float() @ w.float().t(), case, st["x_scale"], st["w_scale"], st["bias"]).to(TYPES[case["out"]])


def plain_linear(st):
    case, x = st["case"], st["x"].float()
    a = x.abs().amax(1)
    q = torch.where(a[:, None] > 0, torch.round(x * 127 / a[:, None]), 0.0)
    return scaled(q @ st["w"].float().t(), case, a / 127, st["w_scale"], st["bias"]).to(TYPES[case["out"]])


def plain_experts(st):
    """Rows padded to the fullest expert's count, one batched product."""
    case, order = st["case"], st["order"].long()
    rows, n = order.numel(), case["n_out"]
    token = order.clamp_min(0) // case["slots"]
    offsets = st["offsets"].long()
    p = torch.arange(rows, device="cuda")
    e = torch.searchsorted(offsets[1:], p, right=True).clamp_max(case["experts"] - 1)
    most = int((offsets[1:] - offsets[:-1]).max())
    used = order >= 0
    slot = torch.where(used, e * most + p - offsets[e], case["experts"] * most)
    padded = torch.zeros((case["experts"] * most + 1, case["n_in"]), device="cuda")
    padded[slot] = torch.where(used[:, None], st["x"][token].float(), 0.0)
    acc = torch.bmm(padded[:-1].view(case["experts"], most, -1), st["w"].float().transpose(1, 2).contiguous())
    acc = torch.cat([acc.view(-1, n), torch.zeros((1, n), device="cuda")])[slot]
    y = acc * st["x_scale"][token][:, None] * st["w_scale"][e]
    if case["bias"]:
        y = y + st["bias"][e]
    if case["relu"]:
        y = torch.clamp_min(y, 0)
    return torch.where(used[:, None], y, 0.0).to(TYPES[case["out"]])


def taken(y, place):
    """Rows of y by place, zeros for dropped pairs, in 32 bits: (tokens, slots, width)."""
    p = place.long()
    return torch.where((p >= 0)[..., None], y[p.clamp_min(0)].float(), 0.0)


def plain_sort(st):
    case = st["case"]
    offsets, order, place = sorted_pairs(st["expert"], case["experts"])
    o = order.long()
    rows = torch.where((o >= 0)[:, None], st["x"][o.clamp_min(0) // case["slots"]], 0.0).to(st["x"].dtype)
    out = {"offsets": offsets, "order": order, "place": place, "rows": rows}
    if case["train"]:
        out["grad_x"] = taken(st["grad"], place.view(-1, case["slots"])).sum(1).to(st["x"].dtype)
    return out


def plain_back(st):
    case, dtype = st["case"], st["y"].dtype
    y = taken(st["y"], st["place"].view(-1, case["slots"]))
    out = {"out": (y * st["weight"][..., None]).sum(1).to(dtype)}
    if case["train"]:
        g, o = st["grad"].float(), st["order"].long()
        pair = o.clamp_min(0)
        dy = st["weight"].view(-1)[pair][:, None] * g[pair // case["slots"]]
        out["grad_y"] = torch.where((o >= 0)[:, None], dy, 0.0).to(dtype)
        out["grad_weight"] = (y * g[:, None, :]).sum(2)
    return out


PLAIN = {"product": plain_product, "linear": plain_linear, "experts": plain_experts, "sort": plain_sort,
         "back": plain_back}


# ------------------------------------------------------------------ the library's operators
def stream(z):
    return torch.cuda.current_stream().cuda_stream or z.LEGACY_STREAM


def empty(*shape, dtype):
    return torch.empty(shape, dtype=dtype, device="cuda")


def own_layer(st):
    z, ctx = library()
    case, kind = st["case"], st["case"]["kind"]
    t, k, n, out = case["tokens"], case["n_in"], case["n_out"], case["out"]
    types = {"i32": z.I32, "f32": z.F32, "f16": z.F16, "bf16": z.BF16}
    more = {"bias": st["bias"], "relu": case["relu"], "stream": stream(z)}
    if kind == "linear":
        y = empty(t, n, dtype=TYPES[out])
        work = empty(ctx.i8_linear_work(t, k), dtype=torch.uint8)
        ctx.i8_linear(st["x"], types[out], st["w"], st["w_scale"], t, n, k, y, types[out], work, **more)
        return y
    if kind == "experts":
        rows = t * case["slots"]
        y = empty(rows, n, dtype=TYPES[out])
        ctx.i8_matmul_experts(st["x"], st["w"], st["offsets"], rows, case["experts"], n, k, y, types[out],
                              x_scale=st["x_scale"], w_scale=st["w_scale"], order=st["order"], slots=case["slots"],
                              tokens=t, **more)
        return y
    y = empty(t, n, dtype=TYPES[out])
    if out == "i32":
        ctx.i8_matmul(st["x"], st["w"], t, n, k, y, types[out], stream=stream(z))
    else:
        ctx.i8_matmul(st["x"], st["w"], t, n, k, y, types[out], x_scale=st["x_scale"], w_scale=st["w_scale"], **more)
    return y


def own_sort(st):
    z, ctx = library()
    case, x = st["case"], st["x"]
    t, s, e, h = case["tokens"], case["slots"], case["experts"], case["width"]
    dtype, on = {"f32": z.F32, "f16": z.F16, "bf16": z.BF16}[case["type"]], stream(z)
    offsets, order, place = (empty(m, dtype=torch.int32) for m in (e + 1, t * s, t * s))
    work = empty(ctx.experts_sort_work(t * s, e), dtype=torch.uint8)
    ctx.experts_sort(st["expert"], t * s, e, offsets, order, place, work, stream=on)
    out = {"offsets": offsets, "order": order, "place": place, "rows": empty(t * s, h, dtype=x.dtype)}
    ctx.experts_gather(x, dtype, h, order, t * s, t, s, out["rows"], stream=on)
    if case["train"]:
        out["grad_x"] = empty(t, h, dtype=x.dtype)
        ctx.experts_combine(st["grad"], dtype, h, place, t * s, t, s, out["grad_x"], stream=on)
    return out


def own_back(st):
    z, ctx = library()
    case, y = st["case"], st["y"]
    t, s, h = case["tokens"], case["slots"], case["width"]
    dtype, on = {"f32": z.F32, "f16": z.F16, "bf16": z.BF16}[case["type"]], stream(z)
    out = {"out": empty(t, h, dtype=y.dtype)}
    ctx.experts_combine(y, dtype, h, st["place"], t * s, t, s, out["out"], weight=st["weight"], stream=on)
    if case["train"]:
        out["grad_y"], out["grad_weight"] = torch.empty_like(y), empty(t, s, dtype=torch.float32)
        ctx.experts_combine_grad(st["grad"], y, dtype, h, st["order"], st["place"], st["weight"], t * s, t, s,
                                 out["grad_y"], out["grad_weight"], stream=on)
    return out


OWN = {"product": own_layer, "linear": own_layer, "experts": own_layer, "sort": own_sort, "back": own_back}


def run(st):
    return (OWN if own else PLAIN)[st["case"]["kind"]](st)


# ------------------------------------------------------------------ work
def work(case):
    kind, t = case["kind"], case["tokens"]
    if kind in ("product", "linear"):
        k, n = case["n_in"], case["n_out"]
        size = SIZE[case["out"]]
        x = t * k * (size if kind == "linear" else 1)
        scale = 0 if case["out"] == "i32" else 4 * n + (4 * t if kind == "product" else 0)
        return {"bytes": x + n * k + scale + t * n * size, "flops": 2 * t * n * k}
    rows = t * case["slots"]
    filled = rows * (1 - case["dropped"])
    if kind == "experts":
        # with this many rows, the experts that have any (evenly spread routes)
        e = case["experts"] * (1 - (1 - 1 / case["experts"]) ** filled)
        k, n = case["n_in"], case["n_out"]
        return {"bytes": t * (k + 4) + e * n * (k + 4) + rows * (n * SIZE[case["out"]] + 4),
                "flops": 2 * filled * n * k}
    size, h = SIZE[case["type"]], case["width"]
    if kind == "sort":
        moved = (t + rows) * h * size + 4 * (3 * rows + case["experts"] + 1)
        return {"bytes": moved + ((filled + t) * h * size if case["train"] else 0),
                "flops": filled * h if case["train"] else 0}
    moved, flops = (filled + t) * h * size + 8 * rows, 2 * filled * h
    if case["train"]:
        moved, flops = moved + (t + rows) * h * size + 8 * rows, flops + 3 * filled * h
    return {"bytes": moved, "flops": flops}


# ------------------------------------------------------------------ in 64 bits
def exact_layer(case, x, x_scale, w, w_scale, bias):
    y = x @ w.double().t()
    if case["out"] == "i32":
        return y.round().to(torch.int32)
    y = y * (x_scale.double()[:, None] * w_scale.double()[None, :])
    if bias is not None:
        y = y + bias.double()
    return torch.where(y > 0, y, 0.0) if case["relu"] else y


def exact(case, seed):
    st, kind = prepare(case, seed), case["kind"]
    if kind == "product":
        return exact_layer(case, st["x"].double(), st.get("x_scale"), st["w"], st["w_scale"], st["bias"])
    if kind == "linear":
        x = st["x"].double()
        a = x.abs().max(dim=1).values
        q = torch.round(127 * x / torch.where(a > 0, a, 1.0)[:, None])
        return exact_layer(case, q, a / 127, st["w"], st["w_scale"], st["bias"])
    slots = case["slots"]
    if kind == "experts":
        at, order = st["offsets"].tolist(), st["order"].long()
        y = torch.zeros((order.numel(), case["n_out"]), dtype=torch.float64, device="cuda")
        for e in range(case["experts"]):
            token = order[at[e]:at[e + 1]] // slots
            if token.numel():
                y[at[e]:at[e + 1]] = exact_layer(case, st["x"][token].double(), st["x_scale"][token], st["w"][e],
                                                 st["w_scale"][e], st["bias"][e] if case["bias"] else None)
        return y
    # each pair's position counted one expert at a time
    expert, pairs = st["expert"].view(-1), case["tokens"] * slots
    place, order = torch.full((pairs,), -1, device="cuda"), torch.full((pairs,), -1, device="cuda")
    offsets, n = [0], 0
    for e in range(case["experts"]):
        mine = torch.nonzero(expert == e).view(-1)
        place[mine] = torch.arange(n, n + mine.numel(), device="cuda")
        order[n:n + mine.numel()] = mine
        n += mine.numel()
        offsets.append(n)
    pair = order[:n]
    if kind == "sort":
        rows = torch.zeros((pairs, case["width"]), dtype=torch.float64, device="cuda")
        rows[:n] = st["x"].double()[pair // slots]
        out = {"offsets": torch.tensor(offsets, dtype=torch.int32), "order": order.to(torch.int32),
               "place": place.to(torch.int32), "rows": rows}
        if case["train"]:
            out["grad_x"] = torch.zeros_like(rows[:case["tokens"]])
            out["grad_x"].index_add_(0, pair // slots, st["grad"][:n].double())
        return out
    y, weight = st["y"][:n].double(), st["weight"].view(-1).double()[pair]
    back = torch.zeros((case["tokens"], case["width"]), dtype=torch.float64, device="cuda")
    back.index_add_(0, pair // slots, y * weight[:, None])
    out = {"out": back}
    if case["train"]:
        g = st["grad"].double()[pair // slots]
        out["grad_y"] = torch.zeros((pairs, case["width"]), dtype=torch.float64, device="cuda")
        out["grad_y"][:n] = g * weight[:, None]
        dw = torch.zeros(pairs, dtype=torch.float64, device="cuda")
        dw[pair] = (g * y).sum(1)
        out["grad_weight"] = dw.view(-1, slots)
    return out
