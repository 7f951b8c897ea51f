"""Performance cases of the layers with 4-bit weights and of the experts' router:
the product of 8-bit rows with 4-bit weights and a scale per group, the linear
layer that quantizes its rows first, the same product over rows grouped by
expert, the choice of each token's experts with their weights, and the balance
loss with the experts' counts, with their gradients.

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

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i32": torch.int32}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i32": 4}

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
        # one token through a square layer whose activations are in 8 bits already: decoding
        {"name": "product 1x4096x4096", "kind": "product", "tokens": 1, "n_in": 4096, "n_out": 4096, "group": 128,
         "scale": "f16", "out": "bf16", "bias": False, "relu": False},
        # a few tokens, odd sizes, small groups, bias and ReLU applied
        {"name": "product 3x1001x1234", "kind": "product", "tokens": 3, "n_in": 1001, "n_out": 1234, "group": 32,
         "scale": "f32", "out": "f32", "bias": True, "relu": True},
        # a decoding batch through a wide layer
        {"name": "product 48x8192x8192", "kind": "product", "tokens": 48, "n_in": 8192, "n_out": 8192, "group": 128,
         "scale": "bf16", "out": "bf16", "bias": False, "relu": False},
        # the largest: a long prompt through a wide layer
        {"name": "product 4096x8192x8192", "kind": "product", "tokens": 4096, "n_in": 8192, "n_out": 8192,
         "group": 128, "scale": "f16", "out": "bf16", "bias": False, "relu": False},
        # one token, its row quantized within the call: latency
        {"name": "linear 1x8192x1024", "kind": "linear", "tokens": 1, "n_in": 8192, "n_out": 1024, "group": 128,
         "scale": "f16", "out": "f16", "bias": True, "relu": False},
        # an ordinary prompt, rows quantized within the call
        {"name": "linear 777x4096x4096", "kind": "linear", "tokens": 777, "n_in": 4096, "n_out": 4096, "group": 64,
         "scale": "f16", "out": "bf16", "bias": False, "relu": False},
        # five tokens in decoding, two experts each: almost every expert that runs has one row
        {"name": "experts 5x2 of 16", "kind": "experts", "tokens": 5, "slots": 2, "experts": 16, "n_in": 4096,
         "n_out": 2048, "group": 128, "scale": "f16", "out": "bf16", "bias": False, "relu": False, "dropped": 0.0},
        # a prompt over many small experts, bias and ReLU applied, unevenly filled
        {"name": "experts 2048x4 of 64", "kind": "experts", "tokens": 2048, "slots": 4, "experts": 64, "n_in": 2048,
         "n_out": 1024, "group": 128, "scale": "f16", "out": "f16", "bias": True, "relu": True, "dropped": 0.0},
        # a decoding batch routed by a gate's integer scores: latency
        {"name": "route 33 to 2 of 8", "kind": "route", "tokens": 33, "slots": 2, "experts": 8, "type": "i32",
         "renormalize": True, "train": False},
        # a training batch routed, its balance loss, and the gradient of both
        {"name": "route 16384 to 8 of 128", "kind": "route", "tokens": 16384, "slots": 8, "experts": 128,
         "type": "bf16", "renormalize": False, "train": True},
        # the balance of a small batch whose routes are given, some dropped for lack of room
        {"name": "balance 500x2 of 60", "kind": "balance", "tokens": 500, "slots": 2, "experts": 60, "type": "f32",
         "dropped": 0.1},
        # the balance of a large batch over many experts
        {"name": "balance 32768x4 of 256", "kind": "balance", "tokens": 32768, "slots": 4, "experts": 256,
         "type": "bf16", "dropped": 0.0},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["product", "product", "linear", "experts", "route", "balance"])
    if kind in ("product", "linear", "experts"):
        case = {"kind": kind, "group": rng.choice([32, 64, 128, 128, 256]), "scale": rng.choice(["f32", "f16", "bf16"]),
                "out": rng.choice(["f32", "f16", "bf16"]), "bias": rng.random() < 0.5, "relu": rng.random() < 0.3}
        if kind != "experts":
            return dict(case, tokens=_log_uniform(rng, 1, 4096), n_in=_log_uniform(rng, 32, 8192),
                        n_out=_log_uniform(rng, 32, 8192))
        return dict(case, tokens=_log_uniform(rng, 1, 2048), slots=rng.choice([1, 2, 4, 8]),
                    experts=_log_uniform(rng, 8, 64), n_in=_log_uniform(rng, 64, 4096),
                    n_out=_log_uniform(rng, 64, 2048), dropped=rng.choice([0.0, 0.0, 0.1]))
    case = {"kind": kind, "tokens": _log_uniform(rng, 1, 32768), "slots": rng.choice([1, 2, 4, 8]),
            "experts": _log_uniform(rng, 8, 256)}
    if kind == "balance":
        return dict(case, type=rng.choice(["f32", "f16", "bf16"]), dropped=rng.choice([0.0, 0.1]))
    train = rng.random() < 0.5
    return dict(case, type=rng.choice(["f32", "f16", "bf16"] + ([] if train else ["i32"])),
                renormalize=rng.random() < 0.5, train=train)


# ------------------------------------------------------------------ inputs
def generator(case, seed):
    sizes = [case.get(k, 0) for k in ("tokens", "slots", "experts", "n_in", "n_out", "group")]
    h = seed
    for s in sizes:
        h = (h * 1000003 + s) % (1 << 61)
    return torch.Generator("cuda").manual_seed(h)


def normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def empty(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="cuda")


def four_bits(g, rows, n_in):
    """Weights as quantizing normal ones by groups gives them, packed: each run of
    128 of a row is 64 bytes, byte b weight b (low four bits) and weight 64 + b."""
    runs = (n_in + 127) // 128
    q = torch.zeros((rows, runs * 128), dtype=torch.int8, device="cuda")
    q[:, :n_in] = normal(g, rows, n_in).mul_(2.6).round_().clamp_(-8, 7).to(torch.int8)
    q = q.view(rows, runs, 2, 64)
    return ((q[:, :, 0] & 15) | (q[:, :, 1] << 4)).view(rows, runs * 64).contiguous()


def scores_of(case, g):
    """A gate's scores, some experts preferred: floats, or integer sums."""
    t, e = case["tokens"], case["experts"]
    s = normal(g, t, e) * 1.5 + normal(g, e) * 0.5
    return (s * 4096).round_().to(torch.int32) if case["type"] == "i32" else s.to(TYPES[case["type"]])


def softmax_scale(case):
    return 1 / 4096 if case["type"] == "i32" else 1.0


def best(scores, slots):
    """The experts of the `slots` largest scores, of equal ones the first; -1 beyond their number."""
    order = torch.sort(scores, dim=1, descending=True, stable=True).indices[:, :slots]
    return torch.nn.functional.pad(order, (0, slots - order.shape[1]), value=-1)


def sorted_pairs(expert, experts):
    """(offsets, order) of the pairs sorted by expert, as the sort defines them."""
    e = expert.reshape(-1).long()
    e = torch.where((e >= 0) & (e < experts), e, experts)
    order = torch.argsort(e, stable=True)
    offsets = torch.zeros(experts + 1, dtype=torch.long, device=e.device)
    offsets[1:] = torch.cumsum(torch.bincount(e, minlength=experts + 1)[:experts], 0)
    order = torch.where(torch.arange(e.numel(), device=e.device) < offsets[-1], order, -1)
    return offsets.to(torch.int32), order.to(torch.int32)


def prepare(case, seed):
    g, kind, t = generator(case, seed), case["kind"], case["tokens"]
    st = {"case": case}
    if kind in ("product", "linear", "experts"):
        k, n = case["n_in"], case["n_out"]
        e = case["experts"] if kind == "experts" else 1
        groups = (k + case["group"] - 1) // case["group"]
        st["w"] = four_bits(g, e * n, k)
        st["w_scale"] = torch.exp(normal(g, e, groups, n) * 0.3 - 3).to(TYPES[case["scale"]])
        st["bias"] = normal(g, e, n) if case["bias"] else None
        if kind == "linear":
            st["x"] = (normal(g, t, k) * torch.exp(normal(g, t, 1))).to(TYPES[case["out"]])
        else:
            st["x"] = normal(g, t, k).mul_(32).round_().clamp_(-127, 127).to(torch.int8)
            st["x_scale"] = torch.exp(normal(g, t) * 0.5 - 4)
        rows = t
        if kind == "experts":
            rows = t * case["slots"]
            gate = normal(g, t, e) + normal(g, e)
            expert = best(gate, case["slots"]).to(torch.int32)
            if case["dropped"]:
                expert[torch.rand(expert.shape, generator=g, device="cuda") < case["dropped"]] = -1
            st["offsets"], st["order"] = sorted_pairs(expert, e)
        st["y"] = empty(rows, n, dtype=TYPES[case["out"]])
        return st
    s, e = case["slots"], case["experts"]
    st["scores"] = scores_of(case, g)
    if kind == "route":
        st["expert"], st["weight"] = empty(t, s, dtype=torch.int32), empty(t, s)
        st["grad_weight"] = normal(g, t, s) if case["train"] else None
    else:
        st["expert"] = best(st["scores"].float(), s).to(torch.int32).contiguous()
        if case["dropped"]:
            st["expert"][torch.rand((t, s), generator=g, device="cuda") < case["dropped"]] = -1
    if kind == "balance" or case["train"]:
        st["count"], st["prob"], st["loss"] = empty(e + 1, dtype=torch.int32), empty(e), empty(1)
        st["grad_loss"] = torch.full((1,), 0.01, device="cuda")
        st["grad_scores"] = torch.empty_like(st["scores"])
    return st


# ------------------------------------------------------------------ plain form
def weights_of(st):
    """The weights in 32-bit floats, [experts *] n_out x n_in."""
    case = st["case"]
    k, n, b = case["n_in"], case["n_out"], st["w"]
    low = b & 15
    low = low - 16 * (low > 7).to(torch.int8)
    q = torch.cat([low.view(b.shape[0], -1, 64), (b >> 4).view(b.shape[0], -1, 64)], 2)
    q = q.view(-1, n, q.shape[1] * 128)[:, :, :k]
    scale = st["w_scale"].float().transpose(1, 2).repeat_interleave(case["group"], dim=2)[:, :, :k]
    return q.float() * scale


def finished(y, case, bias):
    if bias is not None:
        y = y + bias
    return torch.clamp_min(y, 0) if case["relu"] else y


def plain_product(st):
    case = st["case"]
    y = (st["x"].float() @ weights_of(st)[0].t()) * st["x_scale"][:, None]
    return finished(y, case, st["bias"]).to(TYPES[case["out"]])


def plain_linear(st):
    case, x = st["case"], st["x"].float()
    a = x.abs().amax(1, keepdim=True)
    q = torch.where(a > 0, torch.round(x * 127 / a), 0.0)
    return finished((q @ weights_of(st)[0].t()) * (a / 127), case, st["bias"]).to(TYPES[case["out"]])


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
    acc = torch.bmm(padded[:-1].view(case["experts"], most, -1), weights_of(st).transpose(1, 2).contiguous())
    acc = torch.cat([acc.view(-1, n), torch.zeros((1, n), device="cuda")])[slot]
    y = finished(acc * st["x_scale"][token][:, None], case, st["bias"][e] if case["bias"] else None)
    return torch.where(used[:, None], y, 0.0).to(TYPES[case["out"]])


def probabilities(st):
    """Softmax over a token's experts.  (Differences of integer scores are exact first.)"""
    s = st["scores"] if st["case"]["type"] == "i32" else st["scores"].float()
    z = torch.exp((s - s.amax(1, keepdim=True)).float() * softmax_scale(st["case"]))
    return z / z.sum(1, keepdim=True)


def named(expert):
    """(slots that name an expert, indexes to gather by)."""
    return expert >= 0, expert.clamp_min(0).long()


def plain_balance(p, expert, st):
    """Counts (and the number of tokens), mean probabilities, loss, and the loss's
    gradient with regard to the scaled scores."""
    t, s, e = (st["case"][k] for k in ("tokens", "slots", "experts"))
    on, index = named(expert)
    count = torch.zeros(e, device="cuda").index_add_(0, index.view(-1), on.view(-1).float())
    prob, f = p.sum(0) / t, count / (t * s)
    loss = (e * (f * prob).sum()).view(1)
    dz = st["grad_loss"] * (e / t) * p * (f - (p * f).sum(1, keepdim=True))
    count = torch.cat([count, torch.full((1,), t, device="cuda")]).to(torch.int32)
    return {"count": count, "prob": prob, "loss": loss}, dz


def plain_route(st):
    case, p = st["case"], probabilities(st)
    expert = best(st["scores"], case["slots"])
    on, index = named(expert)
    w = torch.where(on, p.gather(1, index), 0.0)
    if case["renormalize"]:
        w = w / w.sum(1, keepdim=True)
    out = {"expert": expert.to(torch.int32), "weight": w}
    if case["train"]:
        more, dz = plain_balance(p, expert, st)
        gw = torch.where(on, st["grad_weight"], 0.0)
        inner = w * (gw - (gw * w).sum(1, keepdim=True))
        if not case["renormalize"]:
            # what softmax's gradient takes from every expert is taken from the others too
            dz = dz - p * (gw * w).sum(1, keepdim=True)
            inner = gw * w
        dz = dz.scatter_add(1, index, torch.where(on, inner, 0.0))
        out.update(more, grad_scores=(dz * softmax_scale(case)).to(TYPES[case["type"]]))
    return out


def plain_given(st):
    out, dz = plain_balance(probabilities(st), st["expert"], st)
    return dict(out, grad_scores=(dz * softmax_scale(st["case"])).to(TYPES[st["case"]["type"]]))


PLAIN = {"product": plain_product, "linear": plain_linear, "experts": plain_experts, "route": plain_route,
         "balance": plain_given}


# ------------------------------------------------------------------ the library's operators
def stream(z):
    return torch.cuda.current_stream().cuda_stream or z.LEGACY_STREAM


def workspace(st, size):
    """A program's own buffer for a call of these sizes, kept."""
    if st.get("work") is None or st["work"].numel() < size:
        st["work"] = empty(max(size, 16), dtype=torch.uint8)
    return st["work"]


def own_layer(st):
    z, ctx = library()
    case, kind, y = st["case"], st["case"]["kind"], st["y"]
    t, k, n, group = case["tokens"], case["n_in"], case["n_out"], case["group"]
    types = {"f32": z.F32, "f16": z.F16, "bf16": z.BF16}
    out, more = types[case["out"]], {"scale_type": types[case["scale"]], "bias": st["bias"], "relu": case["relu"],
                                     "stream": stream(z)}
    if kind == "linear":
        ctx.i4_linear(st["x"], out, st["w"], st["w_scale"], t, n, k, group, y, out,
                      workspace(st, ctx.i4_linear_work(t, k)), **more)
    elif kind == "experts":
        ctx.i4_matmul_experts(st["x"], st["w"], st["w_scale"], st["offsets"], t * case["slots"], case["experts"], n, k,
                              group, y, out, x_scale=st["x_scale"], order=st["order"], slots=case["slots"], tokens=t,
                              **more)
    else:
        ctx.i4_matmul(st["x"], st["w"], st["w_scale"], t, n, k, group, y, out, x_scale=st["x_scale"], **more)
    return y


def own_router(st):
    z, ctx = library()
    case, scores, expert, on = st["case"], st["scores"], st["expert"], stream(z)
    t, s, e = case["tokens"], case["slots"], case["experts"]
    kind = {"f32": z.F32, "f16": z.F16, "bf16": z.BF16, "i32": z.I32}[case["type"]]
    more = {"scale": softmax_scale(case), "stream": on}
    out, balance = {}, {}
    if case["kind"] == "balance" or case["train"]:
        balance = {k: st[k] for k in ("count", "prob", "loss")}
        work = workspace(st, ctx.experts_route_work(t, e))
    if case["kind"] == "route":
        more["renormalize"] = case["renormalize"]
        out = {"expert": expert, "weight": st["weight"]}
        if not case["train"]:
            ctx.experts_route(scores, kind, t, e, s, expert, st["weight"], **more)
            return out
        ctx.experts_route(scores, kind, t, e, s, expert, st["weight"], work=work, **balance, **more)
        more["grad_weight"] = st["grad_weight"]
    else:
        ctx.experts_balance(scores, kind, t, e, s, expert, work=work, **balance, **more)
    ctx.experts_route_grad(scores, kind, t, e, s, expert, st["grad_scores"], count=st["count"],
                           grad_loss=st["grad_loss"], **more)
    return dict(out, **balance, grad_scores=st["grad_scores"])


OWN = {"product": own_layer, "linear": own_layer, "experts": own_layer, "route": own_router, "balance": own_router}


def run(st):
    return (OWN if own else PLAIN)[st["case"]["kind"]](st)


# ------------------------------------------------------------------ work
def work(case):
    kind, t = case["kind"], case["tokens"]
    if kind in ("product", "linear", "experts"):
        k, n = case["n_in"], case["n_out"]
        weights = n * (k / 2 + (k + case["group"] - 1) // case["group"] * SIZE[case["scale"]]
                       + (4 if case["bias"] else 0))
        size = SIZE[case["out"]]
        x = t * (k * size if kind == "linear" else k + 4)
        if kind != "experts":
            return {"bytes": x + weights + t * n * size, "flops": 2 * t * n * k}
        rows = t * case["slots"]
        filled = rows * (1 - case["dropped"])
        # with this many rows, the experts that have any (evenly spread routes)
        e = case["experts"] * (1 - (1 - 1 / case["experts"]) ** filled)
        return {"bytes": x + e * weights + rows * (n * size + 4), "flops": 2 * filled * n * k}
    s, e, size = case["slots"], case["experts"], SIZE[case["type"]]
    scores, pairs = t * e * size, t * s
    if kind == "route" and not case["train"]:
        return {"bytes": scores + 8 * pairs, "flops": 3 * t * e}
    # forward reads the scores once; backward reads them again and writes their gradient
    moved = 3 * scores + 4 * pairs + 8 * e + (12 * pairs if kind == "route" else 4 * pairs)
    return {"bytes": moved, "flops": 12 * t * e}


# ------------------------------------------------------------------ in 64 bits
def exact_weights(case, packed, scale):
    """n_out x n_in weights of one expert, a run of 128 at a time."""
    k, n = case["n_in"], case["n_out"]
    b = packed.view(torch.uint8).to(torch.int64)
    q = torch.empty((n, b.shape[1] * 2), dtype=torch.float64, device="cuda")
    for r in range(b.shape[1] // 64):
        part = b[:, 64 * r:64 * r + 64]
        q[:, 128 * r:128 * r + 64] = ((part % 16 + 8) % 16 - 8).double()
        q[:, 128 * r + 64:128 * r + 128] = ((part // 16 + 8) % 16 - 8).double()
    return q[:, :k] * scale.double()[torch.arange(k, device="cuda") // case["group"]].t()


def exact_layer(case, x, x_scale, w, bias):
    y = (x @ w.t()) * x_scale.double()[:, None]
    if bias is not None:
        y = y + bias.double()
    return torch.where(y > 0, y, 0.0) if case["relu"] else y


def exact(case, seed):
    st, kind = prepare(case, seed), case["kind"]
    if kind in ("product", "linear"):
        x = st["x"].double()
        x_scale = st.get("x_scale")
        if kind == "linear":
            a = x.abs().max(dim=1).values
            x = torch.round(127 * x / torch.where(a > 0, a, 1.0)[:, None])
            x_scale = a / 127
        return exact_layer(case, x, x_scale, exact_weights(case, st["w"], st["w_scale"][0]),
                           st["bias"][0] if case["bias"] else None)
    slots, experts, t = case["slots"], case["experts"], case["tokens"]
    if kind == "experts":
        at, order = st["offsets"].tolist(), st["order"].long()
        y = torch.zeros((order.numel(), case["n_out"]), dtype=torch.float64, device="cuda")
        w = st["w"].view(experts, case["n_out"], -1)
        for e in range(experts):
            token = order[at[e]:at[e + 1]] // slots
            if token.numel():
                y[at[e]:at[e + 1]] = exact_layer(case, st["x"][token].double(), st["x_scale"][token],
                                                 exact_weights(case, w[e], st["w_scale"][e]),
                                                 st["bias"][e] if case["bias"] else None)
        return y
    z = st["scores"].double() * softmax_scale(case)
    p = torch.softmax(z, dim=1)
    out, dz = {}, torch.zeros_like(p)
    if kind == "route":
        # one slot after the other: the largest that is left, the first of equal ones
        left, at = st["scores"].double(), torch.arange(t, device="cuda")
        index = torch.arange(experts, device="cuda")
        chosen, w = [], []
        for _ in range(slots):
            top = left.max(dim=1, keepdim=True).values
            e = torch.where(left == top, index, experts).min(dim=1).values
            some = top[:, 0] > -math.inf
            e = torch.where(some, e, -1)
            chosen.append(e)
            w.append(torch.where(some, p[at, e.clamp_min(0)], 0.0))
            left = torch.where(index == e[:, None], -math.inf, left)
        expert, w = torch.stack(chosen, 1), torch.stack(w, 1)
        total = w.sum(1, keepdim=True)
        out = {"expert": expert.to(torch.int32), "weight": w / total if case["renormalize"] else w}
        if not case["train"]:
            return out
        gw = st["grad_weight"].double()
        for j in range(slots):
            # d weight_j / d score of every expert, one slot at a time
            on = (expert[:, j] >= 0)[:, None]
            mine = (index == expert[:, j:j + 1]).double()
            d = w[:, j:j + 1] * (mine - p)
            if case["renormalize"]:
                among = torch.zeros_like(p)
                for i in range(slots):
                    hit = (index == expert[:, i:i + 1]).double()
                    among += hit * w[:, i:i + 1]
                d = w[:, j:j + 1] / total * (mine - among / total)
            dz += torch.where(on, gw[:, j:j + 1] * d, 0.0)
    else:
        expert = st["expert"]
    count = torch.stack([(expert == e).sum() for e in range(experts)])
    f, prob = count.double() / (t * slots), p.mean(0)
    gl = st["grad_loss"].double()
    dz += gl * experts / t * p * (f[None] - (p @ f)[:, None])
    out.update(count=torch.cat([count, count.new_tensor([t])]).to(torch.int32), prob=prob,
               loss=(experts * (f @ prob)).view(1), grad_scores=dz * softmax_scale(case))
    return out
