"""Operators of the MoE block: the calls that performance is measured on, with their plain forms and
their values in 64 bits.

Five kinds of call, each through the package's public entry points:

  route          ``route_tokens``: scores, a bias for balance, groups, top-k and weights (serving)
  route_step     the same with the gradient of the router's logits (training)
  fp4            ``fp4_linear``: every expert's product of 16-bit rows with weights in 4 bits that have a
                 scale for 32 of them, the rows read through the dispatch's reverse map or in place, with
                 the bias and GELU between the experts' two products (serving)
  sandwich       ``sandwich_norm``: the norm after a block, its gate and residual scale, the addition
                 to the stream, and the norm before the next block (serving)
  sandwich_step  the same with its gradients (training)
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
PITCH = 128   # columns that a row of weights in 4 bits is padded to, with zeros
BLOCK = 32    # weights that share a scale
EPS = 1e-6
FP4 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]  # magnitudes of the eight codes; the fourth bit is the sign


def _route(kind, name, T, E, k, dtype, score, bias=False, groups=1, top_groups=1, group_score="max",
           renormalize=True, scale=1.0, masked=0):
    return {"name": name, "kind": kind, "T": T, "E": E, "k": k, "dtype": dtype, "score": score,
            "bias": bias, "groups": groups, "top_groups": top_groups, "group_score": group_score,
            "renormalize": renormalize, "scale": scale, "masked": masked}


def _fp4(name, T, k, E, K, N, dtype, gather=True, skew=0.0, gelu=False, bias=False):
    return {"name": name, "kind": "fp4", "T": T, "k": k, "E": E, "K": K, "N": N, "dtype": dtype,
            "gather": gather, "skew": skew, "gelu": gelu, "bias": bias}


def _sandwich(kind, name, T, D, dtype, gates=0, scale=1.0):
    return {"name": name, "kind": kind, "T": T, "D": D, "dtype": dtype, "gates": gates, "scale": scale}


def listed():
    return [
        # A decoding step of a few sequences over 256 experts in groups, with the bias: latency.
        _route("route", "route-decode", 8, 256, 8, "fp32", "sigmoid", bias=True, groups=8, top_groups=4,
               group_score="top2", scale=2.5),
        # The same router over a long prompt.
        _route("route", "route-prefill", 32768, 256, 8, "fp32", "sigmoid", bias=True, groups=8,
               top_groups=4, group_score="top2", scale=2.5),
        # A training step of a softmax router whose weights keep their share of all experts.
        _route("route_step", "route-step", 32768, 64, 6, "bf16", "softmax", renormalize=False),
        # Odd everything; some experts masked out.
        _route("route_step", "route-odd-step", 3001, 60, 5, "fp16", "softmax", groups=6, top_groups=3,
               masked=7),
        # First product of a single token over 256 experts: eight of them are read.
        _fp4("fp4-token", 1, 8, 256, 7168, 2048, "bf16", gelu=True),
        # Second product of a few hundred tokens on one rank of 32 experts: packed rows in place.
        _fp4("fp4-rank", 256, 8, 32, 2048, 7168, "bf16", gather=False),
        # First product of a prompt.
        _fp4("fp4-prefill", 8192, 6, 64, 4096, 2048, "bf16", gelu=True),
        # Odd everything, a few experts with most of the rows, one with none of them likely.
        _fp4("fp4-odd", 1501, 3, 13, 1001, 1003, "fp16", skew=2.0, bias=True),
        # Between two blocks in one decoding step of a few sequences: latency.
        _sandwich("sandwich", "sandwich-decode", 8, 7168, "bf16", gates=1),
        # The same for a prompt.
        _sandwich("sandwich", "sandwich-prefill", 8192, 4096, "bf16", gates=1),
        # A training step at the widest hidden size, with a constant scale.
        _sandwich("sandwich_step", "sandwich-step", 4096, 16384, "bf16", scale=0.25),
        # Odd everything, and a gate for each of three sequences.
        _sandwich("sandwich_step", "sandwich-odd-step", 3003, 1001, "fp16", gates=3),
    ]


def _log(rng, lo, hi):
    """An integer between lo and hi, spread evenly over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A row's length: usually a multiple of 64, sometimes of 8, sometimes any number."""
    d, p = _log(rng, lo, hi), rng.random()
    return d if p < 0.25 else max(8, d // 8 * 8) if p < 0.5 else max(64, d // 64 * 64)


def draw(rng):
    kind = rng.choice(["route", "route_step", "fp4", "fp4", "sandwich", "sandwich_step"])
    if kind in ("route", "route_step"):
        groups = rng.choice([1, 1, 2, 4, 6, 8])
        E = groups * _log(rng, 2, 512 // groups)
        top_groups = rng.randint(1, groups)
        k = rng.randint(1, min(8, top_groups * (E // groups)))
        T = _log(rng, 1, min(32768, 32768 * 256 // (2 * E)))
        return _route(kind, None, T, E, k, rng.choice(["bf16", "fp16", "fp32"]),
                      rng.choice(["softmax", "sigmoid"]), rng.random() < 0.5, groups, top_groups,
                      rng.choice(["max", "top2"]), rng.random() < 0.7, rng.choice([1.0, 2.5]),
                      rng.choice([0, 0, E // 3]))
    dtype = rng.choice(["bf16", "fp16"])
    if kind == "fp4":
        E = _log(rng, 1, 256)
        k = rng.randint(1, min(8, E))
        K, N = _width(rng, 256, 8192), _width(rng, 256, 8192)
        E = max(k, min(E, (256 * 2048 * 7168) // (K * N)))
        most = 49152 * 4096 * 2048 // (K * N * k)  # no more products than the largest listed case
        skew = rng.choice([0.0, 0.0, 2.0])
        T = _log(rng, 1, max(1, min(2048 if skew else 8192, most)))
        return _fp4(None, T, k, E, K, N, dtype, rng.random() < 0.5, skew, rng.random() < 0.5,
                    rng.random() < 0.3)
    D = _width(rng, 256, 16384)
    T = _log(rng, 1, min(16384, (4096 * 16384) // D))
    gates = rng.choice([0, 1, rng.randint(2, 9)])
    if gates:
        T = -(-T // gates) * gates if T >= gates else gates
    if kind == "sandwich_step" and rng.random() < 0.3:
        dtype, T = "fp32", max(1, gates, T // 2 // max(1, gates) * max(1, gates))
    return _sandwich(kind, None, T, D, dtype, gates, rng.choice([1.0, 0.25]))


# ---- inputs ---------------------------------------------------------------------------------

def _pad(n):
    return -(-n // PITCH) * PITCH


def _activation(shape, dtype, gen):
    """~N(0, 1) with a few columns many times larger, as hidden states have them."""
    x = torch.randn(shape, generator=gen, device="cuda")
    loud = torch.rand(shape[-1], generator=gen, device="cuda") < 0.01
    return (x * torch.where(loud, 8.0, 1.0)).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, kind = DTYPES[case["dtype"]], case["kind"]
    s = {"case": case, "dtype": dtype}

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    if kind in ("route", "route_step"):
        T, E, k = case["T"], case["E"], case["k"]
        logits = 1.5 * randn(T, E) + 0.5 * randn(E)
        if case["masked"]:  # experts that some tokens may not take
            away = torch.rand(T, E, generator=gen, device="cuda") < case["masked"] / E
            logits.masked_fill_(away, float("-inf"))
        s["logits"] = logits.to(dtype)
        s["bias"] = 0.05 * randn(E) if case["bias"] else None
        if kind == "route_step":
            s["logits"].requires_grad_(True)
            s["grad"] = randn(T, k).to(dtype)
    elif kind == "fp4":
        T, k, E, K, N = (case[n] for n in ("T", "k", "E", "K", "N"))
        logits = randn(T, E) + case["skew"] * randn(E)
        expert = torch.topk(logits, k, dim=-1).indices.reshape(-1)
        order = torch.argsort(expert, stable=True)
        counts = torch.bincount(expert, minlength=E)
        s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
        s["index"] = order // k if case["gather"] else None  # the token of each packed row
        s["x"] = _activation((T if case["gather"] else T * k, K), dtype, gen)
        # two codes a byte, the earlier column in the low half
        s["weight"] = torch.randint(0, 256, (E, N, _pad(K) // 2), generator=gen, device="cuda",
                                    dtype=torch.uint8)
        s["weight"][..., -(-K // 2):] = 0
        if K % 2:
            s["weight"][..., K // 2] &= 15
        # exponents of two, 127 of them standing for one
        s["weight_scales"] = torch.randint(117, 122, (E, N, _pad(K) // BLOCK), generator=gen,
                                           device="cuda", dtype=torch.uint8)
        s["bias"] = 0.1 * randn(E, N).to(dtype) if case["bias"] else None
        # what a program that runs the experts knows of its routing: the experts with rows, and for
        # each packed row which of them it belongs to and its place there
        host = counts.tolist()
        s["most"] = max(host)
        s["active"] = torch.tensor([e for e in range(E) if host[e]], device="cuda")
        sizes = counts[s["active"]]
        s["batch"] = torch.arange(len(sizes), device="cuda").repeat_interleave(sizes)
        s["place"] = torch.arange(T * k, device="cuda") - s["offsets"][s["active"]][s["batch"]]
    else:
        T, D = case["T"], case["D"]
        s["x"], s["residual"] = _activation((T, D), dtype, gen), _activation((T, D), dtype, gen)
        s["post"], s["pre"] = ((1 + 0.1 * randn(D)).to(dtype) for _ in range(2))
        s["gate"] = (0.5 + 0.2 * randn(case["gates"], D)).to(dtype) if case["gates"] else None
        if kind == "sandwich_step":
            s["grad_y"], s["grad_h"] = randn(T, D).to(dtype), randn(T, D).to(dtype)
            for name in ("x", "residual", "post", "pre", "gate"):
                if s[name] is not None:
                    s[name].requires_grad_(True)
    return s


# ---- plain forms: elementary operations in 32 bits, rounded once ----------------------------

def _choose(choice, case):
    """The k best of each row, the best first and the lowest index first among equals, in the groups
    whose best (or two best) choices are highest."""
    T, E, G = case["T"], case["E"], case["groups"]
    if G > 1:
        per = choice.view(T, G, E // G)
        best = torch.sort(per, dim=-1, descending=True).values
        two = case["group_score"] == "top2" and E // G > 1
        score = best[..., 0] + best[..., 1] if two else best[..., 0]
        kept = torch.sort(score, dim=-1, descending=True, stable=True).indices[:, :case["top_groups"]]
        stays = torch.zeros(T, G, dtype=torch.bool, device=choice.device).scatter_(1, kept, True)
        ranked = torch.sort(choice, dim=-1, descending=True, stable=True).indices
        left_out = ~stays.gather(1, ranked // (E // G))
        order = torch.sort(left_out.to(torch.int8), dim=-1, stable=True).indices
        return ranked.gather(1, order[:, :case["k"]])
    return torch.sort(choice, dim=-1, descending=True, stable=True).indices[:, :case["k"]]


def _by_score(case):
    """Where a bias or a sum of two enters, the scores themselves are compared; else they rank experts
    as the logits do."""
    return case["bias"] or (case["groups"] > 1 and case["group_score"] == "top2")


def _plain_route(s):
    case = s["case"]
    logits = s["logits"].detach().double()  # scores next to a border decide: in 64 bits, kept in 32
    if case["score"] == "sigmoid":
        score = torch.sigmoid(logits)
    else:  # where the mask leaves no expert, none has a share
        empty = torch.isneginf(logits).all(-1, keepdim=True)
        score = torch.softmax(logits.masked_fill(empty, 0.0), -1).masked_fill(empty, 0.0)
    choice = logits.float()
    if _by_score(case):
        choice = score.float() if s["bias"] is None else score.float() + s["bias"]
    ids = _choose(choice, case)
    w = score.gather(1, ids)
    if case["renormalize"]:
        total = w.sum(-1, keepdim=True)
        w = torch.where(total > 0, w / total, torch.zeros_like(w))
    return score, ids, w


def _plain_sandwich(s):
    dtype, case = s["dtype"], s["case"]
    x, r, post, pre = (s[n].detach().float() for n in ("x", "residual", "post", "pre"))
    cx = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    hat = x * cx
    g = torch.full((1, case["D"]), case["scale"], device=x.device)
    if s["gate"] is not None:
        g = s["gate"].detach().float() * case["scale"]
    g = g.repeat_interleave(case["T"] // g.shape[0], 0) if g.shape[0] > 1 else g
    h = (r + g * (hat * post)).to(dtype)
    ch = torch.rsqrt(h.float().square().mean(-1, keepdim=True) + EPS)
    return cx, hat, post, g, h, ch, pre


def _plain(s):
    case, dtype, kind = s["case"], s["dtype"], s["case"]["kind"]
    if kind in ("route", "route_step"):
        score, ids, w = _plain_route(s)
        out = {"weights": (w * case["scale"]).to(dtype), "ids": ids}
        if kind == "route_step":
            g = s["grad"].double() * case["scale"]
            taken = score.gather(1, ids)
            slope = 1 - taken if case["score"] == "sigmoid" else torch.ones_like(taken)
            grad = torch.zeros_like(score)
            if case["renormalize"]:
                grad.scatter_(1, ids, w * slope * (g - (g * w).sum(-1, keepdim=True)))
            elif case["score"] == "sigmoid":
                grad.scatter_(1, ids, g * taken * slope)
            else:
                grad.scatter_(1, ids, g)
                grad = score * (grad - (g * taken).sum(-1, keepdim=True))
            out["grad"] = grad.to(dtype)
        return out
    if kind == "fp4":
        return _plain_fp4(s)
    cx, hat, post, g, h, ch, pre = _plain_sandwich(s)
    hhat = h.float() * ch
    out = {"h": h, "y": (hhat * pre).to(dtype)}
    if kind == "sandwich":
        return out
    gy = s["grad_y"].float()
    t = gy * pre
    gh = s["grad_h"].float() + ch * (t - hhat * (t * hhat).mean(-1, keepdim=True))
    gn = gh * g
    t = gn * post
    gx = cx * (t - hat * (t * hat).mean(-1, keepdim=True))
    out.update(grad_x=gx.to(dtype), grad_residual=gh.to(dtype), grad_post=(gn * hat).sum(0).to(dtype),
               grad_pre=(gy * hhat).sum(0).to(dtype))
    if s["gate"] is not None:
        gg = (gh * hat * post * case["scale"]).view(case["gates"], -1, case["D"]).sum(1)
        out["grad_gate"] = gg.to(dtype)
    return out


def _fp4_values(s, which):
    """The weights of some experts in 32 bits, with their padding."""
    codes = s["weight"][which]
    pair = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()
    table = torch.tensor(FP4 + [-v for v in FP4], device=codes.device)
    scale = torch.ldexp(torch.ones((), device=codes.device), s["weight_scales"][which].int() - 127)
    return (table[pair].unflatten(-1, (-1, BLOCK)) * scale.unsqueeze(-1)).flatten(-2)


def _plain_fp4(s):
    # every expert that has rows, as one batch of products, each padded to the largest
    case = s["case"]
    x = s["x"] if s["index"] is None else s["x"][s["index"]]
    batch = torch.zeros(len(s["active"]), s["most"], case["K"], device="cuda")
    batch[s["batch"], s["place"]] = x.float()
    w = _fp4_values(s, s["active"])[..., :case["K"]]
    y = torch.matmul(batch, w.transpose(1, 2).contiguous())
    if s["bias"] is not None:
        y = y + s["bias"][s["active"]].float().unsqueeze(1)
    y = y[s["batch"], s["place"]]
    if case["gelu"]:
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    return y.to(s["dtype"])


# ---- the framework's calls ------------------------------------------------------------------

def _kernels(s):
    import fastmoe_amd as fm

    case, dtype, kind = s["case"], s["dtype"], s["case"]["kind"]
    if kind in ("route", "route_step"):
        routing = fm.Routing(score=case["score"], groups=case["groups"], top_groups=case["top_groups"],
                             group_score=case["group_score"], renormalize=case["renormalize"],
                             scale=case["scale"])
        w, ids = fm.route_tokens(s["logits"], case["k"], routing, bias=s["bias"])
        if kind == "route":
            return {"weights": w, "ids": ids}
        (grad,) = torch.autograd.grad(w, s["logits"], s["grad"])
        return {"weights": w, "ids": ids, "grad": grad}
    if kind == "fp4":
        return fm.fp4_linear(s["x"], fm.Fp4Weights(s["weight"], s["weight_scales"], case["K"]),
                             s["offsets"], rows=s["index"], bias=s["bias"],
                             activation="gelu" if case["gelu"] else None, out_dtype=dtype)
    y, h = fm.sandwich_norm(s["x"], s["post"], s["residual"], s["pre"], gate=s["gate"],
                            scale=case["scale"], eps=EPS)
    if kind == "sandwich":
        return {"h": h, "y": y}
    names = ["x", "residual", "post", "pre"] + (["gate"] if s["gate"] is not None else [])
    grads = torch.autograd.grad([y, h], [s[n] for n in names], [s["grad_y"], s["grad_h"]])
    return {"h": h, "y": y, **{"grad_" + n: g for n, g in zip(names, grads)}}


def run(state):
    return _kernels(state) if own else _plain(state)


# ---- what the path cannot do without --------------------------------------------------------

def work(case):
    b, kind = BYTES[case["dtype"]], case["kind"]
    if kind in ("route", "route_step"):
        n, slots = case["T"] * case["E"], case["T"] * case["k"]
        if kind == "route":
            return {"bytes": n * b + slots * (b + 8), "flops": 20 * n}
        return {"bytes": 2 * n * b + slots * (2 * b + 8), "flops": 30 * n}
    if kind == "fp4":
        T, k, E, K, N = (case[n] for n in ("T", "k", "E", "K", "N"))
        R = T * k
        # the experts that have rows, were the routing even
        active = E * (1 - (1 - k / E) ** T) if k < E else E
        weights = active * N * (-(-K // 2) + -(-K // BLOCK))
        return {"bytes": weights + (T if case["gather"] else R) * K * b + R * N * b,
                "flops": 2 * R * N * K}
    n, D = case["T"] * case["D"], case["D"]
    parameters = (2 + case["gates"]) * D * b
    if kind == "sandwich":  # x, residual, h, y
        return {"bytes": 4 * n * b + parameters, "flops": 12 * n}
    # and grad_y, grad_h, x, h; grad_x, grad_residual
    return {"bytes": 10 * n * b + 2 * parameters, "flops": 40 * n}


# ---- the same from the definitions, in 64 bits ----------------------------------------------

def _exact_route(s):
    case = s["case"]
    T, E, G = case["T"], case["E"], case["groups"]
    l = s["logits"].detach().double()
    if case["score"] == "sigmoid":
        score = 1 / (1 + torch.exp(-l))
    else:
        e = torch.exp(l - l.max(-1, keepdim=True).values.clamp_min(-1e300))
        score = e / e.sum(-1, keepdim=True).clamp_min(1e-300)  # nothing left: no shares
    choice = l.clone()
    if _by_score(case):  # scores are kept, and the bias added, in 32 bits
        choice = score.float()
        choice = (choice if s["bias"] is None else choice + s["bias"]).double()
    if G > 1:
        left, total = choice.view(T, G, -1).clone(), 0
        for _ in range(2 if case["group_score"] == "top2" and E > G else 1):
            top, at = left.max(-1, keepdim=True)
            total = top if isinstance(total, int) else (total + top).float().double()
            left.scatter_(-1, at, float("-inf"))
        total = total.squeeze(-1)
        place = torch.arange(G, device=l.device)
        ahead = (total.unsqueeze(1) > total.unsqueeze(2)) | (
            (total.unsqueeze(1) == total.unsqueeze(2)) & (place.view(1, 1, G) < place.view(1, G, 1)))
        allowed = (ahead.sum(-1) < case["top_groups"]).repeat_interleave(E // G, 1)
    else:
        allowed = torch.ones_like(choice, dtype=torch.bool)
    picked = []
    lowest = torch.arange(E, device=l.device)
    for _ in range(case["k"]):
        top = choice.masked_fill(~allowed, float("-inf")).max(-1, keepdim=True).values
        first = torch.where(allowed & (choice == top), lowest, E).min(-1, keepdim=True).values
        picked.append(first)
        allowed = allowed.scatter(1, first, False)
    return score, torch.cat(picked, 1)


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind in ("route", "route_step"):
        score, ids = _exact_route(s)
        if kind == "route":
            part = torch.take_along_dim(score, ids, 1)
            if case["renormalize"]:
                part = torch.nan_to_num(part / part.sum(-1, keepdim=True), nan=0.0)
            return {"weights": part * case["scale"], "ids": ids}
        # the gradient by differentiating the definition
        l = s["logits"].detach().double().requires_grad_(True)
        if case["renormalize"]:
            chosen = torch.take_along_dim(l, ids, 1)
            if case["score"] == "sigmoid":
                part = torch.sigmoid(chosen)
                w = part / part.sum(-1, keepdim=True)
            else:
                w = torch.softmax(chosen, -1)
        else:
            every = torch.sigmoid(l) if case["score"] == "sigmoid" else torch.softmax(l, -1)
            w = torch.take_along_dim(every, ids, 1)
        w = w * case["scale"]
        (grad,) = torch.autograd.grad(w, l, s["grad"].double())
        if case["renormalize"] and case["k"] == 1:
            grad = torch.zeros_like(grad)  # one share is whole, whatever the logits
        # where every expert that is taken (or that there is) is masked, 0 / 0 stands for no weight
        which = torch.take_along_dim(l.detach(), ids, 1) if case["renormalize"] else l.detach()
        none = torch.isneginf(which).all(-1, keepdim=True)
        w, grad = w.masked_fill(none, 0.0), grad.masked_fill(none, 0.0)
        return {"weights": w.detach(), "ids": ids, "grad": grad}
    if kind == "fp4":
        at = s["offsets"].tolist()
        out = torch.zeros(at[-1], case["N"], dtype=torch.float64, device="cuda")
        for e in range(case["E"]):
            if at[e + 1] > at[e]:
                here = torch.arange(at[e], at[e + 1], device="cuda")
                token = here if s["index"] is None else s["index"][here]
                y = s["x"][token].double() @ _exact_fp4(s, e)[:, :case["K"]].t()
                if s["bias"] is not None:
                    y += s["bias"][e].double()
                out[here] = y * 0.5 * torch.erfc(-y / math.sqrt(2.0)) if case["gelu"] else y
        return out
    with torch.enable_grad():
        return _exact_sandwich(s)


def _exact_fp4(s, e):
    """Expert e's weights from the format: sign, two bits of exponent, one of mantissa."""
    out = torch.empty(*s["weight"][e].shape, 2, dtype=torch.float64, device="cuda")
    for half in range(2):
        code = s["weight"][e].long() // 16 ** half % 16
        sign, exponent, mantissa = 1.0 - 2.0 * (code // 8), code // 2 % 4, code % 2
        out[..., half] = sign * torch.where(exponent > 0, (2.0 + mantissa) * 2.0 ** (exponent - 2.0),
                                            mantissa * 0.5)
    block = 2.0 ** (s["weight_scales"][e].double() - 127)
    return out.flatten(1) * block.repeat_interleave(BLOCK, 1)


def _exact_sandwich(s):
    case, D = s["case"], s["case"]["D"]
    names = ["x", "residual", "post", "pre"] + (["gate"] if s["gate"] is not None else [])
    d = {n: s[n].detach().double().requires_grad_(True) for n in names}

    def norm(v, w):
        return v / torch.sqrt((v * v).sum(-1, keepdim=True) / D + EPS) * w

    term = norm(d["x"], d["post"]) * case["scale"]
    if "gate" in d:
        gates = case["gates"]
        term = (term.view(gates, -1, D) * d["gate"].view(gates, 1, D)).view(-1, D)
    h = d["residual"] + term
    # the stream is normalised as it is stored; its rounding has the slope one
    stored = h + (h.detach().to(s["dtype"]).double() - h.detach())
    y = norm(stored, d["pre"])
    out = {"h": h.detach(), "y": y.detach()}
    if case["kind"] == "sandwich_step":
        grads = torch.autograd.grad([y, h], list(d.values()), [s["grad_y"].double(), s["grad_h"].double()])
        out.update({"grad_" + n: g for n, g in zip(names, grads)})
    return out
