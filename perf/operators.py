"""Operators of the MoE layer in 8 bits: the calls that performance is measured on, with their plain
forms and their values in 64 bits.

Six kinds of call, each through the package's public entry points:

  norm       ``add_rms_norm_int8``: the residual's addition and the root-mean-square norm at the
             layer's entry, with the 8-bit rows that the experts' product reads and the 16-bit rows
             that the router reads (serving)
  norm_step  ``add_rms_norm`` and its gradients (training)
  rows       ``quantize_rows(activation="gelu")``: GELU and 8 bits between the experts' two products
  linear     ``int8_linear``: every expert's product on its own rows, which it reads through the
             dispatch's reverse map (tokens) or in place (the second product)
  gelu_step  ``gelu_compress`` and ``gelu_compressed_backward``: the GELU of a training step whose
             input is held in 8 bits until the backward, which makes both the GELU again (for the
             second weights' gradient) and the gradient
  hold       ``compress_rows`` and ``restore_rows``: any activation held in 8 bits

Rows in 8 bits are returned as the values that they stand for, in the type of what they came from.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
PITCH = 128   # rows in 8 bits are padded with zeros to a multiple of this
BLOCK = 128   # columns of a held activation that share a scale
EPS = 1e-6


def _norm(kind, name, T, D, dtype):
    return {"name": name, "kind": kind, "T": T, "D": D, "dtype": dtype}


def _rows(kind, name, R, F, dtype):
    return {"name": name, "kind": kind, "R": R, "F": F, "dtype": dtype}


def _linear(name, T, k, E, K, N, dtype, gather=True, skew=0.0):
    return {"name": name, "kind": "linear", "T": T, "k": k, "E": E, "K": K, "N": N,
            "dtype": dtype, "gather": gather, "skew": skew}


def listed():
    return [
        # The layer's entry in one decoding step of a few sequences: latency.
        _norm("norm", "norm-decode", 8, 7168, "bf16"),
        # The same for a prompt.
        _norm("norm", "norm-prefill", 8192, 4096, "bf16"),
        # A training step at the widest hidden size.
        _norm("norm_step", "norm-step", 4096, 16384, "bf16"),
        # Odd everything.
        _norm("norm_step", "norm-odd-step", 3001, 1001, "fp16"),
        # Between the experts' products: a decoding step's 64 rows, and a prompt's.
        _rows("rows", "rows-decode", 64, 2048, "bf16"),
        _rows("rows", "rows-prefill", 49152, 2048, "bf16"),
        # First product of a decoding step: 64 rows over 256 experts, about one row for each.
        _linear("linear-decode", 8, 8, 256, 7168, 2048, "bf16"),
        # Second product of a few hundred tokens on one rank of 32 experts: packed rows in place.
        _linear("linear-rank", 256, 8, 32, 2048, 7168, "bf16", gather=False),
        # First product of a prompt.
        _linear("linear-prefill", 8192, 6, 64, 4096, 2048, "bf16"),
        # Odd everything, a few experts with most of the rows, one with none of them likely.
        _linear("linear-odd", 1501, 3, 13, 1001, 1003, "fp16", skew=2.0),
        # A training step's hidden rows: forward and backward of the held GELU.
        _rows("gelu_step", "gelu-step", 32768, 2048, "bf16"),
        # An odd activation held and restored.
        _rows("hold", "hold-odd", 9003, 1001, "fp16"),
    ]


def _log(rng, lo, hi):
    """An integer between lo and hi, spread evenly over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A row's length: usually a multiple of 64, sometimes of 8, sometimes any number."""
    d, p = _log(rng, lo, hi), rng.random()
    return d if p < 0.25 else max(8, d // 8 * 8) if p < 0.5 else max(64, d // 64 * 64)


def draw(rng):
    kind = rng.choice(["norm", "norm_step", "rows", "linear", "linear", "gelu_step", "hold"])
    c = {"kind": kind, "dtype": rng.choice(["bf16", "fp16"])}
    if kind in ("norm", "norm_step"):
        D = _width(rng, 256, 16384)
        c.update(T=_log(rng, 1, min(16384, (4096 * 16384) // D)), D=D)
        if kind == "norm_step" and rng.random() < 0.3:
            c.update(dtype="fp32", T=max(1, c["T"] // 2))
    elif kind in ("rows", "gelu_step", "hold"):
        F = _width(rng, 256, 16384)
        c.update(R=_log(rng, 1, min(65536, (32768 * 2048) // F)), F=F)
    else:
        E = _log(rng, 1, 256)
        k = rng.randint(1, min(8, E))
        K, N = _width(rng, 256, 8192), _width(rng, 256, 8192)
        E = max(k, min(E, (256 * 2048 * 7168) // (K * N)))
        most = 49152 * 4096 * 2048 // (K * N * k)  # no more products than the largest listed case
        skew = rng.choice([0.0, 0.0, 2.0])
        T = _log(rng, 1, max(1, min(2048 if skew else 8192, most)))
        c.update(k=k, E=E, K=K, N=N, T=T, gather=rng.random() < 0.5, skew=skew)
    return c


# ---- inputs ---------------------------------------------------------------------------------

def _pad(n):
    return -(-n // PITCH) * PITCH


def _activation(shape, dtype, gen):
    """~N(0, 1) with a few columns many times larger, as hidden states have them."""
    x = torch.randn(shape, generator=gen, device="cuda")
    loud = torch.rand(shape[-1], generator=gen, device="cuda") < 0.01
    return (x * torch.where(loud, 8.0, 1.0)).to(dtype)


def _int8(rows, width, gen):
    """Rows of whole values from a normal distribution, padded with zeros."""
    q = torch.randn(rows, _pad(width), generator=gen, device="cuda", dtype=torch.bfloat16)
    q = q.mul_(32).round_().clamp_(-127, 127).to(torch.int8)
    q[:, width:] = 0
    return q


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, kind = DTYPES[case["dtype"]], case["kind"]
    s = {"case": case, "dtype": dtype}
    if kind in ("norm", "norm_step"):
        shape = (case["T"], case["D"])
        s["x"], s["residual"] = _activation(shape, dtype, gen), _activation(shape, dtype, gen)
        s["weight"] = (1 + 0.1 * torch.randn(case["D"], generator=gen, device="cuda")).to(dtype)
        if kind == "norm_step":
            s["grad_y"] = torch.randn(shape, generator=gen, device="cuda").to(dtype)
            s["grad_h"] = torch.randn(shape, generator=gen, device="cuda").to(dtype)
            for name in ("x", "residual", "weight"):
                s[name].requires_grad_(True)
    elif kind in ("rows", "gelu_step", "hold"):
        shape = (case["R"], case["F"])
        s["x"] = _activation(shape, dtype, gen)
        if kind == "gelu_step":
            s["grad"] = torch.randn(shape, generator=gen, device="cuda").to(dtype)
    else:
        T, k, E, K, N = (case[n] for n in ("T", "k", "E", "K", "N"))
        logits = torch.randn(T, E, generator=gen, device="cuda")
        logits += case["skew"] * torch.randn(E, generator=gen, device="cuda")
        expert = torch.topk(logits, k, dim=-1).indices.reshape(-1)
        order = torch.argsort(expert, stable=True)
        counts = torch.bincount(expert, minlength=E)
        s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
        rows = T if case["gather"] else T * k
        s["index"] = order // k if case["gather"] else None  # the token of each packed row
        s["q"] = _int8(rows, K, gen)
        s["scales"] = torch.rand(rows, generator=gen, device="cuda") * 0.02 + 0.01
        s["weight"] = _int8(E * N, K, gen).view(E, N, _pad(K))
        s["weight_scales"] = torch.rand(E, N, generator=gen, device="cuda") * 2e-4 + 1e-4
        # what a program that runs the experts knows of its routing: the experts with rows, and for
        # each packed row which of them it belongs to and its place there
        host = counts.tolist()
        s["most"] = max(host)
        s["active"] = torch.tensor([e for e in range(E) if host[e]], device="cuda")
        sizes = counts[s["active"]]
        s["batch"] = torch.arange(len(sizes), device="cuda").repeat_interleave(sizes)
        s["place"] = torch.arange(T * k, device="cuda") - s["offsets"][s["active"]][s["batch"]]
        s["counts"] = host
    return s


# ---- plain forms: elementary operations in 32 bits, rounded once ----------------------------

def _plain_gelu(x):
    return 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))


def _plain_int8(v):
    """(whole values, scale of each row) of the last axis."""
    top = v.abs().amax(-1, keepdim=True)
    q = torch.where(top > 0, v * (127 / top), torch.zeros_like(v)).round()
    return q, top / 127


def _plain_blocks(x):
    """As _plain_int8, for blocks of the last axis; the values have their padding."""
    R, F = x.shape
    padded = x.new_zeros(R, -(-F // BLOCK) * BLOCK)
    padded[:, :F] = x
    return _plain_int8(padded.view(R, -1, BLOCK))


def _plain_norm(s):
    dtype = s["dtype"]
    h = (s["x"].detach().float() + s["residual"].detach().float()).to(dtype)
    rstd = torch.rsqrt(h.float().square().mean(-1, keepdim=True) + EPS)
    return h, rstd, h.float() * rstd * s["weight"].detach().float()


def _plain(s):
    case, dtype, kind = s["case"], s["dtype"], s["case"]["kind"]
    if kind == "norm":
        h, _, y = _plain_norm(s)
        q, scale = _plain_int8(y)
        return {"h": h, "y": y.to(dtype), "q": (q * scale).to(dtype), "scales": scale.view(-1)}
    if kind == "norm_step":
        h, rstd, y = _plain_norm(s)
        gy, hat = s["grad_y"].float(), h.float() * rstd
        t = gy * s["weight"].detach().float()
        gx = s["grad_h"].float() + rstd * (t - hat * (t * hat).mean(-1, keepdim=True))
        return {"h": h, "y": y.to(dtype), "grad_x": gx.to(dtype), "grad_residual": gx.to(dtype),
                "grad_weight": (gy * hat).sum(0).to(dtype)}
    if kind == "rows":
        q, scale = _plain_int8(_plain_gelu(s["x"].float()))
        return {"q": (q * scale).to(dtype), "scales": scale.view(-1)}
    if kind == "gelu_step":
        x = s["x"].float()
        q, scale = _plain_blocks(x)
        held = (q * scale).view(x.shape[0], -1)[:, :x.shape[1]]
        cdf = 0.5 * (1 + torch.erf(held * math.sqrt(0.5)))
        pdf = torch.exp(-0.5 * held * held) * (1 / math.sqrt(2 * math.pi))
        return {"a": _plain_gelu(x).to(dtype), "again": (held * cdf).to(dtype),
                "grad": (s["grad"].float() * (cdf + held * pdf)).to(dtype)}
    if kind == "hold":
        q, scale = _plain_blocks(s["x"].float())
        return {"x": (q * scale).view(case["R"], -1)[:, :case["F"]].to(dtype).contiguous(),
                "scales": scale.squeeze(-1)}
    # every expert that has rows, as one batch of products, each padded to the largest
    rows = s["q"] if s["index"] is None else s["q"][s["index"]]
    scales = s["scales"] if s["index"] is None else s["scales"][s["index"]]
    batch = torch.zeros(len(s["active"]), s["most"], rows.shape[1], device="cuda")
    batch[s["batch"], s["place"]] = rows.float()
    y = torch.matmul(batch, s["weight"][s["active"]].float().transpose(1, 2))
    y = y * s["weight_scales"][s["active"]].unsqueeze(1)
    return (y[s["batch"], s["place"]] * scales.unsqueeze(1)).to(dtype)


# ---- the framework's calls ------------------------------------------------------------------

def _kernels(s):
    import fastmoe_amd as fm

    case, dtype, kind = s["case"], s["dtype"], s["case"]["kind"]
    if kind == "norm":
        r = fm.add_rms_norm_int8(s["x"], s["weight"], s["residual"], eps=EPS)
        return {"h": r.residual, "y": r.normed, "q": r.rows.dequantize(dtype),
                "scales": r.rows.scales}
    if kind == "norm_step":
        y, h = fm.add_rms_norm(s["x"], s["weight"], s["residual"], eps=EPS)
        gx, gr, gw = torch.autograd.grad([y, h], [s["x"], s["residual"], s["weight"]],
                                         [s["grad_y"], s["grad_h"]])
        return {"h": h, "y": y, "grad_x": gx, "grad_residual": gr, "grad_weight": gw}
    if kind == "rows":
        r = fm.quantize_rows(s["x"], activation="gelu")
        return {"q": r.dequantize(dtype), "scales": r.scales}
    if kind == "gelu_step":
        a, held = fm.gelu_compress(s["x"])
        again, grad = fm.gelu_compressed_backward(held, s["grad"])
        return {"a": a, "again": again, "grad": grad}
    if kind == "hold":
        held = fm.compress_rows(s["x"])
        return {"x": fm.restore_rows(held, dtype), "scales": held.scales}
    return fm.int8_linear(fm.QuantizedRows(s["q"], s["scales"], case["K"]),
                          fm.Int8Weights(s["weight"], s["weight_scales"], case["K"]),
                          s["offsets"], rows=s["index"], out_dtype=dtype)


def run(state):
    return _kernels(state) if own else _plain(state)


# ---- what the path cannot do without --------------------------------------------------------

def work(case):
    b, kind = BYTES[case["dtype"]], case["kind"]
    if kind in ("norm", "norm_step"):
        n, D = case["T"] * case["D"], case["D"]
        if kind == "norm":  # x, residual, h, y; the 8-bit rows and their scales
            return {"bytes": n * (4 * b + 1) + 4 * case["T"] + b * D, "flops": 8 * n}
        return {"bytes": 8 * n * b + 2 * b * D, "flops": 20 * n}
    if kind in ("rows", "gelu_step", "hold"):
        n, blocks = case["R"] * case["F"], case["R"] * -(-case["F"] // BLOCK)
        if kind == "rows":
            return {"bytes": n * (b + 1) + 4 * case["R"], "flops": 20 * n}
        if kind == "gelu_step":  # h, a, held; held, grad, GELU again, grad
            return {"bytes": n * (5 * b + 2) + 8 * blocks, "flops": 50 * n}
        return {"bytes": n * (2 * b + 2) + 8 * blocks, "flops": 5 * n}
    T, k, E, K, N = (case[n] for n in ("T", "k", "E", "K", "N"))
    R = T * k
    # the experts that have rows, were the routing even
    active = E * (1 - (1 - k / E) ** T) if k < E else E
    return {"bytes": active * N * (K + 4) + (T if case["gather"] else R) * (K + 4) + R * N * b,
            "flops": 2 * R * N * K}


# ---- the same from the definitions, in 64 bits ----------------------------------------------

def _exact_cdf(x):
    return 0.5 * torch.erfc(-x / math.sqrt(2.0))


def _exact_held(v):
    """The values that 8 bits with one scale hold, and the scale."""
    scale = v.abs().max(dim=-1, keepdim=True).values / 127
    return torch.where(scale > 0, torch.round(v / scale), 0.0) * scale, scale


def _exact_blocks(x):
    parts = [_exact_held(x[:, c:c + BLOCK]) for c in range(0, x.shape[1], BLOCK)]
    return torch.cat([p[0] for p in parts], 1), torch.cat([p[1] for p in parts], 1)


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind in ("norm", "norm_step"):
        x, r, w = (s[n].detach().double() for n in ("x", "residual", "weight"))
        h = (x + r).to(s["dtype"]).double()  # the stream is normalised as it is stored
        norm = torch.sqrt((h * h).sum(-1, keepdim=True) / case["D"] + EPS)
        if kind == "norm":
            held, scale = _exact_held(h / norm * w)
            return {"h": h, "y": h / norm * w, "q": held, "scales": scale.view(-1)}
        gy, gh = s["grad_y"].double(), s["grad_h"].double()
        inner = (gy * w * h).sum(-1, keepdim=True)
        g = gh + gy * w / norm - h * inner / (case["D"] * norm ** 3)
        return {"h": h, "y": h / norm * w, "grad_x": g, "grad_residual": g,
                "grad_weight": (gy * h / norm).sum(0)}
    if kind == "rows":
        x = s["x"].double()
        held, scale = _exact_held(x * _exact_cdf(x))
        return {"q": held, "scales": scale.view(-1)}
    if kind == "gelu_step":
        x = s["x"].double()
        held = _exact_blocks(x)[0]
        slope = _exact_cdf(held) + held * torch.exp(-held ** 2 / 2) / math.sqrt(2 * math.pi)
        return {"a": x * _exact_cdf(x), "again": held * _exact_cdf(held),
                "grad": s["grad"].double() * slope}
    if kind == "hold":
        held, scale = _exact_blocks(s["x"].double())
        return {"x": held, "scales": scale}
    at = s["offsets"].tolist()
    out = torch.zeros(at[-1], case["N"], dtype=torch.float64, device="cuda")
    for e in range(case["E"]):
        if at[e + 1] > at[e]:
            here = torch.arange(at[e], at[e + 1], device="cuda")
            token = here if s["index"] is None else s["index"][here]
            x = s["q"][token].double() * s["scales"][token].double().unsqueeze(1)
            w = s["weight"][e].double() * s["weight_scales"][e].double().unsqueeze(1)
            out[here] = x @ w.t()
    return out
