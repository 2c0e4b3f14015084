"""Performance cases of the operators in front of a block's linears and experts.

A case is one call (with gradients where it trains) that a transformer's forward
makes before its quantized linears or its mixture of experts:

  choose    a router's logits -> the experts of each token and their weights:
            softmax or sigmoid scores, a bias for balance, groups, renormalized
  norm      root-mean-square norm, with the residual's addition in front
  norm8     the same norm, rotated and quantized to 8 bits with a scale for each
            row, as the 8-bit linears take it, and read back as 16-bit values

Activations are N(0, 1) with 1% of the channels scaled by 20, logits N(0, 2^2)
over a taste of the router's own.
"""
from __future__ import annotations

import importlib
import math

import torch

own = False

_PKG = "comfyui-int4-convrot-rdna4_amd"
_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_ES = {"bf16": 2, "f16": 2, "f32": 4}
_EPS = 1e-6


def _choose(name, T, E, k, dtype="bf16", scoring="softmax", bias=False, groups=1, top_groups=1, group_score="max",
            renormalize=True, scale=1.0, masked=False, grad=False):
    return {"name": name, "kind": "choose", "T": T, "E": E, "k": k, "dtype": dtype, "scoring": scoring, "bias": bias,
            "groups": groups, "top_groups": top_groups, "group_score": group_score, "renormalize": renormalize,
            "scale": scale, "masked": masked, "grad": grad}


def _norm(name, M, D, dtype="bf16", weight="bf16", residual=True, grad=False):
    return {"name": name, "kind": "norm", "M": M, "D": D, "dtype": dtype, "weight": weight, "residual": residual,
            "grad": grad}


def _norm8(name, M, D, G=256, dtype="bf16", residual=True):
    return {"name": name, "kind": "norm8", "M": M, "D": D, "G": G, "dtype": dtype, "weight": dtype, "residual": residual}


def listed():
    return [
        # one token through a router of few experts: launch latency
        _choose("choose_t1", 1, 32, 4),
        # a serving step's few tokens, balanced sigmoid scores in groups
        _choose("choose_groups_t16", 16, 256, 8, scoring="sigmoid", bias=True, groups=8, top_groups=4, group_score="sum2",
                scale=2.5),
        # an odd number of tokens and of experts, single precision, softmax as it is, some experts away, with gradients
        _choose("choose_odd_f32_t3001", 3001, 100, 6, dtype="f32", renormalize=False, masked=True, grad=True),
        # a training step's tokens over many experts in groups, with gradients
        _choose("choose_train_t16384", 16384, 256, 8, scoring="sigmoid", bias=True, groups=8, top_groups=4,
                group_score="sum2", scale=2.5, grad=True),
        # one token between two blocks: launch latency
        _norm("norm_m1", 1, 5120),
        # an odd width, fp16, no residual
        _norm("norm_odd_f16_m777", 777, 1605, dtype="f16", weight="f16", residual=False),
        # a training step's tokens with gradients
        _norm("norm_train_m8192", 8192, 4096, weight="f32", grad=True),
        # a large image's tokens between two blocks
        _norm("norm_image_m16384", 16384, 5120),
        # one token in front of its 8-bit linears
        _norm8("norm8_m1", 1, 5120),
        # an odd number of tokens, 64-wide rotation groups, fp16, no residual
        _norm8("norm8_ragged_f16_m777", 777, 1600, G=64, dtype="f16", residual=False),
        # a prompt's tokens
        _norm8("norm8_text_m512", 512, 4096),
        # an image's tokens
        _norm8("norm8_image_m8192", 8192, 5120),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same ranges: 1 to 16384 tokens, 8 to 256 experts with 1 to 8 a token, rows of 64 to 13824, every
    type and rotation group, with and without bias, groups, residual and gradients."""
    kind = rng.choice(("choose", "norm", "norm8"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if kind == "choose":
        groups = rng.choice((1, 1, 2, 4, 8))
        E = max(1, _log_int(rng, 8, 256) // groups) * groups
        top_groups = rng.randint(1, groups)
        k = rng.randint(1, min(8, E // groups * top_groups))
        scoring = rng.choice(("softmax", "sigmoid"))
        case = _choose("", _log_int(rng, 1, 16384), E, k, dtype, scoring, rng.random() < 0.5, groups, top_groups,
                       rng.choice(("max", "sum2")), rng.random() < 0.7, rng.choice((1.0, 1.0, 2.5)), rng.random() < 0.3,
                       rng.random() < 0.5)
        if dtype == "f32":
            case["T"] = max(1, case["T"] // 2)
    elif kind == "norm":
        M, D = _log_int(rng, 1, 16384), _log_int(rng, 64, 13824)
        if rng.random() < 0.6:
            D = max(64, D // 64 * 64)
        case = _norm("", M, D, dtype, rng.choice((dtype, "f32")), rng.random() < 0.6, rng.random() < 0.5)
        share = (2 if case["grad"] else 1) * (2 if dtype == "f32" else 1)
        while share * case["M"] * D > 16384 * 5120:
            case["M"] = max(1, case["M"] // 2)
    else:
        G = rng.choice((16, 64, 256, 256))
        unit = G if rng.random() < 0.5 else 256
        case = _norm8("", _log_int(rng, 1, 16384), max(1, _log_int(rng, 256, 13824) // unit) * unit, G, dtype,
                      rng.random() < 0.6)
        while (2 if dtype == "f32" else 1) * case["M"] * case["D"] > 8192 * 5120:
            case["M"] = max(1, case["M"] // 2)
    del case["name"]
    return case


# --------------------------------------------------------------------------
# inputs (made from the seed alone, on the GPU)
# --------------------------------------------------------------------------

def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + salt) % (1 << 62))
    return g


def _randn(shape, seed, salt):
    return torch.randn(shape, generator=_gen(seed, salt), device="cuda")


def _activations(M, D, dtype, seed, salt):
    x = _randn((M, D), seed, salt)
    channels = torch.randperm(D, generator=_gen(seed, 100), device="cuda")[:max(1, round(0.01 * D))]
    x[:, channels] *= 20.0
    return x.to(_DT[dtype])


def prepare(case, seed):
    kind, dtype = case["kind"], _DT[case["dtype"]]
    s = {"case": case}
    if kind == "choose":
        T, E = case["T"], case["E"]
        logits = 2.0 * _randn((T, E), seed, 1) + 0.7 * _randn((E,), seed, 2)
        if case["masked"]:           # experts of a group that is not reached, one in sixteen
            away = torch.randperm(E, generator=_gen(seed, 3), device="cuda")[:max(1, E // 16)]
            if E - away.numel() >= case["k"]:
                logits[:, away] = -math.inf
        s["logits"] = logits.to(dtype)
        # what steps of 0.001 towards the mean load leave
        s["bias"] = torch.randint(-100, 101, (E,), generator=_gen(seed, 4), device="cuda") * 0.001 if case["bias"] else None
        if case["grad"]:
            s["logits"].requires_grad_(True)
            s["d_weights"] = _randn((T, case["k"]), seed, 5)
        return s
    M, D = case["M"], case["D"]
    s["x"] = _activations(M, D, case["dtype"], seed, 1)
    s["residual"] = (4.0 * _randn((M, D), seed, 2)).to(dtype) if case["residual"] else None
    s["weight"] = (1.0 + 0.2 * _randn((D,), seed, 3)).to(_DT[case["weight"]])
    if kind == "norm" and case["grad"]:
        for name in ("x", "residual", "weight"):
            if s[name] is not None:
                s[name].requires_grad_(True)
        s["d_y"] = _randn((M, D), seed, 6).to(dtype)
        s["d_h"] = _randn((M, D), seed, 7).to(dtype) if case["residual"] else None
    return s


# --------------------------------------------------------------------------
# the plain forms, in 32 bits; in 64 what decides between neighbours (the order
# of experts, the nearest 8-bit code)
# --------------------------------------------------------------------------

def _greatest(v, n):
    """Indexes of the n greatest along the last axis, greatest first, ties to the lowest index."""
    return torch.sort(v, dim=-1, descending=True, stable=True).indices[..., :n]


def _plain_choose(s):
    c, logits = s["case"], s["logits"].detach()
    T, E, k = c["T"], c["E"], c["k"]
    wide = logits.to(torch.float64)
    if c["scoring"] == "softmax":
        e = torch.exp(wide - wide.amax(dim=-1, keepdim=True))
        scores = e / e.sum(dim=-1, keepdim=True)
    else:
        scores = 1.0 / (1.0 + torch.exp(-wide))
    choice = scores if s["bias"] is None else scores + s["bias"].to(torch.float64)
    choice = torch.where(wide == -math.inf, -math.inf, choice)
    if c["groups"] > 1:
        parts = choice.reshape(T, c["groups"], E // c["groups"])
        group = parts.amax(dim=-1)
        if c["group_score"] == "sum2" and parts.shape[-1] > 1:
            two = torch.sort(parts, dim=-1, descending=True).values[..., :2]
            group = torch.where(two[..., 1] == -math.inf, two[..., 0], two.sum(dim=-1))
        kept = torch.zeros_like(group, dtype=torch.bool).scatter_(1, _greatest(group, c["top_groups"]), True)
        choice = torch.where(kept[..., None], parts, -math.inf).reshape(T, E)
    ids = _greatest(choice, k)
    there = choice.gather(1, ids) > -math.inf
    picked = torch.where(there, scores.gather(1, ids), 0.0).to(torch.float32)
    total = picked.sum(dim=-1, keepdim=True)
    p = picked / torch.where(total > 0, total, 1.0) if c["renormalize"] else picked
    out = {"ids": torch.where(there, ids, -1).to(torch.int32), "weights": p * c["scale"]}
    if c["grad"]:
        g = s["d_weights"] * c["scale"]
        mean = (p * g).sum(dim=-1, keepdim=True)
        if c["scoring"] == "sigmoid":
            d = p * (1.0 - picked) * (g - mean if c["renormalize"] else g)
        else:
            d = p * (g - mean) if c["renormalize"] else p * g
        d_logits = torch.zeros((T, E), device=logits.device).scatter_(1, ids, torch.where(there, d, 0.0))
        if c["scoring"] == "softmax" and not c["renormalize"]:
            d_logits = d_logits - scores.to(torch.float32) * mean
        out["d_logits"] = d_logits.to(logits.dtype)
    return out


def _sum_kept(s):
    """The stream as it is kept: x, or x + residual in its type."""
    x, r = s["x"].detach(), s["residual"]
    return x if r is None else (x.to(torch.float32) + r.detach().to(torch.float32)).to(x.dtype)


def _plain_norm(s):
    c, kept = s["case"], _sum_kept(s)
    h, w = kept.to(torch.float32), s["weight"].detach().to(torch.float32)
    rstd = 1.0 / torch.sqrt((h * h).mean(dim=-1, keepdim=True) + _EPS)
    out = {"y": (h * rstd * w).to(kept.dtype)}
    if c["residual"]:
        out["h"] = kept
    if c["grad"]:
        dy = s["d_y"].to(torch.float32)
        g, n = dy * w, h * rstd
        d = rstd * (g - n * (g * n).mean(dim=-1, keepdim=True))
        if c["residual"]:
            d = d + s["d_h"].to(torch.float32)
        out["d_x"] = d.to(kept.dtype)
        if c["residual"]:
            out["d_residual"] = out["d_x"]
        out["d_weight"] = (dy * n).sum(dim=0).to(s["weight"].dtype)
    return out


def _rotation(G, device, dtype):
    h4 = torch.tensor([[1, 1, 1, -1], [1, 1, -1, 1], [1, -1, 1, 1], [-1, 1, 1, 1]], dtype=dtype, device=device)
    h = h4
    while h.shape[0] < G:
        h = torch.kron(h, h4)
    return h / G ** 0.5


def _plain_norm8(s):
    c, kept = s["case"], _sum_kept(s)
    h, G = kept.to(torch.float64), c["G"]
    rstd = 1.0 / torch.sqrt((h * h).mean(dim=-1, keepdim=True) + _EPS)
    z = (h * s["weight"].to(torch.float64)).reshape(-1, G) @ _rotation(G, h.device, torch.float64)
    z = z.reshape(h.shape) * rstd
    scale = (z.abs().amax(dim=-1, keepdim=True).clamp(min=1e-10) / 127.0).to(torch.float32)
    q = torch.round(z / scale.to(torch.float64)).clamp(-127.0, 127.0).to(torch.float32)
    back = (q.reshape(-1, G) @ _rotation(G, h.device, torch.float32)).reshape(h.shape)
    out = {"values": (back * scale).to(torch.bfloat16), "scales": scale.reshape(-1)}
    if c["residual"]:
        out["h"] = kept
    return out


def _own_pass(s):
    q = importlib.import_module(_PKG + "._int4")
    c = s["case"]
    if c["kind"] == "choose":
        ids, weights = q.choose_experts(
            s["logits"], c["k"], s["bias"], scoring=c["scoring"], num_groups=c["groups"], top_groups=c["top_groups"],
            group_score=c["group_score"], renormalize=c["renormalize"], scale=c["scale"])
        out = {"ids": ids, "weights": weights.detach()}
        if c["grad"]:
            out["d_logits"], = torch.autograd.grad(weights, s["logits"], s["d_weights"])
        return out
    if c["kind"] == "norm8":
        int8 = importlib.import_module(_PKG + "._int4.int8_eager")
        rows = q.rms_norm_int8(s["x"], s["weight"], s["residual"], _EPS, convrot_groupsize=c["G"])
        rows, h = rows if c["residual"] else (rows, None)
        out = {"values": int8.dequantize_convrot_w8a8_weight(rows.codes, rows.scales, c["G"], torch.bfloat16),
               "scales": rows.scales}
        if c["residual"]:
            out["h"] = h
        return out
    y = q.rms_norm(s["x"], s["weight"], s["residual"], _EPS)
    y, h = y if c["residual"] else (y, None)
    out = {"y": y.detach()}
    if c["residual"]:
        out["h"] = h.detach()
    if c["grad"]:
        if c["residual"]:
            out["d_x"], out["d_residual"], out["d_weight"] = torch.autograd.grad(
                (y, h), (s["x"], s["residual"], s["weight"]), (s["d_y"], s["d_h"]))
        else:
            out["d_x"], out["d_weight"] = torch.autograd.grad(y, (s["x"], s["weight"]), s["d_y"])
    return out


def run(state):
    if own:
        return _own_pass(state)
    return {"choose": _plain_choose, "norm": _plain_norm, "norm8": _plain_norm8}[state["case"]["kind"]](state)


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------

def work(case):
    c, es = case, _ES[case["dtype"]]
    if c["kind"] == "choose":
        T, E, k = c["T"], c["E"], c["k"]
        moved = es * T * E + 8 * T * k + (4 * E if c["bias"] else 0)
        if c["grad"]:
            moved += es * T * E + 4 * T * k
        return {"bytes": moved, "flops": (8 if c["grad"] else 4) * T * E}
    n, tensors = c["M"] * c["D"], 3 if c["residual"] else 1         # x; residual and the sum
    ws = _ES[c["weight"]] * c["D"]
    if c["kind"] == "norm8":
        # codes out and in again, 16-bit values out
        return {"bytes": n * (es * tensors + 4) + 8 * c["M"] + ws, "flops": n * (10 + 2 * int(math.log(c["G"], 4)))}
    moved = es * n * (tensors + 1) + ws
    if c["grad"]:
        # d_y (and d_h) in, d_x out, d_weight
        moved += es * n * (3 if c["residual"] else 2) + ws
    return {"bytes": moved, "flops": n * (14 if c["grad"] else 5)}


# --------------------------------------------------------------------------
# the definitions, in 64 bits
# --------------------------------------------------------------------------

def _first_greatest(v):
    """Greatest along the last axis and the lowest index that has it."""
    best = v.amax(dim=-1, keepdim=True)
    at = torch.arange(v.shape[-1], device=v.device).expand_as(v)
    return best.squeeze(-1), torch.where(v == best, at, v.shape[-1]).amin(dim=-1)


def _exact_choose(c, s):
    l = s["logits"].detach().double().requires_grad_(c["grad"])
    T, E = c["T"], c["E"]
    score = torch.softmax(l, dim=-1) if c["scoring"] == "softmax" else torch.sigmoid(l)
    left = score.detach() + (0.0 if s["bias"] is None else s["bias"].double())
    left = left.masked_fill(torch.isneginf(l.detach()), -math.inf)
    if c["groups"] > 1:
        size, of = E // c["groups"], torch.arange(E, device=l.device) // (E // c["groups"])
        rank = torch.full((T, c["groups"]), -math.inf, dtype=torch.float64, device=l.device)
        for g in range(c["groups"]):
            part = left[:, g * size:(g + 1) * size].clone()
            first, at = _first_greatest(part)
            rank[:, g] = first
            if c["group_score"] == "sum2" and size > 1:
                part.scatter_(1, at[:, None], -math.inf)
                second = part.amax(dim=-1)
                rank[:, g] += torch.where(torch.isneginf(second), 0.0, second)
        kept = torch.zeros((T, c["groups"]), dtype=torch.bool, device=l.device)
        for _ in range(c["top_groups"]):
            _, at = _first_greatest(rank)
            kept.scatter_(1, at[:, None], True)
            rank.scatter_(1, at[:, None], -math.inf)
        left = left.masked_fill(~kept[:, of], -math.inf)
    ids, weights = [], []
    for _ in range(c["k"]):
        best, at = _first_greatest(left)
        at = at.clamp(max=E - 1)
        left = left.scatter(1, at[:, None], -math.inf)
        there = ~torch.isneginf(best)
        ids.append(torch.where(there, at, -1))
        weights.append(torch.where(there, score.gather(1, at[:, None]).squeeze(1), torch.zeros_like(best)))
    w = torch.stack(weights, dim=1)
    if c["renormalize"]:
        total = w.sum(dim=1, keepdim=True)
        w = w / torch.where(total > 0, total, torch.ones_like(total))
    w = w * c["scale"]
    out = {"ids": torch.stack(ids, dim=1).to(torch.int32), "weights": w.detach()}
    if c["grad"]:
        out["d_logits"], = torch.autograd.grad(w, l, s["d_weights"].double())
    return out


def _exact_norm(c, s):
    h = _sum_kept(s).double().requires_grad_(c["grad"])
    w = s["weight"].detach().double().requires_grad_(c["grad"])
    y = h / torch.sqrt(h.square().sum(dim=-1, keepdim=True) / c["D"] + _EPS) * w
    out = {"y": y.detach()}
    if c["residual"]:
        out["h"] = s["x"].detach().double() + s["residual"].detach().double()
    if c["grad"]:
        d_h, d_w = torch.autograd.grad(y, (h, w), s["d_y"].double())
        if c["residual"]:
            d_h = d_h + s["d_h"].double()
        out["d_x"] = d_h
        if c["residual"]:
            out["d_residual"] = d_h
        out["d_weight"] = d_w
    return out


def _exact_norm8(c, s):
    h, G = _sum_kept(s).double(), c["G"]
    y = h * s["weight"].double() / torch.sqrt(h.square().sum(dim=-1, keepdim=True) / c["D"] + _EPS)
    # +1 or -1 of the rotation's element (i, j): a factor -1 for every base-4 digit pair that adds up to 3
    i, turn = torch.arange(G, device=h.device), torch.ones((G, G), dtype=torch.float64, device=h.device)
    for digit in range(round(math.log(G, 4))):
        d = (i >> 2 * digit) & 3
        turn = torch.where(d[:, None] + d[None, :] == 3, -turn, turn)
    turn /= math.sqrt(G)
    z = (y.reshape(-1, G) @ turn).reshape(h.shape)
    scale = (z.abs().amax(dim=-1).clamp(min=1e-10) / 127.0).float()
    steps = z / scale[:, None].double()
    low = torch.floor(steps)
    up = (steps - low > 0.5) | ((steps - low == 0.5) & (low % 2 != 0))
    q = (low + up).clamp(-127, 127)
    out = {"values": (q.reshape(-1, G) @ turn.T).reshape(h.shape) * scale[:, None].double(), "scales": scale.double()}
    if c["residual"]:
        out["h"] = s["x"].double() + s["residual"].double()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"choose": _exact_choose, "norm": _exact_norm, "norm8": _exact_norm8}[case["kind"]](case, s)
