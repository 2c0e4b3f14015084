"""Performance cases of the microscaled 4-bit operators and of the expert routing.

A case is one call that a quantized transformer's forward (or a training step
over its router) makes:

  quantize  activations or weights -> 4-bit codes with a power-of-two scale for
            every 32 values of a row, and back to 16-bit values
  linear    y = x W^T + b on such weights, x rotated and quantized on the way
  experts   the same for a mixture of experts: every token's row times the
            weights of the experts it was sent to
  route     tokens sorted by expert, their rows gathered, and the experts'
            outputs added up per token with the router's weights; with ``grad``
            also the gradients of the tokens, the outputs and the weights

Activations are N(0, 1) with 1% of the channels scaled by 20, weights N(0, 1/K).
"""
from __future__ import annotations

import importlib
import math

import torch

own = False

_PKG = "comfyui-int4-convrot-rdna4_amd"
_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_ES = {"bf16": 2, "f16": 2, "f32": 4}


def _quant(name, M, K, dtype="bf16"):
    return {"name": name, "kind": "quantize", "M": M, "K": K, "dtype": dtype}


def _linear(name, M, K, N, G=256, dtype="bf16", bias=True):
    return {"name": name, "kind": "linear", "M": M, "K": K, "N": N, "G": G, "dtype": dtype, "bias": bias}


def _experts(name, T, k, E, K, N, G=256, dtype="bf16", bias=False, rows=False):
    return {"name": name, "kind": "experts", "T": T, "k": k, "E": E, "K": K, "N": N, "G": G, "dtype": dtype,
            "bias": bias, "sorted": rows}


def _route(name, T, k, E, D, dtype="bf16", grad=True):
    return {"name": name, "kind": "route", "T": T, "k": k, "E": E, "D": D, "dtype": dtype, "grad": grad}


def listed():
    return [
        # one conditioning vector before its linear: launch latency
        _quant("quantize_m1", 1, 5120),
        # a large image's tokens, kept in 4 bits and read back
        _quant("quantize_m16384", 16384, 5120),
        # one vector through a wide layer: weight bytes and latency
        _linear("linear_m1", 1, 5120, 13824),
        # an odd number of tokens, a width that is no multiple of 128, fp16
        _linear("linear_ragged_f16_m333", 333, 1600, 4800, G=64, dtype="f16"),
        # a prompt's tokens
        _linear("linear_text_m512", 512, 4096, 10240),
        # an image's tokens through the widest layer
        _linear("linear_image_m8192", 8192, 5120, 13824),
        # one token through its four experts
        _experts("experts_t1", 1, 4, 32, 2048, 4096),
        # the experts' second layer on rows that are already sorted, odd counts, fp16, biases
        _experts("experts_ragged_f16_t777", 777, 3, 13, 1600, 2400, G=64, dtype="f16", bias=True, rows=True),
        # a long prompt or an image through the first layer
        _experts("experts_t4096", 4096, 4, 32, 2048, 4096),
        # a serving step's few tokens: sort, gather, combine
        _route("route_t16", 16, 4, 32, 2048, grad=False),
        # odd sizes, many experts, single precision, with gradients
        _route("route_odd_f32_t3001", 3001, 6, 100, 1000, dtype="f32"),
        # a training step's tokens with gradients
        _route("route_train_t8192", 8192, 4, 32, 4096),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same ranges: 1 to 16384 rows, widths in whole blocks of 32 from 512 to 13824, every rotation
    group and none, 2 to 128 experts, 1 to 8 of them a token."""
    kind = rng.choice(("quantize", "linear", "linear", "experts", "experts", "route", "route"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if kind == "quantize":
        M, K = _log_int(rng, 1, 16384), max(1, _log_int(rng, 512, 13824) // 32) * 32
        while M * K > 16384 * 5120:
            M //= 2
        return {"kind": kind, "M": M, "K": K, "dtype": dtype}
    if kind == "route":
        T, k, E = _log_int(rng, 1, 16384), rng.randint(1, 8), _log_int(rng, 8, 128)
        D = _log_int(rng, 256, 8192)
        if rng.random() < 0.7:
            D = max(1, D // 64) * 64
        size = 2 if dtype == "f32" else 1
        while size * T * k * D > 8192 * 4 * 4096:
            T = max(1, T // 2)
        return {"kind": kind, "T": T, "k": k, "E": E, "D": D, "dtype": dtype, "grad": rng.random() < 0.7}
    # rotated rows are rounded to 4 bits from sums: a 32-bit output would show the order of those sums
    G = 0 if dtype == "f32" else rng.choice((0, 16, 64, 256, 256))
    unit = max(G, 32) if rng.random() < 0.5 else 256
    N = _log_int(rng, 512, 13824)
    if rng.random() < 0.7:
        N = max(1, N // 64) * 64
    if kind == "linear":
        M, K = _log_int(rng, 1, 16384), max(1, _log_int(rng, 512, 13824) // unit) * unit
        share = 2 if dtype == "f32" else 1
        while share * M * K * N > 8192 * 5120 * 13824:
            M = max(1, M // 2)
        return {"kind": kind, "M": M, "K": K, "N": N, "G": G, "dtype": dtype, "bias": rng.random() < 0.7}
    T, k, E = _log_int(rng, 1, 8192), rng.randint(1, 6), _log_int(rng, 8, 64)
    K = max(1, _log_int(rng, 512, 4096) // unit) * unit
    N = min(N, 8192)
    while E * K * N > 32 * 2048 * 4096:
        N = max(64, N // 2)
        E = max(8, E * 3 // 4)
    while T * k * K * N > 4096 * 4 * 2048 * 4096:
        T = max(1, T // 2)
    return {"kind": kind, "T": T, "k": k, "E": E, "K": K, "N": N, "G": G, "dtype": dtype,
            "bias": rng.random() < 0.5, "sorted": rng.random() < 0.5}


# --------------------------------------------------------------------------
# inputs (made from the seed alone, on the GPU)
# --------------------------------------------------------------------------

def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + salt) % (1 << 62))
    return g


def _activations(M, K, dtype, seed, salt=1):
    g = _gen(seed, salt)
    x = torch.randn((M, K), generator=g, device="cuda")
    channels = torch.randperm(K, generator=g, device="cuda")[:max(1, round(0.01 * K))]
    x[:, channels] *= 20.0
    return x.to(_DT[dtype])


def _weight(shape, seed, salt=2):
    """Codes [.., K/2] (value 2j in the low half of byte j) and scales [.., K/32] of a weight N(0, 1/K)."""
    w = torch.randn(shape, generator=_gen(seed, salt), device="cuda") * shape[-1] ** -0.5
    v, e = _to_fp4(w)
    level = torch.tensor([0, 1, 2, 3, 4, 0, 5, 0, 6, 0, 0, 0, 7], device="cuda", dtype=torch.uint8)   # 2 |v| -> code
    code = level[(2 * v.abs()).to(torch.int64)] | ((v < 0).to(torch.uint8) << 3)
    code = code.reshape(shape)
    return (code[..., 0::2] | (code[..., 1::2] << 4)), (e + 127).to(torch.uint8)


def _ids(T, k, E, seed):
    """The k experts of each token, by the scores of a router with a taste of its own; 2% of the slots (capacity,
    padding) are not used: -1."""
    g = _gen(seed, 5)
    scores = torch.randn((T, E), generator=g, device="cuda") + 0.7 * torch.randn((E,), generator=g, device="cuda")
    top, ids = scores.topk(k, dim=-1)
    ids[torch.rand((T, k), generator=g, device="cuda") < 0.02] = -1
    return ids, torch.softmax(top, dim=-1)


def prepare(case, seed):
    kind, dtype = case["kind"], case["dtype"]
    if kind == "quantize":
        return {"case": case, "x": _activations(case["M"], case["K"], dtype, seed)}
    if kind == "linear":
        codes, scales = _weight((case["N"], case["K"]), seed)
        bias = torch.randn((case["N"],), generator=_gen(seed, 3), device="cuda").to(_DT[dtype]) if case["bias"] else None
        return {"case": case, "x": _activations(case["M"], case["K"], dtype, seed), "codes": codes, "scales": scales,
                "bias": bias}
    ids, weights = _ids(case["T"], case["k"], case["E"], seed)
    T, R = case["T"], case["T"] * case["k"]
    state = {"case": case, "ids": ids, "weights": weights}
    if kind == "experts":
        state["codes"], state["scales"] = _weight((case["E"], case["N"], case["K"]), seed)
        state["x"] = _activations(R if case["sorted"] else T, case["K"], dtype, seed)
        state["bias"] = torch.randn((case["E"], case["N"]), generator=_gen(seed, 3), device="cuda").to(_DT[dtype]) \
            if case["bias"] else None
        # the most rows of any expert: what a plain program pads the experts' rows to
        state["capacity"] = int(torch.bincount(ids[ids >= 0], minlength=1).max()) if bool((ids >= 0).any()) else 1
        return state
    state["x"] = _activations(T, case["D"], dtype, seed)
    state["rows"] = torch.randn((R, case["D"]), generator=_gen(seed, 6), device="cuda").to(_DT[dtype])
    if case["grad"]:
        state["d_rows"] = torch.randn((R, case["D"]), generator=_gen(seed, 7), device="cuda").to(_DT[dtype])
        state["d_out"] = torch.randn((T, case["D"]), generator=_gen(seed, 8), device="cuda").to(_DT[dtype])
        for name in ("x", "rows", "weights"):
            state[name].requires_grad_(True)
    return state


# --------------------------------------------------------------------------
# the plain forms, in 32 bits
# --------------------------------------------------------------------------

def _to_fp4(x):
    """x [.., K] -> values on the 4-bit grid [.., K/32, 32] in units of the scale 2^e, and e [.., K/32]."""
    b = x.to(torch.float32).reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    amax = b.abs().amax(dim=-1)
    e = torch.where(amax > 0, torch.frexp(amax).exponent - 3, -127).clamp(-127, 127)
    v = torch.ldexp(b, -e.unsqueeze(-1))
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.copysign((torch.round(a / step) * step).clamp(max=6.0), v), e


def _rotation(G, device):
    h4 = torch.tensor([[1, 1, 1, -1], [1, 1, -1, 1], [1, -1, 1, 1], [-1, 1, 1, 1]], dtype=torch.float32, device=device)
    h = h4
    while h.shape[0] < G:
        h = torch.kron(h, h4)
    return h / G ** 0.5


def _rounded(x, G=0):
    """x, rotated in groups of G, on its 4-bit grid, in 32 bits."""
    x = x.to(torch.float32)
    if G:
        x = torch.matmul(x.reshape(-1, G), _rotation(G, x.device)).reshape(x.shape)
    v, e = _to_fp4(x)
    return torch.ldexp(v, e.unsqueeze(-1)).reshape(x.shape)


def _values(codes, scales):
    """Codes [.., K/2] and scales [.., K/32] -> values [.., K]."""
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    byte = torch.arange(256, device=codes.device)
    v = torch.stack((grid[byte & 15], grid[byte >> 4]), dim=-1)[codes.to(torch.int32)].reshape(*scales.shape, 32)
    scale = torch.ldexp(torch.ones((), device=codes.device), scales.to(torch.int32) - 127)
    return (v * scale.unsqueeze(-1)).reshape(*codes.shape[:-1], -1)


def _sort(ids, E):
    """order [T k]: the slot of each sorted row; position [T, k]: the sorted row of each slot; offsets [E + 1]."""
    flat = ids.reshape(-1)
    used = (flat >= 0) & (flat < E)
    key = torch.where(used, flat, E)
    order = torch.argsort(key, stable=True)
    rows = torch.arange(flat.numel(), device=ids.device)
    position = torch.empty_like(order)
    position[order] = rows
    counts = torch.zeros(E + 1, dtype=torch.int64, device=ids.device).index_add_(0, key, torch.ones_like(key))
    offsets = torch.cat((counts.new_zeros(1), counts[:E].cumsum(0)))
    order = torch.where(rows < offsets[E], order, -1)
    position = torch.where(used, position, -1).reshape(ids.shape)
    return order.to(torch.int32), position.to(torch.int32), offsets.to(torch.int32)


def _plain_experts(s):
    c, x = s["case"], s["x"]
    order, _, offsets = _sort(s["ids"], c["E"])
    a = _rounded(x, c["G"])
    if not c["sorted"]:
        a = a[(order // c["k"]).clamp(min=0).long()]
    # [E, C] row numbers: every expert's rows, padded to the fullest expert's
    place = offsets[:-1, None].long() + torch.arange(s["capacity"], device=x.device)
    there = place < offsets[1:, None]
    y = torch.bmm(a[torch.where(there, place, 0)], _values(s["codes"], s["scales"]).transpose(1, 2))
    if s["bias"] is not None:
        y = y + s["bias"].to(torch.float32)[:, None]
    out = torch.zeros((c["T"] * c["k"] + 1, c["N"]), device=x.device)
    out[torch.where(there, place, c["T"] * c["k"])] = y
    out[-1] = 0
    return out[:-1].to(x.dtype)


def _plain_route(s):
    c, x, rows, w = s["case"], s["x"].detach(), s["rows"].detach(), s["weights"].detach()
    order, position, offsets = _sort(s["ids"], c["E"])
    token = (order // c["k"]).clamp(min=0).long()
    used_row, used = (order >= 0)[:, None], (position >= 0)[..., None]
    at = position.clamp(min=0).long()
    out = {"order": order, "position": position, "offsets": offsets}
    out["gathered"] = torch.where(used_row, x[token], 0)
    picked = torch.where(used, rows[at].to(torch.float32), 0.0)
    out["combined"] = (picked * w[..., None]).sum(dim=1).to(x.dtype)
    if c["grad"]:
        out["d_x"] = torch.where(used, s["d_rows"][at].to(torch.float32), 0.0).sum(dim=1).to(x.dtype)
        d_out = s["d_out"].to(torch.float32)
        out["d_weights"] = (picked * d_out[:, None]).sum(dim=-1)
        of_row = w.reshape(-1)[order.clamp(min=0).long()][:, None]
        out["d_rows"] = torch.where(used_row, of_row * d_out[token], 0.0).to(x.dtype)
    return out


def _plain(s):
    c = s["case"]
    if c["kind"] == "quantize":
        v, e = _to_fp4(s["x"])
        return {"values": torch.ldexp(v, e.unsqueeze(-1)).reshape(s["x"].shape).to(torch.bfloat16)}
    if c["kind"] == "linear":
        y = torch.matmul(_rounded(s["x"], c["G"]), _values(s["codes"], s["scales"]).T)
        if s["bias"] is not None:
            y = y + s["bias"].to(torch.float32)
        return y.to(s["x"].dtype)
    return _plain_experts(s) if c["kind"] == "experts" else _plain_route(s)


def _own(s):
    q = importlib.import_module(_PKG + "._int4")
    c = s["case"]
    if c["kind"] == "quantize":
        codes, scales = q.quantize_mxfp4(s["x"])
        return {"values": q.dequantize_mxfp4(codes, scales, output_dtype=torch.bfloat16)}
    if c["kind"] == "linear":
        return q.mxfp4_linear(s["x"], s["codes"], s["scales"], s["bias"], convrot_groupsize=c["G"] or None)
    plan = q.sort_tokens_by_expert(s["ids"], c["E"])
    if c["kind"] == "experts":
        return q.mxfp4_expert_linear(s["x"], s["codes"], s["scales"], plan, s["bias"], convrot_groupsize=c["G"] or None,
                                     sorted_rows=c["sorted"])
    gathered = q.gather_expert_rows(s["x"], plan)
    combined = q.combine_expert_rows(s["rows"], s["weights"], plan)
    out = {"order": plan.order, "position": plan.position, "offsets": plan.offsets, "gathered": gathered.detach(),
           "combined": combined.detach()}
    if c["grad"]:
        grads = torch.autograd.grad((gathered, combined), (s["x"], s["rows"], s["weights"]), (s["d_rows"], s["d_out"]))
        out["d_x"], out["d_rows"], out["d_weights"] = grads
    return out


def run(state):
    return _own(state) if own else _plain(state)


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------

def work(case):
    c, es = case, _ES[case["dtype"]]
    if c["kind"] == "quantize":
        # the values in, codes and scales out and in again, 16-bit values out
        n = c["M"] * c["K"]
        return {"bytes": n * (es + 2) + 2 * (n // 2 + n // 32), "flops": 4 * n}
    if c["kind"] == "linear":
        M, K, N = c["M"], c["K"], c["N"]
        return {"bytes": es * M * (K + N) + N * K // 2 + N * K // 32 + (es * N if c["bias"] else 0), "flops": 2 * M * N * K}
    T, R = c["T"], c["T"] * c["k"]
    if c["kind"] == "experts":
        K, N, busy = c["K"], c["N"], min(c["E"], R)
        rows = R if c["sorted"] else T
        return {"bytes": es * (rows * K + R * N) + busy * (N * K // 2 + N * K // 32 + (es * N if c["bias"] else 0)) + 8 * R,
                "flops": 2 * R * N * K}
    D = c["D"]
    moved = es * (T * D + R * D + R * D + T * D) + 20 * R          # gather and combine, ids, weights, plan
    if c["grad"]:
        moved += es * (R * D + T * D + T * D + R * D) + 4 * R      # d_rows -> d_x; d_out -> d_rows, d_weights
    return {"bytes": moved, "flops": (6 if c["grad"] else 2) * R * D}


# --------------------------------------------------------------------------
# the definitions, in 64 bits
# --------------------------------------------------------------------------

def _sign(i, j):
    """+1 or -1 of the rotation's element (i, j): a factor -1 for every base-4 digit pair that adds up to 3."""
    s = torch.ones(torch.broadcast_shapes(i.shape, j.shape), dtype=torch.float64, device=i.device)
    for shift in (0, 2, 4, 6):
        s = torch.where(((i >> shift) & 3) + ((j >> shift) & 3) == 3, -s, s)
    return s


def _exact_rotated(x, G):
    x = x.double()
    if not G:
        return x
    n = torch.arange(G, device=x.device)
    h = _sign(n[:, None], n[None, :])
    if G < 256:       # the digits past the group's add up to 3 nowhere: both are 0
        assert G in (16, 64)
    return (x.reshape(-1, G) @ h).reshape(x.shape) / math.sqrt(G)


def _exact_values(x):
    """The nearest of the 4-bit values in units of 2^(floor(log2(max)) - 2), ties to the even code."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    amax = b.abs().amax(dim=-1, keepdim=True)
    e = torch.floor(torch.log2(amax.clamp(min=2.0 ** -140)))
    e = torch.where(torch.exp2(e) > amax, e - 1, e)
    e = torch.where(torch.exp2(e + 1) <= amax, e + 1, e)
    scale = torch.exp2((e - 2).clamp(min=-127, max=127))
    v = b.abs() / scale
    out = torch.zeros_like(v)
    # the middles between neighbours, the step up at each, and whether the middle itself goes up
    for middle, rise, up in ((.25, .5, False), (.75, .5, True), (1.25, .5, False), (1.75, .5, True), (2.5, 1., False),
                             (3.5, 1., True), (5., 2., False)):
        out += rise * ((v >= middle) if up else (v > middle))
    return (torch.where(b < 0, -out, out) * scale).reshape(x.shape)


def _exact_weight(codes, scales):
    low, high = codes & 15, codes >> 4
    both = torch.empty((*codes.shape[:-1], 2 * codes.shape[-1]), dtype=torch.int64, device=codes.device)
    both[..., 0::2], both[..., 1::2] = low.long(), high.long()
    exponent, mantissa = (both >> 1) & 3, both & 1
    v = torch.where(exponent == 0, 0.5 * mantissa, (1 + 0.5 * mantissa) * torch.exp2(exponent.double() - 1))
    v = torch.where(both >= 8, -v, v)
    return v * torch.exp2(scales.double() - 127).repeat_interleave(32, dim=-1)


def _exact_plan(ids, E):
    rows = ids.reshape(-1).tolist()
    per = [[] for _ in range(E)]
    for slot, e in enumerate(rows):
        if 0 <= e < E:
            per[e].append(slot)
    order, offsets, position = [], [0], [-1] * len(rows)
    for slots in per:
        for slot in slots:
            position[slot] = len(order)
            order.append(slot)
        offsets.append(len(order))
    return order, position, offsets


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "quantize":
        return {"values": _exact_values(s["x"].double())}
    if c["kind"] == "linear":
        y = _exact_values(_exact_rotated(s["x"], c["G"])) @ _exact_weight(s["codes"], s["scales"]).T
        return y if s["bias"] is None else y + s["bias"].double()
    order, position, offsets = _exact_plan(s["ids"], c["E"])
    dev = s["x"].device
    slots = torch.tensor(order, device=dev, dtype=torch.int64)
    R = c["T"] * c["k"]
    if c["kind"] == "experts":
        a = _exact_values(_exact_rotated(s["x"], c["G"]))
        out = torch.zeros((R, c["N"]), dtype=torch.float64, device=dev)
        for e in range(c["E"]):
            r0, r1 = offsets[e], offsets[e + 1]
            if r1 > r0:
                rows = a[r0:r1] if c["sorted"] else a[slots[r0:r1] // c["k"]]
                out[r0:r1] = rows @ _exact_weight(s["codes"][e], s["scales"][e]).T
                if s["bias"] is not None:
                    out[r0:r1] += s["bias"][e].double()
        return out
    x, rows, w = s["x"].detach().double(), s["rows"].detach().double(), s["weights"].detach().double()
    n = len(order)
    token = slots // c["k"]
    out = {"order": None, "position": None, "offsets": None}
    out["gathered"] = torch.zeros((R, c["D"]), dtype=torch.float64, device=dev)
    out["gathered"][:n] = x[token]
    of_row = w.reshape(-1)[slots][:, None]
    out["combined"] = torch.zeros_like(x).index_add_(0, token, of_row * rows[:n])
    if c["grad"]:
        d_out = s["d_out"].double()
        out["d_x"] = torch.zeros_like(x).index_add_(0, token, s["d_rows"][:n].double())
        out["d_rows"] = torch.zeros((R, c["D"]), dtype=torch.float64, device=dev)
        out["d_rows"][:n] = of_row * d_out[token]
        out["d_weights"] = torch.zeros(R, dtype=torch.float64, device=dev)
        out["d_weights"][slots] = (rows[:n] * d_out[token]).sum(dim=-1)
        out["d_weights"] = out["d_weights"].reshape(c["T"], c["k"])
    return out
