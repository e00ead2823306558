"""Cases of the operators that serve a few tokens from block-float weights: the product of a few rows with a Bfp8_b /
Bfp4_b / Bfp2_b queue image, the router of a mixture of experts, its experts' products, and the whole layer.

Each operator has a plain form here (`own` false: elementary torch operations in 32 or 64 bits on the same inputs) and
the framework's call (`own` true).  Weights are queue images of tilized tensors: 32x32 tiles of four 16x16 faces, one
shared 8-bit exponent for each face row of 16 values, sign and 7 / 3 / 1 magnitude bits, tile records in row-major
order of the tiles, the experts of a layer one after another.
"""
import math
import os
import sys

import torch

own = False

MANT = {"Bfp8_b": 7, "Bfp4_b": 3, "Bfp2_b": 1}        # magnitude bits
RECORD = {"Bfp8_b": 1088, "Bfp4_b": 576, "Bfp2_b": 320}  # bytes of a tile record
CODE = {"Bfp8_b": 6, "Bfp4_b": 7, "Bfp2_b": 15}       # data format numbers
DTYPE = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token through an attention projection of BERT-large: the smallest call, latency counts
        {"name": "matvec 1x1024x1024 Bfp4_b", "op": "matvec", "m": 1, "k": 1024, "n": 1024, "df": "Bfp4_b", "out": "bf16"},
        # a small batch through its feed-forward matrix, binary32 result for a residual sum
        {"name": "matvec 8x4096x1024 Bfp8_b", "op": "matvec", "m": 8, "k": 4096, "n": 1024, "df": "Bfp8_b", "out": "fp32"},
        # sizes that fill no tile
        {"name": "matvec 5x1000x2500 Bfp2_b", "op": "matvec", "m": 5, "k": 1000, "n": 2500, "df": "Bfp2_b", "out": "bf16"},
        # the benchmark's weight matrix: one token, and a decoding batch
        {"name": "matvec 1x4096x16384 Bfp4_b", "op": "matvec", "m": 1, "k": 4096, "n": 16384, "df": "Bfp4_b", "out": "bf16"},
        {"name": "matvec 32x4096x16384 Bfp8_b", "op": "matvec", "m": 32, "k": 4096, "n": 16384, "df": "Bfp8_b", "out": "bf16"},
        # routing of one token among a few experts, and of a decoding batch among many
        {"name": "route 1 of 8", "op": "route", "t": 1, "h": 1024, "e": 8, "top": 2, "router": "fp32", "renorm": True},
        {"name": "route 16 of 128", "op": "route", "t": 16, "h": 4096, "e": 128, "top": 8, "router": "bf16", "renorm": False},
        # experts' products on their own, as a caller with its own routing has them: ragged sizes, dropped
        # slots, experts without a gate matrix; and a batch in the gated form
        {"name": "experts 7 ragged Bfp8_b", "op": "experts", "t": 7, "h": 1000, "i": 1500, "e": 6, "top": 3, "df": "Bfp8_b",
         "act": "gelu", "gated": False, "drop": True},
        {"name": "experts 32 Bfp2_b", "op": "experts", "t": 32, "h": 2048, "i": 1024, "e": 16, "top": 2, "df": "Bfp2_b",
         "act": "silu", "gated": True, "drop": False},
        # the whole layer for one token: few wide experts of BERT-large's feed-forward size, many narrow ones
        {"name": "layer 1 of 8 experts", "op": "layer", "t": 1, "h": 1024, "i": 4096, "e": 8, "top": 2, "df": "Bfp4_b",
         "act": "gelu", "gated": True, "router": "fp32", "renorm": True},
        {"name": "layer 1 of 64 experts", "op": "layer", "t": 1, "h": 2048, "i": 1024, "e": 64, "top": 8, "df": "Bfp4_b",
         "act": "silu", "gated": True, "router": "bf16", "renorm": True},
        # and for a decoding batch that reaches most experts
        {"name": "layer 16 of 32 experts", "op": "layer", "t": 16, "h": 4096, "i": 2048, "e": 32, "top": 4, "df": "Bfp4_b",
         "act": "silu", "gated": True, "router": "fp32", "renorm": False},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm; every other one a multiple of 32 where that fits."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    v = max(lo, min(hi, v))
    return max(32, v // 32 * 32) if v >= 64 and rng.random() < 0.5 else v


def draw(rng):
    op = rng.choice(["matvec", "matvec", "route", "experts", "layer"])
    df = rng.choice(["Bfp8_b", "Bfp4_b", "Bfp2_b"])
    if op == "matvec":
        k = _spread(rng, 32, 16384)
        return {"op": op, "m": _spread(rng, 1, 32), "k": k, "n": _spread(rng, 32, min(16384, (1 << 26) // k)), "df": df,
                "out": rng.choice(["bf16", "fp32"])}
    t, e = _spread(rng, 1, 16), _spread(rng, 2, 64)
    top = min(e, rng.randint(1, 8))
    case = {"op": op, "t": t, "h": _spread(rng, 64, 4096), "e": e, "top": top}
    if op == "route":
        return {**case, "router": rng.choice(["bf16", "fp32"]), "renorm": rng.random() < 0.5}
    # the weights of all experts stay below those of the largest listed layer
    case["i"] = _spread(rng, 64, max(64, min(4096, 120_000_000 // (e * case["h"]))))
    case.update(df=df, act=rng.choice(["silu", "gelu"]), gated=rng.random() < 0.7)
    if op == "experts":
        return {**case, "drop": rng.random() < 0.3}
    return {**case, "router": rng.choice(["bf16", "fp32"]), "renorm": rng.random() < 0.5}


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed, which):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1009 + which) % (1 << 62))


def _weight(case, seed, which, expert=0):
    """One weight matrix in binary32, as a checkpoint has it: normal values, each output's variance kept."""
    rows, cols = {0: lambda c: (c["k"], c["n"]), 1: lambda c: (c["h"], c["i"]), 2: lambda c: (c["h"], c["i"]),
                  3: lambda c: (c["i"], c["h"])}[which](case)
    g = _generator(seed, 16 + 4 * expert + which)
    return torch.randn(rows, cols, generator=g, device="cuda") * rows ** -0.5


def _pack(w, df, out):
    """The queue image of one matrix: tile padding with zeros, shared exponents, magnitudes to nearest even."""
    m = MANT[df]
    rows, cols = -(-w.shape[0] // 32), -(-w.shape[1] // 32)
    w = torch.nn.functional.pad(w, (0, 32 * cols - w.shape[1], 0, 32 * rows - w.shape[0]))
    w = w.view(rows, 2, 16, cols, 2, 16).permute(0, 3, 1, 4, 2, 5).reshape(rows * cols, 4, 16, 16)
    e = w.view(torch.int32).bitwise_right_shift(23).bitwise_and(255).amax(-1, keepdim=True)
    q = torch.round(torch.ldexp(w.abs(), 127 + m - 1 - e)).clamp(max=2 ** m - 1).to(torch.uint8)
    d = q | ((w < 0) & (q > 0)).to(torch.uint8) << m
    per = 8 // (m + 1)
    d = d.view(rows * cols, 4, 16, 16 // per, per)
    d = (d << (torch.arange(per, device=w.device, dtype=torch.uint8) * (m + 1))).sum(-1, dtype=torch.uint8)
    out = out.view(rows * cols, RECORD[df])
    out[:, :64] = e.to(torch.uint8).view(-1, 64)
    out[:, 64:] = d.view(rows * cols, -1)


def _image_bytes(rows, cols, df):
    return -(-rows // 32) * -(-cols // 32) * RECORD[df]


def _tokens(case, seed):
    """Activations as a norm leaves them: unit variance, a few strong channels."""
    rows, width = (case["m"], case["k"]) if case["op"] == "matvec" else (case["t"], case["h"])
    g = _generator(seed, 1)
    x = torch.randn(rows, width, generator=g, device="cuda")
    x *= 1 + 7 * (torch.rand(width, generator=g, device="cuda") < 0.01)
    return x.bfloat16()


def _router(case, seed):
    w = torch.randn(case["e"], case["h"], generator=_generator(seed, 2), device="cuda") * (1.5 * case["h"] ** -0.5)
    return w.to(DTYPE[case["router"]])


def _selection(case, seed):
    """Routing that a caller made itself: distinct experts for each token, weights that add up to one, dropped slots as -1."""
    g = _generator(seed, 3)
    ids = torch.rand(case["t"], case["e"], generator=g, device="cuda").argsort(1)[:, :case["top"]].to(torch.int32)
    weights = torch.softmax(torch.randn(case["t"], case["top"], generator=g, device="cuda"), 1)
    if case["drop"]:
        ids = torch.where(torch.rand(ids.shape, generator=g, device="cuda") < 0.25, -1, ids)
    return weights, ids.to(torch.int32)


def prepare(case, seed):
    state = dict(case, x=_tokens(case, seed))
    if case["op"] == "matvec":
        image = torch.empty(_image_bytes(case["k"], case["n"], case["df"]), dtype=torch.uint8, device="cuda")
        _pack(_weight(case, seed, 0), case["df"], image)
        return {**state, "image": image}
    if case["op"] in ("route", "layer"):
        state["w_router"] = _router(case, seed)
    if case["op"] in ("experts", "layer"):
        state["up"] = None
        for name, which in (("gate", 1), ("up", 2), ("down", 3)) if case["gated"] else (("gate", 1), ("down", 3)):
            rows, cols = (case["i"], case["h"]) if name == "down" else (case["h"], case["i"])
            state[name] = torch.empty(case["e"], _image_bytes(rows, cols, case["df"]), dtype=torch.uint8, device="cuda")
            for e in range(case["e"]):
                _pack(_weight(case, seed, which, e), case["df"], state[name][e])
    if case["op"] == "experts":
        state["weights"], state["ids"] = _selection(case, seed)
    return state


# ------------------------------------------------------------------------------------------------ one pass
def _ops():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tt-buda_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from pybuda import cuda_ops

    return cuda_ops


def _decode(images, rows, cols, df):
    """[n, bytes] queue images -> [n, rows, cols] binary32 values."""
    m = MANT[df]
    n, rt, ct = images.shape[0], -(-rows // 32), -(-cols // 32)
    rec = images.view(n, rt, ct, RECORD[df])
    exps = rec[..., :64].reshape(n, rt, ct, 4, 16, 1).to(torch.int32)
    shifts = torch.arange(8 // (m + 1), device=images.device, dtype=torch.uint8) * (m + 1)
    d = (rec[..., 64:].unsqueeze(-1) >> shifts).reshape(n, rt, ct, 4, 16, 16)
    q = (d & (2 ** m - 1)).float()
    q = torch.where((d >> m & 1) == 1, -q, q)
    w = torch.ldexp(q, exps - (126 + m))
    w = w.view(n, rt, ct, 2, 2, 16, 16).permute(0, 1, 3, 5, 2, 4, 6).reshape(n, rt * 32, ct * 32)
    return w[:, :rows, :cols]


def _act(x, act):
    return x * torch.sigmoid(x) if act == "silu" else 0.5 * x * (1 + torch.erf(x * 0.7071067811865476))


def _plain_route(x, w_router, top, renorm):
    logits = x.double() @ w_router.double().T                     # 64 bits: neighbours of the last place are near
    order = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :top]
    p = torch.exp(logits - logits.amax(1, keepdim=True))
    chosen = p.gather(1, order)
    total = chosen.sum(1, keepdim=True) if renorm else p.sum(1, keepdim=True)
    return (chosen / total).float(), order.to(torch.int32)


def _plain_experts(s, weights, ids):
    t, top, e = s["t"], s["top"], s["e"]
    x = s["x"].float()
    if t * top < e:   # the experts that slots name, one matrix for each slot
        chosen = ids.reshape(-1).clamp(min=0).long()
        pick = lambda images: images[chosen]
        x = x.repeat_interleave(top, 0).view(t * top, 1, -1)
        scale = torch.where(ids < 0, 0.0, weights).reshape(-1, 1, 1)
    else:             # every expert on every token
        pick = lambda images: images
        x = x.expand(e, -1, -1)
        hit = ids.unsqueeze(-1) == torch.arange(e, device=ids.device)
        scale = (hit * weights.unsqueeze(-1)).sum(1).T.unsqueeze(-1)
    h = _act(x @ _decode(pick(s["gate"]), s["h"], s["i"], s["df"]), s["act"])
    if s["up"] is not None:
        h = h * (x @ _decode(pick(s["up"]), s["h"], s["i"], s["df"]))
    y = h @ _decode(pick(s["down"]), s["i"], s["h"], s["df"]) * scale
    return (y.view(t, top, -1).sum(1) if t * top < e else y.sum(0)).to(s["x"].dtype)


def run(state):
    s = state
    if own:
        ops = _ops()
        if s["op"] == "matvec":
            return ops.bfp_matvec(s["x"], s["image"], s["n"], CODE[s["df"]], out_dtype=DTYPE[s["out"]])
        if s["op"] == "route":
            return ops.moe_route(s["x"], s["w_router"], s["top"], s["renorm"])
        if s["op"] == "experts":
            return ops.moe_experts(s["x"], s["weights"], s["ids"], s["gate"], s["up"], s["down"], s["i"], CODE[s["df"]], s["act"])
        return ops.moe_layer(s["x"], s["w_router"], s["top"], s["gate"], s["up"], s["down"], s["i"], CODE[s["df"]], s["act"],
                             s["renorm"])
    if s["op"] == "matvec":
        return (s["x"].float() @ _decode(s["image"].view(1, -1), s["k"], s["n"], s["df"])[0]).to(DTYPE[s["out"]])
    if s["op"] == "route":
        return _plain_route(s["x"], s["w_router"], s["top"], s["renorm"])
    if s["op"] == "experts":
        return _plain_experts(s, s["weights"], s["ids"])
    return _plain_experts(s, *_plain_route(s["x"], s["w_router"], s["top"], s["renorm"]))


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    if c["op"] == "matvec":
        return {"bytes": _image_bytes(c["k"], c["n"], c["df"]) + 2 * c["m"] * c["k"] + (2 if c["out"] == "bf16" else 4) * c["m"] * c["n"],
                "flops": 2 * c["m"] * c["k"] * c["n"]}
    route = c["e"] * c["h"] * (4 if c.get("router") == "fp32" else 2)
    if c["op"] == "route":
        return {"bytes": route + 2 * c["t"] * c["h"] + 8 * c["t"] * c["top"], "flops": 2 * c["t"] * c["e"] * c["h"]}
    # the experts that t tokens with independent choices reach, on average
    slots = c["t"] * c["top"] * (0.75 if c.get("drop") else 1.0)
    reached = c["e"] * (1 - (1 - slots / c["t"] / c["e"]) ** c["t"])
    matrices = 3 if c["gated"] else 2
    nbytes = reached * ((matrices - 1) * _image_bytes(c["h"], c["i"], c["df"]) + _image_bytes(c["i"], c["h"], c["df"]))
    nbytes += 4 * c["t"] * c["h"] + (route if c["op"] == "layer" else 8 * c["t"] * c["top"])
    flops = 2 * slots * matrices * c["h"] * c["i"] + (2 * c["t"] * c["e"] * c["h"] if c["op"] == "layer" else 0)
    return {"bytes": nbytes, "flops": flops}


# ------------------------------------------------------------------------------------------------ 64 bits, from the definitions
def _stored(w, df):
    """What a block-float format keeps of a matrix: for each run of 16 columns the values to nearest even on a grid of
    2^-m times the power of two above the largest one, none past 2^m - 1 steps."""
    m = MANT[df]
    w = w.double()
    cols = w.shape[1]
    b = torch.nn.functional.pad(w, (0, -cols % 16)).view(w.shape[0], -1, 16)
    top = torch.frexp(b.abs().amax(-1, keepdim=True)).exponent    # largest magnitude in [2^(top-1), 2^top)
    step = torch.pow(2.0, (top - m).double())
    steps = torch.round(b / step)
    return (torch.clamp(steps, -(2 ** m - 1), 2 ** m - 1) * step).view(w.shape[0], -1)[:, :cols]


def _exact_route(x, w_router, top, renorm):
    scores = (x.double().unsqueeze(1) * w_router.double().unsqueeze(0)).sum(-1)
    p = torch.softmax(scores, 1)
    at = torch.arange(scores.shape[1], device=scores.device)
    # an expert's place: those that score more, and those that score the same and stand before it
    before = (scores.unsqueeze(1) > scores.unsqueeze(2)) | ((scores.unsqueeze(1) == scores.unsqueeze(2)) & (at < at.unsqueeze(1)))
    ids = before.sum(-1).argsort(1)[:, :top]
    chosen = p.gather(1, ids)
    return chosen / chosen.sum(1, keepdim=True) if renorm else chosen, ids


def exact(case, seed):
    c, x = case, _tokens(case, seed).double()
    if c["op"] == "matvec":
        return x @ _stored(_weight(c, seed, 0), c["df"])
    if c["op"] == "experts":
        weights, ids = _selection(c, seed)
    else:
        weights, ids = _exact_route(x, _router(c, seed), c["top"], c["renorm"])
    if c["op"] == "route":
        return weights, ids
    y = torch.zeros_like(x)
    for e in range(c["e"]):
        a = x @ _stored(_weight(c, seed, 1, e), c["df"])
        h = torch.nn.functional.silu(a) if c["act"] == "silu" else a * torch.special.ndtr(a)
        if c["gated"]:
            h = h * (x @ _stored(_weight(c, seed, 2, e), c["df"]))
        share = torch.where(ids == e, weights.double(), 0.0).sum(1, keepdim=True)
        y += share * (h @ _stored(_weight(c, seed, 3, e), c["df"]))
    return y
