"""The measured calls of the experts' products in 16 and 32 bits with both gradients, and of activations kept in 8 bits for the backward
pass.

listed() names the cases, draw() gives more of the same ranges. Each case is one pass:
  product         out[r] = w_g a(r) for the sorted rows r of each expert g; a(r) is row r, or the token of row r
  product_grad    da[r] = w_g^T dout[r]
  product_wgrad   dw_g = the sum of dout[r] a(r)^T over the expert's rows; a in 16 or 32 bits, or in the 8-bit form
  checkpoint      rows to 8-bit codes with one power-of-two scale per 32 values, given as their values
  swiglu          h = silu(gate) up with the 8-bit copy of gate | up kept, then its backward pass from that copy: the gradient of
                  gate | up, and h again (which the down weights' gradient reads)
Rows behind the last sorted one (a slot without an expert has no row) stay as they were, zero here. A block of 32 values whose largest
magnitude is m 2^k (1 <= m < 2) has the scale 2^(k - 6) and the codes round(x / scale), at most 127 in magnitude.

Where `own` is false, run() computes the pass from elementary torch operations in 32 bits; where it is true it makes the
library's calls. exact() restates each pass in 64 bits from its definition.
"""
import math

import torch

own = False

BENCH = dict(n=2048, ff=512, E=512, K=10)    # the benchmark's layer
MODEL = dict(n=2560, ff=640, E=512, K=10)    # the model's
FEW = dict(n=1024, ff=1024, E=128, K=8)      # fewer, wider experts
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one decoded token through its ten experts' gate and up rows: ten groups of one row, the weights' bytes count
        dict(name="product_1", op="product", T=1, K=10, E=512, N=1024, C=2048, type="bf16", out="bf16", skew="flat", drop=0.0, gather=True),
        # a short prompt in an odd width, dropped slots, fp16 operands
        dict(name="product_203_odd", op="product", T=203, K=8, E=128, N=1021, C=1019, type="f16", out="f32", skew="zipf", drop=0.05, gather=False),
        # a prefill chunk's gate and up products: every expert is read, forty rows each on average
        dict(name="product_2048", op="product", T=2048, K=10, E=512, N=1024, C=2048, type="bf16", out="bf16", skew="zipf", drop=0.0, gather=True),
        # a few large experts: bound by the matrix cores
        dict(name="product_dense", op="product", T=8192, K=2, E=8, N=4096, C=4096, type="bf16", out="bf16", skew="flat", drop=0.0, gather=True),
        # back through the down products of a ragged chunk
        dict(name="product_grad_1777", op="product_grad", T=1777, K=10, E=512, N=2048, C=512, type="bf16", out="bf16", skew="zipf", drop=0.05),
        # back through the gate and up products of fewer, wider experts, fp16
        dict(name="product_grad_8192", op="product_grad", T=8192, K=8, E=128, N=2048, C=1024, type="f16", out="f16", skew="flat", drop=0.0),
        # the gate and up weights' gradients of a chunk in fp32: the results' bytes count
        dict(name="product_wgrad_2048", op="product_wgrad", T=2048, K=10, E=512, N=1280, C=2560, type="bf16", out="f32", skew="zipf", drop=0.05, gather=True, eight=False),
        # the same of fewer, wider experts from tokens that were kept in 8 bits
        dict(name="product_wgrad_8bit", op="product_wgrad", T=8192, K=8, E=128, N=2048, C=1024, type="bf16", out="bf16", skew="zipf", drop=0.0, gather=True, eight=True),
        # one token's activation kept in 8 bits and read back
        dict(name="checkpoint_1", op="checkpoint", rows=1, cols=2048, type="f32", spread=0.0),
        # a chunk's tokens, magnitudes differing from row to row
        dict(name="checkpoint_8192", op="checkpoint", rows=8192, cols=2560, type="bf16", spread=2.0),
        # a token's ten hidden rows
        dict(name="swiglu_10", op="swiglu", rows=10, ff=512, type="bf16", drop=0.0),
        # the hidden rows of the largest chunk, some slots without an expert
        dict(name="swiglu_81920", op="swiglu", rows=81920, ff=640, type="bf16", drop=0.05),
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def _cost(case):
    w = work(case)
    return w["bytes"] / 5e12 + w["flops"] / (1e14 if case["type"] == "f32" else 1.4e15)


def draw(rng):
    op = rng.choice(["product", "product", "product", "product_grad", "product_grad", "product_wgrad", "product_wgrad", "checkpoint", "swiglu"])
    shape = rng.choice([BENCH, MODEL, FEW])
    kind = rng.choice(["bf16", "f16", "bf16", "f16", "f32"])
    if op == "checkpoint":
        cols = rng.choice([shape["n"], 2 * shape["ff"], 32 * _between(rng, 1, 128)])
        return dict(op=op, rows=min(_between(rng, 1, 81920), 8192 * 2560 * 2 // cols), cols=cols, type=kind, spread=rng.choice([0.0, 2.0, 8.0]))
    if op == "swiglu":
        ff = rng.choice([shape["ff"], shape["ff"], 32 * _between(rng, 1, 64)])
        return dict(op=op, rows=min(_between(rng, 1, 81920), 81920 * 640 * 2 // (BYTES[kind] * ff)), ff=ff, type=kind, drop=rng.choice([0.0, 0.05, 0.3]))
    case = dict(op=op, T=_between(rng, 1, 8192), K=shape["K"], E=shape["E"], skew=rng.choice(["flat", "zipf"]), drop=rng.choice([0.0, 0.0, 0.05, 0.3]))
    case["N"], case["C"] = rng.choice([(2 * shape["ff"], shape["n"]), (shape["n"], shape["ff"]), (_between(rng, 33, 2048), _between(rng, 33, 2560))])
    if rng.random() < 0.3:   # one group, or few
        case.update(E=rng.choice([1, 1, 8, 16]), skew="flat")
        case["K"] = min(2, case["E"])
        if rng.random() < 0.5:
            case.update(N=128 * rng.randint(4, 32), C=128 * rng.randint(4, 32))
    case.update(type=kind, out=rng.choice([kind, "f32"]))
    if op != "product_grad":
        case["gather"] = rng.random() < 0.5
    if op == "product_wgrad":
        case["eight"] = rng.random() < 0.4
        if case["eight"]:
            case["C"] = max(32, case["C"] // 32 * 32)
    most = max(_cost(c) for c in listed() if c["op"].startswith("product"))
    while case["T"] > 1 and _cost(case) > most:
        case["T"] = case["T"] * 3 // 4
    return case


# ---------------------------------------------------------------- inputs, from the seed alone

def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + what) & 0x7FFFFFFF)
    return g


def _normal(shape, g, sd=1.0):
    return torch.randn(shape, generator=g, device="cuda") * sd


def _rows(shape, kind, g, sd=1.0):
    return _normal(shape, g, sd).to(TYPES[kind])


def _routing(case, seed):
    """ids [T][K] int32: distinct experts of each token under the case's popularity; a share `drop` of the slots has no expert (half
    of it the batch's padded end, half single slots over an expert's capacity)."""
    T, K, E = case["T"], case["K"], case["E"]
    g = _gen(seed, 1)
    lg = _normal((T, E), g)
    if case["skew"] == "zipf":
        order = torch.randperm(E, generator=g, device="cuda")
        lg[:, order] -= 0.5 * torch.log(torch.arange(1, E + 1, device="cuda").float())
    ids = torch.topk(lg, K, dim=1).indices.to(torch.int32)
    if case["drop"]:
        ids[torch.rand((T, K), generator=g, device="cuda") < case["drop"] / 2] = -1
        ids[T - int(T * case["drop"] / 2):] = -1
    return ids.contiguous()


def _plan(ids, E):
    """(bounds, tok_of) of a stable sort of the slots by expert, slots without one left out."""
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < E), flat, E)
    order = torch.argsort(key, stable=True)
    counts = torch.zeros(E + 1, dtype=torch.int64, device="cuda").index_add_(0, key, torch.ones_like(key))
    bounds = torch.cat([counts.new_zeros(1), torch.cumsum(counts, 0)[:E]])
    tok_of = torch.where(torch.arange(flat.numel(), device="cuda") < bounds[E], order // ids.shape[1], 0)
    return bounds.to(torch.int32), tok_of.to(torch.int32)


def _steps():
    """The value of a scale byte [256], in fp32."""
    return torch.tensor([math.ldexp(1.0, b - 127) for b in range(255)] + [math.nan], dtype=torch.float32, device="cuda")


def _eight(x, steps):
    """(codes, scales) of x in 8 bits."""
    v = x.float().reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    top = v.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(top)
    e = torch.where(top == 0, -127, torch.frexp(torch.where(bad, 1.0, top)).exponent - 7).clamp_min(-127)
    codes = torch.round(v * steps[127 - e]).clamp(-127, 127)
    codes = torch.where(bad, 0.0, codes).to(torch.int8).reshape(x.shape)
    return codes, torch.where(bad, 255, e + 127).squeeze(-1).to(torch.uint8)


def _values(codes, scales, steps):
    """The fp32 values of 8-bit codes and their scales."""
    return (codes.reshape(*scales.shape, 32).float() * steps[scales.int()].unsqueeze(-1)).view(codes.shape)


def _product_inputs(case, seed):
    """bounds, tok_of (None: rows in expert order) and the operands: activations and weights, output gradients and weights, or output
    gradients and activations (in 8 bits where the case says so)."""
    bounds, tok_of = _plan(_routing(case, seed), case["E"])
    op, kind, N, C = case["op"], case["type"], case["N"], case["C"]
    S = case["T"] * case["K"]
    tok_of = tok_of if case.get("gather") else None
    g = _gen(seed, 2)
    first = _rows((S, N), kind, g, 0.01) if op != "product" else None   # gradients of the results
    if op != "product_grad":
        a = _rows((S if tok_of is None else case["T"], C), kind, g)
        if op == "product_wgrad":
            return bounds, tok_of, first, _eight(a, _steps()) if case["eight"] else a
        first = a
    w = torch.empty((case["E"], N, C), dtype=TYPES[kind], device="cuda")
    each = max(1, (1 << 28) // (N * C))
    for e in range(0, case["E"], each):
        w[e:e + each] = _normal((min(each, case["E"] - e), N, C), g, 0.02)
    return bounds, tok_of, first, w


def _checkpoint_input(case, seed):
    g = _gen(seed, 2)
    x = _normal((case["rows"], case["cols"]), g)
    if case["spread"]:   # rows of different magnitude, zeros for a whole block now and then
        x *= torch.exp2(_normal((case["rows"], 1), g, case["spread"] / 2).clamp(-12, 12))
        x.view(case["rows"], -1, 32)[torch.rand((case["rows"], case["cols"] // 32), generator=g, device="cuda") < 0.01] = 0
    return x.to(TYPES[case["type"]])


def _swiglu_inputs(case, seed):
    """gate | up, the gradient of h, and the number of rows that an expert has (one int32)."""
    g, rows, ff = _gen(seed, 2), case["rows"], case["ff"]
    live = torch.tensor([rows - int(rows * case["drop"])], dtype=torch.int32, device="cuda")
    return _rows((rows, 2 * ff), case["type"], g, 1.5), _rows((rows, ff), case["type"], g, 0.01), live


def prepare(case, seed):
    op, kind = case["op"], TYPES[case["type"]]
    s = dict(case=dict(case), steps=_steps())
    zeros = lambda *shape, dtype=kind: torch.zeros(shape, dtype=dtype, device="cuda")  # noqa: E731
    if op == "checkpoint":
        rows, cols = case["rows"], case["cols"]
        s.update(x=_checkpoint_input(case, seed), codes=zeros(rows, cols, dtype=torch.int8), scales=zeros(rows, cols // 32, dtype=torch.uint8), out=zeros(rows, cols))
        return s
    if op == "swiglu":
        rows, ff = case["rows"], case["ff"]
        s["z"], s["dh"], s["live"] = _swiglu_inputs(case, seed)
        s.update(n_live=int(s["live"]), h=zeros(rows, ff), codes=zeros(rows, 2 * ff, dtype=torch.int8), scales=zeros(rows, ff // 16, dtype=torch.uint8),
                 dz=zeros(rows, 2 * ff), again=zeros(rows, ff))
        return s
    s["bounds"], s["rows"], s["left"], s["right"] = _product_inputs(case, seed)
    S, E, N, C = case["T"] * case["K"], case["E"], case["N"], case["C"]
    shape = {"product": (S, N), "product_grad": (S, C), "product_wgrad": (E, N, C)}[op]
    at = s["bounds"].tolist()
    s.update(out=zeros(*shape, dtype=TYPES[case["out"]]), groups=[(e, at[e], at[e + 1]) for e in range(E) if at[e] < at[e + 1]])
    s["used"] = torch.tensor([e for e, _, _ in s["groups"]], dtype=torch.int64, device="cuda")
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    return _library(s) if own else _plain(s)


def _library(s):
    import flashrt_amd as F
    op = s["case"]["op"]
    if op == "checkpoint":
        F.mx8_quantize(s["x"], s["codes"], s["scales"])
        F.mx8_dequantize(s["codes"], s["scales"], s["out"])
        return {"values": s["out"]}
    if op == "swiglu":
        F.moe_swiglu(s["z"], s["h"], codes=s["codes"], scales=s["scales"], live=s["live"])
        F.moe_swiglu_grad(s["dh"], s["dz"], codes=s["codes"], scales=s["scales"], h=s["again"], live=s["live"])
        return {"h": s["h"], "dz": s["dz"], "again": s["again"]}
    if op == "product":
        F.moe_product(s["left"], s["right"], s["out"], bounds=s["bounds"], rows=s["rows"])
    elif op == "product_grad":
        F.moe_product_grad(s["left"], s["right"], s["out"], bounds=s["bounds"])
    else:
        F.moe_product_wgrad(s["left"], s["right"], s["out"], bounds=s["bounds"], rows=s["rows"])
    return {"out": s["out"]}


def _gate(z, ff):
    """silu(g) u and what its gradient needs, in 32 bits: (h, g, u, the sigmoid of g)."""
    g, u = z[:, :ff], z[:, ff:]
    sig = 1 / (1 + torch.exp(-g))
    return g * sig * u, g, u, sig


def _plain(s):
    case, op = s["case"], s["case"]["op"]
    kind = TYPES[case["type"]]
    if op == "checkpoint":
        return {"values": _values(*_eight(s["x"], s["steps"]), s["steps"]).to(kind)}
    if op == "swiglu":
        n, rows, ff = s["n_live"], case["rows"], case["ff"]
        z, dh = s["z"][:n].float(), s["dh"][:n].float()
        h = _gate(z, ff)[0]
        again, g, u, sig = _gate(_values(*_eight(z, s["steps"]), s["steps"]), ff)
        dz = torch.cat([dh * u * sig * (1 + g * (1 - sig)), dh * g * sig], 1)
        fill = lambda v: torch.cat([v.to(kind), torch.zeros((rows - n, v.shape[1]), dtype=kind, device="cuda")])  # noqa: E731
        return {"h": fill(h), "dz": fill(dz), "again": fill(again)}
    out = torch.zeros(s["out"].shape, dtype=torch.float32, device="cuda")
    left = s["left"].float()
    if op == "product_wgrad":
        right = _values(*s["right"], s["steps"]).to(kind).float() if case["eight"] else s["right"].float()
        if s["rows"] is not None:
            right = right[s["rows"].long()]
        for e, lo, hi in s["groups"]:   # one product per expert with rows
            torch.mm(left[lo:hi].t(), right[lo:hi], out=out[e])
        return {"out": out.to(s["out"].dtype)}
    if s["rows"] is not None:
        left = left[s["rows"].long()]
    w = s["right"][s["used"]].float()
    for i, (_, lo, hi) in enumerate(s["groups"]):
        torch.mm(left[lo:hi], w[i].t() if op == "product" else w[i], out=out[lo:hi])
    return {"out": out.to(s["out"].dtype)}


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    op, b = case["op"], BYTES[case["type"]]
    if op == "checkpoint":
        return {"bytes": case["rows"] * case["cols"] * 2 * b, "flops": 0}
    if op == "swiglu":   # z, dh in; h, dz, h again out; the 8-bit copy written and read
        return {"bytes": (case["rows"] - int(case["rows"] * case["drop"])) * case["ff"] * (7 * b + 4 * 33 / 32), "flops": 0}
    T, K, E, N, C = (case[k] for k in ("T", "K", "E", "N", "C"))
    live = T * K * (1 - case["drop"])
    p = [r ** -0.5 for r in range(1, E + 1)] if case["skew"] == "zipf" else [1.0] * E
    hit = max(min(E, K), sum(1 - (1 - q / sum(p)) ** live for q in p))   # the experts that have rows
    a_bytes = (T if case.get("gather") else live) * C * (33 / 32 if case.get("eight") else b)
    ob = BYTES[case["out"]]
    moved = {"product": a_bytes + hit * N * C * b + live * N * ob, "product_grad": live * N * b + hit * N * C * b + live * C * ob,
             "product_wgrad": live * N * b + a_bytes + E * N * C * ob}[op]
    return {"bytes": moved + 4 * (E + 1), "flops": 2.0 * live * N * C}


# ---------------------------------------------------------------- the same in 64 bits, from the definitions

def _exact_eight(x):
    """The float64 values of x in 8 bits."""
    v = x.double().view(x.shape[0], -1, 32)
    top = v.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.where(top > 0, torch.floor(torch.log2(top)) - 6, -127.0).clamp_min(-127))
    return (torch.round(v / scale).clamp(-127, 127) * scale).view(x.shape)


def exact(case, seed):
    op = case["op"]
    if op == "checkpoint":
        return {"values": _exact_eight(_checkpoint_input(case, seed))}
    if op == "swiglu":
        z, dh, live = _swiglu_inputs(case, seed)
        n, ff = int(live), case["ff"]
        out = {k: torch.zeros((case["rows"], w), dtype=torch.float64, device="cuda") for k, w in (("h", ff), ("dz", 2 * ff), ("again", ff))}
        g, u = z[:n].double().split(ff, 1)
        out["h"][:n] = g * torch.sigmoid(g) * u
        g, u = _exact_eight(z[:n]).split(ff, 1)
        sig, d = torch.sigmoid(g), dh[:n].double()
        out["again"][:n] = g * sig * u
        out["dz"][:n, :ff] = d * u * (sig + g * sig * (1 - sig))
        out["dz"][:n, ff:] = d * g * sig
        return out
    bounds, rows, left, right = _product_inputs(case, seed)
    S, E, N, C = case["T"] * case["K"], case["E"], case["N"], case["C"]
    shape = {"product": (S, N), "product_grad": (S, C), "product_wgrad": (E, N, C)}[op]
    out, at = torch.zeros(shape, dtype=torch.float64, device="cuda"), bounds.tolist()
    if case.get("eight"):
        codes, scales = right
        right = (codes.double().view(*scales.shape, 32) * torch.exp2(scales.double() - 127).unsqueeze(-1)).view(codes.shape)
    for e in range(E):
        lo, hi = at[e], at[e + 1]
        if lo == hi:
            continue
        pick = slice(lo, hi) if rows is None else rows[lo:hi].long()
        if op == "product":
            out[lo:hi] = left[pick].double() @ right[e].double().T
        elif op == "product_grad":
            out[lo:hi] = left[lo:hi].double() @ right[e].double()
        else:
            out[e] = left[lo:hi].double().T @ right[pick].double()
    return {"out": out}
