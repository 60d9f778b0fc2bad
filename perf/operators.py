"""The measured calls of the expert sort's moves and of the 4-bit products: token rows moved into expert order and back with
their gradients, microscaled 4-bit quantisation, and the grouped product of 4-bit operands.

listed() names the cases, draw() gives more of the same ranges. Each case is one pass:
  permute         ids -> the sort (bounds, tok_of, row_of) and the rows in expert order
  permute_grad    gradients of the sorted rows summed back into their tokens
  unpermute       expert outputs summed back into their tokens with the routing weights
  unpermute_grad  gradients of the expert outputs and of the routing weights
  quantize        rows rounded to 4-bit floats with one power-of-two scale per 32 values, given as their values
  product         out = a w^T of 4-bit operands, each group of rows with its own expert's w
A slot whose id is outside [0, E) (a padded token, an expert over its capacity) has no row; row_of is -1 there, and the rows
behind the last sorted one stay as they were (zero here).

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


def listed():
    return [
        # one decoded token's activation sent to its ten experts: the smallest call, all latency
        dict(name="permute_1", op="permute", T=1, K=10, E=512, n=2048, type="f32", skew="flat", drop=0.0),
        # the largest prefill chunk in training precision
        dict(name="permute_8192", op="permute", T=8192, K=10, E=512, n=2560, type="bf16", skew="zipf", drop=0.0),
        # the backward pass of a 2048-token chunk with experts over their capacity and a padded tail
        dict(name="permute_grad_2048", op="permute_grad", T=2048, K=10, E=512, n=2048, type="f32", skew="zipf", drop=0.1),
        # a verify window's combine, fp16, an odd width
        dict(name="unpermute_8_odd", op="unpermute", T=8, K=8, E=128, n=1021, type="f16", skew="flat", drop=0.0),
        # a prefill chunk's combine
        dict(name="unpermute_2048", op="unpermute", T=2048, K=10, E=512, n=2560, type="bf16", skew="zipf", drop=0.0),
        # its backward pass on a ragged batch: gradients of the expert outputs and of the routing weights
        dict(name="unpermute_grad_3777", op="unpermute_grad", T=3777, K=10, E=512, n=2048, type="bf16", skew="zipf", drop=0.05),
        # one token's activation before the 4-bit products
        dict(name="quantize_1", op="quantize", rows=1, cols=2048, type="f32", spread=0.0),
        # the sorted hidden values of a chunk, magnitudes differing from row to row
        dict(name="quantize_20480", op="quantize", rows=20480, cols=2560, type="bf16", spread=2.0),
        # one decoded token through its ten experts' gate and up rows: ten groups of one row, the weights' bytes count
        dict(name="product_1", op="product", T=1, K=10, E=512, N=1024, C=2048, out="f32", skew="flat", drop=0.0, gather=True),
        # a short prompt's down products, four rows to an expert on average, dropped slots
        dict(name="product_203", op="product", T=203, K=10, E=512, N=2560, C=640, out="f32", skew="zipf", drop=0.05, gather=False),
        # a prefill chunk's gate and up products: every expert is read
        dict(name="product_2048", op="product", T=2048, K=10, E=512, N=1024, C=2048, out="bf16", skew="zipf", drop=0.0, gather=True),
        # one group: a dense projection of a whole chunk, bound by the matrix cores
        dict(name="product_dense", op="product", T=8192, K=1, E=1, N=8192, C=4096, out="bf16", skew="flat", drop=0.0, gather=False),
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["permute", "permute_grad", "unpermute", "unpermute_grad", "quantize", "product", "product", "product"])
    shape = rng.choice([BENCH, MODEL, FEW])
    routed = dict(T=_between(rng, 1, 8192), K=shape["K"], E=shape["E"], skew=rng.choice(["flat", "zipf"]), drop=rng.choice([0.0, 0.0, 0.05, 0.3]))
    if rng.random() < 0.3:
        routed["K"] = rng.randint(1, 12)
    if op == "quantize":
        cols = rng.choice([shape["n"], shape["ff"], 32 * _between(rng, 1, 128)])
        return dict(op=op, rows=min(_between(rng, 1, 81920), 20480 * 2560 // cols), cols=cols, type=rng.choice(list(TYPES)), spread=rng.choice([0.0, 2.0, 8.0]))
    if op != "product":
        n = rng.choice([shape["n"], shape["n"], _between(rng, 65, 4096)])
        kind = rng.choice(list(TYPES))
        most = 8192 * 11 * 2560 // ((routed["K"] + 1) * n * (2 if kind == "f32" else 1) * (2 if op == "unpermute_grad" else 1))
        return dict(op=op, n=n, type=kind, **dict(routed, T=min(routed["T"], most)))
    N, C = rng.choice([(2 * shape["ff"], shape["n"]), (shape["n"], shape["ff"]), (_between(rng, 33, 2048), 32 * _between(rng, 2, 80))])
    if rng.random() < 0.3:   # one group, or few
        routed.update(E=rng.choice([1, 1, 8, 16]), skew="flat")
        routed["K"] = min(routed["K"], 2, routed["E"])
    return dict(op=op, N=N, C=C, out=rng.choice(list(TYPES)), gather=rng.random() < 0.5, **routed)


# ---------------------------------------------------------------- inputs, from the seed alone

def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + what) & 0x7FFFFFFF)
    return g


def _normal(shape, g, sd=1.0):
    return torch.randn(shape, generator=g, device="cuda") * sd


def _routing(case, seed):
    """(ids [T][K] int32, weights [T][K] fp32): distinct experts of each token under the case's popularity; a share `drop` of the
    slots has no expert (half of it the batch's padded end, half single slots over an expert's capacity)."""
    T, K, E = case["T"], case["K"], case["E"]
    g = _gen(seed, 1)
    lg = _normal((T, E), g)
    if case["skew"] == "zipf":
        order = torch.randperm(E, generator=g, device="cuda")
        lg[:, order] -= 0.5 * torch.log(torch.arange(1, E + 1, device="cuda").float())
    top = torch.topk(lg, K, dim=1)
    ids, wts = top.indices.to(torch.int32), torch.softmax(top.values, 1)
    if case["drop"]:
        ids[torch.rand((T, K), generator=g, device="cuda") < case["drop"] / 2] = -1
        ids[T - int(T * case["drop"] / 2):] = -1
    return ids.contiguous(), wts.contiguous()


def _plan(ids, E):
    """(bounds, tok_of, row_of) of a stable sort of the slots by expert, slots without one left out."""
    flat = ids.reshape(-1).long()
    S, K = flat.numel(), ids.shape[1]
    key = torch.where((flat >= 0) & (flat < E), flat, E)
    order = torch.argsort(key, stable=True)
    counts = torch.zeros(E + 1, dtype=torch.int64, device="cuda").index_add_(0, key, torch.ones_like(key))
    bounds = torch.cat([counts.new_zeros(1), torch.cumsum(counts, 0)[:E]])
    rank = torch.empty_like(order)
    rank[order] = torch.arange(S, device="cuda")
    row_of = torch.where(key < E, rank, -1)
    tok_of = torch.where(torch.arange(S, device="cuda") < bounds[E], order // K, 0)
    return bounds.to(torch.int32), tok_of.to(torch.int32), row_of.to(torch.int32)


def _rows(shape, kind, g, sd=1.0):
    return _normal(shape, g, sd).to(TYPES[kind])


def _tables():
    """The values of a byte's two 4-bit codes [256][2] and of a scale byte [256], in fp32."""
    grid = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    grid += [-v for v in grid]
    pair = torch.tensor([[grid[b & 15], grid[b >> 4]] for b in range(256)], dtype=torch.float32, device="cuda")
    step = torch.tensor([math.ldexp(1.0, b - 127) for b in range(255)] + [math.nan], dtype=torch.float32, device="cuda")
    return pair, step


def _encode(x, tables):
    """(codes [..][cols / 2], scales [..][cols / 32]) of x, in 32 bits."""
    v = x.float().reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    top = v.abs().amax(-1)
    bad = ~torch.isfinite(top)
    e = torch.where(top == 0, -127, torch.frexp(torch.where(bad, 1.0, top)).exponent - 3).clamp(-127, 125)
    y = v.abs() * tables[1][127 - e].unsqueeze(-1)
    code = ((y > 0.25).to(torch.uint8) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5)) | (torch.signbit(v).to(torch.uint8) << 3)
    code = torch.where(bad.unsqueeze(-1), 0, code).to(torch.uint8).reshape(*x.shape[:-1], x.shape[-1] // 2, 2)
    return code[..., 0] | (code[..., 1] << 4), torch.where(bad, 255, e + 127).to(torch.uint8)


def _values(codes, scales, tables):
    """The fp32 values of 4-bit codes and their scales."""
    v = tables[0].index_select(0, codes.reshape(-1).int()).view(*scales.shape, 32)
    return (v * tables[1].index_select(0, scales.reshape(-1).int()).view(*scales.shape, 1)).view(*codes.shape[:-1], codes.shape[-1] * 2)


def _product_inputs(case, seed):
    ids, _ = _routing(case, seed)
    bounds, tok_of, _ = _plan(ids, case["E"])
    g, tables = _gen(seed, 2), _tables()
    aq, asc = _encode(_normal((case["T"] if case["gather"] else ids.numel(), case["C"]), g), tables)
    E, N, C = case["E"], case["N"], case["C"]
    wq = torch.empty((E, N, C // 2), dtype=torch.uint8, device="cuda")
    wsc = torch.empty((E, N, C // 32), dtype=torch.uint8, device="cuda")
    each = max(1, (1 << 27) // (N * C))
    for e in range(0, E, each):
        wq[e:e + each], wsc[e:e + each] = _encode(_normal((min(each, E - e), N, C), g, 0.02), tables)
    return bounds, tok_of if case["gather"] else None, aq, asc, wq, wsc


def _quantize_input(case, seed):
    g = _gen(seed, 2)
    x = _normal((case["rows"], case["cols"]), g)
    if case["spread"]:   # rows of different magnitude, in steps of a block now and then
        x *= torch.exp2(_normal((case["rows"], 1), g, case["spread"] / 2).clamp(-12, 12))
        x.view(case["rows"], -1, 32)[torch.rand((case["rows"], case["cols"] // 32), generator=g, device="cuda") < 0.01] = 0
    return x.to(TYPES[case["type"]])


def prepare(case, seed):
    op = case["op"]
    s = dict(case=dict(case))
    zeros = lambda *shape, dtype=torch.int32: torch.zeros(shape, dtype=dtype, device="cuda")  # noqa: E731
    if op == "quantize":
        rows, cols = case["rows"], case["cols"]
        s.update(tables=_tables(), x=_quantize_input(case, seed), codes=zeros(rows, cols // 2, dtype=torch.uint8), scales=zeros(rows, cols // 32, dtype=torch.uint8),
                 out=zeros(rows, cols, dtype=TYPES[case["type"]]))
        return s
    if op == "product":
        bounds, rows, aq, asc, wq, wsc = _product_inputs(case, seed)
        at = bounds.tolist()
        s.update(tables=_tables(), bounds=bounds, rows=rows, aq=aq, asc=asc, wq=wq, wsc=wsc, groups=[(e, at[e], at[e + 1]) for e in range(case["E"]) if at[e] < at[e + 1]],
                 out=zeros(case["T"] * case["K"], case["N"], dtype=TYPES[case["out"]]))
        s["used"] = torch.tensor([e for e, _, _ in s["groups"]], dtype=torch.int64, device="cuda")
        return s
    T, K, E, n, kind = case["T"], case["K"], case["E"], case["n"], TYPES[case["type"]]
    ids, wts = _routing(case, seed)
    g = _gen(seed, 2)
    s.update(ids=ids, wts=wts)
    if op == "permute":
        s.update(x=_rows((T, n), case["type"], g), bounds=zeros(E + 1), tok_of=zeros(T * K), slot_of=zeros(T * K), row_of=zeros(T * K),
                 xs=zeros(T * K, n, dtype=kind))
        return s
    s["bounds"], s["tok_of"], s["row_of"] = _plan(ids, E)
    if op == "permute_grad":
        s.update(dxs=_rows((T * K, n), case["type"], g), dx=zeros(T, n, dtype=kind))
    elif op == "unpermute":
        s.update(ys=_rows((T * K, n), case["type"], g), y=zeros(T, n, dtype=kind))
    else:
        s.update(ys=_rows((T * K, n), case["type"], g), dy=_rows((T, n), case["type"], g), dys=zeros(T * K, n, dtype=kind),
                 dwts=zeros(T, K, dtype=torch.float32))
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    return _library(s) if own else _plain(s)


def _library(s):
    import flashrt_amd as F
    case, op = s["case"], s["case"]["op"]
    if op == "quantize":
        F.mx4_quantize(s["x"], s["codes"], s["scales"])
        F.mx4_dequantize(s["codes"], s["scales"], s["out"])
        return {"values": s["out"]}
    if op == "product":
        F.mx4_product(s["aq"], s["asc"], s["wq"], s["wsc"], s["out"], bounds=s["bounds"], rows=s["rows"])
        return {"out": s["out"]}
    T, K, E = case["T"], case["K"], case["E"]
    if op == "permute":
        F.moe_sort(s["ids"], T, K, E, s["bounds"], s["tok_of"], s["slot_of"], s["row_of"])
        F.moe_permute(s["x"], T, K, s["row_of"], s["xs"])
        return {"bounds": s["bounds"], "tok_of": s["tok_of"], "row_of": s["row_of"], "xs": s["xs"]}
    if op == "permute_grad":
        F.moe_permute_grad(s["dxs"], T, K, s["row_of"], s["dx"])
        return {"dx": s["dx"]}
    if op == "unpermute":
        F.moe_unpermute(s["ys"], T, K, s["row_of"], s["wts"], s["y"])
        return {"y": s["y"]}
    F.moe_unpermute_grad(s["dy"], s["ys"], T, K, s["row_of"], s["wts"], s["dys"], s["dwts"])
    return {"dys": s["dys"], "dwts": s["dwts"]}


def _plain(s):
    case, op = s["case"], s["case"]["op"]
    if op == "quantize":
        return {"values": _values(*_encode(s["x"], s["tables"]), s["tables"]).to(s["x"].dtype)}
    if op == "product":
        a = _values(s["aq"], s["asc"], s["tables"])
        if s["rows"] is not None:
            a = a[s["rows"].long()]
        w = _values(s["wq"][s["used"]], s["wsc"][s["used"]], s["tables"])
        out = torch.zeros(s["out"].shape, dtype=torch.float32, device="cuda")
        for i, (_, lo, hi) in enumerate(s["groups"]):   # one product per expert with rows
            torch.mm(a[lo:hi], w[i].t(), out=out[lo:hi])
        return {"out": out.to(s["out"].dtype)}
    T, K, E, n = (case[k] for k in ("T", "K", "E", "n"))
    if op == "permute":
        bounds, tok_of, row_of = _plan(s["ids"], E)
        live = torch.arange(T * K, device="cuda") < bounds[E]
        xs = torch.where(live[:, None], s["x"][tok_of.long()], 0)
        return {"bounds": bounds, "tok_of": tok_of, "row_of": row_of, "xs": xs}
    row = s["row_of"].long()
    live = (row >= 0)[:, None]
    row = row.clamp_min(0)
    if op == "permute_grad":
        v = torch.where(live, s["dxs"][row].float(), 0)
        return {"dx": v.view(T, K, n).sum(1).to(s["dxs"].dtype)}
    y = torch.where(live, s["ys"][row].float(), 0).view(T, K, n)
    if op == "unpermute":
        return {"y": (y * s["wts"][:, :, None]).sum(1).to(s["ys"].dtype)}
    dy = s["dy"].float()[:, None, :]
    grad = (dy * s["wts"][:, :, None]).to(s["ys"].dtype).view(T * K, n)
    dys = torch.zeros((T * K + 1, n), dtype=s["ys"].dtype, device="cuda")
    dys[torch.where(live[:, 0], row, T * K)] = grad
    return {"dys": dys[:T * K], "dwts": (y * dy).sum(2)}


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    op = case["op"]
    if op == "quantize":
        return {"bytes": case["rows"] * case["cols"] * 2 * (4 if case["type"] == "f32" else 2), "flops": 0}
    T, K, E = (case[k] for k in ("T", "K", "E"))
    live = T * K * (1 - case["drop"])
    if op == "product":
        N, C = case["N"], case["C"]
        p = [r ** -0.5 for r in range(1, E + 1)] if case["skew"] == "zipf" else [1.0] * E
        hit = max(min(E, K), sum(1 - (1 - q / sum(p)) ** live for q in p))   # the experts that have rows
        a_rows = T if case["gather"] else live
        return {"bytes": 17 / 32 * C * (a_rows + hit * N) + live * N * (4 if case["out"] == "f32" else 2) + 4 * (E + 1), "flops": 2.0 * live * N * C}
    n, b = case["n"], 4 if case["type"] == "f32" else 2
    moved = (T + live) * n * b
    if op == "permute":
        return {"bytes": moved + 4 * (3 * T * K + E + 1), "flops": 0}
    if op == "unpermute_grad":
        return {"bytes": moved + live * n * b + 12 * T * K, "flops": 3.0 * live * n}
    return {"bytes": moved + (8 if op == "unpermute" else 4) * T * K, "flops": (2.0 if op == "unpermute" else 1.0) * live * n}


# ---------------------------------------------------------------- the same in 64 bits, from the definitions

def _exact_decode(codes, scales):
    codes, scales = codes.long(), scales.long()
    v = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    mag, m = (v >> 1) & 3, v & 1
    mag = torch.where(mag == 0, 0.5 * m.double(), (1 + 0.5 * m.double()) * torch.exp2(mag.double() - 1))
    step = torch.where(scales == 255, math.nan, torch.exp2(scales.double() - 127))
    return torch.where(v >= 8, -mag, mag) * step.repeat_interleave(32, -1)


def exact(case, seed):
    op = case["op"]
    if op == "quantize":
        x = _quantize_input(case, seed).double().view(case["rows"], -1, 32)
        top = x.abs().amax(-1, keepdim=True)
        e = torch.where(top > 0, torch.floor(torch.log2(top)) - 2, -127.0).clamp_min(-127)
        y = x / torch.exp2(e)
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(1))) - 1)
        return {"values": ((torch.round(y / step) * step).clamp(-6, 6) * torch.exp2(e)).view(case["rows"], -1)}
    if op == "product":
        bounds, rows, aq, asc, wq, wsc = _product_inputs(case, seed)
        a, at = _exact_decode(aq, asc), bounds.tolist()
        out = torch.zeros((case["T"] * case["K"], case["N"]), dtype=torch.float64, device="cuda")
        for e in range(case["E"]):
            if at[e] < at[e + 1]:
                part = a[at[e]:at[e + 1]] if rows is None else a[rows[at[e]:at[e + 1]].long()]
                out[at[e]:at[e + 1]] = part @ _exact_decode(wq[e], wsc[e]).T
        return {"out": out}
    T, K, E, n = (case[k] for k in ("T", "K", "E", "n"))
    ids, wts = _routing(case, seed)
    g = _gen(seed, 2)
    experts, slot = torch.sort(torch.where(ids < 0, E, ids).reshape(-1), stable=True)   # the slots in expert order
    slot = slot[experts < E]
    tok = slot // K
    if op == "permute":
        xs = torch.zeros((T * K, n), dtype=torch.float64, device="cuda")
        xs[:slot.numel()] = _rows((T, n), case["type"], g).double()[tok]
        return {"xs": xs}
    v = _rows((T * K, n), case["type"], g)[:slot.numel()].double()
    w = wts.double().view(-1)[slot, None]
    if op == "permute_grad":
        return {"dx": torch.zeros((T, n), dtype=torch.float64, device="cuda").index_add_(0, tok, v)}
    if op == "unpermute":
        return {"y": torch.zeros((T, n), dtype=torch.float64, device="cuda").index_add_(0, tok, v * w)}
    dy = _rows((T, n), case["type"], g).double()[tok]
    dys = torch.zeros((T * K, n), dtype=torch.float64, device="cuda")
    dys[:slot.numel()] = dy * w
    dw = torch.zeros(T * K, dtype=torch.float64, device="cuda")
    dw[slot] = (dy * v).sum(1)
    return {"dys": dys, "dwts": dw.view(T, K)}
