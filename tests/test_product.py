"""The products of sorted rows with their experts' matrices and both gradients (moe_product, moe_product_grad, moe_product_wgrad) against
64-bit restatements, through the Python mirror.

Tolerances: products of two 16-bit values are exact in fp32, of two fp32 values they round with their addition. The matrix instructions do
not say how a sum rounds, so a whole step of fp32 (2^-23, relative to the partial sum, at most sum |x y|) is counted for each of the m
additions: m 2^-23 sum |x y|, first order; the result's rounding adds h |value| (h half a step of its type: fp32 2^-24, fp16 2^-11 and at
least 2^-25, bf16 2^-8); 1.01 covers the higher orders (m 2^-23 < 1e-2 at every size here). Inputs that no result may depend on (the
padding between rows, rows of no group) are NaN, outputs that no call may write hold 77."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

STEP = 2.0 ** -23
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
H_ABS = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]


def near(got, want, mag, m, kind):
    got, want, mag = got.detach().double().cpu(), want.cpu(), mag.cpu()
    err = (got - want).abs()
    bad = ~(err <= 1.01 * (m * STEP * mag + HALF[kind] * want.abs()) + H_ABS[kind])
    assert not bad.any(), (int(bad.sum()), float(err[bad].max()), np.argwhere(bad.numpy())[:4].tolist())


def rows_of(rows, cols, kind, seed, pad=0, sd=1.0):
    """A [rows][cols] matrix whose rows lie cols + pad apart, NaN between them."""
    g = torch.Generator().manual_seed(seed)
    buf = torch.full((rows + 1, cols + pad), float("nan"), dtype=kind)
    buf[:rows, :cols] = (torch.randn(rows, cols, generator=g) * sd).to(kind)
    return buf.cuda()[:rows, :cols]


def out_of(rows, cols, kind, pad=0):
    return torch.full((rows + 1, cols + pad), 77.0, dtype=kind, device="cuda")


def untouched(buf, rows, cols):
    assert (buf[rows:] == 77).all() and (buf[:, cols:] == 77).all()


def cut(sizes):
    return [0] + np.cumsum(sizes).tolist()


def i32(v):
    return None if v is None else torch.as_tensor(np.asarray(v, np.int32)).cuda()


def picked(a, rows, M):
    """The float64 rows that the products read: a[rows], zeros for an index outside."""
    if rows is None:
        return a[:M].double()
    rows = torch.as_tensor(np.asarray(rows)).to(a.device)
    ok = (rows >= 0) & (rows < a.shape[0])
    return torch.where(ok[:, None], a.double()[torch.where(ok, rows, 0)], 0.0)


def quantized(F, a):
    """a in 8 bits on the GPU, and the values that stands for in a's type."""
    codes = torch.zeros(a.shape, dtype=torch.int8, device="cuda")
    scales = torch.zeros(a.shape[0], a.shape[1] // 32, dtype=torch.uint8, device="cuda")
    F.mx8_quantize(a, codes, scales)
    back = torch.empty(a.shape, dtype=a.dtype, device="cuda")
    F.mx8_dequantize(codes, scales, back)
    return (codes, scales), back


def run(op, sizes, N, C, kind, out_kind, gather=0, eight=False, add=False, pad=0, behind=7, stream=None, seed=0):
    """One call on groups of the given sizes (None: one group without bounds, of `behind` rows) against the definition."""
    import flashrt_amd as F
    bounds = [0, behind] if sizes is None else cut(sizes)
    E, live = len(bounds) - 1, bounds[-1]
    M = live + (behind if sizes is not None else 0)
    rows = None
    if gather:
        rows = np.random.default_rng(M + seed).integers(0, gather, M)
        rows[::9], rows[1::13] = -1, gather
    b = None if sizes is None else i32(bounds)
    out_rows, out_cols = {"product": (M, N), "grad": (M, C), "wgrad": (E * N, C)}[op]
    x = rows_of(gather or M, C, kind, M + N, pad) if op != "grad" else None
    dout = rows_of(M, N, kind, M + C + 1, pad, 0.1) if op != "product" else None
    for v in (x if not gather else None, dout):
        if v is not None:
            v[live:] = float("nan")
    if op != "wgrad":
        g = torch.Generator(device="cuda").manual_seed(N + C)
        w = (torch.randn(E, N, C, generator=g, device="cuda") * 0.1).to(kind)
        arg = w if sizes is not None else w[0]
    buf = out_of(out_rows, out_cols, out_kind, 0 if op == "wgrad" else pad)
    got = buf[:out_rows, :out_cols]
    if op == "product":
        F.moe_product(x, arg, got, bounds=b, rows=i32(rows), stream=stream)
    elif op == "grad":
        F.moe_product_grad(dout, arg, got, bounds=b, stream=stream)
    else:
        a, x = quantized(F, x) if eight else (x, x)
        dw = got.view(E, N, C)
        F.moe_product_wgrad(dout, a, dw if sizes is not None else dw[0], bounds=b, rows=i32(rows), add=add, stream=stream)
    torch.cuda.synchronize()
    untouched(buf, out_rows, out_cols)
    a64 = picked(x, rows, M) if x is not None else None
    want = torch.full((out_rows, out_cols), 0.0 if op == "wgrad" else 77.0, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(want)
    m = {"product": C, "grad": N, "wgrad": max(np.diff(bounds).tolist() + [0]) + 1}[op]
    for e in range(E):
        lo, hi = bounds[e], bounds[e + 1]
        if lo == hi:
            continue
        if op == "wgrad":
            l, r, at = dout[lo:hi].double().t(), a64[lo:hi], slice(e * N, (e + 1) * N)
        else:
            l, r, at = (a64[lo:hi], w[e].double().t(), slice(lo, hi)) if op == "product" else (dout[lo:hi].double(), w[e].double(), slice(lo, hi))
        want[at], mag[at] = l @ r, l.abs() @ r.abs()
    if add:
        want, mag = want + 77.0, mag + 77.0
    near(got, want, mag, m, out_kind)
    if op == "wgrad" and add:
        for e in range(E):
            if bounds[e] == bounds[e + 1]:
                assert (got[e * N:(e + 1) * N] == 77).all()
    return got


# ---------------------------------------------------------------- refusals, on the CPU

def test_refusals_before_any_launch():
    """Shapes, types, alignments and null pointers are refused with the library's codes; nothing is launched."""
    from flashrt_amd import _lib
    L = _lib.lib()
    p = 1 << 20
    a = [None, p, 24, 5, p, p, p, 4, 9, 16, 24, 1, p, 16, 0]
    d = [None, p, 16, p, p, 4, 9, 16, 24, 30, p, 24, 0]
    w = [None, p, 16, p, 32, p, 5, p, p, 4, 9, 16, 32, 1, p, 0, 0]
    big = (1 << 30) + 1
    for fn, good, bad in ((L.frt_moe_product, a, [(1, None, -4), (1, p + 1, -1), (2, 23, -1), (3, 0, -1), (4, p + 2, -1), (5, None, -4), (5, p + 1, -1), (6, p + 2, -1),
                                                  (6, None, -1), (7, 0, -1), (7, 4097, -1), (8, -1, -1), (8, big, -1), (9, 0, -1), (9, big, -1), (10, 0, -1), (10, big, -1),
                                                  (11, 8, -1), (12, None, -4), (12, p + 2, -1), (13, 15, -1), (14, 7, -1)]),
                          (L.frt_moe_product_grad, d, [(1, None, -4), (2, 15, -1), (3, None, -4), (4, None, -1), (4, p + 1, -1), (5, 0, -1), (5, 4097, -1), (6, -1, -1),
                                                       (7, 0, -1), (8, 0, -1), (9, 3, -1), (10, None, -4), (11, 23, -1), (12, 2, -1)]),
                          (L.frt_moe_product_wgrad, w, [(1, None, -4), (2, 15, -1), (3, None, -4), (3, p + 8, -1), (4, 33, -1), (6, 0, -1), (7, p + 2, -1), (8, None, -1),
                                                        (9, 0, -1), (10, -1, -1), (11, 0, -1), (12, 48, -1), (12, 0, -1), (13, 3, -1), (14, None, -4), (14, p + 2, -1),
                                                        (15, 9, -1)])):
        for i, v, rc in bad:
            args = list(good)
            args[i] = v
            assert fn(*args) == rc, (fn.__name__, i, v, L.frt_last_error())
            assert L.frt_last_error()
    a[4], a[3] = None, 8   # fewer rows of activations than M, and none picked
    assert L.frt_moe_product(*a) == -1
    w[5], w[4] = None, 31  # rows of 16 bits closer than they are wide
    assert L.frt_moe_product_wgrad(*w) == -1
    for fn, args, i in ((L.frt_moe_product, a, 8), (L.frt_moe_product_grad, d, 6)):
        args[i] = 0
        assert fn(*args) == 0   # no rows: nothing to do


def test_python_refusals():
    import flashrt_amd as F
    z = torch.zeros
    a, w, out, b = z(4, 24), z(2, 16, 24), z(4, 16), z(3, dtype=torch.int32)
    dw = z(2, 16, 24)
    for call in (lambda: F.moe_product(a, w, out, bounds=b), lambda: F.moe_product_grad(out, w, a, bounds=b), lambda: F.moe_product_wgrad(out, a, dw, bounds=b)):
        with pytest.raises(ValueError, match="device"):
            call()
    for call in (lambda: F.moe_product(a.half(), w, out, bounds=b), lambda: F.moe_product(a, w.transpose(1, 2), out, bounds=b), lambda: F.moe_product(a, w, z(4, 17), bounds=b),
                 lambda: F.moe_product(z(4, 25), w, out, bounds=b), lambda: F.moe_product(a, w, out, bounds=b[:2]), lambda: F.moe_product(a, w, out, bounds=b.long()),
                 lambda: F.moe_product(a.double(), w.double(), out, bounds=b), lambda: F.moe_product(a, w, out, bounds=b, rows=z(3, dtype=torch.int32)),
                 lambda: F.moe_product(a, w, out.int(), bounds=b), lambda: F.moe_product(a, w[None], out, bounds=b),
                 lambda: F.moe_product_grad(out, w.half(), a, bounds=b), lambda: F.moe_product_grad(z(5, 16), w, a, bounds=b), lambda: F.moe_product_grad(out, w, z(4, 23), bounds=b),
                 lambda: F.moe_product_wgrad(out, a.half(), dw, bounds=b), lambda: F.moe_product_wgrad(out, a, dw.transpose(0, 1), bounds=b),
                 lambda: F.moe_product_wgrad(out, (z(4, 32, dtype=torch.int8), z(4, dtype=torch.uint8)), dw, bounds=b),
                 lambda: F.moe_product_wgrad(out, (z(4, 24), z(4, dtype=torch.uint8)), dw, bounds=b),
                 lambda: F.moe_product_wgrad(out, (z(4, 32, dtype=torch.int8), z(3, dtype=torch.uint8)), z(2, 16, 32), bounds=b)):
        with pytest.raises(ValueError):
            call()


def test_tensors_that_require_a_gradient_are_refused():
    import flashrt_amd as F
    z = torch.zeros
    a, w, out, b = z(4, 24), z(2, 16, 24), z(4, 16), z(3, dtype=torch.int32)
    for fn, args in ((F.moe_product, (a, w, out, b)), (F.moe_product_grad, (out, w, a, b)), (F.moe_product_wgrad, (out, a, w, b))):
        for i in range(3):
            with_grad = [v.clone().requires_grad_() if j == i else v for j, v in enumerate(args)]
            with pytest.raises(ValueError, match="requires a gradient"):
                fn(*with_grad)
            with torch.no_grad(), pytest.raises(ValueError, match="device"):
                fn(*with_grad)


# ---------------------------------------------------------------- sizes, groups, types

SIZES = [(1, 1, 1), (1, 1024, 2048), (1, 17, 96), (2, 3, 5), (3, 130, 160), (15, 16, 128), (16, 33, 64), (17, 15, 224), (40, 257, 512), (64, 64, 1056), (65, 128, 256),
         (129, 300, 1048), (200, 1000, 640), (257, 129, 357), (512, 512, 1024)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("op", ["product", "grad", "wgrad"])
@pytest.mark.parametrize("M,N,C", SIZES)
def test_one_group(M, N, C, op, kind):
    run(op, None, N, C, kind, kind if M % 2 else F32, pad=0 if M % 3 else 8, behind=M)


GROUPS = {
    "singles": [1, 0, 0, 1, 0, 1, 1, 0],
    "edges": [15, 0, 16, 17, 1, 31, 32, 33],
    "wide": [0, 63, 64, 65, 0, 127, 129, 0],
    "wider": [255, 256, 257, 3],
    "one": [0, 0, 0, 300, 0, 0, 0, 0],
    "last": [0, 0, 0, 0, 0, 0, 0, 5],
    "many": [i % 5 for i in range(203)],
    "empty": [0] * 9,
}


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("groups", list(GROUPS))
@pytest.mark.parametrize("N,C", [(96, 256), (136, 72), (131, 737)])
@pytest.mark.parametrize("op,gather", [("product", 0), ("product", 23), ("grad", 0), ("wgrad", 0), ("wgrad", 23)])
def test_groups(op, gather, groups, N, C, kind):
    """Groups of every size with rows of no group behind them; with rows: tokens picked more than once, and indices outside."""
    run(op, GROUPS[groups], N, C, kind, kind, gather=gather, pad=C % 2)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("out_kind", TYPES)
@pytest.mark.parametrize("op", ["product", "grad", "wgrad"])
@pytest.mark.parametrize("N,C,pad", [(72, 136, 8), (72, 136, 1), (33, 35, 0)])
def test_result_types(op, N, C, pad, out_kind, kind):
    run(op, [3, 0, 70, 1], N, C, kind, out_kind, pad=pad)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("groups", ["edges", "wide", "wider", "many", "empty"])
@pytest.mark.parametrize("N,C", [(96, 256), (131, 96), (200, 32)])
@pytest.mark.parametrize("gather", [0, 23])
def test_weight_gradient_from_8_bits(groups, N, C, gather, kind):
    run("wgrad", GROUPS[groups], N, C, kind, F32, gather=gather, eight=True)


@pytest.mark.gpu
@pytest.mark.parametrize("out_kind", TYPES)
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("N,C,eight", [(96, 256, False), (131, 73, False), (96, 256, True)])
def test_weight_gradient_added(N, C, eight, kind, out_kind):
    """add: the sums go on what is there, and groups without rows stay as they were."""
    run("wgrad", [5, 0, 130, 1, 0], N, C, kind, out_kind, eight=eight, add=True)


@pytest.mark.gpu
def test_weight_gradient_without_rows():
    """No rows at all (M = 0): every expert's gradient is zero; with add it stays as it was."""
    import flashrt_amd as F
    for sizes in (None, 3):
        dw = torch.full((1 if sizes is None else sizes, 20, 40), 77.0, dtype=BF16, device="cuda")
        b = None if sizes is None else torch.zeros(sizes + 1, dtype=torch.int32, device="cuda")
        dout, a = torch.empty(0, 20, dtype=BF16, device="cuda"), torch.empty(0, 40, dtype=BF16, device="cuda")
        F.moe_product_wgrad(dout, a, dw, bounds=b, add=True)
        assert (dw == 77).all()
        F.moe_product_wgrad(dout, a, dw, bounds=b)
        assert (dw == 0).all()


def ragged(n, lo, hi):
    """n group sizes between lo and hi, with an empty one and the ends among them."""
    return [lo + (37 * i) % (hi - lo + 1) for i in range(n - 3)] + [0, hi, lo]


# Shapes that each of the kernels for whole, aligned rows takes (op, group sizes, N, C, gather): the rows that are read straight into registers by
# four, two and one wave to a row, the tiles of 64 x 128, 128 x 256 and 256 x 256, with contracted values that end inside a stage.
KERNELS = {
    "rows, four waves": ("product", [1, 0, 3, 16, 17], 136, 520, 0),
    "rows, two waves": ("product", [1] * 40, 328, 264, 9),
    "rows, one wave": ("product", [2, 0, 1, 33], 200, 136, 9),
    "rows, one wave, many": ("product", ragged(30, 1, 20), 1000, 648, 0),
    "product 64": ("product", ragged(40, 0, 30), 4100, 1928, 50),
    "product 128": ("product", ragged(33, 1, 140), 1000, 1096, 0),
    "product 128, picked": ("product", ragged(33, 1, 140), 1004, 1032, 300),
    "product 256": ("product", [1111, 1300], 13320, 264, 0),
    "product 256, picked": ("product", [1536, 1027], 13316, 136, 600),
    "grad 64": ("grad", ragged(90, 0, 70), 200, 328, 0),
    "grad 128": ("grad", ragged(33, 1, 300), 264, 1000, 0),
    "grad 256": ("grad", [1111, 1300], 200, 13320, 0),
    "wgrad 64": ("wgrad", ragged(24, 0, 300), 200, 328, 0),
    "wgrad 64, picked": ("wgrad", ragged(24, 0, 300), 328, 136, 70),
    "wgrad 256": ("wgrad", ragged(70, 0, 400), 328, 520, 0),
    "wgrad 256, picked": ("wgrad", ragged(70, 0, 400), 264, 776, 70),
}


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("shape", list(KERNELS))
def test_every_kernel(shape, kind):
    op, sizes, N, C, gather = KERNELS[shape]
    run(op, sizes, N, C, kind, F32 if kind is F16 else BF16, gather=gather, pad=8)


@pytest.mark.gpu
@pytest.mark.parametrize("out_kind", TYPES)
@pytest.mark.parametrize("shape", ["rows, four waves", "product 64", "product 128", "grad 128", "wgrad 64", "wgrad 256"])
def test_result_types_of_every_kernel(shape, out_kind):
    op, sizes, N, C, gather = KERNELS[shape]
    run(op, sizes, N, C, BF16, out_kind, gather=gather, pad=8)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("shape,C", [("wgrad 64", 352), ("wgrad 64, picked", 160), ("wgrad 256", 544), ("wgrad 256, picked", 800)])
def test_8_bit_rows_in_every_kernel(shape, C, kind):
    op, sizes, N, _, gather = KERNELS[shape]
    run(op, sizes, N, C, kind, kind, gather=gather, eight=True)


@pytest.mark.gpu
@pytest.mark.parametrize("out_kind", TYPES)
@pytest.mark.parametrize("shape,eight", [("wgrad 64", False), ("wgrad 256", False), ("wgrad 256", True)])
def test_added_in_every_kernel(shape, eight, out_kind):
    op, sizes, N, C, _ = KERNELS[shape]
    run(op, sizes, N, C // 32 * 32, BF16, out_kind, eight=eight, add=True)


# Shapes that each form of the kernel for rows at any alignment takes, by tile and shares of the summed values; beside these, every call of few tiles
ANY = {
    "32 x 64 over 8, fp32": ("product", ragged(40, 0, 20), 201, 333, 0),
    "32 x 64 over 8, fp32, picked": ("product", ragged(40, 0, 20), 201, 333, 50),
    "32 x 64 over 8, fp32, gradient": ("grad", ragged(40, 0, 20), 333, 201, 0),
    "64 x 64 over 4": ("product", [70, 0, 130], 1801, 1300, 0),
    "64 x 64 over 4, gradient": ("grad", [70, 0, 130], 1300, 1801, 0),
    "64 x 64 over 4, weights": ("wgrad", [300, 0, 77], 500, 501, 0),
    "64 x 64 over 2": ("product", ragged(20, 0, 90), 1275, 1111, 60),
    "64 x 64 over 2, gradient": ("grad", ragged(20, 0, 90), 1111, 1275, 0),
    "64 x 64 over 2, weights": ("wgrad", [300, 0, 77], 700, 801, 200),
    "128 x 128": ("product", [300, 0, 411], 8261, 137, 0),
    "128 x 128, gradient": ("grad", [300, 0, 411], 137, 8261, 0),
    "128 x 128, weights": ("wgrad", ragged(6, 0, 300), 1021, 1019, 0),
}


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("shape", list(ANY))
def test_every_form_at_any_alignment(shape, kind):
    op, sizes, N, C, gather = ANY[shape]
    run(op, sizes, N, C, kind, kind, gather=gather, pad=1)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("shape,N,C", [("64 x 64 over 4, weights", 501, 480), ("64 x 64 over 2, weights", 701, 800), ("128 x 128, weights", 1021, 1024)])
def test_8_bit_rows_in_every_form(shape, N, C, add, kind):
    op, sizes, _, _, gather = ANY[shape]
    run(op, sizes, N, C, kind, F32, gather=gather, eight=True, add=add)


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["product", "grad", "wgrad"])
def test_fp32_sums_of_long_rows(op):
    """8192 values summed in fp32 in two steps, of 256 and of these, and over shares: within 300 half steps of the sum of the products' sizes, where one
    after the other may take 8192."""
    m, n = 8192, 40
    N, C, M = {"product": (n, m, 70), "grad": (m, n, 70), "wgrad": (n, n, m)}[op]
    import flashrt_amd as F
    g = torch.Generator(device="cuda").manual_seed(5)
    x, d, w = (torch.rand(*s, generator=g, device="cuda") for s in ((M, C), (M, N), (1, N, C)))
    out = torch.empty({"product": (M, N), "grad": (M, C), "wgrad": (1, N, C)}[op], device="cuda")
    if op == "product":
        F.moe_product(x, w[0], out)
        want = x.double() @ w[0].double().t()
    elif op == "grad":
        F.moe_product_grad(d, w[0], out)
        want = d.double() @ w[0].double()
    else:
        F.moe_product_wgrad(d, x, out[0])
        want = (d.double().t() @ x.double())[None]
    assert ((out.double() - want).abs() <= 300 * 2.0 ** -24 * want).all()


# ---------------------------------------------------------------- values, bounds, offsets

@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("N,C", [(72, 136), (71, 133), (5512, 5512)])
def test_infinities_and_nan_stay_in_their_rows(N, C, kind):
    """An infinity or a NaN reaches the results that it is a term of, and no other row, feature or group; the values a step past the
    end would take are not zero times it either."""
    import flashrt_amd as F
    bounds, M = [0, 3, 70, 75], 80
    a, dout = rows_of(M, C, kind, 1), rows_of(M, N, kind, 2)
    w = rows_of(3 * N, C, kind, 3).contiguous().view(3, N, C)
    b = i32(bounds)
    a[4, 7], a[69, C - 1], a[75:] = float("inf"), float("nan"), float("inf")
    out = out_of(M, N, F32)[:M]
    F.moe_product(a, w, out, bounds=b)
    bad = ~torch.isfinite(out[:75])
    assert bad[[4, 69]].all() and bad.sum() == 2 * N and out[69].isnan().all()
    assert torch.equal(out[4], torch.where(w[1, :, 7] > 0, torch.inf, -torch.inf).float())
    dout[2, N - 1], dout[74, 0], dout[75:] = float("-inf"), float("nan"), float("nan")
    da = out_of(M, C, F32)[:M]
    F.moe_product_grad(dout, w, da, bounds=b)
    bad = ~torch.isfinite(da[:75])
    assert bad[[2, 74]].all() and bad.sum() == 2 * C
    a = rows_of(M, C, kind, 1)
    a[4, 7], a[75:] = float("inf"), float("inf")
    dw = torch.empty(3, N, C, device="cuda")
    F.moe_product_wgrad(dout, a, dw, bounds=b)
    bad = ~torch.isfinite(dw)
    want = torch.zeros_like(bad)
    want[0, N - 1], want[1, :, 7], want[2, 0] = True, True, True
    assert torch.equal(bad, want) and torch.equal(dw[1, :, 7], torch.where(dout[4] > 0, torch.inf, -torch.inf).float())


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["product", "grad", "wgrad"])
@pytest.mark.parametrize("M,N,C", [(40, 64, 128), (40, 61, 127), (400, 1704, 520), (400, 520, 1704)])
def test_bounds_out_of_order_stay_inside(op, M, N, C):
    """Bounds that do not ascend, or leave [0, M], lead nowhere outside the operands and results (their results are unspecified)."""
    import flashrt_amd as F
    E = 5
    x, dout, w = rows_of(M, C, BF16, 1), rows_of(M, N, BF16, 2), rows_of(E * N, C, BF16, 3).contiguous().view(E, N, C)
    for bounds in ([0, 30, 10, 35, 20, 40], [-9, 5, 90, 7, 1 << 30, 40], [40, 30, 20, 10, 5, 0], [-(1 << 31), (1 << 31) - 1, 0, 3, -1, 50]):
        b = i32(bounds)
        rows, cols = {"product": (M, N), "grad": (M, C), "wgrad": (E * N, C)}[op]
        buf = out_of(rows + 300, cols, BF16)
        if op == "product":
            F.moe_product(x, w, buf[:M], bounds=b)
        elif op == "grad":
            F.moe_product_grad(dout, w, buf[:M], bounds=b)
        else:
            F.moe_product_wgrad(dout, x, buf[:rows].view(E, N, C), bounds=b)
        torch.cuda.synchronize()
        assert (buf[rows:] == 77).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [6, 70])
@pytest.mark.parametrize("op", ["product", "grad", "wgrad"])
def test_weights_past_32_bits(op, M):
    """The last experts of a matrix tensor of more than 2^32 values."""
    import flashrt_amd as F
    E, N, C = 1030, 2048, 2056
    big = torch.zeros((E, N, C), dtype=BF16, device="cuda")
    assert big.numel() > 2 ** 32
    x, dout, w = rows_of(M, C, BF16, 1), rows_of(M, N, BF16, 2), rows_of(2 * N, C, BF16, 3).contiguous().view(2, N, C)
    bounds = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    bounds[E - 1], bounds[E] = 4, M
    if op == "wgrad":
        big.fill_(77)
        F.moe_product_wgrad(dout, x, big, bounds=bounds)
        assert (big[:E - 2:50] == 0).all()
        for e, (lo, hi) in ((E - 2, (0, 4)), (E - 1, (4, M))):
            l, r = dout[lo:hi].double().t(), x[lo:hi].double()
            near(big[e], l @ r, l.abs() @ r.abs(), hi - lo, BF16)
        return
    big[E - 2:] = w
    out = torch.empty(M, N if op == "product" else C, device="cuda")
    if op == "product":
        F.moe_product(x, big, out, bounds=bounds)
    else:
        F.moe_product_grad(dout, big, out, bounds=bounds)
    for e, (lo, hi) in enumerate(((0, 4), (4, M))):
        l, r = (x[lo:hi].double(), w[e].double().t()) if op == "product" else (dout[lo:hi].double(), w[e].double())
        near(out[lo:hi], l @ r, l.abs() @ r.abs(), C if op == "product" else N, F32)


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["product", "grad", "wgrad"])
def test_rows_far_apart(op):
    """Operands and results whose rows lie so far apart that their offsets pass 32 bits, also in bytes within one tile."""
    import flashrt_amd as F
    M, N, C, far = 70, 40, 72, 1 << 26
    base = torch.empty(M * far, dtype=BF16, device="cuda")   # 9.4 GB
    spread = lambda at, cols: base[at:].as_strided((M, cols), (far, 1))  # noqa: E731
    w = rows_of(2 * N, C, BF16, 3).contiguous().view(2, N, C)
    b, bounds = i32([0, 3, M]), [0, 3, M]
    x, dout, out = spread(0, C), spread(1000, N), spread(3000, C if op == "grad" else N)
    x.copy_(rows_of(M, C, BF16, 1))
    dout.copy_(rows_of(M, N, BF16, 2))
    dw = torch.empty(2, N, C, device="cuda")
    if op == "product":
        F.moe_product(x, w, out, bounds=b)
    elif op == "grad":
        F.moe_product_grad(dout, w, out, bounds=b)
    else:
        F.moe_product_wgrad(dout, x, dw, bounds=b)
    for e in range(2):
        lo, hi = bounds[e], bounds[e + 1]
        l, r, got = {"product": (x[lo:hi], w[e].t(), out[lo:hi]), "grad": (dout[lo:hi], w[e], out[lo:hi]), "wgrad": (dout[lo:hi].t(), x[lo:hi], dw[e])}[op]
        l, r = l.double(), r.double()
        near(got, l @ r, l.abs() @ r.abs(), {"product": C, "grad": N, "wgrad": hi - lo}[op], got.dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,N,M", [(BF16, 8, (1 << 30) - 3), (F32, 8, (1 << 28) + 5), (F32, 2, (1 << 30) - 3)])
def test_more_rows_than_one_grid_dimension(kind, N, M):
    """Nearly 2^30 rows of eight values (two, or 2^28 rows, in fp32): more workgroups than one dimension of a launch holds, offsets past 32 bits. The
    rows repeat, in small whole numbers, so that every sum is exact."""
    import flashrt_amd as F
    n = 1 << 16
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = torch.randint(-8, 9, (n, N), generator=g, device="cuda").to(kind)
    w = torch.randint(-8, 9, (N, N), generator=g, device="cuda").to(kind)
    a = rows.repeat((M + n - 1) // n, 1)[:M]
    out = torch.empty(M, N, dtype=kind, device="cuda")
    F.moe_product(a, w, out)
    want = (rows.double() @ w.double().t()).to(kind)
    for r in range(0, M, n):
        m = min(n, M - r)
        if r // n % 64 == 0 or m < n:
            assert torch.equal(out[r:r + m], want[:m]), r


@pytest.mark.gpu
def test_largest_weights_of_the_type():
    """fp16 results beyond the type's range become infinities as a conversion's do, and sums stay in fp32 on the way."""
    import flashrt_amd as F
    M, N, C = 40, 48, 256
    x, w = torch.full((M, C), 256.0, dtype=F16, device="cuda"), torch.full((N, C), 256.0, dtype=F16, device="cuda")
    w[1::2, 1::2] = -256
    out = torch.empty(M, N, dtype=F16, device="cuda")
    F.moe_product(x, w, out)
    assert (out[:, ::2] == torch.inf).all() and (out[:, 1::2] == 0).all()


# ---------------------------------------------------------------- in use

@pytest.mark.gpu
@pytest.mark.parametrize("N,C", [(136, 264), (4104, 4104)])
def test_other_stream_and_graph(N, C):
    """The three calls on a stream of their own, and captured and replayed on new inputs with eager work between; results are the same
    bits every time."""
    import flashrt_amd as F
    M, E = 90, 5
    v = dict(a=torch.zeros(M, C, dtype=BF16, device="cuda"), d=torch.zeros(M, N, dtype=BF16, device="cuda"), w=rows_of(E * N, C, BF16, 3).contiguous().view(E, N, C),
             b=torch.zeros(E + 1, dtype=torch.int32, device="cuda"), out=torch.zeros(M, N, dtype=BF16, device="cuda"), da=torch.zeros(M, C, dtype=BF16, device="cuda"),
             dw=torch.zeros(E, N, C, device="cuda"))

    def step(v, stream=None):
        F.moe_product(v["a"], v["w"], v["out"], bounds=v["b"], stream=stream)
        F.moe_product_grad(v["d"], v["w"], v["da"], bounds=v["b"], stream=stream)
        F.moe_product_wgrad(v["d"], v["a"], v["dw"], bounds=v["b"], stream=stream)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(v)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(v)
    for seed in range(4):
        v["a"].copy_(rows_of(M, C, BF16, seed))
        v["d"].copy_(rows_of(M, N, BF16, seed + 9))
        v["b"].copy_(torch.tensor([0, 0, 10 + seed, 30, 30, 80 - seed], dtype=torch.int32))
        for k in ("out", "da", "dw"):
            v[k].fill_(5)
        want = {k: t.clone() for k, t in v.items()}
        side.wait_stream(torch.cuda.current_stream())
        step(want, side)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for k in v:
            assert torch.equal(v[k], want[k]), (seed, k)


@pytest.mark.gpu
def test_written_tensors_count_as_changed():
    import flashrt_amd as F
    a, w, out, da, dw = (torch.zeros(s, device="cuda") for s in ((4, 8), (6, 8), (4, 6), (4, 8), (6, 8)))
    everything = [a, w, out, da, dw]
    for o, call in ((out, lambda: F.moe_product(a, w, out)), (da, lambda: F.moe_product_grad(out, w, da)), (dw, lambda: F.moe_product_wgrad(out, a, dw))):
        was = [v._version for v in everything]
        call()
        for v, old in zip(everything, was):
            assert v._version == old + (v is o)


@pytest.mark.gpu
def test_gradients_against_differences():
    """Directional derivatives of sum(out * r) by the activations and the weights. The products are linear in each, so a difference over
    any step is the derivative but for rounding: both sides are sums of fp32 results whose error the bound counts."""
    import flashrt_amd as F
    sizes, N, C = [4, 0, 33], 40, 56
    bounds, M = cut(sizes), 37
    b = i32(bounds)
    a, da, r = rows_of(M, C, F32, 1), rows_of(M, C, F32, 2), rows_of(M, N, F32, 3)
    w, dwt = (rows_of(3 * N, C, F32, s).contiguous().view(3, N, C) for s in (4, 5))

    def f(a, w):
        out = torch.empty(M, N, device="cuda")
        F.moe_product(a, w, out, bounds=b)
        return (out.double() * r.double()).sum()

    ga, gw = torch.empty(M, C, device="cuda"), torch.empty(3, N, C, device="cuda")
    F.moe_product_grad(r, w, ga, bounds=b)
    F.moe_product_wgrad(r, a, gw, bounds=b)
    size = lambda x, y: float(sum((x[lo:hi].abs().double() @ y[e].abs().double().t() * r[lo:hi].abs().double()).sum() for e, (lo, hi) in enumerate(zip(bounds, bounds[1:]))))  # noqa: E731
    # one step of fp32 for the input's own addition and C + 1 for the sum, twice; the derivative's own sums: N or M terms
    for got, want, mag in (((f(a + da, w) - f(a, w)), (ga.double() * da.double()).sum(), size(a.abs() + da.abs(), w)),
                           ((f(a, w + dwt) - f(a, w)), (gw.double() * dwt.double()).sum(), size(a, w.abs() + dwt.abs()))):
        assert abs(float(got - want)) <= 1.01 * (2 * (C + 2) + M + N) * STEP * mag, (float(got), float(want))


def missing(M, tokens):
    """Row indices of which every third lies outside [0, tokens), and which those are."""
    rows = np.random.default_rng(M).integers(0, tokens, M)
    rows[::3] = np.resize([-1, tokens, -(2 ** 31), 2 ** 31 - 1], rows[::3].size)
    out = np.zeros(M, bool)
    out[::3] = True
    return i32(rows), torch.from_numpy(out).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("shape", [k for k, v in {**KERNELS, **ANY}.items() if v[0] == "product"])
def test_missing_rows_times_infinities(shape, kind):
    """A row whose index lies outside is zeros in the sums of every kernel: an infinite or NaN weight times it gives NaN, a finite one 0. (fp32
    rows of any of these shapes take the kernel for rows at any alignment.)"""
    import flashrt_amd as F
    _, sizes, N, C, _ = {**KERNELS, **ANY}[shape]
    pad, E, M, tokens = 1 if shape in ANY else 8, len(sizes), sum(sizes), 50
    x, (rows, out_rows) = rows_of(tokens, C, kind, 1, pad), missing(M, tokens)
    w = rows_of(E * N, C, kind, 2).contiguous().view(E, N, C)
    w[:, 1, 3], w[:, N - 1, C - 1] = float("inf"), float("nan")
    out = out_of(M, N, F32)[:M]
    F.moe_product(x, w, out, bounds=i32(cut(sizes)), rows=rows)
    lost = out[out_rows]
    assert lost[:, [1, N - 1]].isnan().all()
    lost[:, [1, N - 1]] = 0
    assert (lost == 0).all()
    there, a = out[~out_rows], x[rows[~out_rows].long(), 3].float()
    assert torch.equal(there[:, 1], torch.where(a > 0, torch.inf, -torch.inf)) and there[:, N - 1].isnan().all()
    there[:, [1, N - 1]] = 0
    assert torch.isfinite(there).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("shape", [k for k, v in {**KERNELS, **ANY}.items() if v[0] == "wgrad"])
def test_missing_rows_in_the_weight_gradient(shape, eight, kind):
    """The same in the weights' gradient: an infinity or a NaN of such a row's output gradient gives NaN in its feature, and its finite ones add
    nothing."""
    import flashrt_amd as F
    _, sizes, N, C, _ = {**KERNELS, **ANY}[shape]
    pad, E, M, tokens = 1 if shape in ANY else 8, len(sizes), sum(sizes), 50
    C = C // 32 * 32 if eight else C
    x, (rows, out_rows) = rows_of(tokens, C, kind, 1, 0 if eight else pad), missing(M, tokens)
    dout = rows_of(M, N, kind, 3, pad)
    dout[out_rows, 1], dout[out_rows, N - 1] = float("-inf"), float("nan")
    clean = dout.clone()
    clean[out_rows] = 0
    a = quantized(F, x)[0] if eight else x
    dw, want = (torch.full((E, N, C), 77.0, device="cuda") for _ in range(2))
    F.moe_product_wgrad(dout, a, dw, bounds=i32(cut(sizes)), rows=rows)
    F.moe_product_wgrad(clean, a, want, bounds=i32(cut(sizes)), rows=rows.clamp(0, tokens - 1))
    at = cut(sizes)
    hit = torch.tensor([bool(out_rows[lo:hi].any()) for lo, hi in zip(at, at[1:])], device="cuda")
    assert dw[hit][:, [1, N - 1]].isnan().all()
    dw[hit, 1], dw[hit, N - 1] = want[hit, 1], want[hit, N - 1]
    assert torch.isfinite(want).all() and torch.equal(dw, want)


# The last feature tile (1, 3 or 5 features in it) ends inside a piece of 16 bytes: its results leave value by value, by as few instructions as one.
CUT_SHORT = {
    "product 64": (ragged(40, 0, 30), 4096, 1928),
    "product 128": (ragged(33, 1, 140), 1024, 1096),
    "product 256": ([1111, 1300], 13312, 264),
}


@pytest.mark.gpu
@pytest.mark.parametrize("out_kind", TYPES)
@pytest.mark.parametrize("more", [1, 3, 5])
@pytest.mark.parametrize("shape", list(CUT_SHORT))
def test_feature_tiles_cut_inside_a_piece(shape, more, out_kind):
    """Such a workgroup waits for all its loads into LDS before it ends, which its own results do not show: the same call eight times without a pause,
    whose workgroups follow one another in the same LDS, gives the same bits eight times, and the values are right."""
    import flashrt_amd as F
    sizes, N, C = CUT_SHORT[shape]
    want = run("product", sizes, N + more, C, BF16, out_kind, behind=0)
    M, b = sum(sizes), i32(cut(sizes))
    x = rows_of(M, C, BF16, M + N + more)
    g = torch.Generator(device="cuda").manual_seed(N + more + C)
    w = (torch.randn(len(sizes), N + more, C, generator=g, device="cuda") * 0.1).to(BF16)
    outs = torch.empty(8, M, N + more, dtype=out_kind, device="cuda")
    for o in outs:
        F.moe_product(x, w, o, bounds=b)
    assert all(torch.equal(o, want) for o in outs)


# Shapes of which a workgroup takes several feature tiles one after another, as one sequence of stages: (op, group sizes, N, C), the tile, the feature
# tiles of a row tile and of a workgroup (the last workgroup of a row tile has fewer in those of 5 / 3 and 5 / 2), the stages of an average group
SEQUENCES = {
    "wgrad 256: 3 / 3, 7": ("wgrad", ragged(128, 0, 400), 1032, 544),
    "wgrad 256: 4 / 4, 1 (short groups)": ("wgrad", ragged(300, 0, 60), 520, 800),
    "wgrad 64: 5 / 3, 3": ("wgrad", ragged(64, 0, 300), 200, 640),
    "grad 128: 5 / 2, 4": ("grad", ragged(200, 17, 60), 200, 1040),
    "grad 64: 9 / 5, 4": ("grad", ragged(300, 0, 30), 200, 1032),
    "grad 64: 5 / 5, 3": ("grad", ragged(600, 0, 25), 136, 520),
    "grad 64: 8 / 1, 4 (several row tiles to a group)": ("grad", ragged(20, 0, 200), 200, 1000),
    "product 128: 4 / 2, 3": ("product", ragged(200, 17, 60), 1021, 136),
    "product 64: 8 / 3, 11": ("product", ragged(600, 0, 25), 1021, 648),
}


@pytest.mark.gpu
@pytest.mark.parametrize("kind,out_kind", [(F16, F32), (BF16, BF16)])
@pytest.mark.parametrize("gather", [0, 70])
@pytest.mark.parametrize("shape", [k for k, v in SEQUENCES.items() if v[0] != "grad"])
def test_sequences_of_feature_tiles(shape, gather, kind, out_kind):
    op, sizes, N, C = SEQUENCES[shape]
    run(op, sizes, N, C, kind, out_kind, gather=gather, pad=8)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,out_kind", [(F16, F32), (BF16, BF16)])
@pytest.mark.parametrize("shape", [k for k, v in SEQUENCES.items() if v[0] == "grad"])
def test_sequences_of_feature_tiles_in_the_row_gradient(shape, kind, out_kind):
    op, sizes, N, C = SEQUENCES[shape]
    run(op, sizes, N, C, kind, out_kind, pad=8)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,out_kind", [(F16, F16), (BF16, F32)])
@pytest.mark.parametrize("gather", [0, 70])
@pytest.mark.parametrize("eight,add", [(True, False), (False, True), (True, True)])
@pytest.mark.parametrize("shape", [k for k, v in SEQUENCES.items() if v[0] == "wgrad"])
def test_sequences_of_feature_tiles_from_8_bits_and_added(shape, eight, add, gather, kind, out_kind):
    op, sizes, N, C = SEQUENCES[shape]
    run(op, sizes, N, C, kind, out_kind, gather=gather, eight=eight, add=add, pad=8)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("N", [768, 769, 1536, 1537])
@pytest.mark.parametrize("C", [256, 512, 1160])
def test_few_rows_at_the_limits_of_their_waves(C, N, kind):
    """Sixteen groups of one row, of as many tiles of 16 x 16 as four or two waves to a row are taken for, and of one more."""
    run("product", [1] * 16, N, C, kind, kind, gather=9, pad=8)
