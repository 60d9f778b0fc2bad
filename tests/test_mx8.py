"""Activations in 8 bits (mx8_quantize, mx8_dequantize) and the experts' gated activation with its backward pass from them (moe_swiglu,
moe_swiglu_grad) against 64-bit restatements.

Codes and scales are compared bit for bit. swiglu's tolerances: u = 2^-24 is half a step of fp32. exp is taken to be off by at most 4 steps of
its result plus what its argument's own rounding to a multiple of log2(e) moves it: |g| u relative, |g| < 90 here. In s = 1 / (1 + e) that
error counts with e / (1 + e) < 1, the addition and the reciprocal add 3 u, so s is off by (8 + 3 + 2 |g|) u relative: S. 1 - s then by S s + u.
h has three more roundings, dg the errors of its parts; the result's rounding adds h |value| (h half a step of the type: fp32 2^-24, fp16
2^-11 and at least 2^-25, bf16 2^-8)."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
H_ABS = {F32: 2.0 ** -149, F16: 2.0 ** -25, BF16: 2.0 ** -134}
TYPES = [F32, F16, BF16]


def near(got, want, bound, kind):
    err = (got.detach().cpu().double() - want).abs()
    bad = ~(err <= 1.01 * (bound + HALF[kind] * want.abs()) + H_ABS[kind])
    assert not bad.any(), (int(bad.sum()), float(err[bad].max()), np.argwhere(bad.numpy())[:4].tolist())


def ref_quantize(x):
    """(codes, scales) of float64 rows from the definition."""
    rows, cols = x.shape
    v = x.reshape(rows, cols // 32, 32)
    top = np.abs(v).max(2)
    bad = ~np.isfinite(top)
    with np.errstate(all="ignore"):
        k = np.where(top > 0, np.floor(np.log2(np.where(bad, 1.0, top))), -1000)
        b = np.maximum(k - 6, -127) + 127
        codes = np.clip(np.rint(np.where(bad[:, :, None], 0.0, v) * np.exp2(127 - b)[:, :, None]), -127, 127)
    return codes.reshape(rows, cols).astype(np.int8), np.where(bad, 255, b).astype(np.uint8)


def values(codes, scales):
    step = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return codes.astype(np.float64) * np.repeat(step, 32, -1)


def gpu_quantize(F, x):
    codes = torch.full(x.shape, 0x5E, dtype=torch.int8, device="cuda")
    scales = torch.full((x.shape[0], x.shape[1] // 32), 0xEE, dtype=torch.uint8, device="cuda")
    F.mx8_quantize(x, codes, scales)
    return codes, scales


def same(got, codes, scales):
    assert np.array_equal(got[1].cpu().numpy(), scales), np.argwhere(got[1].cpu().numpy() != scales)[:4]
    assert np.array_equal(got[0].cpu().numpy(), codes), np.argwhere(got[0].cpu().numpy() != codes)[:4]


def matrix(rows, cols, kind, seed, pad=0, sd=1.0):
    g = torch.Generator().manual_seed(seed)
    buf = torch.full((rows + 1, cols + pad), float("nan"), dtype=kind)
    buf[:rows, :cols] = (torch.randn(rows, cols, generator=g) * sd).to(kind)
    return buf.cuda()[:rows, :cols]


# ---------------------------------------------------------------- refusals, on the CPU

def test_refusals_before_any_launch():
    from flashrt_amd import _lib
    L = _lib.lib()
    p = 1 << 20
    q = [None, p, 64, 0, 3, 64, p, p]
    d = [None, p, p, 3, 64, p, 64, 0]
    s = [None, p, 64, 1, 3, 32, p, p, 32, p, p]
    g = [None, p, 32, None, 0, p, p, 1, 3, 32, p, p, 64, p, 32]
    for fn, good, bad in ((L.frt_mx8_quantize, q, [(2, 63, -1), (3, 8, -1), (4, -1, -1), (5, 48, -1), (5, 0, -1), (1, None, -4), (6, None, -4), (7, None, -4), (6, p + 8, -1),
                                                   (1, p + 2, -1)]),
                          (L.frt_mx8_dequantize, d, [(6, 63, -1), (7, 2, -1), (3, -1, -1), (4, 16, -1), (1, None, -4), (2, None, -4), (5, None, -4), (1, p + 1, -1),
                                                     (5, p + 1, -1)]),
                          (L.frt_moe_swiglu, s, [(1, None, -4), (1, p + 1, -1), (2, 63, -1), (3, 8, -1), (4, -1, -1), (5, 0, -1), (5, 48, -1), (5, (1 << 29) + 32, -1), (6, p + 2, -1),
                                                 (7, None, -4), (8, 31, -1), (9, None, -4), (10, None, -4), (9, p + 4, -1)]),
                          (L.frt_moe_swiglu_grad, g, [(1, None, -4), (2, 31, -1), (3, p, -1), (5, None, -4), (6, None, -4), (5, p + 8, -1), (7, 2, -1), (8, -1, -1), (9, 0, -1),
                                                      (9, 48, -1), (10, p + 1, -1), (11, None, -4), (12, 63, -1), (13, p + 1, -1), (14, 31, -1)])):
        for i, v, rc in bad:
            a = list(good)
            a[i] = v
            assert fn(*a) == rc, (fn.__name__, i, v, L.frt_last_error())
            assert L.frt_last_error()
    g[5] = g[6] = None   # neither z nor its codes
    assert L.frt_moe_swiglu_grad(*g) == -4
    for fn, good, i in ((L.frt_mx8_quantize, q, 4), (L.frt_mx8_dequantize, d, 3), (L.frt_moe_swiglu, s, 4), (L.frt_moe_swiglu_grad, g, 8)):
        a = list(good)
        a[i] = 0
        assert fn(*a) == 0   # no rows: nothing to do


def test_python_refusals():
    import flashrt_amd as F
    z = torch.zeros
    i8, u8 = (lambda *s: z(s, dtype=torch.int8)), (lambda *s: z(s, dtype=torch.uint8))
    x, h, dz = z(4, 64), z(4, 32), z(4, 64)
    for call in (lambda: F.mx8_quantize(x, i8(4, 64), u8(4, 2)), lambda: F.mx8_dequantize(i8(4, 64), u8(4, 2), x), lambda: F.moe_swiglu(x, h),
                 lambda: F.moe_swiglu(x, h, i8(4, 64), u8(4, 2)), lambda: F.moe_swiglu_grad(h, dz, z=x), lambda: F.moe_swiglu_grad(h, dz, codes=i8(4, 64), scales=u8(4, 2), h=h)):
        with pytest.raises(ValueError, match="device"):
            call()
    for call in (lambda: F.mx8_quantize(x, i8(4, 63), u8(4, 2)), lambda: F.mx8_quantize(x, i8(4, 64), u8(4, 1)), lambda: F.mx8_quantize(x.double(), i8(4, 64), u8(4, 2)),
                 lambda: F.mx8_quantize(x, u8(4, 64), u8(4, 2)), lambda: F.mx8_quantize(x.t(), i8(64, 4), u8(64, 1)), lambda: F.moe_swiglu(x, z(4, 31)), lambda: F.moe_swiglu(x, h.half()),
                 lambda: F.moe_swiglu(x, h, codes=i8(4, 64)), lambda: F.moe_swiglu(x, h, scales=u8(4, 2)), lambda: F.moe_swiglu(x, h, live=z(1)),
                 lambda: F.moe_swiglu(x, h, live=z(0, dtype=torch.int32)), lambda: F.moe_swiglu_grad(h, dz), lambda: F.moe_swiglu_grad(h, dz, z=x, codes=i8(4, 64), scales=u8(4, 2)),
                 lambda: F.moe_swiglu_grad(h, dz, codes=i8(4, 64)), lambda: F.moe_swiglu_grad(h, z(4, 63), z=x), lambda: F.moe_swiglu_grad(h, dz, z=x, h=z(3, 32))):
        with pytest.raises(ValueError):
            call()
    for i in range(3):   # a gradient that would be lost
        z_, h_, d_ = (v.clone().requires_grad_() if j == i else v for j, v in enumerate((x, h, dz)))
        with pytest.raises(ValueError, match="requires a gradient"):
            F.moe_swiglu_grad(h_, d_, z=z_)
        with torch.no_grad(), pytest.raises(ValueError, match="device"):
            F.moe_swiglu_grad(h_, d_, z=z_)


def test_reference_rounds_to_even_codes():
    """The restatement itself: ties, the clipped end, zeros."""
    x = np.zeros((1, 32))
    x[0, :9] = [64, 0.5, 1.5, 2.5, -0.5, -1.5, 127.5, -127.9, 126.5]
    codes, scales = ref_quantize(x)
    assert scales[0, 0] == 127 and codes[0, :9].tolist() == [64, 0, 2, 2, 0, -2, 127, -127, 126]


# ---------------------------------------------------------------- quantisation

@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,cols,pad", [(1, 32, 0), (1, 2048, 0), (3, 96, 0), (7, 640, 5), (129, 2560, 0), (1000, 544, 3)])
def test_quantize(rows, cols, pad, kind):
    import flashrt_amd as F
    x = matrix(rows, cols, kind, rows, pad)
    x *= torch.exp2(torch.arange(rows, device="cuda") % 17 - 8)[:, None].to(kind)
    got = gpu_quantize(F, x)
    codes, scales = ref_quantize(x.cpu().double().numpy())
    same(got, codes, scales)
    buf = torch.full((rows, cols + pad), 77.0, dtype=kind, device="cuda")
    F.mx8_dequantize(*got, buf[:, :cols])
    assert torch.equal(buf[:, :cols].cpu().double(), torch.from_numpy(values(codes, scales)).to(kind).double())
    assert (buf[:, cols:] == 77).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
def test_quantize_every_exponent(kind):
    """Blocks whose largest value takes every exponent of the type, with ties, their neighbours, both ends and both zeros. What was
    kept of a finite value of the type is finite in the type."""
    import flashrt_amd as F
    fi = torch.finfo(kind)
    lo, hi = int(np.log2(fi.smallest_normal)) - int(-np.log2(fi.eps)), int(np.log2(fi.max))
    eps = float(fi.eps)
    tie = np.array([0.5, 1.5, 2.5, 63.5, 64.5, 126.5, 127.5])
    pat = np.concatenate([[64.0, 128 * (1 - eps / 2), 127.0, 1.0, 0.0, -0.0], tie, -tie, tie[:5] * (1 + eps), tie[:5] * (1 - eps)])
    assert pat.size <= 32
    blk = np.zeros((hi - lo + 1, 32))
    for i, k in enumerate(range(lo, hi + 1)):
        blk[i, :pat.size] = np.clip(pat * 2.0 ** (k - 6), -float(fi.max), float(fi.max))
    x = torch.from_numpy(blk).to(kind)
    got = gpu_quantize(F, x.cuda())
    codes, scales = ref_quantize(x.double().numpy())
    same(got, codes, scales)
    back = torch.empty(x.shape, dtype=kind, device="cuda")
    F.mx8_dequantize(*got, back)
    assert torch.isfinite(back).all() and torch.equal(back.cpu().double(), torch.from_numpy(values(codes, scales)).to(kind).double())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
def test_quantize_zeros_infinities_nan(kind):
    import flashrt_amd as F
    x = torch.ones(6, 96, dtype=kind)
    x[0], x[1, 40], x[2, 33], x[3, 63], x[4, 32:64] = 0, float("inf"), float("nan"), float("-inf"), -0.0
    codes, scales = gpu_quantize(F, x.cuda())
    s = scales.cpu()
    assert (s[0] == 0).all() and s[4, 1] == 0 and (s[1:4, 1] == 255).all() and (s[1:4, ::2] == 121).all()
    assert (codes.cpu()[1:5, 32:64] == 0).all()
    y = torch.empty(6, 96, dtype=kind, device="cuda")
    F.mx8_dequantize(codes, scales, y)
    y = y.cpu()
    assert y[1:4, 32:64].isnan().all() and (y[1:4, :32] == 1).all() and (y[1:4, 64:] == 1).all() and (y[0] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
def test_dequantize_every_code_and_scale(kind):
    import flashrt_amd as F
    scales = np.arange(256, dtype=np.uint8).repeat(8).reshape(256, 8)
    codes = np.tile(np.arange(-128, 128).astype(np.int8), (256, 1))
    out = torch.empty(256, 256, dtype=kind, device="cuda")
    F.mx8_dequantize(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), out)
    with np.errstate(over="ignore", invalid="ignore"):
        want = torch.from_numpy(values(codes, scales).astype(np.float32)).to(kind)   # (every value but the largest is an fp32 number)
    assert torch.equal(out.cpu().isnan(), want.isnan()) and torch.equal(out.cpu().nan_to_num(0.25), want.nan_to_num(0.25))


# ---------------------------------------------------------------- the gated activation

def ref_swiglu(z, dh):
    """(h, its error, dz, its error) of float64 z and dh, the errors relative to the roundings named above and without the results' own."""
    ff = z.shape[1] // 2
    g, u = z[:, :ff], z[:, ff:]
    s = torch.sigmoid(g)
    S = (11 + 2 * g.abs()) * U
    h, dg, du = g * s * u, dh * u * s * (1 + g * (1 - s)), dh * g * s
    inner = g.abs() * (S * s + U + U) + U * (1 + (g * (1 - s)).abs())   # of 1 + g (1 - s)
    e_dg = (dh * u).abs() * s * (inner + (S + 4 * U) * (1 + g * (1 - s)).abs())
    return h, h.abs() * (S + 3 * U), torch.cat([dg, du], 1), torch.cat([e_dg, du.abs() * (S + 3 * U)], 1)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,ff,pad", [(1, 1, 0), (1, 512, 0), (2, 5, 1), (3, 8, 0), (5, 33, 3), (64, 96, 0), (130, 640, 8), (700, 61, 0)])
@pytest.mark.parametrize("kept", [False, True])
def test_swiglu(kept, rows, ff, pad, kind):
    """h, the 8-bit copy, and the gradient from z or from the copy; rows behind `live` stay as they were, whatever they hold."""
    import flashrt_amd as F
    if kept:
        ff = (ff + 31) // 32 * 32
    live = rows - rows // 3
    z, dh = matrix(rows, 2 * ff, kind, rows + ff, pad, 3.0), matrix(rows, ff, kind, ff, pad)
    z[live:], dh[live:] = float("nan"), float("inf")
    n = torch.tensor([live], dtype=torch.int32, device="cuda")
    new = lambda cols: torch.full((rows + 1, cols + pad), 77.0, dtype=kind, device="cuda")  # noqa: E731
    h, dz, again = new(ff), new(2 * ff), new(ff)
    got_h, got_dz, got_again = h[:rows, :ff], dz[:rows, :2 * ff], again[:rows, :ff]
    src = z[:live].cpu().double()
    if kept:
        codes = torch.full((rows, 2 * ff), 0x5E, dtype=torch.int8, device="cuda")
        scales = torch.full((rows, ff // 16), 0xEE, dtype=torch.uint8, device="cuda")
        F.moe_swiglu(z, got_h, codes, scales, live=n)
        rc, rs = ref_quantize(src.numpy())
        same((codes[:live], scales[:live]), rc, rs)
        assert (codes[live:] == 0x5E).all() and (scales[live:] == 0xEE).all()
        F.moe_swiglu_grad(dh, got_dz, codes=codes, scales=scales, h=got_again, live=n)
        back = torch.from_numpy(values(rc, rs))
    else:
        F.moe_swiglu(z, got_h, live=n)
        F.moe_swiglu_grad(dh, got_dz, z=z, h=got_again, live=n)
        back = src
    d64 = dh[:live].cpu().double()
    want_h, e_h, _, _ = ref_swiglu(src, d64)
    near(got_h[:live], want_h, e_h, kind)
    want_again, e_again, want_dz, e_dz = ref_swiglu(back, d64)
    near(got_again[:live], want_again, e_again, kind)
    near(got_dz[:live], want_dz, e_dz, kind)
    for buf, cols in ((h, ff), (dz, 2 * ff), (again, ff)):
        assert (buf[live:] == 77).all() and (buf[:, cols:] == 77).all()
    # all rows, without the count
    z.copy_(matrix(rows, 2 * ff, kind, 5, 0, 3.0))
    F.moe_swiglu(z, got_h)
    want_h, e_h, _, _ = ref_swiglu(z.cpu().double(), torch.zeros(rows, ff, dtype=torch.float64))
    near(got_h, want_h, e_h, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
def test_swiglu_of_large_gates(kind):
    """Gates far from zero: the sigmoid is 0 or 1 to the type's precision, exp overflows without a NaN, an infinity stays in its place."""
    import flashrt_amd as F
    g = torch.tensor([-3e4, -200.0, -90.0, -20.0, 20.0, 90.0, 200.0, 3e4], dtype=kind)
    z = torch.cat([g, torch.full((8,), 2.0, dtype=kind)])[None].cuda()
    h, dz, dh = torch.empty(1, 8, dtype=kind, device="cuda"), torch.empty(1, 16, dtype=kind, device="cuda"), torch.ones(1, 8, dtype=kind, device="cuda")
    F.moe_swiglu(z, h)
    F.moe_swiglu_grad(dh, dz, z=z)
    want = (g.double() * torch.sigmoid(g.double()) * 2)[None]
    assert torch.isfinite(h).all() and torch.isfinite(dz).all()
    assert torch.allclose(h.cpu().double(), want, rtol=2e-2, atol=1e-6) and torch.equal(h[0, 4:].cpu(), (g[4:].float() * 2).to(kind))
    assert torch.equal(dz[0, 4:8].cpu(), torch.full((4,), 2.0, dtype=kind)) and torch.equal(dz[0, 12:].cpu(), g[4:])
    z[0, 1], z[0, 6], z[0, 8 + 3] = float("nan"), float("inf"), float("inf")
    F.moe_swiglu(z, h)
    assert h[0, 1].isnan() and h[0, 6] == torch.inf and h[0, 3] == -torch.inf and torch.isfinite(h[0, [0, 2, 4, 5, 7]]).all()


@pytest.mark.gpu
def test_swiglu_gradient_against_differences():
    """Central differences of the fp32 call over a step t: the definition's third derivatives are below 1 in g for |u dh| <= 1, so the
    difference is off by t^2 / 6 and by the calls' errors over t."""
    import flashrt_amd as F
    rows, ff, t = 6, 40, 2.0 ** -6
    z, dh = matrix(rows, 2 * ff, F32, 3).clamp(-1, 1), matrix(rows, ff, F32, 4).clamp(-1, 1)
    dz = torch.empty(rows, 2 * ff, device="cuda")
    F.moe_swiglu_grad(dh, dz, z=z)
    up, down = torch.empty(rows, ff, device="cuda"), torch.empty(rows, ff, device="cuda")
    for half in (slice(0, ff), slice(ff, 2 * ff)):
        for s, h in ((t, up), (-t, down)):
            moved = z.clone()
            moved[:, half] += s
            F.moe_swiglu(moved, h)
        diff = (up.double() - down.double()) / (2 * t) * dh.double()
        err = (diff - dz[:, half].double()).abs()
        assert (err <= t * t / 6 + 40 * U * 2 / t).all(), float(err.max())


@pytest.mark.gpu
def test_live_counts_past_the_ends():
    """A count below zero leaves every row, one beyond the rows takes them all."""
    import flashrt_amd as F
    z, h = matrix(3, 64, BF16, 1), torch.full((3, 32), 77.0, dtype=BF16, device="cuda")
    for n, hit in ((0, 0), (-5, 0), (-2 ** 31, 0), (2, 2), (3, 3), (2 ** 31 - 1, 3)):
        h.fill_(77)
        F.moe_swiglu(z, h, live=torch.tensor([n], dtype=torch.int32, device="cuda"))
        assert (h[hit:] == 77).all() and not (h[:hit] == 77).any()


@pytest.mark.gpu
def test_rows_past_32_bits():
    """2^19 rows of 8256 values, 4.3 G codes: offsets past 32 bits, in the first and last rows."""
    import flashrt_amd as F
    rows, ff = 2 ** 19, 4128
    z = torch.empty(rows, 2 * ff, dtype=BF16, device="cuda")
    assert z.numel() > 2 ** 32
    few = matrix(4, 2 * ff, BF16, 1)
    for at in (0, rows - 2):
        z[at:at + 2] = few[:2] if at == 0 else few[2:]
    z[2:rows - 2] = 0
    h = torch.empty(rows, ff, dtype=BF16, device="cuda")
    codes, scales = torch.empty(rows, 2 * ff, dtype=torch.int8, device="cuda"), torch.empty(rows, ff // 16, dtype=torch.uint8, device="cuda")
    F.moe_swiglu(z, h, codes, scales)
    rc, rs = ref_quantize(few.cpu().double().numpy())
    same((torch.cat([codes[:2], codes[-2:]]), torch.cat([scales[:2], scales[-2:]])), rc, rs)
    assert not codes[2:-2:999].any() and not h[2:-2:999].any()
    dz = z
    F.moe_swiglu_grad(h, dz, codes=codes, scales=scales)
    one = torch.empty(4, 2 * ff, dtype=BF16, device="cuda")
    F.moe_swiglu_grad(torch.cat([h[:2], h[-2:]]), one, codes=torch.cat([codes[:2], codes[-2:]]), scales=torch.cat([scales[:2], scales[-2:]]))
    assert torch.equal(torch.cat([dz[:2], dz[-2:]]), one) and not dz[2:-2:999].any()


@pytest.mark.gpu
def test_other_stream_and_graph():
    import flashrt_amd as F
    rows, ff = 50, 96
    i8, u8 = (lambda *s: torch.zeros(s, dtype=torch.int8, device="cuda")), (lambda *s: torch.zeros(s, dtype=torch.uint8, device="cuda"))
    f = lambda *s: torch.zeros(s, dtype=BF16, device="cuda")  # noqa: E731
    v = dict(z=f(rows, 2 * ff), dh=f(rows, ff), h=f(rows, ff), c=i8(rows, 2 * ff), s=u8(rows, ff // 16), dz=f(rows, 2 * ff), again=f(rows, ff), hc=i8(rows, ff), hs=u8(rows, ff // 32),
             back=f(rows, ff), n=torch.zeros(1, dtype=torch.int32, device="cuda"))

    def step(v, stream=None):
        F.moe_swiglu(v["z"], v["h"], v["c"], v["s"], live=v["n"], stream=stream)
        F.moe_swiglu_grad(v["dh"], v["dz"], codes=v["c"], scales=v["s"], h=v["again"], live=v["n"], stream=stream)
        F.mx8_quantize(v["h"], v["hc"], v["hs"], stream=stream)
        F.mx8_dequantize(v["hc"], v["hs"], v["back"], stream=stream)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(v)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(v)
    for seed in range(4):
        v["z"].copy_(matrix(rows, 2 * ff, BF16, seed))
        v["dh"].copy_(matrix(rows, ff, BF16, seed + 9))
        v["n"].fill_(rows - seed)
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
    z, h, dz, dh, again = (torch.zeros(4, c, device="cuda") for c in (64, 32, 64, 32, 32))
    c, s = torch.zeros(4, 64, dtype=torch.int8, device="cuda"), torch.zeros(4, 2, dtype=torch.uint8, device="cuda")
    everything = [z, h, dz, dh, again, c, s]
    for outs, call in (((h,), lambda: F.moe_swiglu(z, h)), ((h, c, s), lambda: F.moe_swiglu(z, h, c, s)), ((dz,), lambda: F.moe_swiglu_grad(dh, dz, z=z)),
                       ((dz, again), lambda: F.moe_swiglu_grad(dh, dz, codes=c, scales=s, h=again)), ((c, s), lambda: F.mx8_quantize(z, c, s)),
                       ((dz,), lambda: F.mx8_dequantize(c, s, dz))):
        was = [v._version for v in everything]
        call()
        for v, old in zip(everything, was):
            assert v._version == old + any(v is o for o in outs)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,u", [(F32, 2.0), (F32, 1e30), (F16, 2.0), (BF16, 2.0), (BF16, 1e30)])
def test_swiglu_of_subnormal_sigmoids(kind, u):
    """Gates below -87.3, whose sigmoid is a subnormal number of fp32: off by a step of these (2^-149) more, here times |g u|."""
    import flashrt_amd as F
    g = -torch.arange(86.0, 89.0, 0.5, dtype=torch.float64).to(kind)   # (exp(88.5) is the last that fp32 holds)
    ff, tiny = g.numel(), 2.0 ** -149
    z = torch.cat([g, torch.full((ff,), u, dtype=kind)])[None]
    dh = torch.full((1, ff), 0.5, dtype=kind)
    h, dz = torch.empty(1, ff, dtype=kind, device="cuda"), torch.empty(1, 2 * ff, dtype=kind, device="cuda")
    F.moe_swiglu(z.cuda(), h)
    F.moe_swiglu_grad(dh.cuda(), dz, z=z.cuda())
    want_h, e_h, want_dz, e_dz = ref_swiglu(z.double(), dh.double())
    assert (want_h != 0).all()
    near(h, want_h, e_h + tiny * 90 * u, kind)
    near(dz, want_dz, e_dz + tiny * 90 * max(u, 1.0), kind)
