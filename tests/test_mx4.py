"""Microscaled 4-bit floats (mx4_quantize, mx4_dequantize) and their grouped product (mx4_product) against 64-bit restatements.

Codes and scales are compared bit for bit. A product of two codes and their scales is exact in fp32 (4 significant bits), so a sum
of m products is off by at most m u sum |a w| (u = 2^-24, half a step of fp32, first order), and the result's rounding by h |out|
(h half a step of the type: fp32 2^-24, fp16 2^-11 and at least 2^-25, bf16 2^-8); 1.01 covers the higher orders."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
H_ABS = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}
TYPES = [torch.float32, torch.float16, torch.bfloat16]
GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def near(got, want, bound):
    err = (got.detach().cpu().double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), (int(bad.sum()), float(err[bad].max()), np.argwhere(bad.numpy())[:4].tolist())


def ref_quantize(x):
    """(codes, scales) of float64 rows from the definition: nearest of the grid, ties to the even code."""
    rows, cols = x.shape
    v = x.reshape(rows, cols // 32, 32)
    top = np.abs(v).max(2)
    bad = ~np.isfinite(top)
    with np.errstate(all="ignore"):
        k = np.where(top > 0, np.floor(np.log2(np.where(bad, 1.0, top))), -1000)
    b = np.maximum(k - 2, -127) + 127
    y = np.abs(np.where(bad[:, :, None], 0.0, v)) * np.exp2(127 - b)[:, :, None]
    dist = np.abs(y[..., None] - GRID)
    code = dist.argmin(-1)
    tie = (code < 7) & (np.take_along_axis(dist, np.minimum(code + 1, 7)[..., None], -1)[..., 0] == dist.min(-1))
    code = code + (tie & (code % 2 == 1))
    code = np.where(bad[:, :, None], 0, code | (np.signbit(v).astype(np.int64) << 3)).reshape(rows, cols)
    return (code[:, ::2] | code[:, 1::2] << 4).astype(np.uint8), np.where(bad, 255, b).astype(np.uint8)


def values(codes, scales):
    """The float64 values of codes [..][c / 2] and scales [..][c / 32] (uint8 arrays)."""
    c = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1).astype(np.int64)
    step = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return np.where(c >= 8, -1.0, 1.0) * GRID[c & 7] * np.repeat(step, 32, -1)


def gpu_quantize(F, x):
    codes = torch.full((x.shape[0], x.shape[1] // 2), 0xEE, dtype=torch.uint8, device="cuda")
    scales = torch.full((x.shape[0], x.shape[1] // 32), 0xEE, dtype=torch.uint8, device="cuda")
    F.mx4_quantize(x, codes, scales)
    return codes, scales


# ---------------------------------------------------------------- refusals, on the CPU

def test_refusals_before_any_launch():
    """Shapes, types, alignments and null pointers are refused with the library's codes; nothing is launched."""
    from flashrt_amd import _lib
    L = _lib.lib()
    p = 1 << 20
    q = [None, p, 64, 0, 3, 64, p, p]
    d = [None, p, p, 3, 64, p, 64, 0]
    m = [None, p, p, 5, p, p, p, p, 4, 5, 24, 64, p, 24, 0]
    for fn, good, bad in ((L.frt_mx4_quantize, q, [(2, 63, -1), (3, 8, -1), (4, -1, -1), (5, 48, -1), (5, 0, -1), (1, None, -4), (6, None, -4),
                                                   (7, None, -4), (6, p + 8, -1), (1, p + 2, -1)]),
                          (L.frt_mx4_dequantize, d, [(6, 63, -1), (7, 2, -1), (3, -1, -1), (4, 16, -1), (1, None, -4), (2, None, -4), (5, None, -4),
                                                     (1, p + 1, -1), (5, p + 1, -1)]),
                          (L.frt_mx4_product, m, [(14, 7, -1), (13, 23, -1), (8, 0, -1), (8, 4097, -1), (9, -1, -1), (10, 0, -1), (10, (1 << 30) + 1, -1), (11, 48, -1),
                                                  (3, 0, -1), (1, None, -4), (2, None, -4), (5, None, -4), (6, None, -4), (12, None, -4), (1, p + 4, -1),
                                                  (5, p + 4, -1), (12, p + 1, -1), (7, None, -1)])):
        for i, v, rc in bad:
            a = list(good)
            a[i] = v
            assert fn(*a) == rc, (fn.__name__, i, v, L.frt_last_error())
            assert L.frt_last_error()
    a = list(m)
    a[4], a[3] = None, 4   # fewer rows of activations than M, and none picked
    assert L.frt_mx4_product(*a) == -1
    for fn, good, i in ((L.frt_mx4_quantize, q, 4), (L.frt_mx4_dequantize, d, 3), (L.frt_mx4_product, m, 9)):
        a = list(good)
        a[i] = 0
        assert fn(*a) == 0   # no rows: nothing to do


def test_product_refuses_more_rows_than_it_numbers():
    from flashrt_amd import _lib
    L, p = _lib.lib(), 1 << 20
    assert L.frt_mx4_product(None, p, p, 5, p, p, p, p, 4, (1 << 30) + 1, 24, 64, p, 24, 0) == -1
    assert L.frt_mx4_product(None, p, p, 0x7fffffff, None, p, p, None, 1, 0x7fffffff, 24, 64, p, 24, 0) == -1


def test_python_refusals():
    import flashrt_amd as F
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)  # noqa: E731
    x, out = torch.zeros(4, 64), torch.zeros(4, 24)
    with pytest.raises(ValueError, match="device"):
        F.mx4_quantize(x, u8(4, 32), u8(4, 2))
    with pytest.raises(ValueError, match="device"):
        F.mx4_product(u8(4, 32), u8(4, 2), u8(24, 32), u8(24, 2), out)
    for call in (lambda: F.mx4_quantize(x, u8(4, 31), u8(4, 2)), lambda: F.mx4_quantize(x, u8(4, 32), u8(4, 1)), lambda: F.mx4_quantize(x.double(), u8(4, 32), u8(4, 2)),
                 lambda: F.mx4_quantize(x.t(), u8(64, 2), u8(64, 1)), lambda: F.mx4_dequantize(u8(4, 32).int(), u8(4, 2), x),
                 lambda: F.mx4_product(u8(4, 32), u8(4, 2), u8(24, 16), u8(24, 2), out), lambda: F.mx4_product(u8(4, 32), u8(4, 2), u8(23, 32), u8(24, 2), out),
                 lambda: F.mx4_product(u8(4, 32), u8(4, 1), u8(24, 32), u8(24, 2), out), lambda: F.mx4_product(u8(4, 32), u8(4, 2), u8(24, 32), u8(24, 1), out),
                 lambda: F.mx4_product(u8(4, 32), u8(4, 2), u8(2, 24, 32), u8(2, 24, 2), out, bounds=torch.zeros(2, dtype=torch.int32)),
                 lambda: F.mx4_product(u8(4, 32), u8(4, 2), u8(24, 32), u8(24, 2), out, rows=torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(ValueError):
            call()


def test_reference_rounds_to_even_codes():
    """The restatement itself, at every midpoint and end of the grid."""
    x = np.zeros((1, 32))
    x[0, :16] = [4, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.99, -0.25, -5.0, 0.2500001, 0.7499999, -0.0]
    codes, scales = ref_quantize(x)
    assert scales[0, 0] == 127
    assert values(codes, scales)[0, :16].tolist() == [4, 0, 1, 1, 2, 2, 4, 4, 6, 6, 6, -0.0, -4, 0.5, 0.5, -0.0]


def _client(arg):
    import os
    import subprocess
    exe = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "_build", "test_ops")
    assert os.path.exists(exe), "build first: make -C flashrt_amd/csrc"
    r = subprocess.run([exe, arg], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "all passed" in r.stdout, r.stdout + r.stderr


def test_cpp_client_host():
    """The C++ mirror's calls turn refusals into std::runtime_error."""
    _client("--host")


@pytest.mark.gpu
def test_cpp_client_gpu():
    """The C++ mirror's calls in a run: sort, permute, quantize, product, unpermute and the gradients, exact values."""
    _client("--gpu")


# ---------------------------------------------------------------- quantisation

@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,cols,pad", [(1, 32, 0), (1, 2048, 0), (3, 96, 0), (7, 640, 5), (129, 2560, 0), (1000, 544, 3)])
def test_quantize(rows, cols, pad, kind):
    import flashrt_amd as F
    g = torch.Generator().manual_seed(rows)
    x = (torch.randn(rows, cols + pad, generator=g) * torch.exp2(torch.randn(rows, 1, generator=g) * 4)).to(kind).cuda()[:, :cols]
    codes, scales = gpu_quantize(F, x)
    rc, rs = ref_quantize(x.cpu().double().numpy())
    assert np.array_equal(scales.cpu().numpy(), rs) and np.array_equal(codes.cpu().numpy(), rc)
    buf = torch.full((rows, cols + pad), 77.0, dtype=kind, device="cuda")
    F.mx4_dequantize(codes, scales, buf[:, :cols])
    assert torch.equal(buf[:, :cols].cpu().double(), torch.from_numpy(values(rc, rs)).to(kind).double())
    assert (buf[:, cols:] == 77).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
def test_quantize_every_exponent(kind):
    """Blocks whose largest value takes every exponent of the type, with the grid's midpoints, their neighbours and both zeros."""
    import flashrt_amd as F
    fi = torch.finfo(kind)
    lo, hi = int(np.log2(fi.smallest_normal)) - int(-np.log2(fi.eps)), int(np.log2(fi.max))
    mid = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0])
    eps = float(fi.eps)
    pat = np.concatenate([mid, -mid, [0.0, -0.0, 0.5, 1.0, 4.0], mid[:4] * (1 + eps), mid[:4] * (1 - eps)])
    assert pat.size <= 32
    blk = np.zeros((hi - lo + 1, 32))
    for i, k in enumerate(range(lo, hi + 1)):
        blk[i, :pat.size] = np.clip(pat * 2.0 ** (k - 2), -float(fi.max), float(fi.max))
    x = torch.from_numpy(blk).to(kind)
    codes, scales = gpu_quantize(F, x.cuda())
    rc, rs = ref_quantize(x.double().numpy())
    assert np.array_equal(scales.cpu().numpy(), rs), np.argwhere(scales.cpu().numpy() != rs)[:4]
    assert np.array_equal(codes.cpu().numpy(), rc), np.argwhere(codes.cpu().numpy() != rc)[:4]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
def test_quantize_zeros_infinities_nan(kind):
    """A block of zeros has the scale byte 0; one infinity or NaN makes its own block NaN and leaves its neighbours."""
    import flashrt_amd as F
    x = torch.ones(6, 96, dtype=kind)
    x[0], x[1, 40], x[2, 33], x[3, 63], x[4, 32:64] = 0, float("inf"), float("nan"), float("-inf"), -0.0
    codes, scales = gpu_quantize(F, x.cuda())
    s = scales.cpu()
    assert (s[0] == 0).all() and s[4, 1] == 0 and (s[1:4, 1] == 255).all() and (s[1:4, ::2] == 125).all()
    assert (codes.cpu()[1:4, 16:32] == 0).all() and (codes.cpu()[4, 16:32] == 0x88).all()
    y = torch.empty(6, 96, dtype=kind, device="cuda")
    F.mx4_dequantize(codes, scales, y)
    y = y.cpu()
    assert y[1:4, 32:64].isnan().all() and (y[1:4, :32] == 1).all() and (y[1:4, 64:] == 1).all() and (y[0] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
def test_dequantize_every_code_and_scale(kind):
    import flashrt_amd as F
    scales = np.arange(256, dtype=np.uint8).reshape(256, 1)
    codes = np.tile(np.arange(16, dtype=np.uint8) * 16 + np.arange(15, -1, -1, dtype=np.uint8), (256, 1))
    out = torch.empty(256, 32, dtype=kind, device="cuda")
    F.mx4_dequantize(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), out)
    want = torch.from_numpy(values(codes, scales)).to(torch.float32).to(kind)   # (every value is an fp32 number)
    assert torch.equal(out.cpu().isnan(), want.isnan()) and torch.equal(out.cpu().nan_to_num(0.25), want.nan_to_num(0.25))


# ---------------------------------------------------------------- the product

def operands(a_rows, E, N, C, seed, sd=1.0):
    """Random codes of every kind with scales around one, as (codes, scales) arrays of the activations and weights."""
    r = np.random.default_rng(seed)
    byte = lambda *s: r.integers(0, 256, s, dtype=np.uint8)  # noqa: E731
    scale = lambda *s: r.integers(121, 131, s).astype(np.uint8)  # noqa: E731
    return byte(a_rows, C // 2), scale(a_rows, C // 32), byte(E, N, C // 2), scale(E, N, C // 32)


def run_product(F, ops, M, kind, bounds=None, rows=None, pad=0, stream=None):
    aq, asc, wq, wsc = (torch.from_numpy(v).cuda() for v in ops)
    N = wq.shape[1]
    buf = torch.full((M + 1, N + pad), 77.0, dtype=kind, device="cuda")
    i32 = lambda v: None if v is None else torch.from_numpy(np.asarray(v, np.int32)).cuda()  # noqa: E731
    F.mx4_product(aq, asc, wq if bounds is not None else wq[0], wsc, buf[:M, :N], bounds=i32(bounds), rows=i32(rows), stream=stream)
    assert (buf[:, N:] == 77).all() and (buf[M] == 77).all()
    return buf[:M, :N]


def check_product(got, ops, M, kind, bounds=None, rows=None):
    aq, asc, wq, wsc = ops
    a, w = values(aq, asc), values(wq, wsc)
    rows = np.arange(M) if rows is None else np.asarray(rows)
    ok = (rows >= 0) & (rows < a.shape[0])
    a = np.where(ok[:, None], a[np.where(ok, rows, 0)], 0.0)
    bounds = [0, M] if bounds is None else bounds
    want, mag = np.full((M, w.shape[1]), 77.0), np.zeros((M, w.shape[1]))
    for g in range(w.shape[0]):
        lo, hi = bounds[g], bounds[g + 1]
        want[lo:hi], mag[lo:hi] = a[lo:hi] @ w[g].T, np.abs(a[lo:hi]) @ np.abs(w[g]).T
    C = a.shape[1]
    near(got, torch.from_numpy(want), torch.from_numpy(1.01 * (C * U * mag + HALF[kind] * np.abs(want)) + H_ABS[kind]))
    live = bounds[-1]
    if kind is torch.float32 and live:   # and near the float64 result as a whole
        err = np.linalg.norm(got.cpu().double().numpy()[:live] - want[:live]) / max(np.linalg.norm(want[:live]), 1e-30)
        assert err < 1e-6, err


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("M,N,C", [(1, 1, 32), (1, 1024, 2048), (1, 17, 96), (3, 130, 160), (15, 16, 128), (16, 33, 64), (17, 15, 224), (40, 257, 512),
                                   (64, 64, 1056), (65, 128, 256), (129, 300, 2048), (200, 1000, 640), (257, 129, 352), (512, 512, 1024)])
def test_product_one_group(M, N, C, kind):
    import flashrt_amd as F
    ops = operands(M, 1, N, C, M + N + C)
    check_product(run_product(F, ops, M, kind, pad=3), ops, M, kind)


def cut(sizes):
    return [0] + np.cumsum(sizes).tolist()


GROUPS = {
    "singles": [1, 0, 0, 1, 0, 1, 1, 0],
    "edges": [15, 0, 16, 17, 1, 31, 32, 33],
    "wide": [0, 63, 64, 65, 0, 127, 129, 0],
    "one": [0, 0, 0, 300, 0, 0, 0, 0],
    "last": [0, 0, 0, 0, 0, 0, 0, 5],
    "many": [i % 5 for i in range(203)],
    "empty": [0] * 9,
}


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("groups", list(GROUPS))
@pytest.mark.parametrize("N,C", [(96, 256), (131, 736)])
@pytest.mark.parametrize("gather", [False, True])
def test_product_groups(groups, N, C, gather, kind):
    """Groups of every size with rows of no group behind them; with rows: tokens picked more than once, and indices outside."""
    import flashrt_amd as F
    bounds = cut(GROUPS[groups])
    M = bounds[-1] + 7
    ops = operands(23 if gather else M, len(bounds) - 1, N, C, M)
    rows = None
    if gather:
        rows = np.random.default_rng(M).integers(0, 23, M)
        rows[::9], rows[1::13] = -1, 23
    check_product(run_product(F, ops, M, kind, bounds, rows, pad=1), ops, M, kind, bounds, rows)


# (rows of the groups, features) for the tiles of 32, 64, 128 and 256 rows; ragged, with empty and far larger groups among them. The
# groups are repeated until their weights, read by tiles of 16 rows, are over the 16 MB below which the values are split instead.
TILES = {
    "rows32": ([(5 * i) % 9 for i in range(90)] + [70, 0], 395),
    "rows64": ([17 + (7 * i) % 23 for i in range(62)] + [0, 129], 424),
    "rows128": ([60 + (31 * i) % 150 for i in range(20)] + [0, 300], 1608),
    "rows256": ([4200], 4104),
}


@pytest.mark.gpu
@pytest.mark.parametrize("tile", list(TILES))
@pytest.mark.parametrize("C,kind", [(64, torch.bfloat16), (256, torch.float32), (544, torch.float16), (544, torch.float32), (640, torch.bfloat16),
                                    (1408, torch.float32), (1408, torch.float16)])
def test_product_tiles(tile, C, kind):
    """Every tile size, with rows of fewer than one stage (256 values) to several, whole words of scales (C % 128 = 0) and not; tokens
    picked by index, some outside, and rows behind the last group."""
    import flashrt_amd as F
    sizes, N = TILES[tile]
    if len(sizes) > 1:
        avg = sum(sizes) // len(sizes)
        sizes = sizes * max(1, -(-(17 << 20) // (-(-avg // 16) * len(sizes) * N * C // 2)))
    bounds = cut(sizes)
    M = bounds[-1] + 5
    gather = kind is not torch.float16
    ops = operands(57 if gather else M, len(sizes), N, C, C)
    rows = None
    if gather:
        rows = np.random.default_rng(C).integers(0, 57, M)
        rows[::29], rows[1::31] = -1, 57
    check_product(run_product(F, ops, M, kind, bounds, rows, pad=3), ops, M, kind, bounds, rows)


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [1, 2, 3])
@pytest.mark.parametrize("tile", list(TILES))
def test_product_scales_at_any_byte(tile, shift):
    """Every tile size with 17 scales to a row that start at every byte of a word, bytes of NaN scales beside both tensors; activations
    picked by index."""
    import flashrt_amd as F
    sizes, N = TILES[tile]
    C = 544
    if len(sizes) > 1:
        avg = sum(sizes) // len(sizes)
        sizes = sizes * max(1, -(-(17 << 20) // (-(-avg // 16) * len(sizes) * N * C // 2)))
    bounds = cut(sizes)
    M = bounds[-1]
    ops = operands(301, len(sizes), N, C, shift)
    aq, asc, wq, wsc = (torch.from_numpy(v).cuda() for v in ops)

    def moved(v, by):
        buf = torch.full((v.numel() + 8,), 255, dtype=torch.uint8, device="cuda")
        buf[by:by + v.numel()] = v.reshape(-1)
        return buf[by:by + v.numel()].view(v.shape)

    rows = np.random.default_rng(shift).integers(0, 301, M).astype(np.int32)
    out = torch.empty(M, N, device="cuda")
    F.mx4_product(aq, moved(asc, shift), wq, moved(wsc, 4 - shift), out, bounds=torch.tensor(bounds, dtype=torch.int32, device="cuda"),
                  rows=torch.from_numpy(rows).cuda())
    check_product(out, ops, M, torch.float32, bounds, rows)


@pytest.mark.gpu
def test_product_many_groups():
    """More than 512 groups (their bounds are read in blocks): 1500, most of one row or none, over tiles and over few features."""
    import flashrt_amd as F
    sizes = [(i * 7) % 3 for i in range(1500)]
    bounds = cut(sizes)
    for N in (8, 300):
        ops = operands(bounds[-1], 1500, N, 96, N)
        check_product(run_product(F, ops, bounds[-1], torch.float32, bounds), ops, bounds[-1], torch.float32, bounds)


@pytest.mark.gpu
def test_product_tiles_captured():
    """The tile kernels in a graph, replayed on other activations and bounds with eager work between, each replay equal to the eager call."""
    import flashrt_amd as F
    E, N, C, M = 128, 512, 512, 3000   # (two tiles of 16 rows to a group: 34 MB)
    ops = operands(M, E, N, C, 3)
    aq, asc, wq, wsc = (torch.from_numpy(v).cuda() for v in ops)
    bounds = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    out, want = torch.zeros(M, N, device="cuda"), torch.zeros(M, N, device="cuda")
    F.mx4_product(aq, asc, wq, wsc, out, bounds=bounds)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        F.mx4_product(aq, asc, wq, wsc, out, bounds=bounds)
    for seed in range(3):
        aq.copy_(torch.from_numpy(operands(M, 1, 1, C, 40 + seed)[0]))
        cuts = np.sort(np.random.default_rng(seed).integers(0, M + 1, E + 1)).astype(np.int32)
        bounds.copy_(torch.from_numpy(cuts))
        out.zero_(), want.zero_()
        F.mx4_product(aq, asc, wq, wsc, want, bounds=bounds)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and bool((out[:int(cuts[0])] == 0).all()) and bool((out[int(cuts[-1]):] == 0).all())


@pytest.mark.gpu
def test_product_scales():
    """Scales far apart whose products stay in range; and a NaN block reaches its own row, or its own feature, alone."""
    import flashrt_amd as F
    M, N, C = 33, 70, 288
    ops = operands(M, 1, N, C, 9)
    for a, w in ((1, 253), (253, 1), (60, 190), (250, 4)):
        o = (ops[0], np.full_like(ops[1], a), ops[2], np.full_like(ops[3], w))
        check_product(run_product(F, o, M, torch.float32), o, M, torch.float32)
    o = [v.copy() for v in ops]
    o[1][5, 8], o[3][0, 66, 0], o[1][32, 0] = 255, 255, 255
    got = run_product(F, o, M, torch.float32).cpu()
    nan = torch.zeros(M, N, dtype=torch.bool)
    nan[5], nan[32], nan[:, 66] = True, True, True
    assert torch.equal(got.isnan(), nan)
    clean = run_product(F, ops, M, torch.float32).cpu()
    assert torch.equal(got[~nan], clean[~nan])


@pytest.mark.gpu
def test_product_rows_do_not_depend_on_their_neighbours():
    """A row's result is the same bits whether it is alone in its group, among few or among many."""
    import flashrt_amd as F
    N, C = 200, 1056
    ops = operands(300, 1, N, C, 4)
    whole = run_product(F, ops, 300, torch.float32)
    for m in (1, 9, 40, 130):
        part = (ops[0][:m], ops[1][:m], ops[2], ops[3])
        err = (run_product(F, part, m, torch.float32).double() - whole[:m].double()).norm() / whole[:m].double().norm()
        assert float(err) < 1e-6


@pytest.mark.gpu
def test_bounds_out_of_order_stay_inside():
    """Bounds that no sort gives (past the rows, negative, descending): nothing outside the operands is read or written (the kernel
    clamps them to the rows; the results are unspecified)."""
    import flashrt_amd as F
    ops = operands(40, 4, 64, 128, 1)
    for bounds in ([0, 100, 200, 300, 1 << 30], [-5, 3, 3, 9, 40], [0, 30, 10, 20, 40], [40, 40, 40, 40, 40]):
        got = run_product(F, ops, 40, torch.float32, bounds)
        assert got.shape == (40, 64)
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [6, 70])
def test_weights_past_32_bits(M):
    """The last experts of a weight tensor of more than 2^32 bytes, 1100 experts of 2048 x 4096: for few rows, and in tiles with the
    weights streamed."""
    import flashrt_amd as F
    E, N, C = 1100, 2048, 4096
    wq = torch.zeros((E, N, C // 2), dtype=torch.uint8, device="cuda")
    wsc = torch.full((E, N, C // 32), 127, dtype=torch.uint8, device="cuda")
    assert wq.numel() > 2 ** 32
    ops = operands(M, 2, N, C, 8)
    aq, asc, q, s = (torch.from_numpy(v).cuda() for v in ops)
    wq[E - 2:], wsc[E - 2:] = q, s
    bounds = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    bounds[E - 1], bounds[E] = 4, M
    out = torch.empty(M, N, device="cuda")
    F.mx4_product(aq, asc, wq, wsc, out, bounds=bounds)
    check_product(out, ops, M, torch.float32, [0, 4, M])


@pytest.mark.gpu
def test_results_past_32_bits():
    """2^20 rows of the same few activations against 8200 features, 8.6 G results: offsets
    past 32 bits. The columns' extremes over the rows with activations are the one row's results; the others are 0."""
    import flashrt_amd as F
    M, N, C = 2 ** 20, 8200, 32
    ops = operands(1, 1, N, C, 11)
    aq, asc, wq, wsc = (torch.from_numpy(v).cuda() for v in ops)
    rows = torch.where(torch.arange(M, device="cuda") % 5 == 2, -1, 0).to(torch.int32)
    one, out = torch.empty(1, N, device="cuda"), torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
    F.mx4_product(aq, asc, wq, wsc, one)
    check_product(one, ops, 1, torch.float32)
    F.mx4_product(aq, asc, wq, wsc, out, rows=rows)
    want, step = one.to(torch.bfloat16), 2 ** 16
    for r in range(0, M, step):
        none = (rows[r:r + step] < 0)[:, None]
        assert torch.equal(out[r:r + step], torch.where(none, torch.zeros_like(want), want)), r


@pytest.mark.gpu
def test_rows_past_31_bits_apart():
    """Results too far apart for the tiles' offsets (rows of 2^22 half-precision features), so that the kernel of few rows takes 33 row
    tiles: more workgroups than one grid dimension holds. Small codes at scale one: every sum is exact in fp32, whatever its order."""
    import flashrt_amd as F
    M, N, C, n = 528, 2 ** 22, 2048, 300
    g = torch.Generator(device="cuda").manual_seed(3)
    wq = torch.empty((N, C // 2), dtype=torch.uint8, device="cuda")   # 0 to 1.5 in halves, and every other value 0: sums below 2^12
    for f in range(0, N, N // 16):
        wq[f:f + N // 16] = torch.randint(0, 4, (N // 16, C // 2), generator=g, device="cuda", dtype=torch.uint8)
    aq = torch.randint(0, 4, (3, C // 2), generator=g, device="cuda", dtype=torch.uint8)
    wsc, asc = (torch.full((r, C // 32), 127, dtype=torch.uint8, device="cuda") for r in (N, 3))
    rows = (torch.arange(M, device="cuda") * 7 % 4 - 1).to(torch.int32)
    out = torch.empty(M, N, dtype=torch.float16, device="cuda")
    F.mx4_product(aq, asc, wq, wsc, out, rows=rows)
    few = torch.zeros(4, N, dtype=torch.float16, device="cuda")   # row 0: none
    F.mx4_product(aq, asc, wq, wsc, few[1:])
    assert torch.equal(out, few[rows.long() + 1])
    for f in (0, N // 2, N - n):
        a, w = values(aq.cpu().numpy(), asc.cpu().numpy()), values(wq[f:f + n].cpu().numpy(), wsc[f:f + n].cpu().numpy())
        assert torch.equal(few[1:, f:f + n].cpu().double(), torch.from_numpy(a @ w.T).half().double())


@pytest.mark.gpu
def test_other_stream_and_graph():
    """Quantise, product and dequantise on a stream of their own, and captured and replayed on new inputs with eager work between."""
    import flashrt_amd as F
    M, N, C, E = 50, 130, 256, 5
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8, device="cuda")  # noqa: E731
    ops = operands(1, E, N, C, 3)
    wq, wsc = torch.from_numpy(ops[2]).cuda(), torch.from_numpy(ops[3]).cuda()
    v = dict(x=torch.zeros(M, C, device="cuda"), q=u8(M, C // 2), s=u8(M, C // 32), b=torch.zeros(E + 1, dtype=torch.int32, device="cuda"),
             out=torch.zeros(M, N, device="cuda"), back=torch.zeros(M, C, device="cuda"))

    def step(v, stream=None):
        F.mx4_quantize(v["x"], v["q"], v["s"], stream=stream)
        F.mx4_product(v["q"], v["s"], wq, wsc, v["out"], bounds=v["b"], stream=stream)
        F.mx4_dequantize(v["q"], v["s"], v["back"], stream=stream)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(v)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(v)
    for seed in range(4):
        g = torch.Generator().manual_seed(seed)
        v["x"].copy_(torch.randn(M, C, generator=g))
        v["b"].copy_(torch.tensor([0, 0, 10 + seed, 30, 30, 50 - seed], dtype=torch.int32))
        v["out"].zero_()
        want = {k: t.clone() for k, t in v.items()}
        side.wait_stream(torch.cuda.current_stream())
        step(want, side)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for k in v:
            assert torch.equal(v[k], want[k]), (seed, k)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 5, 70, 300])
def test_experts_in_a_run(T):
    """A layer's experts with 4-bit weights, as they are used together: route, sort, quantize the tokens, the gate and up products
    picking each row's token, SwiGLU, quantize, the down products, and the weighted sum back; the sorted rows once more through
    moe_permute. Every call is held to a 64-bit restatement on its own inputs, so that a code at a rounding border cannot
    move what follows."""
    import flashrt_amd as F
    K, E, n, ff = 6, 24, 256, 96
    S = T * K
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, n, generator=g).cuda()
    logits = torch.randn(T, E, generator=g).cuda()
    ids, wts = torch.zeros(T, K, dtype=torch.int32, device="cuda"), torch.zeros(T, K, device="cuda")
    F.moe_route_topk(None, logits, T, E, K, ids, wts)
    i32 = lambda m: torch.zeros(m, dtype=torch.int32, device="cuda")  # noqa: E731
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8, device="cuda")  # noqa: E731
    b, tok, slot, row = i32(E + 1), i32(S), i32(S), i32(S)
    F.moe_sort(ids, T, K, E, b, tok, slot, row)
    up, down = operands(1, E, 2 * ff, n, 1)[2:], operands(1, E, n, ff, 2)[2:]
    (uq, us), (dq, ds) = ([torch.from_numpy(v).cuda() for v in p] for p in (up, down))
    xq, xsc = gpu_quantize(F, x)
    h = torch.zeros(S, 2 * ff, device="cuda")
    F.mx4_product(xq, xsc, uq, us, h, bounds=b, rows=tok)
    bounds = b.tolist()
    check_product(h, (xq.cpu().numpy(), xsc.cpu().numpy(), *up), S, torch.float32, bounds, tok.cpu().numpy())
    act = (torch.nn.functional.silu(h[:, :ff]) * h[:, ff:]).bfloat16()
    aq, asc = gpu_quantize(F, act)
    rc, rs = ref_quantize(act.cpu().double().numpy())
    assert np.array_equal(aq.cpu().numpy(), rc) and np.array_equal(asc.cpu().numpy(), rs)
    ys = torch.zeros(S, n, device="cuda")
    F.mx4_product(aq, asc, dq, ds, ys, bounds=b)
    check_product(ys, (rc, rs, *down), S, torch.float32, bounds)
    y = torch.zeros(T, n, device="cuda")
    F.moe_unpermute(ys, T, K, row, wts, y)
    terms = ys.cpu().double()[row.cpu().long().view(T, K)] * wts.cpu().double()[:, :, None]
    near(y, terms.sum(1), 1.01 * (K * U * terms.abs().sum(1) + U * terms.sum(1).abs()))
    # the sorted tokens quantized themselves give the same first product
    xs = torch.zeros(S, n, device="cuda")
    F.moe_permute(x, T, K, row, xs)
    sq, ssc = gpu_quantize(F, xs)
    h2 = torch.zeros_like(h)
    F.mx4_product(sq, ssc, uq, us, h2, bounds=b)
    assert torch.equal(h, h2)


# ---------------------------------------------------------------- the product's limits, for every kernel

def tile_groups(tile, C):
    """(bounds, features) of a row of TILES at C values, over the 16 MB from which the tiles are taken."""
    sizes, N = TILES[tile]
    if len(sizes) > 1:
        avg = sum(sizes) // len(sizes)
        sizes = sizes * max(1, -(-(17 << 20) // (-(-avg // 16) * len(sizes) * N * C // 2)))
    return cut(sizes), N


# one group: few rows, and the tiles of 32, 64, 128 and 256 rows by the rule of product_t
DENSE = {"few": (20, 130, 1056), "rows32": (24, 8200, 2112), "rows64": (48, 20500, 640), "rows128": (200, 16300, 352), "rows256": (300, 16200, 1056)}


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.float16])
@pytest.mark.parametrize("shape", list(DENSE))
def test_one_group_in_every_kernel(shape, kind):
    """Neither bounds nor rows: one group, each row its own activations."""
    import flashrt_amd as F
    M, N, C = DENSE[shape]
    ops = operands(M, 1, N, C, M)
    check_product(run_product(F, ops, M, kind, pad=5), ops, M, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("C,kind", [(352, torch.float32), (1024, torch.bfloat16), (1056, torch.float32)])
def test_largest_tile_with_ragged_groups(C, kind):
    """Eight groups of 0 to 700 rows, 269 on average: the tiles of 256 rows."""
    import flashrt_amd as F
    bounds = cut([257, 700, 0, 1, 512, 300, 255, 130])
    M, N = bounds[-1] + 3, 1801
    ops = operands(400, 8, N, C, C)
    rows = np.random.default_rng(C).integers(-1, 401, M)
    check_product(run_product(F, ops, M, kind, bounds, rows, pad=2), ops, M, kind, bounds, rows)


@pytest.mark.gpu
@pytest.mark.parametrize("C", [544, 640])
@pytest.mark.parametrize("tile", ["few"] + list(TILES))
def test_scale_extremes(tile, C):
    """The smallest and largest scale bytes with every code, products in range: 2^-127 times 2^127 is one, 2^-127 times one leaves
    fp32 results below 2^-126, which are exact (multiples of 2^-129, fewer than 2^24 of them)."""
    import flashrt_amd as F
    bounds, N = tile_groups(tile, C) if tile in TILES else (cut([1, 0, 16, 3]), 70)
    M = bounds[-1]
    ops = operands(M, len(bounds) - 1, N, C, 9)
    for a, w in ((0, 254), (254, 0), (1, 253), (0, 127), (127, 0)):
        o = (ops[0], np.full_like(ops[1], a), ops[2], np.full_like(ops[3], w))
        got = run_product(F, o, M, torch.float32, bounds)
        check_product(got, o, M, torch.float32, bounds)


@pytest.mark.gpu
@pytest.mark.parametrize("C", [544, 640])
@pytest.mark.parametrize("tile", list(TILES))
def test_nan_scales_in_tiles(tile, C):
    """A NaN block of a row, in a whole stage or in the last, shorter one, makes that row NaN alone; one of a feature, that feature of its
    group's rows alone. Everything else is bit for bit what it is without them."""
    import flashrt_amd as F
    bounds, N = tile_groups(tile, C)
    M, nb = bounds[-1], C // 32
    ops = operands(M, len(bounds) - 1, N, C, 9)
    o = [v.copy() for v in ops]
    nan = torch.zeros(M, N, dtype=torch.bool)
    for r, b in ((0, 0), (7, nb - 1), (M // 2, 3), (M - 1, nb - 1)):
        o[1][r, b], nan[r] = 255, True
    for g, f, b in ((0, N - 1, nb - 1), (len(bounds) - 2, 0, 0), (len(bounds) // 3, 67, nb - 2)):
        o[3][g, f, b], nan[bounds[g]:bounds[g + 1], f] = 255, True
    got, clean = run_product(F, o, M, torch.float32, bounds).cpu(), run_product(F, ops, M, torch.float32, bounds).cpu()
    assert torch.equal(got.isnan(), nan) and torch.equal(got[~nan], clean[~nan])


@pytest.mark.gpu
@pytest.mark.parametrize("tile", ["few"] + list(TILES))
def test_half_precision_results_that_overflow(tile):
    """fp16 results past its largest number are infinities of their sign; the others keep their bound."""
    import flashrt_amd as F
    C = 544
    bounds, N = tile_groups(tile, C) if tile in TILES else (cut([1, 0, 16, 3]), 70)
    M = bounds[-1]
    ops = operands(M, len(bounds) - 1, N, C, 2)
    ops = (ops[0], np.full_like(ops[1], 134), ops[2], np.full_like(ops[3], 128))   # 2^8: sums around 2^16
    got = run_product(F, ops, M, torch.float16, bounds).cpu()
    a, w = values(ops[0], ops[1]), values(ops[2], ops[3])
    seen = 0
    for g in range(len(bounds) - 1):
        lo, hi = bounds[g], bounds[g + 1]
        want = torch.from_numpy(a[lo:hi] @ w[g].T)   # (multiples of 2^6 below 2^30: exact in fp32, whatever the order)
        assert torch.equal(got[lo:hi], want.half())
        seen += int(got[lo:hi].isinf().sum())
    assert 0 < seen < M * N


@pytest.mark.gpu
@pytest.mark.parametrize("tile", list(TILES))
def test_bounds_out_of_order_in_tiles(tile):
    """Bounds that no sort gives (past the rows, negative, descending, all the same), in the tile kernels: nothing before or behind the
    rows is written, and no index leaves the operands (the kernel clamps the bounds to the rows; the results are unspecified)."""
    import flashrt_amd as F
    C = 544
    bounds, N = tile_groups(tile, C)
    E, M = len(bounds) - 1, bounds[-1]
    aq, asc, wq, wsc = (torch.from_numpy(v).cuda() for v in operands(M, E, N, C, 1))
    buf = torch.full((M + 64, N + 3), 77.0, device="cuda")
    r = np.random.default_rng(E)
    for cuts in (np.array(bounds) + M // 2, np.array(bounds) - M // 2, np.array(bounds)[::-1], r.integers(-M, 2 * M, E + 1),
                 np.full(E + 1, M), np.full(E + 1, 2 ** 31 - 1), np.full(E + 1, -2 ** 31), np.resize([0, M], E + 1), np.resize([-2 ** 31, 2 ** 31 - 1], E + 1)):
        F.mx4_product(aq, asc, wq, wsc, buf[32:32 + M, :N], bounds=torch.from_numpy(cuts.astype(np.int32)).cuda())
        assert (buf[:32] == 77).all() and (buf[32 + M:] == 77).all() and (buf[:, N:] == 77).all()


@pytest.mark.gpu
def test_few_rows_of_weights_past_32_bits():
    """The kernel of few rows (four rows: 16 MB of weights to read) on the last two of 1100 experts of 2048 x 4096."""
    import flashrt_amd as F
    E, N, C, M = 1100, 2048, 4096, 4
    wq = torch.zeros((E, N, C // 2), dtype=torch.uint8, device="cuda")
    wsc = torch.full((E, N, C // 32), 127, dtype=torch.uint8, device="cuda")
    ops = operands(M, 2, N, C, 8)
    aq, asc, q, s = (torch.from_numpy(v).cuda() for v in ops)
    wq[E - 2:], wsc[E - 2:] = q, s
    bounds = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    bounds[E - 1], bounds[E] = 1, M
    out = torch.empty(M, N, device="cuda")
    F.mx4_product(aq, asc, wq, wsc, out, bounds=bounds)
    check_product(out, ops, M, torch.float32, [0, 1, M])


@pytest.mark.gpu
def test_rows_in_one_kernel_and_across_kernels():
    """A row's bits do not depend on the rows beside it where the same kernel takes them (few rows: 1 to 300; the tiles of 256: 2049
    and 4200). Across kernels the order of the sums differs: each is within C u sum |a w| of the exact one."""
    import flashrt_amd as F
    N, C = 200, 1056
    ops = operands(300, 1, N, C, 4)
    whole = run_product(F, ops, 300, torch.float32)
    for m in (1, 9, 40, 130):
        assert torch.equal(run_product(F, (ops[0][:m], ops[1][:m], ops[2], ops[3]), m, torch.float32), whole[:m])
    N = 4104
    ops = operands(4200, 1, N, C, 5)
    whole = run_product(F, ops, 4200, torch.float32)
    assert torch.equal(run_product(F, (ops[0][:2049], ops[1][:2049], ops[2], ops[3]), 2049, torch.float32), whole[:2049])
    few = run_product(F, (ops[0][:5], ops[1][:5], ops[2], ops[3]), 5, torch.float32)
    mag = torch.from_numpy(np.abs(values(ops[0][:5], ops[1][:5])) @ np.abs(values(ops[2][0], ops[3][0])).T)
    near(few, whole[:5].cpu().double(), 2 * 1.01 * C * U * mag)


@pytest.mark.gpu
@pytest.mark.parametrize("tile", ["few"] + list(TILES))
def test_scales_far_apart_in_a_row(tile):
    """Blocks of a row whose scales differ by up to 2^60, large ones that cancel among them: the sums keep 24 bits of the largest."""
    import flashrt_amd as F
    C = 544
    bounds, N = tile_groups(tile, C) if tile in TILES else (cut([1, 0, 16, 3]), 70)
    M = bounds[-1]
    ops = operands(M, len(bounds) - 1, N, C, 6)
    r = np.random.default_rng(6)
    ops = (ops[0], r.integers(112, 143, ops[1].shape).astype(np.uint8), ops[2], r.integers(112, 143, ops[3].shape).astype(np.uint8))
    got = run_product(F, ops, M, torch.float32, bounds)
    a, w = values(ops[0], ops[1]), values(ops[2], ops[3])
    for g in range(len(bounds) - 1):
        lo, hi = bounds[g], bounds[g + 1]
        want, mag = a[lo:hi] @ w[g].T, np.abs(a[lo:hi]) @ np.abs(w[g]).T
        near(got[lo:hi], torch.from_numpy(want), torch.from_numpy(1.01 * (C * U * mag + U * np.abs(want))))
