"""The expert sort and the row moves with their gradients (moe_sort, moe_permute, moe_permute_grad, moe_unpermute,
moe_unpermute_grad) against 64-bit restatements, through the Python mirror.

Tolerances: u = 2^-24 is half a step of fp32, h half a step of the row type (fp32 2^-24, fp16 2^-11, bf16 2^-8), relative to the
value; a fp16 result also has h_abs = 2^-25, half its smallest step. A sum of m fp32 terms is off by at most m u times the sum of
the terms' magnitudes (first order; the products round with their addition), the result's rounding adds h |y|. The factor 1.01 covers
the higher orders (m u < 1e-3 at every size here)."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
H_ABS = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def near(got, want, bound):
    """|got - want| <= bound everywhere, in float64."""
    err = (got.detach().cpu().double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), (int(bad.sum()), float(err[bad].max()), np.argwhere(bad.numpy())[:4].tolist())


def slots(T, K, E, kind, seed):
    """ids [T][K]: "flat" any expert (twice in a token now and then), "hot" one expert nearly always, "drop" a third without one
    (also ids far outside), "none" no slot with an expert."""
    r = np.random.default_rng(seed)
    ids = r.integers(0, E, (T, K))
    if kind == "hot":
        ids[r.random((T, K)) < 0.9] = E - 1
    elif kind == "drop":
        out = r.random((T, K)) < 0.33
        ids[out] = r.choice([-1, E, -2 ** 31, 2 ** 31 - 1], out.sum())
        ids[T // 2] = -1
    elif kind == "none":
        ids[:] = -1
    return ids.astype(np.int32)


def sorted_slots(ids, E):
    """(bounds, slot_of, row_of) of a stable sort of the slots that have an expert."""
    flat = ids.reshape(-1).astype(np.int64)
    live = np.flatnonzero((flat >= 0) & (flat < E))
    slot_of = live[np.argsort(flat[live], kind="stable")]
    row_of = np.full(flat.size, -1, np.int64)
    row_of[slot_of] = np.arange(slot_of.size)
    return np.concatenate([[0], np.cumsum(np.bincount(flat[live], minlength=E))]), slot_of, row_of


def gpu_sort(F, ids, E, fill=-7):
    T, K = ids.shape
    new = lambda n: torch.full((n,), fill, dtype=torch.int32, device="cuda")  # noqa: E731
    b, tok, slot, row = new(E + 1), new(T * K), new(T * K), new(T * K)
    F.moe_sort(torch.from_numpy(ids).cuda(), T, K, E, b, tok, slot, row)
    return b, tok, slot, row


def matrix(rows, cols, kind, seed, pad=0, skip=0):
    """A [rows][cols] matrix of N(0, 1) values with pad values behind each row and skip before the first (a view of a flat buffer)."""
    g = torch.Generator().manual_seed(seed)
    flat = torch.randn(skip + rows * (cols + pad), generator=g).to(kind).cuda()
    return flat[skip:].view(rows, cols + pad)[:, :cols]


# ---------------------------------------------------------------- refusals, on the CPU

def test_refusals_before_any_launch():
    """Shapes, types, strides and null pointers are refused with the library's codes; nothing is launched (there is no
    device here: a launch would report FRT_ERR_HIP)."""
    from flashrt_amd import _lib
    L = _lib.lib()
    p = 1 << 20   # an address that is never read
    for T, K, E in ((-1, 1, 4), (1, 0, 4), (1, 1, 0), (1, 1, 1025), (1 << 20, 1 << 12, 4)):
        assert L.frt_moe_sort(None, p, T, K, E, p, p, p, p) == -1, (T, K, E)
    assert L.frt_moe_sort(None, p, 1, 1, 4, None, p, p, p) == -4
    assert L.frt_moe_sort(None, None, 0, 1, 4, None, None, None, None) == -4
    for i in (1, 6, 7, 8):
        a = [None, p, 1, 1, 4, p, p, p, p]
        a[i] = None
        assert L.frt_moe_sort(*a) == -4, i
    calls = [(L.frt_moe_permute, [None, p, 8, 0, 2, 2, 8, p, p, 8], 3, (1, 7, 8), (2, 9)),
             (L.frt_moe_permute_grad, [None, p, 8, 0, 2, 2, 8, p, p, 8], 3, (1, 7, 8), (2, 9)),
             (L.frt_moe_unpermute, [None, p, 8, 0, 2, 2, 8, p, p, p, 8], 3, (1, 7, 8, 9), (2, 10)),
             (L.frt_moe_unpermute_grad, [None, p, 8, p, 8, 0, 2, 2, 8, p, p, p, 8, p], 5, (1, 3, 9, 10, 11, 13), (2, 4, 12))]
    for fn, good, at, ptrs, lds in calls:
        for i, v, rc in [(at, 2, -1), (at, -1, -1), (at + 1, -1, -1), (at + 2, 0, -1), (at + 3, 0, -1), (at + 3, (1 << 30) + 1, -1), (at + 1, 1 << 30, -1)] + \
                [(i, None, -4) for i in ptrs] + [(i, 7, -1) for i in lds]:
            a = list(good)
            a[i] = v
            assert fn(*a) == rc, (fn.__name__, i, v, L.frt_last_error())
            assert L.frt_last_error()
        a = list(good)
        a[1] = p + 2   # half an fp32 value
        assert fn(*a) == -1
        a = list(good)
        a[at + 1], a[1] = 0, None
        assert fn(*a) == 0   # no tokens: nothing to do


def test_python_refusals():
    """Host tensors, and on one device wrong types, shapes and layouts, are ValueErrors."""
    import flashrt_amd as F
    x, xs, row = torch.zeros(4, 8), torch.zeros(8, 8), torch.zeros(8, dtype=torch.int32)
    wts = torch.ones(8)
    with pytest.raises(ValueError, match="device"):
        F.moe_permute(x, 4, 2, row, xs)
    with pytest.raises(ValueError, match="device"):
        F.moe_sort(row, 4, 2, 8, torch.zeros(9, dtype=torch.int32), row, row, row)
    for call in (lambda: F.moe_permute(x, 4, 2, row.long(), xs), lambda: F.moe_permute(x, 4, 2, row, xs.half()),
                 lambda: F.moe_permute(x, 4, 2, row[:7], xs), lambda: F.moe_permute(x, 4, 2, row, xs[:7]),
                 lambda: F.moe_permute(x, 4, 2, row, torch.zeros(8, 8).t()[:, ::1].t().t()), lambda: F.moe_permute(x.int(), 4, 2, row, xs.int()),
                 lambda: F.moe_permute(x.expand(4, 8)[:1].expand(4, 8), 4, 2, row, xs), lambda: F.moe_permute_grad(xs, 4, 2, row, x[:, :7]),
                 lambda: F.moe_unpermute(xs, 4, 2, row, wts.double(), x), lambda: F.moe_unpermute(xs, 4, 2, row[::2], wts, x),
                 lambda: F.moe_unpermute_grad(x, xs, 4, 2, row, wts, xs, wts[:7])):
        with pytest.raises(ValueError):
            call()


# ---------------------------------------------------------------- the sort

@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["flat", "hot", "drop", "none"])
@pytest.mark.parametrize("T,K,E", [(1, 1, 1), (1, 10, 512), (1, 32, 1024), (3, 5, 7), (64, 1, 2), (65, 1, 1), (50, 10, 1024), (93, 11, 65), (128, 8, 128), (205, 10, 1000),
                                   (1024, 1, 1), (2048, 10, 512), (5003, 3, 8)])
def test_sort(T, K, E, kind):
    import flashrt_amd as F
    ids = slots(T, K, E, kind, T * 7 + E)
    b, tok, slot, row = (v.cpu().numpy() for v in gpu_sort(F, ids, E))
    bounds, slot_of, row_of = sorted_slots(ids, E)
    live = slot_of.size
    assert np.array_equal(b, bounds)
    assert np.array_equal(row, row_of)
    assert np.array_equal(slot[:live], slot_of) and np.array_equal(tok[:live], slot_of // K)
    assert (slot[live:] == -7).all() and (tok[live:] == -7).all()   # rows behind the last stay as they were


@pytest.mark.gpu
def test_sort_no_tokens_and_many():
    """No tokens: bounds of zeros. More slots than one batch of each workgroup: 300,000 and 1024 experts."""
    import flashrt_amd as F
    b = gpu_sort(F, np.zeros((0, 4), np.int32), 17)[0]
    assert (b.cpu() == 0).all()
    ids = slots(30000, 10, 1024, "drop", 5)
    b, tok, slot, row = (v.cpu().numpy() for v in gpu_sort(F, ids, 1024))
    bounds, slot_of, row_of = sorted_slots(ids, 1024)
    assert np.array_equal(b, bounds) and np.array_equal(row, row_of) and np.array_equal(slot[:slot_of.size], slot_of)


@pytest.mark.gpu
def test_sort_equals_dispatch():
    """Where every slot has an expert, moe_dispatch's bounds, tok_of and slot_of."""
    import flashrt_amd as F
    for T, K, E in ((9, 10, 512), (777, 10, 512)):
        ids = slots(T, K, E, "flat", T)
        b, tok, slot, _ = gpu_sort(F, ids, E)
        d = [torch.empty_like(v) for v in (b, tok, slot)]
        F.moe_dispatch(torch.from_numpy(ids).cuda(), T, K, E, *d)
        assert all(torch.equal(x, y) for x, y in zip((b, tok, slot), d))


# ---------------------------------------------------------------- the moves

WIDTHS = [1, 3, 8, 9, 127, 512, 513, 1021, 2048, 2560]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("drop", ["flat", "drop"])
@pytest.mark.parametrize("pad,skip", [(0, 0), (5, 3)])
def test_moves(n, kind, drop, pad, skip):
    import flashrt_amd as F
    T, K, E = 37, 6, 16
    ids = slots(T, K, E, drop, n)
    _, slot_of, row_of = sorted_slots(ids, E)
    row = torch.from_numpy(row_of.astype(np.int32)).cuda()
    live = torch.from_numpy(row_of >= 0)
    at = torch.from_numpy(np.where(row_of < 0, 0, row_of))
    x, s = matrix(T, n, kind, 1, pad, skip), matrix(T * K, n, kind, 2, pad, skip)
    wts = torch.rand(T, K, generator=torch.Generator().manual_seed(3))
    wd = wts.cuda()

    def out(rows):   # a result with a border that has to stay as it was
        buf = torch.full((skip + rows * (n + pad),), 77.0, dtype=kind, device="cuda")
        return buf, buf[skip:].view(rows, n + pad)[:, :n]

    def border(buf, rows):
        assert (buf[:skip] == 77).all() and (buf[skip:].view(rows, n + pad)[:, n:] == 77).all()

    # permute: bit for bit; rows without a slot stay
    buf, xs = out(T * K)
    F.moe_permute(x, T, K, row, xs)
    tok = torch.from_numpy(slot_of // K).cuda()
    assert torch.equal(xs[:slot_of.size], x[tok]) and (xs[slot_of.size:] == 77).all()
    border(buf, T * K)

    rows64 = torch.where(live[:, None], s.cpu().double()[at], 0.0).view(T, K, n)
    m = torch.from_numpy((row_of >= 0).reshape(T, K).sum(1)).double()[:, None]
    # permute_grad
    buf, dx = out(T)
    F.moe_permute_grad(s, T, K, row, dx)
    want = rows64.sum(1)
    near(dx, want, 1.01 * m * U * rows64.abs().sum(1) + 1.01 * HALF[kind] * want.abs() + H_ABS[kind])
    border(buf, T)
    # unpermute
    buf, y = out(T)
    F.moe_unpermute(s, T, K, row, wd, y)
    terms = rows64 * wts.double()[:, :, None]
    want = terms.sum(1)
    near(y, want, 1.01 * m * U * terms.abs().sum(1) + 1.01 * HALF[kind] * want.abs() + H_ABS[kind])
    border(buf, T)
    # unpermute_grad
    buf, dys = out(T * K)
    dw = torch.full((T, K), 77.0, device="cuda")
    F.moe_unpermute_grad(x, s, T, K, row, wd, dys, dw)
    dy = x.cpu().double()[:, None, :]
    want = (dy * wts.double()[:, :, None]).view(T * K, n)[torch.from_numpy(slot_of)]
    # (the product rounds to fp32 first where the rows have 16 bits)
    near(dys[:slot_of.size], want, (1.01 * HALF[kind] + (U if kind is not torch.float32 else 0)) * want.abs() + H_ABS[kind])
    assert (dys[slot_of.size:] == 77).all()
    border(buf, T * K)
    terms = rows64 * dy
    near(dw, terms.sum(2), 1.01 * (n + 6) * U * terms.abs().sum(2))
    assert (dw.cpu()[~live.view(T, K)] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,K,n", [(1, 1, 2048), (1, 10, 2048), (1, 32, 515), (2, 13, 64), (600, 10, 2560)])
def test_moves_sizes(T, K, n, kind):
    """One token to a chunk, with up to 32 slots: the round trip with weights 1/K gives the rows back (a token's K equal rows),
    and the two gradients agree with their formulas."""
    import flashrt_amd as F
    ids = slots(T, K, 64, "flat", n)
    b, tok, slot, row = gpu_sort(F, ids, 64)
    x = matrix(T, n, kind, 4)
    xs = torch.empty(T * K, n, dtype=kind, device="cuda")
    F.moe_permute(x, T, K, row, xs)
    assert torch.equal(xs, x[tok.long()])
    y, wts = torch.empty_like(x), torch.full((T, K), 1.0 / K, device="cuda")
    F.moe_unpermute(xs, T, K, row, wts, y)
    want = x.cpu().double() * float(wts[0, 0]) * K
    near(y, want, 1.01 * (K * U + HALF[kind]) * want.abs())
    dys, dw = torch.empty_like(xs), torch.empty_like(wts)
    F.moe_unpermute_grad(x, xs, T, K, row, wts, dys, dw)
    sq = (x.cpu().double() ** 2).sum(1, keepdim=True)
    near(dw, sq.expand(T, K), 1.01 * (n + 6) * U * sq)
    dx = torch.empty_like(x)
    F.moe_permute_grad(dys, T, K, row, dx)
    one = dys.cpu().double()[row.cpu().long().view(T, K)]   # (what the second call reads)
    near(dx, one.sum(1), 1.01 * (K * U * one.abs().sum(1) + HALF[kind] * one.sum(1).abs()))


@pytest.mark.gpu
def test_gradients_against_differences():
    """unpermute is linear in ys and in the weights: the difference of L = <dy, y> between two points 2 d apart is 2 d times the
    gradient, up to the rounding of the two sums (off by at most (K + 1) u sum |dy| sum |w ys| each)."""
    import flashrt_amd as F
    T, K, E, n = 11, 4, 8, 96
    ids = slots(T, K, E, "drop", 3)
    _, _, _, row = gpu_sort(F, ids, E)
    ys, dy = matrix(T * K, n, torch.float32, 1), matrix(T, n, torch.float32, 2)
    wts = torch.rand(T, K, generator=torch.Generator().manual_seed(5)).cuda()
    dys, dw = torch.zeros_like(ys), torch.empty_like(wts)
    F.moe_unpermute_grad(dy, ys, T, K, row, wts, dys, dw)

    def loss(ys, wts):
        y = torch.empty_like(dy)
        F.moe_unpermute(ys, T, K, row, wts, y)
        return float((dy.double() * y.double()).sum())

    d = 0.5
    noise = 4 * (K + 2) * U * float((dy.abs().sum()) * ys.abs().max() * K * 2)
    for s in range(T * K):
        up, down = wts.clone().view(-1), wts.clone().view(-1)
        up[s] += d
        down[s] -= d
        step = float(up[s]) - float(down[s])
        got = (loss(ys, up.view(T, K)) - loss(ys, down.view(T, K))) / step
        assert abs(got - float(dw.view(-1)[s])) <= noise, s
    g = torch.Generator().manual_seed(6)
    for _ in range(20):
        r, c = int(torch.randint(T * K, (1,), generator=g)), int(torch.randint(n, (1,), generator=g))
        up, down = ys.clone(), ys.clone()
        up[r, c] += d
        down[r, c] -= d
        got = (loss(up, wts) - loss(down, wts)) / (float(up[r, c]) - float(down[r, c]))
        assert abs(got - float(dys[r, c])) <= noise, (r, c)
    # permute's gradient: <xs(x), g> = <x, permute_grad(g)>
    xs, dx = torch.zeros_like(ys), torch.empty_like(dy)
    F.moe_permute(dy, T, K, row, xs)
    F.moe_permute_grad(ys, T, K, row, dx)
    a, b = float((xs.double() * ys.double()).sum()), float((dy.double() * dx.double()).sum())
    assert abs(a - b) <= noise


@pytest.mark.gpu
def test_infinities_and_nan():
    """A NaN row reaches its own token only; a dropped slot's weight and a row that no slot has are not read; a weight of zero
    multiplies (0 * inf is NaN)."""
    import flashrt_amd as F
    ids = np.array([[0, 1], [2, -1], [-1, -1], [1, 0]], np.int32)
    _, _, _, row = gpu_sort(F, ids, 4)
    ys = torch.ones(8, 40, device="cuda")
    r = row.cpu().view(4, 2)
    ys[r[0, 0]] = float("nan")
    ys[r[3, 1]] = float("inf")
    ys[5:] = float("nan")   # rows behind the last
    wts = torch.tensor([[1.0, 1.0], [2.0, float("nan")], [float("inf"), 1.0], [1.0, 0.0]], device="cuda")
    y = torch.empty(4, 40, device="cuda")
    F.moe_unpermute(ys, 4, 2, row, wts, y)
    assert y[0].isnan().all() and (y[1] == 2).all() and (y[2] == 0).all() and y[3].isnan().all()
    dx = torch.empty(4, 40, device="cuda")
    F.moe_permute_grad(ys, 4, 2, row, dx)
    assert dx[0].isnan().all() and (dx[1] == 1).all() and (dx[2] == 0).all() and (dx[3] == float("inf")).all()


@pytest.mark.gpu
def test_row_map_out_of_range():
    """Entries of row_of outside [0, T K) count as dropped slots'."""
    import flashrt_amd as F
    T, K, n = 3, 2, 130
    row = torch.tensor([0, 6, 2 ** 31 - 1, -5, -2 ** 31, 5], dtype=torch.int32, device="cuda")
    x = matrix(T, n, torch.bfloat16, 1)
    xs = torch.full((T * K, n), 77.0, dtype=torch.bfloat16, device="cuda")
    F.moe_permute(x, T, K, row, xs)
    assert torch.equal(xs[0], x[0]) and torch.equal(xs[5], x[2]) and (xs[1:5] == 77).all()
    y = torch.empty_like(x)
    F.moe_unpermute(xs, T, K, row, torch.ones(T, K, device="cuda"), y)
    assert torch.equal(y[0], x[0]) and (y[1] == 0).all() and torch.equal(y[2], x[2])


@pytest.mark.gpu
def test_rows_past_32_bits():
    """Sorted rows whose offsets pass 2^32 values' bytes and 2^31 values: 20,000 tokens of 16 slots, rows 8192 apart in bf16."""
    import flashrt_amd as F
    T, K, n, ld = 20000, 16, 64, 8192
    ids = slots(T, K, 16, "flat", 1)
    b, tok, slot, row = gpu_sort(F, ids, 16)
    x = matrix(T, n, torch.bfloat16, 1)
    xs = torch.zeros(T * K, ld, dtype=torch.bfloat16, device="cuda")[:, :n]
    F.moe_permute(x, T, K, row, xs)
    assert torch.equal(xs, x[tok.long()])
    y, dx, dys, dw = torch.empty_like(x), torch.empty_like(x), torch.zeros(T * K, ld, dtype=torch.bfloat16, device="cuda")[:, :n], \
        torch.empty(T, K, device="cuda")
    wts = torch.full((T, K), 1.0 / K, device="cuda")   # (a power of two: exact)
    F.moe_unpermute(xs, T, K, row, wts, y)
    assert torch.equal(y, x)
    F.moe_permute_grad(xs, T, K, row, dx)
    assert torch.equal(dx, x * K)
    F.moe_unpermute_grad(x, xs, T, K, row, wts, dys, dw)
    assert torch.equal(dys, (x / K)[tok.long()])


@pytest.mark.gpu
def test_other_stream_and_graph():
    """On a stream of its own, and captured: sort, permute, unpermute and both gradients replayed on new inputs, with eager work
    between, each replay equal to the eager calls bit for bit."""
    import flashrt_amd as F
    T, K, E, n = 50, 10, 512, 1000
    S = T * K
    i32 = lambda m: torch.zeros(m, dtype=torch.int32, device="cuda")  # noqa: E731
    buf = dict(ids=i32(S), b=i32(E + 1), tok=i32(S), slot=i32(S), row=i32(S), x=torch.zeros(T, n, device="cuda"), xs=torch.zeros(S, n, device="cuda"),
               w=torch.rand(T, K, device="cuda"), y=torch.zeros(T, n, device="cuda"), dys=torch.zeros(S, n, device="cuda"),
               dw=torch.zeros(T, K, device="cuda"), dx=torch.zeros(T, n, device="cuda"))

    def step(v, stream=None):
        F.moe_sort(v["ids"], T, K, E, v["b"], v["tok"], v["slot"], v["row"], stream=stream)
        F.moe_permute(v["x"], T, K, v["row"], v["xs"], stream=stream)
        F.moe_unpermute(v["xs"], T, K, v["row"], v["w"], v["y"], stream=stream)
        F.moe_unpermute_grad(v["y"], v["xs"], T, K, v["row"], v["w"], v["dys"], v["dw"], stream=stream)
        F.moe_permute_grad(v["dys"], T, K, v["row"], v["dx"], stream=stream)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(buf)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(buf)
    for seed in range(4):
        buf["ids"].copy_(torch.from_numpy(slots(T, K, E, ["flat", "drop", "none", "hot"][seed], seed).reshape(-1)))
        buf["x"].copy_(matrix(T, n, torch.float32, seed))
        buf["xs"].zero_()
        buf["dys"].zero_()
        want = {k: v.clone() for k, v in buf.items()}
        for k in ("tok", "slot"):
            buf[k].zero_(), want[k].zero_()
        step(want, side if seed % 2 == 0 and not side.wait_stream(torch.cuda.current_stream()) else None)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for k in buf:
            assert torch.equal(buf[k], want[k]), (seed, k)


@pytest.mark.gpu
def test_more_tokens_than_one_grid_dimension():
    """2^26 + 37 tokens of two values, one slot each: more waves than 2^32 threads in one dimension hold. Powers of two and small
    integers, so every result is exact."""
    import flashrt_amd as F
    T = 2 ** 26 + 37
    x = ((torch.arange(2 * T, device="cuda", dtype=torch.int32) * 7) % 1021).to(torch.float16).reshape(T, 2)
    row = torch.arange(T - 1, -1, -1, dtype=torch.int32, device="cuda")
    w = torch.where(torch.arange(T, device="cuda") % 3 == 0, 2.0, 0.5)
    xs, y, dw = torch.zeros_like(x), torch.zeros_like(x), torch.zeros(T, device="cuda")
    F.moe_permute(x, T, 1, row, xs)
    assert torch.equal(xs, x.flip(0))
    F.moe_permute_grad(xs, T, 1, row, y)
    assert torch.equal(y, x)
    F.moe_unpermute(xs, T, 1, row, w, y)
    assert torch.equal(y, (x * w[:, None]).half())
    F.moe_unpermute_grad(x, xs, T, 1, row, w, y, dw)
    assert torch.equal(y, (x * w[:, None]).half().flip(0))
    assert torch.equal(dw, x[:, 0].float() ** 2 + x[:, 1].float() ** 2)   # (integers below 2^24)


def test_python_refuses_counts_past_the_librarys_ints(monkeypatch):
    """2^32 tokens, which a C int would cut to none, are a ValueError before anything is launched (the tensors' own checks and
    the device's are left out here: there is no memory for such rows)."""
    from flashrt_amd import moe
    monkeypatch.setattr(moe, "_raw_stream", lambda dev: 0)
    monkeypatch.setattr(moe, "_current_device", lambda: 0)
    p = 1 << 20
    for T in (2 ** 31, 2 ** 32):
        with pytest.raises(ValueError, match="C int"):
            moe._enqueue(moe.lib().frt_moe_permute, 0, None, p, 1, 1, T, 1, 1, p, p, 1)
        with pytest.raises(ValueError, match="C int"):
            moe._enqueue(moe.lib().frt_mx4_product, 0, None, p, p, 1, p, p, p, p, 1, T, 8, 32, p, 8, 0)


def test_tensors_that_require_a_gradient_are_refused():
    """The calls record nothing for autograd: with gradients enabled, an input or output that requires one is a ValueError (its
    gradient would be lost without a word); detached, or with gradients disabled, it is taken (here up to the device's check)."""
    import flashrt_amd as F
    x, xs, row = torch.zeros(4, 8), torch.zeros(8, 8), torch.zeros(8, dtype=torch.int32)
    wts, u8 = torch.ones(8), torch.zeros(64, dtype=torch.uint8)
    calls = [(F.moe_permute, (x, 4, 2, row, xs)), (F.moe_permute_grad, (xs, 4, 2, row, x)), (F.moe_unpermute, (xs, 4, 2, row, wts, x)),
             (F.moe_unpermute_grad, (x, xs, 4, 2, row, wts, xs, wts)), (F.mx4_quantize, (torch.zeros(2, 32), u8, u8)),
             (F.mx4_dequantize, (u8, u8, torch.zeros(2, 32))), (F.mx4_product, (u8.view(4, 16), u8, u8.view(4, 16), u8, torch.zeros(4, 4)))]
    for fn, args in calls:
        for i, a in enumerate(args):
            if not (isinstance(a, torch.Tensor) and a.is_floating_point()):
                continue
            with_grad = [b.clone().requires_grad_() if j == i else b for j, b in enumerate(args)]
            with pytest.raises(ValueError, match="requires a gradient"):
                fn(*with_grad)
            with torch.no_grad(), pytest.raises(ValueError, match="device"):
                fn(*with_grad)
            with pytest.raises(ValueError, match="device"):
                fn(*(b.detach() if j == i else b for j, b in enumerate(with_grad)))


class _Permute(torch.autograd.Function):
    """Token rows in expert order, as a user's training code wraps the calls."""

    @staticmethod
    def forward(ctx, x, row, T, K):
        import flashrt_amd as F
        xs = torch.zeros(T * K, x.shape[1], dtype=x.dtype, device=x.device)
        F.moe_permute(x, T, K, row, xs)
        ctx.save_for_backward(row)
        ctx.T, ctx.K = T, K
        return xs

    @staticmethod
    def backward(ctx, dxs):
        import flashrt_amd as F
        dx = torch.empty(ctx.T, dxs.shape[1], dtype=dxs.dtype, device=dxs.device)
        F.moe_permute_grad(dxs.contiguous(), ctx.T, ctx.K, ctx.saved_tensors[0], dx)
        return dx, None, None, None


class _Unpermute(torch.autograd.Function):
    """The weighted sum back into the tokens."""

    @staticmethod
    def forward(ctx, ys, wts, row, T, K):
        import flashrt_amd as F
        y = torch.empty(T, ys.shape[1], dtype=ys.dtype, device=ys.device)
        F.moe_unpermute(ys, T, K, row, wts, y)
        ctx.save_for_backward(ys, wts, row)
        ctx.T, ctx.K = T, K
        return y

    @staticmethod
    def backward(ctx, dy):
        import flashrt_amd as F
        ys, wts, row = ctx.saved_tensors
        dys, dw = torch.zeros_like(ys), torch.empty_like(wts)
        F.moe_unpermute_grad(dy.contiguous(), ys, ctx.T, ctx.K, row, wts, dys, dw)
        return dys, dw, None, None, None


@pytest.mark.gpu
@pytest.mark.parametrize("drop", ["flat", "drop"])
def test_training_step_through_autograd(drop):
    """The moves in autograd Functions around an expert's product (row scales here), against autograd of the same in 64 bits on the
    CPU: the gradients of the tokens, the scales and the routing weights. Errors: a token's row passes the product of three factors
    and two sums of at most K terms, a weight's gradient a sum of n, so (n + 3 K + 8) roundings of the sum of magnitudes at most."""
    T, K, E, n = 29, 4, 8, 72
    ids = slots(T, K, E, drop, 9)
    _, slot_of, row_of = sorted_slots(ids, E)
    row = torch.from_numpy(row_of.astype(np.int32)).cuda()
    g = torch.Generator().manual_seed(2)
    x, dy, scale, wts = torch.randn(T, n, generator=g), torch.randn(T, n, generator=g), torch.randn(T * K, 1, generator=g), torch.rand(T, K, generator=g)
    on = [v.cuda().requires_grad_() for v in (x, scale, wts)]
    y = _Unpermute.apply(_Permute.apply(on[0], row, T, K) * on[1], on[2], row, T, K)
    y.backward(dy.cuda())

    def plain(x, scale, wts, dy):   # the same from indexing, in 64 bits
        at, live = torch.from_numpy(np.where(row_of < 0, 0, row_of)), torch.from_numpy(row_of >= 0)
        leaves = [v.double().requires_grad_() for v in (x, scale, wts)]
        v = leaves[0].repeat_interleave(K, 0) * leaves[1][at]
        out = (torch.where(live[:, None], v, 0.0).view(T, K, n) * leaves[2][:, :, None]).sum(1)
        out.backward(dy.double())
        return [out.detach()] + [v.grad for v in leaves]

    want, mag = plain(x, scale, wts, dy), plain(x.abs(), scale.abs(), wts, dy.abs())
    for got, w, m in zip([y] + [v.grad for v in on], want, mag):
        near(got, w, 1.01 * (n + 3 * K + 8) * U * m)


@pytest.mark.gpu
def test_written_tensors_count_as_changed():
    """Every output's version goes up with a call, and no input's; a backward whose saved row map or rows another call has since
    overwritten says so instead of using them."""
    import flashrt_amd as F
    T, K, E, n = 3, 2, 4, 64
    i32 = lambda m: torch.zeros(m, dtype=torch.int32, device="cuda")  # noqa: E731
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8, device="cuda")  # noqa: E731
    ids = torch.tensor([0, 1, 2, 3, 0, 1], dtype=torch.int32, device="cuda")
    b, tok, slot, row = i32(E + 1), i32(T * K), i32(T * K), i32(T * K)
    x, xs, y, dys = (torch.randn(r, n, device="cuda") for r in (T, T * K, T, T * K))
    w, dw, q, s, h = torch.rand(T, K, device="cuda"), torch.zeros(T, K, device="cuda"), u8(T, n // 2), u8(T, n // 32), torch.zeros(T, T, device="cuda")
    everything = [ids, b, tok, slot, row, x, xs, y, dys, w, dw, q, s, h]
    for outs, call in [((b, tok, slot, row), lambda: F.moe_sort(ids, T, K, E, b, tok, slot, row)), ((xs,), lambda: F.moe_permute(x, T, K, row, xs)),
                       ((y,), lambda: F.moe_permute_grad(xs, T, K, row, y)), ((y,), lambda: F.moe_unpermute(xs, T, K, row, w, y)),
                       ((dys, dw), lambda: F.moe_unpermute_grad(x, xs, T, K, row, w, dys, dw)), ((q, s), lambda: F.mx4_quantize(x, q, s)),
                       ((y,), lambda: F.mx4_dequantize(q, s, y)), ((h,), lambda: F.mx4_product(q, s, q, s, h))]:
        was = [v._version for v in everything]
        call()
        for v, old in zip(everything, was):
            assert v._version == old + any(v is o for o in outs)
    for overwrite in (lambda: F.moe_sort(ids, T, K, E, b, tok, slot, row), lambda: F.moe_permute(x, T, K, row, xs)):
        out = _Unpermute.apply(xs, w.clone().requires_grad_(), row, T, K)
        overwrite()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()
    with torch.inference_mode():   # (tensors without a version)
        z = torch.empty(T * K, n, device="cuda")
        F.moe_permute(x, T, K, row, z)
        assert torch.equal(z, x[tok.long()])


def test_misaligned_words_are_refused():
    """Ids, row maps, bounds, picked rows and weights that are not 4-byte aligned are refused before any launch (the kernels read
    some of them through scalar loads, which drop an address's low bits)."""
    from flashrt_amd import _lib
    L = _lib.lib()
    p = 1 << 20
    for fn, good, ptrs in ((L.frt_moe_sort, [None, p, 2, 2, 4, p, p, p, p], (1, 5, 6, 7, 8)),
                           (L.frt_moe_permute, [None, p, 8, 30, 2, 2, 8, p, p, 8], (7,)),
                           (L.frt_moe_permute_grad, [None, p, 8, 30, 2, 2, 8, p, p, 8], (7,)),
                           (L.frt_moe_unpermute, [None, p, 8, 30, 2, 2, 8, p, p, p, 8], (7, 8)),
                           (L.frt_moe_unpermute_grad, [None, p, 8, p, 8, 30, 2, 2, 8, p, p, p, 8, p], (9, 10, 13)),
                           (L.frt_mx4_product, [None, p, p, 5, p, p, p, p, 4, 5, 24, 64, p, 24, 30], (4, 7))):
        for i in ptrs:
            for off in (1, 2, 3):
                a = list(good)
                a[i] = p + off
                assert fn(*a) == -1, (fn.__name__, i, off, L.frt_last_error())
                assert b"misaligned" in L.frt_last_error()


@pytest.mark.gpu
def test_tokens_of_many_slots():
    """Two tokens of 200,003 slots each (no multiple of the four rows in flight): small integers, so that every sum is exact."""
    import flashrt_amd as F
    T, K, n = 2, 200003, 3
    g = torch.Generator().manual_seed(4)
    row = torch.randperm(T * K, generator=g).to(torch.int32)
    row[::7] = -1
    ys = torch.randint(-2, 3, (T * K, n), generator=g).float()
    wts = torch.randint(0, 3, (T, K), generator=g).float()
    live = (row >= 0)[:, None]
    picked = torch.where(live, ys[row.clamp_min(0).long()], 0.0).double().view(T, K, n)
    y, dx = torch.empty(T, n, device="cuda"), torch.empty(T, n, device="cuda")
    F.moe_unpermute(ys.cuda(), T, K, row.cuda(), wts.cuda(), y)
    F.moe_permute_grad(ys.cuda(), T, K, row.cuda(), dx)
    assert torch.equal(y.cpu().double(), (picked * wts.double()[:, :, None]).sum(1)) and torch.equal(dx.cpu().double(), picked.sum(1))
    x = torch.randint(-9, 9, (T, n), generator=g).float()
    xs = torch.full((T * K, n), 77.0, device="cuda")
    F.moe_permute(x.cuda(), T, K, row.cuda(), xs)
    want = torch.full((T * K, n), 77.0)
    want[row[row >= 0].long()] = x.repeat_interleave(K, 0)[row >= 0]
    assert torch.equal(xs.cpu(), want)
