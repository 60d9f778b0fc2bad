"""The experts of a layer trained through the calls together: sort, product of picked tokens, gated activation with its 8-bit copy, product, weighted
sum; and back through the gradients, the weights' from tokens kept in 8 bits. Every call is held to a 64-bit restatement on its own
inputs (tolerances as in the tests of the single calls), so that a rounding cannot move what follows."""
from __future__ import annotations

import os
import subprocess

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tests.test_mx8 import ref_quantize, ref_swiglu, values  # noqa: E402

STEP, U = 2.0 ** -23, 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
H_ABS = {F32: 2.0 ** -149, F16: 2.0 ** -25, BF16: 2.0 ** -134}


def near(got, want, bound):
    err = (got.detach().cpu().double() - want).abs()
    bad = ~(err <= 1.01 * (bound + HALF[got.dtype] * want.abs()) + H_ABS[got.dtype])
    assert not bad.any(), (int(bad.sum()), float(err[bad].max()), np.argwhere(bad.numpy())[:4].tolist())


def product(got, a, w, bounds, live=None):
    """got[r] = a[r] w_g^T of the groups' rows, w [E] of [out][in]."""
    for e, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        l, r = a[lo:hi], w[e].t()
        near(got[lo:hi], l @ r, a.shape[1] * STEP * (l.abs() @ r.abs()))


def cpu(*tensors):
    return [t.detach().cpu().double() for t in tensors]


class Experts(torch.autograd.Function):
    """y[t] = sum_k wts[t, k] down_e(silu(gate) up), (gate | up) = up_e x[t]; e = ids[t, k]. Keeps the tokens and gate | up in 8 bits."""

    @staticmethod
    def forward(ctx, x, up, down, wts, ids, log):
        import flashrt_amd as F
        (T, n), K, (E, two_ff, _) = x.shape, ids.shape[1], up.shape
        S, ff, kind = T * K, two_ff // 2, x.dtype
        new = lambda *s, dtype=kind: torch.zeros(s, dtype=dtype, device="cuda")  # noqa: E731
        b, tok, slot, row = (new(m, dtype=torch.int32) for m in (E + 1, S, S, S))
        F.moe_sort(ids, T, K, E, b, tok, slot, row)
        z, h, ys, y = new(S, 2 * ff), new(S, ff), new(S, n), new(T, n)
        xc, xs, zc, zs = new(T, n, dtype=torch.int8), new(T, n // 32, dtype=torch.uint8), new(S, 2 * ff, dtype=torch.int8), new(S, ff // 16, dtype=torch.uint8)
        F.moe_product(x, up, z, bounds=b, rows=tok)
        F.moe_swiglu(z, h, zc, zs, live=b[-1:])
        F.moe_product(h, down, ys, bounds=b)
        F.moe_unpermute(ys, T, K, row, wts, y)
        F.mx8_quantize(x, xc, xs)
        ctx.save_for_backward(xc, xs, zc, zs, ys, up, down, wts, b, tok, row)
        ctx.log = log
        if log is not None:
            log.update(b=b, tok=tok, row=row, z=z, h=h, ys=ys, xc=xc, xs=xs, zc=zc, zs=zs)
        return y

    @staticmethod
    def backward(ctx, dy):
        import flashrt_amd as F
        xc, xs, zc, zs, ys, up, down, wts, b, tok, row = ctx.saved_tensors
        (T, n), K, ff, kind = dy.shape, wts.shape[1], down.shape[2], dy.dtype
        S = T * K
        new = lambda *s, dtype=kind: torch.zeros(s, dtype=dtype, device="cuda")  # noqa: E731
        dys, dwts, dh, dz, h, dxs, dx = new(S, n), torch.zeros_like(wts), new(S, ff), new(S, 2 * ff), new(S, ff), new(S, n), new(T, n)
        dup, ddown = torch.empty_like(up), torch.empty_like(down)
        F.moe_unpermute_grad(dy.contiguous(), ys, T, K, row, wts, dys, dwts)
        F.moe_product_grad(dys, down, dh, bounds=b)
        F.moe_swiglu_grad(dh, dz, codes=zc, scales=zs, h=h, live=b[-1:])
        F.moe_product_wgrad(dys, h, ddown, bounds=b)
        F.moe_product_wgrad(dz, (xc, xs), dup, bounds=b, rows=tok)
        F.moe_product_grad(dz, up, dxs, bounds=b)
        F.moe_permute_grad(dxs, T, K, row, dx)
        if ctx.log is not None:
            ctx.log.update(dys=dys, dwts=dwts, dh=dh, dz=dz, again=h, dxs=dxs)
        return dx, dup, ddown, dwts, None, None


def setup(T, K, E, n, ff, kind):
    g = torch.Generator().manual_seed(T + n)
    ids = torch.from_numpy(np.random.default_rng(T).integers(0, E, (T, K)).astype(np.int32))
    if T > 1:
        ids[T // 2, 0], ids[-1] = -1, E   # a dropped slot and a padded token
    leaves = [(torch.randn(s, generator=g) * sd).to(kind).cuda() for s, sd in (((T, n), 1.0), ((E, 2 * ff, n), 2 * n ** -0.5), ((E, n, ff), ff ** -0.5))]
    wts = torch.rand(T, K, generator=g).cuda()
    return [v.requires_grad_() for v in (*leaves, wts)], ids.cuda(), torch.randn(T, n, generator=g).to(kind).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("T,K,E,n,ff", [(1, 6, 24, 256, 96), (5, 2, 3, 64, 32), (70, 6, 24, 256, 96), (300, 4, 9, 160, 64)])
def test_experts_forward_and_backward(T, K, E, n, ff, kind):
    (x, up, down, wts), ids, dy = setup(T, K, E, n, ff, kind)
    v = {}
    y = Experts.apply(x, up, down, wts, ids, v)
    y.backward(dy)
    bounds, tok, row = v["b"].tolist(), v["tok"].cpu().long(), v["row"].cpu().long()
    live = bounds[-1]
    x64, up64, down64, w64, dy64 = cpu(x, up, down, wts, dy)
    z, h, ys, dys, dh, dz, again, dxs = cpu(*(v[k] for k in ("z", "h", "ys", "dys", "dh", "dz", "again", "dxs")))
    xt = x64[tok[:live]]
    product(v["z"], xt, up64, bounds)
    want, e = ref_swiglu(z[:live], dh[:live])[:2]
    near(v["h"][:live], want, e)
    rc, rs = ref_quantize(z[:live].numpy())
    assert np.array_equal(v["zc"][:live].cpu().numpy(), rc) and np.array_equal(v["zs"][:live].cpu().numpy(), rs)
    product(v["ys"], h, down64, bounds)
    xc, xs = ref_quantize(x64.numpy())
    assert np.array_equal(v["xc"].cpu().numpy(), xc) and np.array_equal(v["xs"].cpu().numpy(), xs)
    x8 = torch.from_numpy(values(xc, xs)).to(kind).double()[tok[:live]]
    # back
    product(v["dh"], dys, down64.transpose(1, 2), bounds)
    want, e, want_dz, e_dz = ref_swiglu(torch.from_numpy(values(rc, rs)), dh[:live])
    near(v["again"][:live], want, e)
    near(v["dz"][:live], want_dz, e_dz)
    product(v["dxs"], dz, up64.transpose(1, 2), bounds)
    for e, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        for got, l, r in ((down.grad[e], dys[lo:hi].t(), again[lo:hi]), (up.grad[e], dz[lo:hi].t(), x8[lo:hi])):
            near(got, l @ r, (hi - lo) * STEP * (l.abs() @ r.abs()))
    # the sums over a token's rows
    has = (row >= 0).view(T, K, 1)
    at = lambda m: torch.where(has, m[row.clamp_min(0)].view(T, K, n), 0.0)  # noqa: E731
    terms = at(ys) * w64[:, :, None]
    near(y, terms.sum(1), (K + 1) * U * terms.abs().sum(1))
    near(x.grad, at(dxs).sum(1), K * U * at(dxs).abs().sum(1))
    dot = (at(ys) * dy64[:, None, :])
    near(wts.grad, dot.sum(2), (n + 1) * U * dot.abs().sum(2))
    assert (v["z"][live:] == 0).all() and (v["dz"][live:] == 0).all() and (v["dxs"][live:] == 0).all()


@pytest.mark.gpu
def test_one_token_and_many_in_the_same_rows():
    """A token's results on its own, as it is decoded, and in a batch: the same products through other kernels, within their roundings."""
    (x, up, down, wts), ids, _ = setup(200, 4, 9, 160, 64, BF16)
    ids.clamp_(0, 8)
    with torch.no_grad():
        many = Experts.apply(x, up, down, wts, ids, None)
        for t in (0, 77, 199):
            one = Experts.apply(x[t:t + 1].contiguous(), up, down, wts[t:t + 1].contiguous(), ids[t:t + 1].contiguous(), None)
            # z and ys differ by a step of bf16 here and there, h by what that moves it: three steps of the terms' size
            assert ((one - many[t:t + 1]).abs() <= 3 * 2.0 ** -7 * many.abs().max()).all()


@pytest.mark.gpu
def test_step_on_another_stream_and_captured():
    """Forward and backward captured into a graph and replayed on new tokens, against the eager step, with eager work between."""
    T, K, E, n, ff = 60, 4, 7, 96, 64
    (x, up, down, wts), ids, dy = setup(T, K, E, n, ff, BF16)

    def step():
        y = Experts.apply(x, up, down, wts, ids, None)
        return (y.detach(), *torch.autograd.grad(y, (x, up, down, wts), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, step()):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(4):
        g = torch.Generator().manual_seed(seed)
        with torch.no_grad():
            x.copy_(torch.randn(T, n, generator=g).to(BF16))
            dy.copy_(torch.randn(T, n, generator=g).to(BF16))
            ids.copy_(torch.randint(-1, E, (T, K), generator=g, dtype=torch.int32))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, want):
            assert torch.equal(a, b), seed


def _client(arg):
    exe = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "_build", "test_train")
    assert os.path.exists(exe), "build first: make -C flashrt_amd/csrc"
    r = subprocess.run([exe, arg], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "all passed" in r.stdout, r.stdout + r.stderr


def test_cpp_client_host():
    """The C++ mirror's calls turn refusals into std::runtime_error."""
    _client("--host")


@pytest.mark.gpu
def test_cpp_client_gpu():
    """The C++ mirror's calls in a run, exact values."""
    _client("--gpu")
