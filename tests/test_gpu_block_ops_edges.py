"""GPU tests of the transformer-block operators where their conventions meet: captures before the first eager
call, scratch that is outgrown, values that are not finite, widths without a vector or a TMA form."""
import ctypes

import numpy as np
import pytest

import block_ops_ref as ref
from test_gpu_block_ops import Attn, _dt, _rand, _weight

pytestmark = pytest.mark.gpu


def _own_context():
    """A context of its own on a side stream: nothing has run on it."""
    import torch
    import sa3k
    side = torch.cuda.Stream()
    own = sa3k.Context(0, use_torch_stream=False)
    own.set_stream(side.cuda_stream)
    return own, side


def _capture(side, fn):
    import torch
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        fn()
    return g


# ------------------------------------------------------------------------- split-K and captures
def _leave_ones_in_free_memory():
    """Small device allocations that a later one may be given hold ones: every other chunk of a few MB is freed
    (the rest are returned, for the caller to free), so that their pages stay mapped."""
    rt = ctypes.CDLL("libcudart.so.12")
    chunks = [ctypes.c_void_p() for _ in range(2000)]
    for c in chunks:
        assert rt.cudaMalloc(ctypes.byref(c), ctypes.c_size_t(4096)) == 0
        assert rt.cudaMemset(c, 1, ctypes.c_size_t(4096)) == 0
    assert rt.cudaDeviceSynchronize() == 0
    for c in chunks[::2]:
        assert rt.cudaFree(c) == 0
    return rt, chunks[1::2]


@pytest.mark.parametrize("first", ["eager", "second"])
def test_split_product_captured_before_any_eager_call(ctx, first):
    """A context's first split-K product is recorded, not run: what runs next (an eager call, or another
    recorded one) finds the tiles' counters at zero all the same."""
    import torch
    rt, held = _leave_ones_in_free_memory()
    own, side = _own_context()
    try:
        with torch.cuda.stream(side):
            w, W = _weight(own, "f16", 128, 4096, 3)      # dx: 20 rows, 128 columns, K = 4096
        rnd = _rand(5)
        dys = [rnd(20, 4096).half() for _ in range(3)]
        dxs = [torch.full((20, 128), float("nan"), device="cuda").half() for _ in range(3)]
        call = lambda i: own.linear_act_bwd(w, None, None, dys[i], dxs[i])  # noqa: E731
        torch.cuda.synchronize()
        graphs = [_capture(side, lambda i=i: call(i)) for i in range(2)]
        with torch.cuda.stream(side):
            if first == "eager":
                call(2)
                graphs[1].replay()
                graphs[0].replay()
            else:
                graphs[1].replay()
                call(2)
                graphs[0].replay()
        own.sync()
        for i in range(3):
            want = dys[i].double() @ W
            tol = ref.u(torch.float16) * want.abs() + 4096 * 2.0 ** -24 * (dys[i].double().abs() @ W.abs()) + 2.0 ** -25
            ref.assert_within(f"dx{i}", dxs[i], want, tol)
    finally:
        own.close()
        for c in held:
            rt.cudaFree(c)


# ---------------------------------------------------------------------- values that are not finite
def _sees(Sq, Sk, left, right, sinks):
    import torch
    p, j = torch.arange(Sq, device="cuda")[:, None], torch.arange(Sk, device="cuda")[None]
    return (j <= p + right) & ((j < sinks) | (j >= p - left))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("Sq", [256, 16])      # 128-row tiles; 16-row tiles
def test_attention_sink_nan_in_a_visible_key(ctx, dtype, Sq):
    """One NaN key per head, at every residue of the column: the rows that see it are NaN, the others are what
    they are without it."""
    import torch
    a, clean = (Attn(1, 48, 48, Sq, 256, 100, 0, 8, dtype=dtype, seed=21) for _ in range(2))
    at = [(5 * h) % Sq for h in range(48)]                # sink tile, whole tiles, edges; all residues mod 8
    for h, j in enumerate(at):
        a.k[0, h, j, 7 + h % 3] = float("nan")
    a.fwd(ctx)
    clean.fwd(ctx)
    ctx.sync()
    clean.check(grads=False)
    see = _sees(Sq, 256, 100, 0, 8)
    for h, j in enumerate(at):
        hit = see[:, j]
        assert bool(a.o[0, h, hit].isnan().all()) and bool(a.lse[0, h, hit].isnan().all()), (h, j)
        assert torch.equal(a.o[0, h, ~hit], clean.o[0, h, ~hit]) and torch.equal(a.lse[0, h, ~hit], clean.lse[0, h, ~hit])


@pytest.mark.parametrize("Sq", [256, 16])
def test_attention_sink_huge_values_outside_the_window(ctx, Sq):
    """A value near bf16's largest weighs exactly nothing in the rows that do not see its key.  (Those that do are
    not compared: with probabilities of up to 2^8 before the division, 2^126 leaves the f32 sums' range.)"""
    import torch
    a, clean = (Attn(1, 48, 48, Sq, 256, 20, 0, 0, dtype="bf16", seed=22) for _ in range(2))
    at = [(h * 5) % Sq for h in range(48)]
    for h, j in enumerate(at):
        a.v[0, h, j] = 2.0 ** 126
    a.fwd(ctx)
    clean.fwd(ctx)
    ctx.sync()
    clean.check(grads=False)
    see = _sees(Sq, 256, 20, 0, 0)
    for h, j in enumerate(at):
        assert torch.equal(a.o[0, h, ~see[:, j]], clean.o[0, h, ~see[:, j]]), (h, j)
    assert torch.equal(a.lse, clean.lse)


# ------------------------------------------------------------------------------------ layer norm
@pytest.mark.parametrize("cols", [200, 1000, 1536, 1537, 4100, 9000, 20000, 40000])
@pytest.mark.parametrize("offset", [1e4, -3e5, 0.0])
def test_layernorm_offset_costs_no_digits(ctx, cols, offset):
    """Rows far from zero, every form of the forward.  With m the f32 mean, d = x - m is exact (x and m are
    within a factor of two), and what m is off by is taken out as the mean of d: a chain of 74 additions of
    terms whose mean is about one standard deviation, then a few roundings of the result."""
    import torch
    x = _rand(cols)(5, cols) + offset
    y, mean, rstd = torch.empty_like(x), torch.empty(5, device="cuda"), torch.empty(5, device="cuda")
    ctx.layernorm_fwd(x, y, None, None, 1e-5, mean, rstd)
    ctx.sync()
    w = ref.layernorm(x, None, None, 1e-5, torch.float32, 74)
    c = 74 * 2.0 ** -24
    # (the first mean is off by c |offset| at most, which widens the terms by as much)
    wide = 1 + c * abs(offset)
    ref.assert_within("y", y, w["y"], 2 * c * wide + w["y"].abs() * (c * wide ** 2 + 2 ** -21))
    ref.assert_within("mean", mean, w["mean"], 2 ** -23 * w["mean"].abs() + 2 * c * wide)
    ref.assert_within("rstd", rstd, w["rstd"], w["rstd"] * (2 * c * wide ** 2 + 2 ** -21))


@pytest.mark.parametrize("cols", [7, 200, 1000, 1536, 1537, 9000, 40000])
def test_layernorm_rows_that_are_not_finite(ctx, cols):
    """An infinity or a NaN spoils its own row and no other, forward and backward."""
    import torch
    rnd = _rand(cols)
    x, dy, gamma, beta = rnd(9, cols), rnd(9, cols), 1 + 0.1 * rnd(cols), rnd(cols)
    bad = x.clone()
    bad[1, cols // 2], bad[4, 0], bad[7, cols - 1] = float("inf"), float("nan"), float("-inf")
    rows = torch.tensor([1, 4, 7], device="cuda")
    rest = torch.tensor([0, 2, 3, 5, 6, 8], device="cuda")

    def run(t):
        y, dx, mean, rstd = torch.empty_like(t), torch.empty_like(t), torch.empty(9, device="cuda"), torch.empty(9, device="cuda")
        ctx.layernorm_fwd(t, y, gamma, beta, 1e-5, mean, rstd)
        ctx.layernorm_bwd(t, dy, dx, mean, rstd, gamma)
        ctx.sync()
        return y, mean, rstd, dx

    for got, want in zip(run(bad), run(x)):
        assert torch.equal(got[rest], want[rest])
    y, mean, rstd, dx = run(bad)
    assert bool(y[rows].isnan().all()) and bool(rstd[rows].isnan().all()) and bool(dx[rows].isnan().all())
    assert float(mean[1]) == float("inf") and bool(mean[4].isnan()) and float(mean[7]) == float("-inf")


# ------------------------------------------------------- the layer norm backward's ring of rows
RING = [  # rows, cols: every block refills its slots several times; each of the kernel's forms; odd last pairs
    (30001, 264), (9999, 768), (7001, 1536), (4003, 2048), (2500, 2560), (3001, 4096), (1999, 5120), (2001, 5128), (1201, 8192),
    (296, 8192), (150, 8192),
]


@pytest.mark.parametrize("rows,cols", RING)
@pytest.mark.parametrize("xt,yt", [("f32", "f16"), ("f16", "f16"), ("bf16", "f32"), ("f32", "f32")])
def test_layernorm_backward_of_many_rows(ctx, rows, cols, xt, yt):
    import torch
    rnd = _rand(rows + cols)
    x, gamma = (rnd(rows, cols) + 0.5 * rnd(cols)).to(_dt(xt)), 1 + 0.3 * rnd(cols)
    dy = rnd(rows, cols).to(_dt(yt))
    mean, rstd = x.double().mean(1).float(), (x.double().var(1, unbiased=False) + 1e-5).rsqrt().float()
    dx = torch.full_like(x, float("nan"))
    dg, db = (torch.full((cols,), float("nan"), device="cuda") for _ in range(2))
    ctx.layernorm_bwd(x, dy, dx, mean, rstd, gamma, dg, db)
    g = ref.layernorm_grads(x, dy, gamma, mean, rstd, 74, 64 + rows // 64)
    for n, got in (("dx", dx), ("dgamma", dg), ("dbeta", db)):
        ref.assert_within(n, got, g[n], g[n + "_tol"])
    again = torch.empty_like(dx)
    dg2, db2 = torch.ones_like(dg), torch.ones_like(db)
    ctx.layernorm_bwd(x, dy, again, mean, rstd, gamma, dg2, db2, accumulate=True)
    ctx.sync()
    assert torch.equal(again, dx) and torch.equal(dg2, dg + 1) and torch.equal(db2, db + 1)


# ------------------------------------------------------------------------ widths of quantized bases
ODD_WIDTHS = [  # S, in, out, weight, type
    (5, 128, 77, "q8_0", "f16"), (33, 128, 77, "q8_0", "f16"), (200, 192, 129, "q8_0", "f32"), (40, 128, 520, "q8_0", "f16"),
    (300, 64, 1001, "q8_0", "f16"), (33, 256, 77, "q4_k", "f16"), (300, 256, 1000, "q4_k", "f32"), (130, 512, 264, "q4_k", "f16"),
    (70, 128, 202, "q8_0", "f16"), (520, 256, 3, "q8_0", "f16"),
]


@pytest.mark.parametrize("inside", ["no copy", "forced"])
@pytest.mark.parametrize("S,inn,out,kind,t", ODD_WIDTHS)
def test_linear_act_any_width_without_the_half_copy(ctx, S, inn, out, kind, t, inside):
    """Every output width is taken whether the products dequantize the base themselves or not, few rows and many."""
    import torch
    import sa3k
    option, value = (sa3k.OPT_WEIGHT_F16_CACHE, 0) if inside == "no copy" else (sa3k.OPT_SMEM_DEQUANT, 1)
    ctx.set_option(option, value)
    try:
        w, W = _weight(ctx, kind, inn, out, S + out)
        rnd = _rand(S * 3 + out)
        dt, D = _dt(t), torch.float64
        x, bias, res, zin, dy = rnd(S, inn).to(dt), rnd(out), rnd(S, out).to(dt), rnd(S, out).to(dt), rnd(S, out).to(dt)
        y, z, dx = (torch.full((S, n), float("nan"), device="cuda", dtype=dt) for n in (out, out, inn))
        ctx.linear_act_fwd(w, x, y, "silu", bias=bias, residual=res, z=z)
        ctx.linear_act_bwd(w, None, zin, dy, dx, "silu")
        ctx.sync()
    finally:
        ctx.set_option(option, 1 - value)
    # roundings as in test_linear_act: the weight and (f32) x to half, f32 sums, the result
    eps = 2.0 ** -11 + (2.0 ** -11 if t == "f32" else 0.0)
    small = 2.0 ** -25 if t == "f16" else 1e-30
    zr = x.to(D) @ W.T + bias.to(D)
    zt = (eps + inn * 2.0 ** -24) * (x.to(D).abs() @ W.T.abs() + bias.to(D).abs())
    yr = ref.act(zr, "silu") + res.to(D)
    ref.assert_within("z", z, zr, ref.u(dt) * zr.abs() + zt + small)
    ref.assert_within("y", y, yr, ref.u(dt) * yr.abs() + 1.13 * zt + 2 ** -20 * (zr.abs() + yr.abs()) + small)
    zz = zin.to(D).requires_grad_(True)
    ref.act(zz, "silu").backward(dy.to(D))
    dz = zz.grad
    e2 = 2.0 ** -10 + out * 2.0 ** -24 + 2 ** -19
    lost = (2 ** -25 + 2 ** -19) * W.abs().sum(0)
    dxr = dz @ W
    ref.assert_within("dx", dx, dxr, ref.u(dt) * dxr.abs() + e2 * (dz.abs() @ W.abs()) + lost * dy.abs().max().double() + small)


@pytest.mark.parametrize("dora", [False, True])
def test_linear_act_adapter_widths(ctx, dora):
    """An adapter's backward takes widths of 8 and refuses others before it has written anything."""
    import torch
    import sa3k
    for out in (72, 77):
        w, W = _weight(ctx, "q8_0", 128, out, 5)
        rnd = _rand(out)
        A, Bm = rnd(16, 128) / 128 ** 0.5, 0.1 * rnd(out, 16)
        bns, nrm = torch.empty(out, device="cuda"), torch.empty(out, device="cuda")
        ctx.row_norms(w, 1e-12, bns, nrm)
        m = 1.1 * nrm if dora else None
        ad = ctx.adapter(A, Bm, 0.7, m, bns if dora else None)
        x, dy = rnd(50, 128).half(), rnd(50, out).half()
        y, z, dx = (torch.full((50, n), 9.0, device="cuda").half() for n in (out, out, 128))
        ctx.linear_act_fwd(w, x, y, "silu", z=z, ad=ad)
        leaves = [v.double().requires_grad_(True) for v in (x, A, Bm, *((m,) if dora else ()))]
        V = W + 0.7 * leaves[2] @ leaves[1]
        if dora:
            V = V * (leaves[3] / ((V ** 2).sum(1) + 128 * 1e-12).sqrt())[:, None]
        yr = ref.act(leaves[0] @ V.T, "silu")
        rel = lambda a, b: float((a.double() - b).norm() / b.norm())  # noqa: E731
        assert rel(y, yr.detach()) < 5 * 2.0 ** -11      # (half operands in a chain, see test_linear_act_with_adapter)
        grads = [torch.full(s, 9.0, device="cuda") for s in ((out,), (16, 128), (out, 16), (out,))]
        bwd = lambda: ctx.linear_act_bwd(w, x, z, dy, dx, "silu", dbias=grads[0], ad=ad, dA=grads[1], dB=grads[2],  # noqa: E731
                                         dm=grads[3] if dora else None)
        if out % 8:
            with pytest.raises(sa3k.Sa3kError, match="multiple of 8"):
                bwd()
            ctx.sync()
            assert all(bool((g == 9.0).all()) for g in (*grads, dx))
            continue
        bwd()
        ctx.sync()
        yr.backward(dy.double())
        got = [dx, grads[1], grads[2], *((grads[3],) if dora else ())]
        for g, leaf in zip(got, leaves):
            assert rel(g, leaf.grad) < 5 * 2.0 ** -11


# ------------------------------------------------------------------------------- scratch and captures
def _used():
    import gc
    import torch
    gc.collect()          # (what earlier tests left is not freed between two looks)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    free, total = torch.cuda.mem_get_info()
    return total - free


def test_scratch_of_captures_that_grow(ctx):
    """Captured calls of ever larger sizes hold a few times the largest one's scratch, not the sum of all."""
    import torch
    own, side = _own_context()
    try:
        with torch.cuda.stream(side):
            w, _ = _weight(own, "f16", 64, 2048, 3)
        top = 12000
        z, dy = (torch.zeros(top, 2048, device="cuda").half() for _ in range(2))
        dx, db = torch.zeros(top, 64, device="cuda").half(), torch.zeros(2048, device="cuda")
        call = lambda s: own.linear_act_bwd(w, None, z[:s], dy[:s], dx[:s], "silu", dbias=db)  # noqa: E731
        torch.cuda.synchronize()
        call(64)
        own.sync()
        before, graphs = _used(), []
        for s in range(2000, top + 1, 500):
            graphs.append(_capture(side, lambda s=s: call(s)))
        held = _used() - before
        largest = top * 2048 * 2 + (top // 16 + 1) * 2 * 2048 * 4           # dz in half, partial column sums
        assert held < 4 * largest, (held, largest)
        with torch.cuda.stream(side):
            for g in graphs:
                g.replay()
        own.sync()
        graphs.clear()
    finally:
        own.close()


def test_step_graph_gives_its_scratch_back(ctx):
    """The DiT step's own recorded graph is made anew when its scratch grows: the old scratch is freed."""
    import test_gpu_dit as dit_test
    import sa3k

    def run(lengths):
        own = sa3k.Context(0, use_torch_stream=False)
        try:
            start = _used()
            dit, _, _, _, rng = dit_test._build(own, dict(dit_test.CFG, depth=1))
            for T in lengths:
                f32 = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
                ins = f32(1, T, 64), f32(1, T, 64), f32(1, 64), f32(1, 16, 64), f32(1, 64)
                for _ in range(3):           # eager, recorded, replayed
                    dit.forward_backward(1, T, 16, *ins, loss=np.zeros(1, np.float32))
            own.sync()
            return _used() - start
        finally:
            own.close()

    lengths = list(range(4000, 12001, 1000))
    run(lengths[:1])                                       # (modules are loaded)
    alone, grown = run(lengths[-1:]), run(lengths)
    # the rotation table alone is 512 bytes a token: 32 MB over the shorter lengths
    assert grown - alone < 12 << 20, (grown, alone)


def test_linear_act_backward_scratch(ctx):
    """The partial sums of a backward without a dora adapter take one plane of S / 16 rows."""
    import torch
    own, side = _own_context()
    try:
        with torch.cuda.stream(side):
            w, _ = _weight(own, "f16", 64, 4096, 3)
        S = 64000
        z, dy = (torch.zeros(S, 4096, device="cuda").half() for _ in range(2))
        dx, db = torch.zeros(S, 64, device="cuda").half(), torch.zeros(4096, device="cuda")
        torch.cuda.synchronize()
        own.linear_act_bwd(w, None, z[:64], dy[:64], dx[:64], "silu", dbias=db)
        own.sync()
        before = _used()
        own.linear_act_bwd(w, None, z, dy, dx, "silu", dbias=db)
        own.sync()
        held, plane = _used() - before, S // 16 * 4096 * 4
        assert held < S * 4096 * 2 + plane + plane // 2, (held, plane)
    finally:
        own.close()


# --------------------------------------------------------------------- the same bits, and replays
@pytest.mark.parametrize("kw", [
    dict(B=1, H=1, Hkv=1, Sq=1, Sk=20011, left=-1, right=0, sinks=0, end=True),              # clusters of 16
    dict(B=2, H=24, Hkv=8, Sq=1, Sk=3000, left=800, right=0, sinks=64, end=True, dtype="bf16"),
    dict(B=1, H=3, Hkv=3, Sq=40, Sk=900, left=300, right=0, sinks=4, end=True),
    dict(B=2, H=24, Hkv=8, Sq=600, Sk=600, left=200, right=0, sinks=30, dtype="bf16"),
])
def test_attention_sink_repeats_and_replays(ctx, kw):
    """Twenty calls give the same bits; a captured call gives them too, on inputs that came after the capture."""
    import torch
    own, side = _own_context()
    try:
        a = Attn(**kw, seed=31)
        torch.cuda.synchronize()
        a.fwd(own)
        a.bwd(own)
        own.sync()
        g = _capture(side, lambda: (a.fwd(own), a.bwd(own)))
        with torch.cuda.stream(side):
            a.q.copy_(a.q.flip(1)), a.v.neg_()
            a.fwd(own)
            a.bwd(own)
            first = [t.clone() for t in (a.o, a.lse, a.dq, a.dk, a.dv)]
            for i in range(20):
                for t in (a.o, a.lse, a.dq, a.dk, a.dv):
                    t.fill_(9.0)
                if i % 2:
                    g.replay()
                else:
                    a.fwd(own)
                    a.bwd(own)
                for x, y in zip(first, (a.o, a.lse, a.dq, a.dk, a.dv)):
                    assert torch.equal(x, y)
        own.sync()
        a.check()
    finally:
        own.close()


@pytest.mark.parametrize("S,inn,out", [(1, 1536, 6144), (33, 1536, 6144), (20, 4096, 128), (1100, 1536, 1544), (4352, 512, 1536)])
def test_linear_act_repeats(ctx, S, inn, out):
    """Few rows, split-K and pair tiles: the same bits every time (without an adapter, whose gradients use atomics)."""
    import torch
    w, _ = _weight(ctx, "q8_0", inn, out, 3)
    rnd = _rand(S)
    x, res, dy, bias = rnd(S, inn).half(), rnd(S, out).half(), rnd(S, out).half(), rnd(out)
    runs = []
    for _ in range(6):
        y, z, dx = (torch.full((S, n), float("nan"), device="cuda").half() for n in (out, out, inn))
        db = torch.empty(out, device="cuda")
        ctx.linear_act_fwd(w, x, y, "gelu_tanh", bias=bias, residual=res, z=z)
        ctx.linear_act_bwd(w, None, z, dy, dx, "gelu_tanh", dbias=db)
        runs.append((y, z, dx, db))
    ctx.sync()
    for other in runs[1:]:
        for a, b in zip(runs[0], other):
            assert torch.equal(a, b)


def test_dense_and_windowed_attention_in_turn(ctx):
    """Kernels of 512, 256 and 128 tensor-memory columns follow one another on one stream, each started early."""
    import torch
    a = Attn(1, 16, 16, 500, 500, 100, 100, 0, token_major=False, seed=41)
    o2, lse2 = torch.empty_like(a.q), torch.empty(16 * 500, device="cuda")
    grads = [torch.empty(1, 16, 500, 64, device="cuda") for _ in range(3)]
    for _ in range(30):
        a.fwd(ctx)
        ctx.attention_fwd(1, 16, 500, 500, 0.125, 100, a.t4(a.q), a.t4(a.k), a.t4(a.v), a.t4(o2), lse2)
        a.bwd(ctx)
        ctx.attention_bwd(1, 16, 500, 500, 0.125, 100, a.t4(a.q), a.t4(a.k), a.t4(a.v), a.t4(o2), a.t4(a.dO), lse2,
                          *(a.t4(t) for t in grads))
    ctx.sync()
    a.check()
    assert float((a.o.double() - o2.double()).norm() / o2.double().norm()) < 1e-3   # two roundings of P and o each
    for mine, dense in zip((a.dq, a.dk, a.dv), grads):
        # P, dS and the gradient rounded to half on this side, P and dS on the other
        assert float((mine.double() - dense.double()).norm() / dense.double().norm()) < 3e-3
