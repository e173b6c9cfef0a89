"""GPU tests of layer normalisation, attention with sink tokens and the linear with activation and
residual, through the C ABI, against float64 with derived elementwise bounds (block_ops_ref.py)."""
import itertools

import numpy as np
import pytest

import block_ops_ref as ref
import gguf_blocks

pytestmark = pytest.mark.gpu
T = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}


def _dt(name):
    import torch
    return getattr(torch, T[name])


def _rand(seed):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=g, device="cuda")


# ------------------------------------------------------------------------------------ layer norm
LN_SHAPES = [(1, 1), (3, 7), (5, 8), (2, 40), (33, 64), (7, 255), (9, 256), (4, 257), (3, 1000), (5, 1001), (6, 1536),
             (3, 4100), (2, 8200), (2, 16400), (1, 40000), (700, 96), (1500, 520)]


@pytest.mark.parametrize("rows,cols", LN_SHAPES)
@pytest.mark.parametrize("xt,yt", [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f32"), ("f16", "f32"),
                                   ("bf16", "f16")])
def test_layernorm(ctx, rows, cols, xt, yt):
    import torch
    rnd = _rand(rows * 7 + cols)
    x = (rnd(rows, cols) * 2 + 3 * rnd(cols)).to(_dt(xt))
    gamma, beta = 1 + 0.3 * rnd(cols), 0.2 * rnd(cols)
    y = torch.full((rows, cols), float("nan"), device="cuda", dtype=_dt(yt))
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    ctx.layernorm_fwd(x, y, gamma, beta, 1e-5, mean, rstd)
    # a thread adds at most 64 values of a row, then 10 levels of a tree
    w = ref.layernorm(x, gamma, beta, 1e-5, _dt(yt), 74)
    for n, got in (("mean", mean), ("rstd", rstd), ("y", y)):
        ref.assert_within(n, got, w[n], w[n + "_tol"])
    dy = rnd(rows, cols).to(_dt(yt))
    dx = torch.full_like(x, float("nan"))
    dgamma, dbeta = torch.full((cols,), float("nan"), device="cuda"), torch.full((cols,), float("nan"), device="cuda")
    ctx.layernorm_bwd(x, dy, dx, mean, rstd, gamma, dgamma, dbeta)
    # a column's chain: the rows that one thread walks, the groups of its block and the blocks
    g = ref.layernorm_grads(x, dy, gamma, mean, rstd, 74, 64 + rows // 64)
    for n, got in (("dx", dx), ("dgamma", dgamma), ("dbeta", dbeta)):
        ref.assert_within(n, got, g[n], g[n + "_tol"])
    # accumulated, without dx; and the same bits in a second run
    again = dgamma.clone()
    ctx.layernorm_bwd(x, dy, None, mean, rstd, gamma, again, None, accumulate=True)
    assert torch.equal(again, dgamma + dgamma)
    ctx.sync()


def test_layernorm_strides_and_alignment(ctx):
    import torch
    rnd = _rand(5)
    for off, ld, cols in ((0, 80, 64), (1, 67, 64), (8, 72, 56), (3, 1600, 1536), (0, 1540, 1536)):
        store = rnd(9, ld + 16).half()
        x = store.as_strided((9, cols), (ld, 1), off)
        out = torch.full((9 * ld + 32,), 7.0, device="cuda", dtype=torch.float16)
        y = out.as_strided((9, cols), (ld, 1), off)
        ctx.layernorm_fwd(x, y)
        w = ref.layernorm(x, None, None, 1e-5, torch.float16, 74)
        ref.assert_within("y", y, w["y"], w["y_tol"])
        y.fill_(7.0)
        assert bool((out == 7.0).all()), "written outside the rows"


def test_layernorm_common_offset_and_constant_rows(ctx):
    import torch
    rnd = _rand(6)
    x = rnd(4, 1536) + torch.tensor([[1e4], [-3e3], [0.0], [1.0]], device="cuda")
    x[3] = 2.5                                        # no variance: y = beta
    y = torch.empty_like(x)
    ctx.layernorm_fwd(x, y)
    w = ref.layernorm(x, None, None, 1e-5, torch.float32, 74)
    ref.assert_within("y", y, w["y"], w["y_tol"])
    assert float(y[3].abs().max()) == 0.0


def test_layernorm_gradient_against_differences(ctx):
    import torch
    rnd = _rand(7)
    x, dy, gamma = rnd(3, 24), rnd(3, 24), 1 + 0.2 * rnd(24)
    mean, rstd, y = torch.empty(3, device="cuda"), torch.empty(3, device="cuda"), torch.empty_like(x)
    ctx.layernorm_fwd(x, y, gamma, None, 1e-5, mean, rstd)
    dx = torch.empty_like(x)
    ctx.layernorm_bwd(x, dy, dx, mean, rstd, gamma)
    f = lambda t: float((ref.layernorm(t, gamma, None, 1e-5, torch.float32, 1)["y"] * dy.double()).sum())  # noqa: E731
    h = 1e-4
    for i, j in ((0, 0), (1, 7), (2, 23)):
        e = torch.zeros(3, 24, dtype=torch.float64, device="cuda")
        e[i, j] = h
        num = (f(x.double() + e) - f(x.double() - e)) / (2 * h)
        assert abs(num - float(dx[i, j])) < 1e-5 * (1 + abs(num))   # h^2 and f32 rounding are far below


def test_layernorm_refusals(ctx):
    import torch
    import sa3k
    x = torch.zeros(4, 16, device="cuda")
    m = torch.zeros(4, device="cuda")
    with pytest.raises(sa3k.Sa3kError, match="matrix with contiguous rows"):
        ctx.layernorm_fwd(x, torch.zeros(4, 15, device="cuda"))
    with pytest.raises(sa3k.Sa3kError, match="float32 vector of 16"):
        ctx.layernorm_fwd(x, x.clone(), torch.zeros(15, device="cuda"))
    with pytest.raises(sa3k.Sa3kError, match="unsupported type"):
        ctx.layernorm_fwd(x.double(), x.clone())
    with pytest.raises(sa3k.Sa3kError, match="eps"):
        ctx.layernorm_fwd(x, x.clone(), eps=-1.0)
    with pytest.raises(sa3k.Sa3kError, match="context on"):
        ctx.layernorm_fwd(x, torch.zeros(4, 16))
    with pytest.raises(sa3k.Sa3kError, match="smaller than a row"):
        ctx.layernorm_fwd(x.as_strided((4, 16), (8, 1)), x.clone())
    with pytest.raises(sa3k.Sa3kError, match="x's type"):
        ctx.layernorm_bwd(x, x.clone(), x.half(), m, m)
    # no rows: nothing is launched, fresh parameter gradients are zero
    e, dg = torch.zeros(0, 16, device="cuda"), torch.ones(16, device="cuda")
    ctx.layernorm_fwd(e, e.clone())
    ctx.layernorm_bwd(e, e.clone(), None, m[:0], m[:0], dgamma=dg)
    assert float(dg.abs().max()) == 0.0


# --------------------------------------------------------------------- attention with sink tokens
class Attn:
    """Inputs of one attention in a chosen layout, with NaN behind the sequences' ends."""

    def __init__(self, B, H, Hkv, Sq, Sk, left, right, sinks, end=False, qn=None, kn=None, dtype="f16", token_major=True,
                 seed=0, scale=0.125, pad=0):
        import torch
        import sa3k
        rnd = _rand(seed + 31 * Sq + Sk)
        dt = _dt(dtype)
        self.dims = (B, H, Hkv, Sq, Sk)
        self.win = (scale, left, right, sinks)
        self.end, self.tm, self.pad = end, token_major, pad
        self.qn, self.kn = qn or [Sq] * B, kn or [Sk] * B
        self.q, self.dO = self._lay(rnd(B, H, Sq, 64).to(dt)), self._lay(rnd(B, H, Sq, 64).to(dt))
        self.k, self.v = self._lay(rnd(B, Hkv, Sk, 64).to(dt)), self._lay(rnd(B, Hkv, Sk, 64).to(dt))
        for b in range(B):
            for t, n in ((self.q, self.qn), (self.dO, self.qn), (self.k, self.kn), (self.v, self.kn)):
                t[b, :, min(max(n[b], 0), t.shape[2]):] = float("nan")
        self.o, self.dq = (self._lay(torch.full_like(self.q, 9.0)) for _ in range(2))
        self.dk, self.dv = (self._lay(torch.full_like(self.k, 9.0)) for _ in range(2))
        self.lse = torch.full((B, H, Sq), 9.0, device="cuda")
        i32 = lambda n: torch.tensor(n, dtype=torch.int32, device="cuda")  # noqa: E731
        self.p = sa3k.sink_attn(B, H, Sq, Sk, scale, left, right, sinks, heads_kv=Hkv, dtype=dtype, align_end=end,
                                q_len=i32(qn) if qn else None, kv_len=i32(kn) if kn else None)

    def _lay(self, t):
        """[B][H][S][64] values in token-major or head-major storage (rows `pad` values apart)."""
        import torch
        B, H, S, _ = t.shape
        if self.tm:
            store = torch.zeros(B, S, H * 64 + self.pad, device="cuda", dtype=t.dtype)
            view = store[..., :H * 64].unflatten(-1, (H, 64)).permute(0, 2, 1, 3)
        else:
            view = torch.zeros(B, H, S, 64 + self.pad, device="cuda", dtype=t.dtype)[..., :64]
        view.copy_(t)
        return view

    def t4(self, t):
        import sa3k
        return sa3k.t4(t, t.stride(0), t.stride(1), t.stride(2))

    def fwd(self, ctx):
        ctx.attention_sink_fwd(self.p, *(self.t4(t) for t in (self.q, self.k, self.v, self.o)), self.lse)

    def bwd(self, ctx, kv=True):
        ctx.attention_sink_bwd(self.p, *(self.t4(t) for t in (self.q, self.k, self.v, self.o, self.dO)), self.lse,
                               self.t4(self.dq), self.t4(self.dk) if kv else None, self.t4(self.dv) if kv else None)

    def check(self, grads=True):
        import torch
        scale, left, right, sinks = self.win
        for b in range(self.dims[0]):
            nq, nk = min(max(self.qn[b], 0), self.dims[3]), min(max(self.kn[b], 0), self.dims[4])
            w = ref.attention(self.q[b], self.k[b], self.v[b], scale, left, right, sinks, nq, nk, self.end,
                              self.dO[b] if grads else None, self.o[b], self.lse[b])
            names = ("o", "lse") + (("dq", "dk", "dv") if grads else ())
            for n in names:
                t, rows = getattr(self, n)[b], nk if n in ("dk", "dv") else nq
                ref.assert_within(f"{n}[{b}]", t[:, :rows], w[n], w[n + "_tol"])
                assert bool((t[:, rows:] == 9.0).all()), f"{n}[{b}]: rows behind the end were written"


SINK_CASES = [
    # B, H, Hkv, Sq, Sk, left, right, sinks
    dict(B=1, H=1, Hkv=1, Sq=1, Sk=1, left=0, right=0, sinks=0),
    dict(B=2, H=3, Hkv=3, Sq=200, Sk=200, left=40, right=40, sinks=8),
    dict(B=1, H=4, Hkv=2, Sq=333, Sk=333, left=64, right=0, sinks=4),
    dict(B=1, H=2, Hkv=1, Sq=700, Sk=700, left=100, right=17, sinks=70, dtype="bf16"),
    dict(B=1, H=2, Hkv=2, Sq=513, Sk=513, left=0, right=0, sinks=0),            # each row sees itself
    dict(B=1, H=2, Hkv=2, Sq=513, Sk=513, left=0, right=0, sinks=129),
    dict(B=1, H=2, Hkv=2, Sq=300, Sk=300, left=-1, right=-1, sinks=0),          # dense
    dict(B=1, H=3, Hkv=1, Sq=257, Sk=257, left=-1, right=0, sinks=5, dtype="bf16"),   # causal
    dict(B=1, H=2, Hkv=2, Sq=130, Sk=1000, left=128, right=0, sinks=64, end=True),    # a chunk against a cache
    dict(B=1, H=2, Hkv=2, Sq=1000, Sk=130, left=50, right=50, sinks=3),         # most rows see only the sinks
    dict(B=1, H=2, Hkv=2, Sq=1000, Sk=130, left=50, right=50, sinks=0),         # most rows see nothing
    dict(B=1, H=2, Hkv=2, Sq=200, Sk=60, left=30, right=0, sinks=10, end=True),  # rows in front of the first key
    dict(B=3, H=4, Hkv=2, Sq=260, Sk=260, left=90, right=0, sinks=16, qn=[260, 129, 1], kn=[260, 129, 1], dtype="bf16"),
    dict(B=4, H=2, Hkv=2, Sq=190, Sk=320, left=70, right=3, sinks=20, qn=[190, 0, 64, 65], kn=[320, 100, 0, 63], end=True),
    dict(B=2, H=2, Hkv=1, Sq=256, Sk=256, left=64, right=64, sinks=64, qn=[999, -5], kn=[256, 300]),   # clamped
    dict(B=1, H=8, Hkv=1, Sq=96, Sk=400, left=200, right=0, sinks=64, end=True),
    dict(B=2, H=24, Hkv=24, Sq=320, Sk=320, left=64, right=64, sinks=64),
]
ROW_CASES = [   # few query rows: the single-token form
    dict(B=1, H=1, Hkv=1, Sq=1, Sk=5000, left=-1, right=0, sinks=0, end=True),
    dict(B=3, H=8, Hkv=8, Sq=1, Sk=900, left=255, right=0, sinks=64, end=True, kn=[900, 1, 333]),
    dict(B=3, H=8, Hkv=2, Sq=1, Sk=900, left=255, right=0, sinks=64, end=True, kn=[900, 0, 60], dtype="bf16"),
    dict(B=2, H=12, Hkv=4, Sq=2, Sk=2100, left=1000, right=0, sinks=4, end=True, kn=[2100, 1]),
    dict(B=2, H=16, Hkv=1, Sq=5, Sk=700, left=300, right=0, sinks=1, end=True, qn=[5, 3], kn=[700, 650]),
    dict(B=1, H=6, Hkv=6, Sq=16, Sk=300, left=64, right=64, sinks=7),
    dict(B=1, H=40, Hkv=1, Sq=3, Sk=300, left=64, right=0, sinks=7, end=True),
    dict(B=5, H=2, Hkv=2, Sq=1, Sk=64, left=0, right=0, sinks=0, end=True),
    dict(B=2, H=4, Hkv=4, Sq=1, Sk=129, left=10, right=0, sinks=0),              # position 0
]


@pytest.mark.parametrize("token_major,pad", [(True, 0), (False, 0), (True, 8), (False, 16)])
@pytest.mark.parametrize("case", range(len(SINK_CASES)))
def test_attention_sink(ctx, case, token_major, pad):
    a = Attn(**SINK_CASES[case], token_major=token_major, pad=pad, seed=case)
    a.fwd(ctx)
    a.bwd(ctx)
    ctx.sync()
    a.check()


@pytest.mark.parametrize("token_major", [True, False])
@pytest.mark.parametrize("case", range(1, len(SINK_CASES)))
def test_attention_sink_of_many_heads(ctx, case, token_major):
    """The same masks with enough heads that the forward takes 128-row tiles."""
    kw = dict(SINK_CASES[case])
    more = 48 // (kw["B"] * kw["Hkv"]) + 1
    a = Attn(**{**kw, "H": kw["H"] * more, "Hkv": kw["Hkv"] * more}, token_major=token_major, pad=8, seed=300 + case)
    a.fwd(ctx)
    ctx.sync()
    a.check(grads=False)


@pytest.mark.parametrize("token_major", [True, False])
@pytest.mark.parametrize("case", range(len(ROW_CASES)))
def test_attention_sink_few_rows(ctx, case, token_major):
    a = Attn(**ROW_CASES[case], token_major=token_major, seed=100 + case)
    a.fwd(ctx)
    a.bwd(ctx)
    ctx.sync()
    a.check()


def test_attention_sink_large_scores(ctx):
    """Scores of hundreds: one key takes nearly everything, and the running maximum moves far."""
    a = Attn(1, 2, 2, 300, 300, 80, 80, 16, scale=4.0, seed=3)
    a.fwd(ctx)
    ctx.sync()
    import torch
    # |score| reaches 4 * 64: its f32 error is 64 * 2^-24 of 4 * sum |q k|, about 2^-9.4 in the exponent
    w = ref.attention(a.q[0], a.k[0], a.v[0], 4.0, 80, 80, 16, 300, 300, False)
    ref.assert_within("o", a.o[0], w["o"], w["o_tol"] + 2 ** -9 * float(a.v.abs().max()))
    ref.assert_within("lse", a.lse[0], w["lse"], 2 ** -9 + 2 ** -22 * w["lse"].abs())
    assert torch.isfinite(a.o).all()


def test_attention_sink_is_the_band_without_sinks(ctx):
    """left = right = w without sinks is the band of sa3k_attention_fwd."""
    import torch
    a = Attn(2, 4, 4, 333, 333, 100, 100, 0, token_major=False, seed=9)
    a.fwd(ctx)
    o2, lse2 = torch.empty_like(a.q), torch.empty(2 * 4 * 333, device="cuda")
    ctx.attention_fwd(2, 4, 333, 333, 0.125, 100, a.t4(a.q), a.t4(a.k), a.t4(a.v), a.t4(o2), lse2)
    ctx.sync()
    assert float((a.o.double() - o2.double()).norm() / o2.double().norm()) < 1e-3   # two roundings of P and o each


def test_attention_sink_same_bits_twice_and_without_dkdv(ctx):
    import torch
    a = Attn(2, 4, 2, 400, 400, 90, 0, 32, seed=4)
    a.fwd(ctx)
    a.bwd(ctx)
    first = [t.clone() for t in (a.o, a.lse, a.dq, a.dk, a.dv)]
    a.fwd(ctx)
    a.bwd(ctx)
    for x, y in zip(first, (a.o, a.lse, a.dq, a.dk, a.dv)):
        assert torch.equal(x, y)
    a.dq.fill_(0)
    a.dk.fill_(9)
    a.bwd(ctx, kv=False)
    ctx.sync()
    assert torch.equal(a.dq, first[2]) and bool((a.dk == 9).all())


def test_attention_sink_gradient_against_differences(ctx):
    import torch
    a = Attn(1, 2, 1, 40, 40, 9, 2, 3, seed=11)
    a.fwd(ctx)
    a.bwd(ctx)
    ctx.sync()

    def loss(q, k, v):
        w = ref.attention(q, k, v, 0.125, 9, 2, 3, 40, 40, False)
        return float((w["o"] * a.dO[0].double()).sum())

    base = [t[0].double() for t in (a.q, a.k, a.v)]
    h = 1e-4
    for n, g in enumerate((a.dq, a.dk, a.dv)):
        for idx in ((0, 0, 0), (0, 5, 17), (0, 39, 63)):
            hi, lo = [t.clone() for t in base], [t.clone() for t in base]
            hi[n][idx] += h
            lo[n][idx] -= h
            num = (loss(*hi) - loss(*lo)) / (2 * h)
            # one rounding of the gradient to f16, and of P, dS, o to f16 in sums of about 15 terms
            assert abs(num - float(g[0][idx])) < 2 ** -11 * (abs(num) + 30)


def test_attention_sink_empty_sizes(ctx):
    for dims in (dict(B=0, Sq=8, Sk=8), dict(B=2, Sq=0, Sk=8), dict(B=2, Sq=8, Sk=0), dict(B=2, Sq=300, Sk=0), dict(B=2, Sq=2500, Sk=0)):
        a = Attn(H=2, Hkv=1, left=4, right=0, sinks=2, **dims)
        a.fwd(ctx)
        a.bwd(ctx)
        ctx.sync()
        a.check()


def test_attention_sink_refusals(ctx):
    import torch
    import sa3k
    a = Attn(2, 4, 2, 32, 32, 8, 0, 4)
    ok = [a.t4(t) for t in (a.q, a.k, a.v, a.o)]
    call = lambda p, q=ok[0], k=ok[1], v=ok[2], o=ok[3]: ctx.attention_sink_fwd(p, q, k, v, o, a.lse)  # noqa: E731
    mk = lambda **kw: sa3k.sink_attn(**{**dict(B=2, H=4, Sq=32, Sk=32, scale=0.125, left=8, heads_kv=2), **kw})  # noqa: E731
    for kw, text in ((dict(head_dim=128), "head_dim"), (dict(heads_kv=3), "multiple of H_kv"), (dict(scale=0.0), "scale"),
                     (dict(sinks=-1), "sinks"), (dict(B=-1), "need B"), (dict(B=40000), "65535")):
        with pytest.raises(sa3k.Sa3kError, match=text):
            call(mk(**kw))
    with pytest.raises(sa3k.Sa3kError, match="dtype"):
        mk(dtype="f32")
    t = sa3k.t4(a.q, a.q.stride(0), a.q.stride(1), a.q.stride(2) + 4)
    with pytest.raises(sa3k.Sa3kError, match="multiples of 8"):
        call(mk(), q=t)
    with pytest.raises(sa3k.Sa3kError, match="overlap"):
        call(mk(), o=sa3k.t4(a.o, 0, a.o.stride(1), a.o.stride(2)))
    with pytest.raises(sa3k.Sa3kError, match="from 0 to"):
        call(mk(), k=sa3k.t4(a.k, a.k.stride(0), -64, a.k.stride(2)))
    off = torch.zeros(70000, device="cuda", dtype=torch.float16)[1:]
    with pytest.raises(sa3k.Sa3kError, match="16 bytes"):
        call(mk(), q=sa3k.t4(off, 8192, 64, 256))
    with pytest.raises(sa3k.Sa3kError, match="both dk and dv"):
        ctx.attention_sink_bwd(a.p, *ok[:3], ok[3], a.t4(a.dO), a.lse, a.t4(a.dq), a.t4(a.dk), None)
    with pytest.raises(sa3k.Sa3kError, match="lse"):
        ctx.attention_sink_bwd(a.p, *ok[:3], ok[3], a.t4(a.dO), None, a.t4(a.dq))
    with pytest.raises(sa3k.Sa3kError, match="int32"):
        sa3k.sink_attn(2, 4, 32, 32, 0.125, q_len=torch.zeros(2, device="cuda"))


LONG_TOKENS = [   # one stream, one or two heads: clusters of 8 and 16 blocks; the last has keys of no block
    dict(B=1, H=1, Hkv=1, Sq=1, Sk=20011, left=-1, right=0, sinks=0, end=True),
    dict(B=1, H=4, Hkv=1, Sq=1, Sk=40000, left=30000, right=0, sinks=100, end=True, dtype="bf16"),
    dict(B=9, H=1, Hkv=1, Sq=1, Sk=6000, left=-1, right=0, sinks=3, end=True, kn=[6000, 0, 1, 31, 32, 33, 130, 2049, 5999]),
    dict(B=1, H=1, Hkv=1, Sq=64, Sk=3001, left=2000, right=0, sinks=65, end=True),
    dict(B=1, H=1, Hkv=1, Sq=65, Sk=3001, left=2000, right=0, sinks=65, end=True),
]


@pytest.mark.parametrize("case", range(len(LONG_TOKENS)))
def test_attention_sink_long_cache(ctx, case):
    a = Attn(**LONG_TOKENS[case], seed=200 + case)
    a.fwd(ctx)
    ctx.sync()
    a.check(grads=False)


@pytest.mark.parametrize("B,H,Hkv,S,left,sinks", [(4, 16, 16, 700, 64, 64), (2, 8, 4, 1500, 400, 3), (1, 40, 40, 1100, -1, 0)])
def test_attention_sink_gradients_of_many_tiles(ctx, B, H, Hkv, S, left, sinks):
    """More (head, key tile) items than SMs; the ones that are long go first."""
    a = Attn(B, H, Hkv, S, S, left, 0, sinks, seed=17)
    for _ in range(2):      # the items' counter is set for each call
        a.dq.fill_(9.0), a.dk.fill_(9.0), a.dv.fill_(9.0)
        a.fwd(ctx)
        a.bwd(ctx)
    ctx.sync()
    a.check()


@pytest.mark.parametrize("Hkv,end", [(4, True), (1, True), (2, False)])
def test_attention_sink_token_and_evicted_keys(ctx, Hkv, end):
    """A single token does not read what lies outside its window: NaN and infinities there stay there."""
    import torch
    a = Attn(2, 4, Hkv, 1, 777, 100, 5, 37, end=end, kn=[777, 401], seed=8)
    want = Attn(2, 4, Hkv, 1, 777, 100, 5, 37, end=end, kn=[777, 401], seed=8)
    j = torch.arange(777, device="cuda")
    for b in range(2):
        pos = a.kn[b] - 1 if end else 0
        gone = ~(((j >= pos - 100) | (j < 37)) & (j <= pos + 5))
        a.k[b, :, gone], a.v[b, :, gone] = float("nan"), float("inf")
    a.fwd(ctx)
    want.fwd(ctx)
    ctx.sync()
    want.check(grads=False)
    assert torch.equal(a.o, want.o) and torch.equal(a.lse, want.lse)


def test_attention_sink_unseen_keys(ctx):
    """Keys that no query sees: their gradients are zero, in tiles of their own too."""
    a = Attn(1, 2, 2, 100, 1000, 10, 0, 2, seed=5)
    a.fwd(ctx)
    a.bwd(ctx)
    ctx.sync()
    a.check()
    assert float(a.dk[:, :, 100:].abs().max()) == 0.0 and float(a.dv[:, :, 100:].abs().max()) == 0.0


@pytest.mark.parametrize("Sq", [3, 200])
def test_attention_sink_mixed_layouts_and_broadcast(ctx, Sq):
    """Each tensor in an order of its own ([S][B][H], [H][B][S], ...), keys and values shared by the batch
    (stride 0)."""
    import torch
    B, H, Sk = 3, 4, 260
    a = Attn(B, H, H, Sq, Sk, 50, 0, 9, end=True, seed=Sq)
    order = lambda t, *dims: torch.empty([t.shape[d] for d in dims] + [64], device="cuda", dtype=t.dtype).permute(  # noqa: E731
        *[dims.index(d) for d in range(3)], 3).copy_(t)
    a.q, a.dO, a.o = order(a.q, 2, 0, 1), order(a.dO, 1, 0, 2), order(a.o, 1, 2, 0)
    a.dq, a.dk, a.dv = order(a.dq, 0, 1, 2), order(a.dk, 2, 1, 0), order(a.dv, 1, 0, 2)
    a.k, a.v = a.k[:1].expand(B, -1, -1, -1), order(a.v, 2, 0, 1)[:1].expand(B, -1, -1, -1)
    a.fwd(ctx)
    a.bwd(ctx)
    ctx.sync()
    a.check()


def test_two_contexts_at_once(ctx):
    """Contexts on streams of their own share nothing."""
    import torch
    import sa3k
    own, streams = [sa3k.Context(0, use_torch_stream=False) for _ in range(2)], [torch.cuda.Stream() for _ in range(2)]
    try:
        for c, s in zip(own, streams):
            c.set_stream(s.cuda_stream)
        both = [Attn(2, 8, 8, 500, 500, 100, 0, 16, seed=60 + i) for i in range(2)]
        torch.cuda.synchronize()
        for _ in range(3):
            for c, a in zip(own, both):
                a.fwd(c)
                a.bwd(c)
        for c, a in zip(own, both):
            c.sync()
        for a in both:
            a.check()
    finally:
        for c in own:
            c.close()


def test_attention_sink_wrapper_refusals(ctx):
    import torch
    import sa3k
    a = Attn(1, 2, 2, 32, 32, 8, 0, 4)
    t = [a.t4(x) for x in (a.q, a.k, a.v, a.o)]
    host = torch.zeros(1, 2, 32, 64, dtype=torch.float16)
    with pytest.raises(sa3k.Sa3kError, match="not on the context's device"):
        ctx.attention_sink_fwd(a.p, sa3k.t4(host, 4096, 2048, 64), *t[1:], a.lse)
    with pytest.raises(sa3k.Sa3kError, match="float32 vector of 64"):
        ctx.attention_sink_fwd(a.p, *t, a.lse[..., :31])
    with pytest.raises(sa3k.Sa3kError, match="float32 vector of 64"):
        ctx.attention_sink_fwd(a.p, *t, a.lse.double())


# --------------------------------------------------------------- linear with activation, residual
def _weight(ctx, kind, inn, out, seed):
    """(handle, float64 dequantized weight on the GPU)."""
    import torch
    rng = np.random.default_rng(seed)
    W = rng.normal(0, 0.05, (out, inn)).astype(np.float32)
    w = ctx.upload(gguf_blocks.encode(W, kind), kind, inn, out)
    d = torch.empty(out, inn, device="cuda")
    ctx.dequant(w, d)
    return w, d.double()


def _operand_error(kind, t):
    """Relative rounding of a product's operands to half: the weight's (none when it is half already)
    and, for f32 activations, x's."""
    return (0.0 if kind == "f16" else 2.0 ** -11) + (2.0 ** -11 if t == "f32" else 0.0)


LIN_CASES = [  # S, in, out, weight, type, act, residual, keep z
    (1, 64, 8, "f16", "f16", "none", False, False), (1, 1536, 520, "q8_0", "f16", "silu", True, True),
    (2, 256, 1000, "q4_k", "f16", "gelu", False, True), (4, 512, 77, "q8_0", "f32", "gelu_tanh", True, False),
    (7, 320, 129, "f32", "f16", "silu", True, True), (8, 1024, 2048, "f16", "f16", "gelu_tanh", True, True),
    (9, 1024, 2048, "q8_0", "f16", "silu", False, True), (16, 256, 96, "q4_k", "f32", "silu", True, True),
    (17, 192, 200, "q8_0", "f16", "gelu", True, False), (127, 128, 264, "q8_0", "f16", "none", True, False),
    (200, 512, 385, "f16", "f32", "gelu", True, True), (300, 640, 768, "q8_0", "f16", "gelu_tanh", True, True),
    (513, 256, 1536, "q8_0", "f16", "silu", False, True), (1100, 1536, 1544, "f16", "f16", "gelu", True, True),
    (2500, 128, 2056, "q8_0", "f16", "gelu_tanh", True, True), (2304, 256, 2304, "q4_k", "f32", "silu", True, False),
    (64, 4096, 128, "f16", "f16", "silu", True, True),
]


@pytest.mark.parametrize("cache", [True, False])
@pytest.mark.parametrize("S,inn,out,kind,t,act,residual,keep", LIN_CASES)
def test_linear_act(ctx, S, inn, out, kind, t, act, residual, keep, cache):
    import torch
    import sa3k
    if not cache and kind in ("f16", "f32"):
        pytest.skip("only quantized weights have a form without the half copy")
    if not cache and out % 16:
        pytest.skip("without the half copy, the engine's gradients take widths of 16")
    ctx.set_option(sa3k.OPT_WEIGHT_F16_CACHE, 1 if cache else 0)
    w, W = _weight(ctx, kind, inn, out, S + out)
    ctx.set_option(sa3k.OPT_WEIGHT_F16_CACHE, 1)
    rnd = _rand(S * 3 + out)
    dt, D = _dt(t), torch.float64
    x, bias = rnd(S, inn).to(dt), rnd(out)
    res = rnd(S, out).to(dt) if residual else None
    nan = lambda *s: torch.full(s, float("nan"), device="cuda", dtype=dt)  # noqa: E731
    y, z = nan(S, out), nan(S, out) if keep else None
    ctx.linear_act_fwd(w, x, y, act, bias=bias, residual=res, z=z)
    eps = _operand_error(kind, t)
    zr = x.to(D) @ W.T + bias.to(D)
    terms = x.to(D).abs() @ W.T.abs() + bias.to(D).abs()
    zt = (eps + inn * 2.0 ** -24) * terms
    yr = ref.act(zr, act) + (res.to(D) if residual else 0)
    small = 2.0 ** -25 if t == "f16" else 1e-30
    # no activation's slope is above 1.13; the f32 exponential and division are good to 2^-20
    ref.assert_within("y", y, yr, ref.u(dt) * yr.abs() + 1.13 * zt + 2 ** -20 * (zr.abs() + yr.abs()) + small)
    if keep:
        ref.assert_within("z", z, zr, ref.u(dt) * zr.abs() + zt + small)
    # backward from a given z
    zin, dy = rnd(S, out).to(dt), rnd(S, out).to(dt)
    dx, dbias = nan(S, inn), torch.full((out,), float("nan"), device="cuda")
    ctx.linear_act_bwd(w, None, zin, dy, dx, act, bias=bias, dbias=dbias)
    zz = zin.to(D).clone().requires_grad_(True)
    ref.act(zz, act).backward(dy.to(D))
    dz = zz.grad
    # dz is rounded to half as an operand, the weight as above
    e2 = 2.0 ** -11 + _operand_error(kind, "f16") + out * 2.0 ** -24 + 2 ** -19
    lost = (2 ** -25 + 2 ** -19) * W.abs().sum(0)      # subnormal dz; slopes near zero, absolute
    dxr = dz @ W
    ref.assert_within("dx", dx, dxr, ref.u(dt) * dxr.abs() + e2 * (dz.abs() @ W.abs()) + lost * dy.abs().max().double() + small)
    ref.assert_within("dbias", dbias, dz.sum(0), (64 + S / 32) * 2.0 ** -24 * dz.abs().sum(0) + 2 ** -20 * dy.to(D).abs().sum(0))
    acc = dbias.clone()
    ctx.linear_act_bwd(w, None, zin, dy, None, act, bias=bias, dbias=acc, accumulate=True)
    assert torch.equal(acc, dbias + dbias)
    ctx.sync()


@pytest.mark.parametrize("S", [3, 200, 1030])
@pytest.mark.parametrize("dora", [False, True])
@pytest.mark.parametrize("t", ["f16", "f32"])
def test_linear_act_with_adapter(ctx, S, dora, t):
    """The adapter's forward and gradients through the activation, against autograd in 64 bits."""
    import torch
    inn, out, R, s = 256, 320, 16, 0.7
    w, W = _weight(ctx, "q8_0", inn, out, 5)
    rnd = _rand(S + dora)
    dt, D = _dt(t), torch.float64
    A, Bm = rnd(R, inn) / inn ** 0.5, 0.1 * rnd(out, R)
    bns, nrm = torch.empty(out, device="cuda"), torch.empty(out, device="cuda")
    ctx.row_norms(w, 1e-12, bns, nrm)
    m = nrm * 1.1 if dora else None
    ad = ctx.adapter(A, Bm, s, m, bns if dora else None)
    x, bias, res, dy = rnd(S, inn).to(dt), 0.3 * rnd(out), rnd(S, out).to(dt), rnd(S, out).to(dt)
    y, z, dx = (torch.empty(S, n, device="cuda", dtype=dt) for n in (out, out, inn))
    dA, dB, dm, dbias = (torch.empty(n, device="cuda") for n in ((R, inn), (out, R), (out,), (out,)))
    ctx.linear_act_fwd(w, x, y, "silu", bias=bias, residual=res, z=z, ad=ad)
    ctx.linear_act_bwd(w, x, z, dy, dx, "silu", bias=bias, dbias=dbias, ad=ad, dA=dA, dB=dB, dm=dm if dora else None)
    ctx.sync()
    leaves = [v.to(D).requires_grad_(True) for v in (x, A, Bm, m if dora else torch.ones(out, device="cuda"), bias)]
    xr, Ar, Br, mr, br = leaves
    V = W + s * Br @ Ar
    if dora:
        V = V * (mr / ((V ** 2).sum(1) + inn * 1e-12).sqrt())[:, None]
    yr = ref.act(xr @ V.T + br, "silu") + res.to(D)
    yr.backward(dy.to(D))
    # half operands throughout (x, W, u, A, B, dz, du: relative 2^-11 each, a few of them in a chain) and
    # sums of independent terms: a relative 2-norm error of at most 5 * 2^-11
    tol = 5 * 2.0 ** -11
    rel = lambda a, b: float((a.double() - b).norm() / b.norm())  # noqa: E731
    got = dict(y=(y, yr), dx=(dx, xr.grad), dA=(dA, Ar.grad), dB=(dB, Br.grad), dbias=(dbias, br.grad))
    if dora:
        got["dm"] = (dm, mr.grad)
    errs = {n: rel(a, b.detach()) for n, (a, b) in got.items()}
    assert all(e < tol for e in errs.values()), errs


def test_linear_act_refusals_and_empty(ctx):
    import torch
    import sa3k
    w, _ = _weight(ctx, "f16", 64, 48, 1)
    x, y = torch.zeros(4, 64, device="cuda").half(), torch.zeros(4, 48, device="cuda").half()
    for kw, text in ((dict(act="relu"), "unknown activation"), (dict(bias=torch.zeros(47, device="cuda")), "vector of 48"),
                     (dict(residual=y.float()), "one type"), (dict(z=y[:3]), "contiguous")):
        with pytest.raises(sa3k.Sa3kError, match=text):
            ctx.linear_act_fwd(w, x, y, **kw)
    with pytest.raises(sa3k.Sa3kError, match="F32 or F16"):
        ctx.linear_act_fwd(w, x.bfloat16(), y.bfloat16())
    with pytest.raises(sa3k.Sa3kError, match="16 bytes"):
        ctx.linear_act_fwd(w, torch.zeros(4 * 64 + 1, device="cuda").half()[1:].view(4, 64), y)
    with pytest.raises(sa3k.Sa3kError, match="forward's z"):
        ctx.linear_act_bwd(w, None, None, y, x, "silu")
    with pytest.raises(sa3k.Sa3kError, match="dA and dB"):
        ctx.linear_act_bwd(w, x, y, y, None, "silu",
                           ad=ctx.adapter(torch.zeros(16, 64, device="cuda"), torch.zeros(48, 16, device="cuda"), 1.0))
    with pytest.raises(sa3k.Sa3kError, match="bias must start"):
        ctx.linear_act_fwd(w, x, y, bias=torch.zeros(49, device="cuda")[1:])
    with pytest.raises(sa3k.Sa3kError, match="adapter's arrays"):
        ctx.linear_act_fwd(w, x, y, ad=ctx.adapter(torch.zeros(16 * 64 + 1, device="cuda")[1:].view(16, 64),
                                                   torch.zeros(48, 16, device="cuda"), 1.0))
    db = torch.ones(48, device="cuda")
    ctx.linear_act_fwd(w, x[:0], y[:0], "silu")
    ctx.linear_act_bwd(w, None, y[:0], y[:0], x[:0], "silu", dbias=db)
    assert float(db.abs().max()) == 0.0


@pytest.mark.parametrize("S,t", [(5, "f16"), (40, "f16"), (40, "f32"), (1100, "f16"), (700, "f32")])
def test_linear_act_residual_in_place_and_unaligned(ctx, S, t):
    """The residual may be y itself; y, z and the residual need no more than their type's alignment."""
    import torch
    w, W = _weight(ctx, "q8_0", 128, 520, 6)
    rnd = _rand(S)
    x, res, bias = rnd(S, 128).to(_dt(t)), rnd(S, 520).to(_dt(t)), rnd(520)
    y, z = torch.empty_like(res), torch.empty_like(res)
    ctx.linear_act_fwd(w, x, y, "gelu", bias=bias, residual=res, z=z)
    inplace = res.clone()
    ctx.linear_act_fwd(w, x, inplace, "gelu", bias=bias, residual=inplace)
    assert torch.equal(inplace, y)
    off = lambda: torch.zeros(S * 520 + 1, device="cuda", dtype=_dt(t))[1:].view(S, 520)  # noqa: E731
    y1, z1, r1 = off(), off(), off()
    r1.copy_(res)
    ctx.linear_act_fwd(w, x, y1, "gelu", bias=bias, residual=r1, z=z1)
    # The same f32 products, but the compiler contracts another kernel's sums and activation otherwise: f32
    # values at most 2^-20 (|act| + |residual|) apart (the bound of an activation above), and after rounding
    # a step of the type more; a step is 2 finfo.eps / 2 of the value
    D, step = torch.float64, torch.finfo(_dt(t)).eps
    near = lambda a, b, m: bool(((a.to(D) - b.to(D)).abs() <= 2 ** -20 * m + step * b.to(D).abs() + 2.0 ** -24).all())  # noqa: E731
    mag = res.to(D).abs() * 2 + y.to(D).abs() + x.to(D).abs() @ W.T.abs() + bias.to(D).abs()
    assert near(y1, y, mag) and near(z1, z, mag)
    z1.copy_(z)
    dy, dx, dx1 = rnd(S, 520).to(_dt(t)), torch.empty_like(x), torch.empty_like(x)
    dy1 = off()
    dy1.copy_(dy)
    ctx.linear_act_bwd(w, None, z, dy, dx, "gelu")
    ctx.linear_act_bwd(w, None, z1, dy1, dx1, "gelu")
    # dz (a half operand) a step apart in places, |act'| <= 1.13, then dx's own step
    lim = 2.0 ** -10 * (1.13 * dy.to(D).abs() @ W.abs()) + step * dx.to(D).abs() + 2.0 ** -24
    assert bool(((dx.to(D) - dx1.to(D)).abs() <= lim).all())


# ---------------------------------------------------------------------- together, graphs, streams
class Block:
    """A pre-norm transformer block of the operators over a frozen base: forward and backward."""

    def __init__(self, ctx, B, S, dim=128, H=2, ff=256, seed=0):
        import torch
        import sa3k
        self.ctx, self.B, self.S, self.dim, self.H = ctx, B, S, dim, H
        names = (("qkv", dim, 3 * dim), ("out", dim, dim), ("up", dim, ff), ("down", ff, dim))
        self.w = {n: _weight(ctx, "f16", i, o, seed + k) for k, (n, i, o) in enumerate(names)}
        rnd = _rand(seed)
        self.bias = {n: 0.1 * rnd(o) for n, _, o in names}
        self.gamma, self.beta = [1 + 0.1 * rnd(dim) for _ in range(2)], [0.1 * rnd(dim) for _ in range(2)]
        n = B * S
        e = lambda c, dt=torch.float16: torch.zeros(n, c, device="cuda", dtype=dt)  # noqa: E731
        self.x, self.g = rnd(n, dim).half(), rnd(n, dim).half()
        self.h1, self.h2, self.att, self.x1, self.x2 = (e(dim) for _ in range(5))
        self.qkv, self.z, self.a = e(3 * dim), e(ff), e(ff)
        self.st = [torch.zeros(n, device="cuda") for _ in range(4)]
        self.lse = torch.zeros(B, H, S, device="cuda")
        self.da, self.dh2, self.dx1, self.datt, self.dqkv, self.dh1, self.dx = (e(c) for c in (ff, dim, dim, dim, 3 * dim, dim, dim))
        self.dgamma = [torch.zeros(dim, device="cuda") for _ in range(2)]
        self.dbeta = [torch.zeros(dim, device="cuda") for _ in range(2)]
        self.p = sa3k.sink_attn(B, H, S, S, 0.125, 24, 24, 8)

    def heads(self, t, col, width):
        import sa3k
        view = t.view(self.B, self.S, width)[..., col:]
        return sa3k.t4(view, self.S * width, 64, width)

    def fwd(self):
        c, D = self.ctx, self.dim
        c.layernorm_fwd(self.x, self.h1, self.gamma[0], self.beta[0], 1e-5, self.st[0], self.st[1])
        c.linear_act_fwd(self.w["qkv"][0], self.h1, self.qkv, bias=self.bias["qkv"])
        q, k, v = (self.heads(self.qkv, i * D, 3 * D) for i in range(3))
        c.attention_sink_fwd(self.p, q, k, v, self.heads(self.att, 0, D), self.lse)
        c.linear_act_fwd(self.w["out"][0], self.att, self.x1, bias=self.bias["out"], residual=self.x)
        c.layernorm_fwd(self.x1, self.h2, self.gamma[1], self.beta[1], 1e-5, self.st[2], self.st[3])
        c.linear_act_fwd(self.w["up"][0], self.h2, self.a, "gelu", bias=self.bias["up"], z=self.z)
        c.linear_act_fwd(self.w["down"][0], self.a, self.x2, bias=self.bias["down"], residual=self.x1)

    def bwd(self):
        c, D = self.ctx, self.dim
        c.linear_act_bwd(self.w["down"][0], None, None, self.g, self.da)
        c.linear_act_bwd(self.w["up"][0], None, self.z, self.da, self.dh2, "gelu")
        c.layernorm_bwd(self.x1, self.dh2, self.dx1, self.st[2], self.st[3], self.gamma[1], self.dgamma[1], self.dbeta[1])
        self.dx1.add_(self.g)
        c.linear_act_bwd(self.w["out"][0], None, None, self.dx1, self.datt)
        q, k, v = (self.heads(self.qkv, i * D, 3 * D) for i in range(3))
        dq, dk, dv = (self.heads(self.dqkv, i * D, 3 * D) for i in range(3))
        c.attention_sink_bwd(self.p, q, k, v, self.heads(self.att, 0, D), self.heads(self.datt, 0, D), self.lse, dq, dk, dv)
        c.linear_act_bwd(self.w["qkv"][0], None, None, self.dqkv, self.dh1)
        c.layernorm_bwd(self.x, self.dh1, self.dx, self.st[0], self.st[1], self.gamma[0], self.dgamma[0], self.dbeta[0])
        self.dx.add_(self.dx1)

    def outputs(self):
        return dict(x2=self.x2, dx=self.dx, dg0=self.dgamma[0], dg1=self.dgamma[1], db0=self.dbeta[0], db1=self.dbeta[1])

    def reference(self):
        import torch
        D = torch.float64
        x = self.x.to(D).requires_grad_(True)
        pars = [t.to(D).requires_grad_(True) for t in (*self.gamma, *self.beta)]
        lin = lambda t, n: t @ self.w[n][1].T + self.bias[n].to(D)  # noqa: E731
        ln = lambda t, i: torch.nn.functional.layer_norm(t, (self.dim,), pars[i], pars[2 + i], 1e-5)  # noqa: E731
        B, S, H = self.B, self.S, self.H
        qkv = lin(ln(x, 0), "qkv").view(B, S, 3, H, 64).permute(2, 0, 3, 1, 4)
        i = torch.arange(S, device="cuda")
        see = (i[None] <= i[:, None] + 24) & ((i[None] >= i[:, None] - 24) | (i[None] < 8))
        s = (qkv[0] @ qkv[1].transpose(-1, -2) * 0.125).masked_fill(~see, -torch.inf)
        o = (torch.softmax(s, -1) @ qkv[2]).permute(0, 2, 1, 3).reshape(B * S, self.dim)
        x1 = x + lin(o, "out")
        x2 = x1 + lin(ref.act(lin(ln(x1, 1), "up"), "gelu"), "down")
        x2.backward(self.g.to(D))
        return dict(x2=x2.detach(), dx=x.grad, dg0=pars[0].grad, dg1=pars[1].grad, db0=pars[2].grad, db1=pars[3].grad)


def _close(got, want):
    # each value passes about a dozen roundings to half (2^-11 at most, independent): 2-norm 12 * 2^-11
    for n, w in want.items():
        e = float((got[n].double() - w).norm() / w.norm())
        assert e < 12 * 2.0 ** -11, (n, e)


def test_block_of_the_operators(ctx):
    b = Block(ctx, 2, 150)
    b.fwd()
    b.bwd()
    ctx.sync()
    _close(b.outputs(), b.reference())


def test_block_captured_replayed_and_outgrown(ctx):
    """A captured step replays on new inputs, also after a larger eager step has outgrown its scratch,
    and next to a second captured step of the same context."""
    import torch
    import sa3k
    own = sa3k.Context(0, use_torch_stream=False)
    side = torch.cuda.Stream()
    own.set_stream(side.cuda_stream)
    try:
        with torch.cuda.stream(side):
            blocks, graphs = [Block(own, 1, 70, seed=1), Block(own, 2, 50, seed=2)], []
            for b in blocks:
                b.fwd()
                b.bwd()
                side.synchronize()
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=side):
                    b.fwd()
                    b.bwd()
                graphs.append(g)
            big = Block(own, 3, 400, seed=3)
            big.fwd()
            big.bwd()
            for b in blocks:
                b.x.copy_(_rand(77 + b.S)(*b.x.shape).half())
                b.dx.zero_()
                b.x2.zero_()
            for _ in range(2):
                for g in graphs:
                    g.replay()
        own.sync()
        for b in blocks + [big]:
            _close(b.outputs(), b.reference())
    finally:
        own.close()


def test_first_call_inside_a_capture(ctx):
    """Scratch grows beside a capture without invalidating it; what an earlier capture holds stays valid, and
    the random generator that the capture took is given back."""
    import torch
    import sa3k
    own = sa3k.Context(0, use_torch_stream=False)
    side = torch.cuda.Stream()
    own.set_stream(side.cuda_stream)
    try:
        both = [Attn(1, 2, 2, 64, 64, 8, 0, 4), Attn(3, 8, 8, 400, 400, 70, 0, 4)]
        blocks = [Block(own, 1, 40, seed=5), Block(own, 2, 300, seed=6)]
        torch.cuda.synchronize()
        graphs = []
        for a, b in zip(both, blocks):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=side):
                a.fwd(own)
                a.bwd(own)
                b.fwd()
                b.bwd()
        with torch.cuda.stream(side):
            for g in graphs * 2:
                g.replay()
        own.sync()
        for a, b in zip(both, blocks):
            a.check()
            _close(b.outputs(), b.reference())
        assert torch.isfinite(torch.randn(3, device="cuda")).all()
    finally:
        own.close()


def test_current_device_is_left_alone(ctx):
    import torch
    before = torch.cuda.current_device()
    b = Block(ctx, 1, 20)
    b.fwd()
    assert torch.cuda.current_device() == before


def test_every_activation_and_layout_agrees_between_forms(ctx):
    """The same rows give the same values whether they come alone or among many (other kernels)."""
    import torch
    w, _ = _weight(ctx, "f16", 256, 264, 3)
    rnd = _rand(8)
    x, bias = rnd(300, 256).half(), rnd(264)
    for act, rows in itertools.product(("none", "silu", "gelu", "gelu_tanh"), (1, 5, 40)):
        many, few = torch.empty(300, 264, device="cuda").half(), torch.empty(rows, 264, device="cuda").half()
        ctx.linear_act_fwd(w, x, many, act, bias=bias)
        ctx.linear_act_fwd(w, x[:rows].contiguous(), few, act, bias=bias)
        d = (many[:rows].double() - few.double()).abs()
        # two roundings to half of values a few 2^-14 apart (f32 sums in another order)
        assert bool((d <= 2 ** -10 * many[:rows].double().abs() + 2 ** -13).all())
