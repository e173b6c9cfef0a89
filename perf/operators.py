"""Cases for the transformer-block operators: layer normalisation, attention over a sliding window
with sink tokens, and the frozen linear with bias, activation and residual in its epilogue.

A case is a dict; prepare() makes its inputs on the GPU, run() is one pass (the plain form, or the
library's call where `own` is set), exact() the same result in 64 bits and work() the bytes and
operations that a pass cannot do without.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

LOG2E = 1.4426950408889634
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
HEAD = 64
ACTS = {"none": 0, "silu": 1, "gelu": 2, "gelu_tanh": 3}


# ------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # the norm in front of a projection: residual stream (f32) in, GEMM operand (f16) out, at
        # the training batch of 4 x (1024 frames + 64 memory tokens)
        dict(name="layernorm fwd 4352x1536", op="ln_fwd", rows=4352, cols=1536, x="f32", y="f16"),
        # its backward over a long batch (odd row count) with f16 activations
        dict(name="layernorm bwd 16383x1536", op="ln_bwd", rows=16383, cols=1536, x="f16", y="f16"),
        # the audio transformer's banded self-attention with its 64 memory tokens kept visible
        dict(name="attn fwd band 2048", op="attn_fwd", B=2, H=24, Hkv=24, Sq=2048, Sk=2048, left=256, right=256,
             sinks=64, end=False, ragged=False, dtype="f16"),
        # a long causal stream with shared key / value heads and a few sinks
        dict(name="attn fwd causal 8192", op="attn_fwd", B=1, H=24, Hkv=8, Sq=8192, Sk=8192, left=1023, right=0,
             sinks=4, end=False, ragged=False, dtype="bf16"),
        # the training step's self-attention: batch 4, 64 memory tokens + 1024 frames
        dict(name="attn bwd band 1088", op="attn_bwd", B=4, H=24, Hkv=24, Sq=1088, Sk=1088, left=256, right=256,
             sinks=64, end=False, ragged=False, dtype="f16"),
        # a padded batch of unequal lengths, causal, with shared key / value heads
        dict(name="attn bwd ragged 2047", op="attn_bwd", B=3, H=24, Hkv=8, Sq=2047, Sk=2047, left=511, right=0,
             sinks=16, end=False, ragged=True, dtype="bf16"),
        # one new token of one stream: latency
        dict(name="attn token 1x1500", op="attn_fwd", B=1, H=24, Hkv=24, Sq=1, Sk=1500, left=511, right=0, sinks=64,
             end=True, ragged=False, dtype="f16"),
        # one new token for each of 64 streams with caches of unequal lengths
        dict(name="attn token 64x8192", op="attn_fwd", B=64, H=24, Hkv=8, Sq=1, Sk=8192, left=2047, right=0, sinks=64,
             end=True, ragged=True, dtype="f16"),
        # one row through the MLP's up projection (a single token, or one sample's conditioning)
        dict(name="linear silu 1 row", op="lin_fwd", S=1, inn=1536, out=6144, w="q8_0", act="silu", residual=False,
             keep=False),
        # the up projection of the training batch, pre-activation kept for the backward
        dict(name="linear gelu 4352 up", op="lin_fwd", S=4352, inn=1536, out=6144, w="q8_0", act="gelu_tanh",
             residual=False, keep=True),
        # the down projection with the residual stream added
        dict(name="linear residual 4352 down", op="lin_fwd", S=4352, inn=6144, out=1536, w="q8_0", act="none",
             residual=True, keep=False),
        # the up projection's backward: input gradient and bias gradient, odd row count
        dict(name="linear bwd 2047 up", op="lin_bwd", S=2047, inn=1536, out=6144, w="q8_0", act="silu"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["ln_fwd", "ln_bwd", "attn_fwd", "attn_fwd", "attn_bwd", "token", "lin_fwd", "lin_fwd", "lin_bwd"])
    if kind in ("ln_fwd", "ln_bwd"):
        cols = _log(rng, 32, 5000)
        rows = _log(rng, 1, 25000000 // cols)
        return dict(op=kind, rows=rows, cols=cols, x=rng.choice(list(DTYPES)), y=rng.choice(list(DTYPES)))
    if kind in ("attn_fwd", "attn_bwd"):
        hkv = rng.choice([1, 2, 3, 4, 8])
        H = hkv * rng.choice([1, 1, 2, 3, 4])
        # the plain form works on all B x H x Sq x Sk scores: no more of them than the listed work
        most = 3e8 if kind == "attn_fwd" else 1.2e8
        top = min(4096, int((most / H) ** 0.5))
        Sq = _log(rng, 1, top)
        Sk = Sq if rng.random() < 0.7 else _log(rng, 1, top)
        B = rng.randint(1, max(1, min(8, int(most / (H * max(Sq, 64) * max(Sk, 64))))))
        left = rng.choice([-1, 0]) if rng.random() < 0.15 else _log(rng, 1, 2048)
        right = rng.choice([0, 0, left, -1, rng.randint(0, 300)])
        return dict(op=kind, B=B, H=H, Hkv=hkv, Sq=Sq, Sk=Sk, left=left, right=right,
                    sinks=rng.choice([0, 1, 4, 64, rng.randint(0, 200)]), end=rng.random() < 0.3,
                    ragged=rng.random() < 0.5, dtype=rng.choice(["f16", "bf16"]))
    if kind == "token":
        hkv = rng.choice([1, 2, 4, 8, 24])
        H = hkv * rng.choice([1, 2, 3, 4, 8])
        B = _log(rng, 1, 64)
        return dict(op="attn_fwd", B=B, H=H, Hkv=hkv, Sq=rng.choice([1, 1, 1, 2, 5]),
                    Sk=_log(rng, 64, min(65536, int(64 * 8 * 8192 / (B * hkv)))), left=_log(rng, 64, 4096), right=0,
                    sinks=rng.choice([0, 4, 64]), end=True, ragged=rng.random() < 0.7, dtype=rng.choice(["f16", "bf16"]))
    w = rng.choice(["q8_0", "q8_0", "f16"])
    inn = 64 * _log(rng, 1, 64)
    out = 8 * _log(rng, 1, 768)
    S = _log(rng, 1, max(1, min(8192, int(4.1e10 / (inn * out)))))
    act = rng.choice(list(ACTS))
    if kind == "lin_bwd":
        return dict(op="lin_bwd", S=S, inn=inn, out=out, w=w, act=act)
    return dict(op="lin_fwd", S=S, inn=inn, out=out, w=w, act=act, residual=rng.random() < 0.5, keep=rng.random() < 0.5)


# ------------------------------------------------------------------------------------ the inputs
def _lengths(case):
    """(query rows, key rows) of every batch entry: all of them, or lengths spread over the range."""
    B, Sq, Sk = case["B"], case["Sq"], case["Sk"]
    if not case["ragged"]:
        return [Sq] * B, [Sk] * B
    kv = [max(1, Sk - (b * 7919 + 13) * Sk // (B * 9973) % max(1, Sk // 2 + 1)) for b in range(B)]
    if case["end"]:
        return [Sq] * B, kv
    return [min(Sq, n) if Sq == Sk else Sq for n in kv], kv


def _positions(case, qn, kn):
    """Position of query row 0 of a batch entry with qn query rows and kn keys."""
    return kn - qn if case["end"] else 0


def _handle():
    """The library's module and this program's context (one per process, on torch's stream)."""
    here = os.path.join(os.getcwd(), "sa3.cpp_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import sa3k
    if not hasattr(_handle, "ctx"):
        _handle.ctx = sa3k.Context(0)
    return sa3k, _handle.ctx


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    st = dict(case=case)
    op = case["op"]
    if op in ("ln_fwd", "ln_bwd"):
        rows, cols = case["rows"], case["cols"]
        # activations with a per-channel offset and scale, as a residual stream has them
        x = rnd(rows, cols) * (1 + 0.5 * rnd(cols).abs()) + 0.5 * rnd(cols)
        st["x"] = x.to(DTYPES[case["x"]])
        st["gamma"], st["beta"] = 1 + 0.2 * rnd(cols), 0.1 * rnd(cols)
        st["y"] = torch.empty(rows, cols, device="cuda", dtype=DTYPES[case["y"]])
        st["mean"], st["rstd"] = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
        if op == "ln_bwd":
            xf = st["x"].double()
            mean = xf.mean(1, keepdim=True)
            st["mean"] = mean[:, 0].float()
            st["rstd"] = (((xf - mean) ** 2).mean(1) + 1e-5).rsqrt().float()
            st["dy"] = rnd(rows, cols).to(DTYPES[case["y"]])
            st["dx"] = torch.empty(rows, cols, device="cuda", dtype=DTYPES[case["x"]])
            st["dgamma"], st["dbeta"] = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    elif op in ("attn_fwd", "attn_bwd"):
        B, H, Hkv, Sq, Sk, dt = case["B"], case["H"], case["Hkv"], case["Sq"], case["Sk"], DTYPES[case["dtype"]]
        # token-major projections [B][S][H][64], as a fused projection leaves them
        st["q"] = rnd(B, Sq, H, HEAD).to(dt)
        st["k"], st["v"] = rnd(B, Sk, Hkv, HEAD).to(dt), rnd(B, Sk, Hkv, HEAD).to(dt)
        st["o"] = torch.zeros(B, Sq, H, HEAD, device="cuda", dtype=dt)
        st["lse"] = torch.zeros(B, H, Sq, device="cuda")
        qn, kn = _lengths(case)
        st["q_len"] = torch.tensor(qn, device="cuda", dtype=torch.int32) if case["ragged"] else None
        st["kv_len"] = torch.tensor(kn, device="cuda", dtype=torch.int32) if case["ragged"] else None
        if case["ragged"]:   # what lies behind a sequence's end is whatever the buffer held before
            stale = torch.arange(Sk, device="cuda")[None] >= st["kv_len"][:, None].long()
            st["k"][stale] = float("nan")
            st["v"][stale] = float("inf")
        if op == "attn_bwd":
            st["do"] = rnd(B, Sq, H, HEAD).to(dt)
            for n in ("dq", "dk", "dv"):
                st[n] = torch.zeros_like(st[n[1]])
            st["o"], st["lse"] = _attention_plain(st)
    else:
        S, inn, out = case["S"], case["inn"], case["out"]
        # a frozen base: GGUF Q8_0 blocks of 32 (f16 scale, int8 codes) or f16 rows, about N(0, 0.02)
        if case["w"] == "q8_0":
            q = (rnd(out, inn // 32, 32) * 40).round().clamp(-127, 127).to(torch.int8)
            d = ((0.8 + 0.4 * torch.rand(out, inn // 32, 1, generator=g, device="cuda")) * 0.0005).half()
            st["weight"] = (q.float() * d.float()).reshape(out, inn)
            raw = torch.cat([d.view(torch.uint8).reshape(out, inn // 32, 2), q.view(torch.uint8)], 2).reshape(out, -1)
        else:
            w = (rnd(out, inn) * 0.02).half()
            st["weight"] = w.float()
            raw = w.view(torch.uint8).reshape(out, -1)
        if own:
            st["w"] = _handle()[1].upload(raw.cpu().numpy(), case["w"], inn, out)
        st["bias"] = 0.1 * rnd(out)
        st["x"] = rnd(S, inn).half()
        if op == "lin_fwd":
            st["y"] = torch.empty(S, out, device="cuda", dtype=torch.float16)
            st["residual"] = rnd(S, out).half() if case["residual"] else None
            st["z"] = torch.empty_like(st["y"]) if case["keep"] else None
        else:
            st["z"] = (rnd(S, out) * 0.8).half()
            st["dy"] = rnd(S, out).half()
            st["dx"] = torch.empty(S, inn, device="cuda", dtype=torch.float16)
            st["dbias"] = torch.empty(out, device="cuda")
    if own:
        _handle()
    return st


# ----------------------------------------------------------------------------- the library's calls
def _run_own(st):
    sa3k, ctx = _handle()
    case = st["case"]
    op = case["op"]
    if op == "ln_fwd":
        ctx.layernorm_fwd(st["x"], st["y"], st["gamma"], st["beta"], 1e-5, st["mean"], st["rstd"])
        return st["y"], st["mean"], st["rstd"]
    if op == "ln_bwd":
        ctx.layernorm_bwd(st["x"], st["dy"], st["dx"], st["mean"], st["rstd"], st["gamma"], st["dgamma"], st["dbeta"])
        return st["dx"], st["dgamma"], st["dbeta"]
    if op in ("attn_fwd", "attn_bwd"):
        B, H, Hkv, Sq, Sk = case["B"], case["H"], case["Hkv"], case["Sq"], case["Sk"]
        p = sa3k.sink_attn(B, H, Sq, Sk, HEAD ** -0.5, case["left"], case["right"], case["sinks"], heads_kv=Hkv,
                           dtype=case["dtype"], align_end=case["end"], q_len=st["q_len"], kv_len=st["kv_len"])
        # [B][S][H][64] tensors as the batch, head and row strides that they have
        t4 = lambda t: sa3k.t4(t, t.stride(0), t.stride(2), t.stride(1))  # noqa: E731
        q, k, v, o = t4(st["q"]), t4(st["k"]), t4(st["v"]), t4(st["o"])
        if op == "attn_fwd":
            ctx.attention_sink_fwd(p, q, k, v, o, st["lse"])
            return st["o"], st["lse"]
        ctx.attention_sink_bwd(p, q, k, v, o, t4(st["do"]), st["lse"], t4(st["dq"]), t4(st["dk"]), t4(st["dv"]))
        return st["dq"], st["dk"], st["dv"]
    if op == "lin_fwd":
        ctx.linear_act_fwd(st["w"], st["x"], st["y"], case["act"], bias=st["bias"], residual=st["residual"], z=st["z"])
        return [t for t in (st["y"], st["z"]) if t is not None]
    ctx.linear_act_bwd(st["w"], st["x"], st["z"], st["dy"], st["dx"], case["act"], bias=st["bias"], dbias=st["dbias"])
    return st["dx"], st["dbias"]


# ------------------------------------------------------------------------------- the plain forms
def _valid_rows(case, lens, S):
    """[B, S] truth values: the rows in front of each sequence's end."""
    return torch.arange(S, device="cuda")[None] < torch.tensor(lens, device="cuda")[:, None]


def _visible(case):
    """[B, Sq, Sk] truth values: query row i at position p sees key j when j <= p + right and
    (j < sinks or j >= p - left), both inside their sequences."""
    qn, kn = _lengths(case)
    shift = torch.tensor([_positions(case, a, b) for a, b in zip(qn, kn)], device="cuda")
    p = torch.arange(case["Sq"], device="cuda")[None, :, None] + shift[:, None, None]
    j = torch.arange(case["Sk"], device="cuda")[None, None, :]
    vis = _valid_rows(case, qn, case["Sq"])[:, :, None] & _valid_rows(case, kn, case["Sk"])[:, None, :]
    if case["right"] >= 0:
        vis = vis & (j <= p + case["right"])
    if case["left"] >= 0:
        vis = vis & ((j < case["sinks"]) | (j >= p - case["left"]))
    return vis


def _heads(st, name, rows):
    """[B, Hkv, groups, S, 64] in 32 bits, rows behind the sequence's end as zeros."""
    t = st[name]
    B, S, h, _ = t.shape
    t = torch.where(rows[:, :, None, None], t, torch.zeros((), device="cuda", dtype=t.dtype)).float()
    hkv = st["case"]["Hkv"]
    return t.permute(0, 2, 1, 3).reshape(B, hkv, h // hkv, S, HEAD)


def _scores(st):
    case = st["case"]
    qn, kn = _lengths(case)
    qr, kr = _valid_rows(case, qn, case["Sq"]), _valid_rows(case, kn, case["Sk"])
    q, k, v = _heads(st, "q", qr), _heads(st, "k", kr), _heads(st, "v", kr)
    s = torch.matmul(q * HEAD ** -0.5, k.transpose(-1, -2))
    s.masked_fill_(~_visible(case)[:, None, None], float("-inf"))
    return q, k, v, s, qr, kr


def _token_major(t, like):
    """[B, Hkv, groups, S, 64] -> [B, S, H, 64] in the type of `like`."""
    B, a, b, S, _ = t.shape
    return t.reshape(B, a * b, S, HEAD).permute(0, 2, 1, 3).to(like.dtype)


def _attention_plain(st):
    q, k, v, s, qr, _ = _scores(st)
    m = s.amax(-1, keepdim=True).clamp_min(-1e30)
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / total.clamp_min(1e-30)
    lse = torch.where(total > 0, (m + total.log()) * LOG2E, float("-inf"))
    B, H, Sq = st["lse"].shape
    lse = torch.where(qr[:, None], lse.reshape(B, H, Sq), st["lse"])
    return torch.where(qr[:, :, None, None], _token_major(o, st["q"]), st["o"]), lse


def _attention_grads_plain(st):
    q, k, v, p, qr, kr = _scores(st)
    case = st["case"]
    B, H, Sq = st["lse"].shape
    lse = torch.where(qr[:, None], st["lse"], 0.0)
    lse = torch.where(lse == float("-inf"), 0.0, lse).reshape(B, case["Hkv"], H // case["Hkv"], Sq, 1)
    p.mul_(LOG2E).sub_(lse).exp2_()
    do, o = _heads(st, "do", qr), _heads(st, "o", qr)
    dv = torch.matmul(p.transpose(-1, -2), do).sum(2, keepdim=True)
    ds = torch.matmul(do, v.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p)
    del p
    dq = torch.matmul(ds, k) * HEAD ** -0.5
    dk = torch.matmul(ds.transpose(-1, -2), q).sum(2, keepdim=True) * HEAD ** -0.5
    keep = lambda t, name, rows: torch.where(rows[:, :, None, None], _token_major(t, st[name]), st[name])  # noqa: E731
    return keep(dq, "dq", qr), keep(dk, "dk", kr), keep(dv, "dv", kr)


def _act(z, act):
    if act == "silu":
        return z / (1 + (-z).exp())
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _act_slope(z, act):
    if act == "silu":
        s = 1 / (1 + (-z).exp())
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * (-0.5 * z * z).exp() / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def run(st):
    if own:
        return _run_own(st)
    case = st["case"]
    op = case["op"]
    if op == "ln_fwd":
        x = st["x"].float()
        mean = x.mean(1, keepdim=True)
        c = x - mean
        rstd = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-5)
        return (c * rstd * st["gamma"] + st["beta"]).to(st["y"].dtype), mean[:, 0], rstd[:, 0]
    if op == "ln_bwd":
        xh = (st["x"].float() - st["mean"][:, None]) * st["rstd"][:, None]
        dy = st["dy"].float()
        a = dy * st["gamma"]
        dx = st["rstd"][:, None] * (a - a.mean(1, keepdim=True) - xh * (a * xh).mean(1, keepdim=True))
        return dx.to(st["dx"].dtype), (dy * xh).sum(0), dy.sum(0)
    if op == "attn_fwd":
        return _attention_plain(st)
    if op == "attn_bwd":
        return _attention_grads_plain(st)
    if op == "lin_fwd":
        z = torch.matmul(st["x"].float(), st["weight"].t()) + st["bias"]
        y = _act(z, case["act"])
        if st["residual"] is not None:
            y = y + st["residual"].float()
        return [t for t in (y.half(), z.half() if case["keep"] else None) if t is not None]
    dz = st["dy"].float() * _act_slope(st["z"].float(), case["act"])
    return torch.matmul(dz, st["weight"]).half(), dz.sum(0)


# --------------------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    D = torch.float64
    if op in ("ln_fwd", "ln_bwd"):
        x = st["x"].to(D)
        gamma = st["gamma"].to(D)
        if op == "ln_fwd":
            mu = x.sum(1) / case["cols"]
            var = ((x - mu[:, None]) ** 2).sum(1) / case["cols"]
            r = (var + 1e-5) ** -0.5
            return torch.addcmul(st["beta"].to(D), (x - mu[:, None]) * r[:, None], gamma), mu, r
        mu, r, dy = st["mean"].to(D), st["rstd"].to(D), st["dy"].to(D)
        xh = (x - mu[:, None]) * r[:, None]
        g = dy * gamma
        n = case["cols"]
        dx = (g - (g.sum(1) / n)[:, None] - xh * (torch.einsum("rc,rc->r", g, xh) / n)[:, None]) * r[:, None]
        return dx, torch.einsum("rc,rc->c", dy, xh), dy.sum(0)
    if op in ("attn_fwd", "attn_bwd"):
        return _exact_attention(st)
    x, w = st["x"].to(D), st["weight"].to(D)
    if op == "lin_fwd":
        z = x @ w.T + st["bias"].to(D)
        y = {"none": lambda: z, "silu": lambda: z * torch.sigmoid(z),
             "gelu": lambda: z * 0.5 * torch.special.erfc(-z / 2 ** 0.5),
             "gelu_tanh": lambda: z * torch.sigmoid(2 * (2 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3))}[case["act"]]()
        if st["residual"] is not None:
            y = y + st["residual"].to(D)
        return [y, z] if case["keep"] else [y]
    z = st["z"].to(D)
    # the slope as a sum of products of each activation's factors
    if case["act"] == "silu":
        s = torch.sigmoid(z)
        slope = s + z * s * torch.sigmoid(-z)
    elif case["act"] == "gelu":
        slope = 0.5 * torch.special.erfc(-z / 2 ** 0.5) + z * torch.exp(-z * z / 2) * (2 * math.pi) ** -0.5
    elif case["act"] == "gelu_tanh":
        c = 2 * (2 / math.pi) ** 0.5
        u = c * (z + 0.044715 * z ** 3)
        s = torch.sigmoid(u)
        slope = s + z * s * torch.sigmoid(-u) * c * (1 + 0.134145 * z * z)
    else:
        slope = torch.ones_like(z)
    dz = st["dy"].to(D) * slope
    return dz @ w, dz.sum(0)


def _exact_attention(st):
    """Every batch entry and key / value head by itself, over the rows that its sequence has."""
    case = st["case"]
    D = torch.float64
    backward = case["op"] == "attn_bwd"
    groups = case["H"] // case["Hkv"]
    out = [st[n].to(D).clone() for n in (("dq", "dk", "dv") if backward else ("o", "lse"))]
    qn, kn = _lengths(case)
    for b in range(case["B"]):
        nq, nk = qn[b], kn[b]
        pos = torch.arange(nq, device="cuda") + _positions(case, nq, nk)
        key = torch.arange(nk, device="cuda")
        hi = pos + case["right"] if case["right"] >= 0 else torch.full_like(pos, nk)
        lo = pos - case["left"] if case["left"] >= 0 else torch.zeros_like(pos)
        seen = (key[None] <= hi[:, None]) & ((key[None] >= lo[:, None]) | (key[None] < case["sinks"]))
        some = seen.any(1)
        for h in range(case["Hkv"]):
            hs = slice(h * groups, (h + 1) * groups)
            q = st["q"][b, :nq, hs].to(D).transpose(0, 1)
            k, v = st["k"][b, :nk, h].to(D), st["v"][b, :nk, h].to(D)
            s = torch.einsum("gid,jd->gij", q, k) / 8
            if backward:
                lse = torch.where(some, st["lse"][b, hs, :nq].to(D), 0.0) / LOG2E
                p = torch.where(seen, torch.exp(s - lse[..., None]), 0.0)
                do, o = (st[n][b, :nq, hs].to(D).transpose(0, 1) for n in ("do", "o"))
                ds = p * (torch.einsum("gid,jd->gij", do, v) - (do * o).sum(-1)[..., None]) / 8
                out[0][b, :nq, hs] = torch.einsum("gij,jd->igd", ds, k)
                out[1][b, :nk, h] = torch.einsum("gij,gid->jd", ds, q)
                out[2][b, :nk, h] = torch.einsum("gij,gid->jd", p, do)
            else:
                top = torch.where(seen, s, -torch.inf).amax(-1)
                top = torch.where(some, top, 0.0)
                p = torch.where(seen, torch.exp(s - top[..., None]), 0.0)
                total = p.sum(-1)
                w = p / torch.where(some, total, 1.0)[..., None]
                out[0][b, :nq, hs] = torch.einsum("gij,jd->igd", w, v)
                out[1][b, hs, :nq] = torch.where(some, top * LOG2E + torch.log2(total), -torch.inf)
    return tuple(out)


# -------------------------------------------------------------------------- what a pass has to do
def work(case):
    op = case["op"]
    if op in ("ln_fwd", "ln_bwd"):
        n, bx, by = case["rows"] * case["cols"], SIZES[case["x"]], SIZES[case["y"]]
        if op == "ln_fwd":
            return {"bytes": n * (bx + by) + 8 * case["cols"] + 8 * case["rows"], "flops": 8 * n}
        return {"bytes": n * (2 * bx + by) + 12 * case["cols"] + 8 * case["rows"], "flops": 14 * n}
    if op in ("attn_fwd", "attn_bwd"):
        pairs, rows_k, rows_q = 0, 0, 0
        for nq, nk in zip(*_lengths(case)):
            p = np.arange(nq, dtype=np.int64) + _positions(case, nq, nk)
            hi = np.minimum(p + case["right"], nk - 1) if case["right"] >= 0 else np.full(nq, nk - 1)
            lo = np.maximum(p - case["left"], 0) if case["left"] >= 0 else np.zeros(nq, np.int64)
            n = np.maximum(hi - lo + 1, 0)
            first = np.clip(np.minimum(np.minimum(case["sinks"], lo), hi + 1), 0, None)
            pairs += int((n + first).sum())
            band = max(0, int(hi.max()) - int(lo.min()) + 1)      # keys that some row sees
            rows_k += min(nk, band + min(case["sinks"], int(lo.min())))
            rows_q += nq
        q, k = rows_q * case["H"] * HEAD * 2, rows_k * case["Hkv"] * HEAD * 2
        lse = rows_q * case["H"] * 4
        if op == "attn_fwd":
            return {"bytes": 2 * q + 2 * k + lse, "flops": 4 * HEAD * case["H"] * pairs}
        return {"bytes": 4 * q + 4 * k + lse, "flops": 10 * HEAD * case["H"] * pairs}
    S, inn, out = case["S"], case["inn"], case["out"]
    w = out * inn * 34 // 32 if case["w"] == "q8_0" else out * inn * 2
    if op == "lin_fwd":
        n = 1 + int(case["residual"]) + int(case["keep"])
        return {"bytes": w + 2 * S * inn + 2 * n * S * out + 4 * out, "flops": 2 * S * inn * out}
    return {"bytes": w + 2 * S * inn + 4 * S * out + 4 * out, "flops": 2 * S * inn * out}
