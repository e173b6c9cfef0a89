"""Float64 restatements of the transformer-block operators, with the elementwise error bounds that the
tests hold the kernels to.

u(t) is half a unit in the last place relative to the value (finfo(t).eps / 2).  A result rounded to t
once is off by u |value|.  Products of attention round P (and dS) to the operand type first: one more u
relative to the sum of absolute terms.  f32 arithmetic adds 2^-13 .. 2^-12 of the same sums: a 64-term
dot product is off by at most 64 * 2^-24 of its absolute terms, which are a few tens in the exponent of
the softmax, so a probability is off by about 2^-24 * 64 * 30 = 2^-13.  Values below a half-precision
type's normal range are off by an absolute half step instead (2^-25 for f16; bf16 has f32's range)."""
import torch

LOG2E = 1.4426950408889634


def u(t):
    return torch.finfo(t).eps / 2


def attention(q, k, v, scale, left, right, sinks, qn, kn, end, dO=None, o=None, lse=None):
    """q [H][Sq][64], k / v [Hkv][Sk][64] of one batch entry, cut to its qn / kn rows here.  Returns a
    dict of float64 results and bounds; with dO also the gradients (from the given o and lse)."""
    D = torch.float64
    t = q.dtype
    g = q.shape[0] // k.shape[0]
    qf = q[:, :qn].to(D)
    kf, vf = (x[:, :kn].to(D).repeat_interleave(g, 0) for x in (k, v))
    p = torch.arange(qn, device=q.device) + (kn - qn if end else 0)
    j = torch.arange(kn, device=q.device)
    see = torch.ones(qn, kn, dtype=torch.bool, device=q.device)
    if right >= 0:
        see &= j[None] <= p[:, None] + right
    if left >= 0:
        see &= (j[None] >= p[:, None] - left) | (j[None] < sinks)
    s = (qf @ kf.transpose(1, 2) * scale).masked_fill(~see, -torch.inf)
    some = see.any(1)
    m = torch.where(some, s.amax(-1) if kn else torch.full((q.shape[0], qn), -torch.inf, dtype=D, device=q.device), 0.0)
    e = torch.exp(s - m[..., None])
    l = e.sum(-1)
    P = e / torch.where(some, l, 1.0)[..., None]
    out = dict(o=P @ vf, lse=torch.where(some, m * LOG2E + torch.log2(l), -torch.inf))
    tiny = 2.0 ** -25 if t == torch.float16 else 0.0
    big = lambda x: float(x.abs().max()) if x.numel() else 0.0  # noqa: E731
    out["o_tol"] = u(t) * out["o"].abs() + (u(t) + 2 ** -13) * (P @ vf.abs()) + tiny * (kn * big(vf) + 1)
    # |lse| error: the exponent's error (2^-13 at most, see above) in log2 units, and f32 rounding
    out["lse_tol"] = 2 ** -13 + 2 ** -22 * out["lse"].abs()
    if dO is None:
        return out
    dof, of = dO[:, :qn].to(D), o[:, :qn].to(D)
    ls = torch.where(some, lse[:, :qn].to(D), 0.0)
    P = torch.where(see, torch.exp2(torch.where(see, s, 0.0) * LOG2E - ls[..., None]), 0.0)
    dP = dof @ vf.transpose(1, 2)
    Dr = (dof * of).sum(-1, keepdim=True)
    dS = P * (dP - Dr)
    E = P * (dof.abs() @ vf.abs().transpose(1, 2) + (dof * of).abs().sum(-1, keepdim=True))
    A = dS.abs()
    w = 2 ** -12
    out["dq"] = dS @ kf * scale
    out["dq_tol"] = u(t) * out["dq"].abs() + scale * ((u(t) * A + w * E) @ kf.abs()) + tiny * (kn * scale * big(kf) + 1)
    fold = lambda x: x.reshape(k.shape[0], g, *x.shape[1:]).sum(1)  # noqa: E731
    Et, At, Pt = (x.transpose(1, 2) for x in (E, A, P))
    out["dk"] = fold(dS.transpose(1, 2) @ qf) * scale
    out["dk_tol"] = u(t) * out["dk"].abs() + scale * fold((u(t) * At + w * Et) @ qf.abs()) + tiny * (g * qn * scale * big(qf) + 1)
    out["dv"] = fold(Pt @ dof)
    out["dv_tol"] = u(t) * out["dv"].abs() + (u(t) + w) * fold(Pt @ dof.abs()) + tiny * (g * qn * big(dof) + 1)
    return out


def layernorm(x, gamma, beta, eps, yt, n_seq):
    """n_seq: the longest chain of f32 additions behind a row's sum."""
    D = torch.float64
    xf = x.to(D)
    mu = xf.mean(1)
    var = ((xf - mu[:, None]) ** 2).mean(1)
    r = (var + eps) ** -0.5
    xh = (xf - mu[:, None]) * r[:, None]
    gm = gamma.to(D) if gamma is not None else torch.ones(x.shape[1], dtype=D, device=x.device)
    bt = beta.to(D) if beta is not None else torch.zeros(x.shape[1], dtype=D, device=x.device)
    y = xh * gm + bt
    c = n_seq * 2.0 ** -24
    mu_tol = c * xf.abs().mean(1) + 1e-30
    # xh: the mean's error over the standard deviation, and the variance's relative error
    dxh = (mu_tol * r)[:, None] * (1 + xh.abs()) + xh.abs() * (c + 2 ** -22)
    return dict(y=y, mean=mu, rstd=r, mean_tol=mu_tol, rstd_tol=r * (c + 2 ** -22 + 2 * mu_tol * r),
                y_tol=u(yt) * y.abs() + gm.abs() * dxh + 2 ** -23 * (y.abs() + bt.abs()) + 1e-7 * (yt == torch.float16))


def layernorm_grads(x, dy, gamma, mean, rstd, n_row, n_col):
    D = torch.float64
    n = x.shape[1]
    xh = (x.to(D) - mean.to(D)[:, None]) * rstd.to(D)[:, None]
    d = dy.to(D)
    g = d * (gamma.to(D) if gamma is not None else 1.0)
    dx = rstd.to(D)[:, None] * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    c = (n_row + 8) * 2.0 ** -24
    a = rstd.to(D)[:, None] * (g.abs() + g.abs().mean(1, keepdim=True) + xh.abs() * (g * xh).abs().mean(1, keepdim=True))
    cc = (n_col + 8) * 2.0 ** -24
    return dict(dx=dx, dgamma=(d * xh).sum(0), dbeta=d.sum(0),
                dx_tol=u(x.dtype) * dx.abs() + c * a + 1e-7 * (x.dtype == torch.float16),
                dgamma_tol=cc * (d * xh).abs().sum(0) + 1e-30, dbeta_tol=cc * d.abs().sum(0) + 1e-30)


def act(z, name):
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return 0.5 * z * torch.special.erfc(-z * 0.5 ** 0.5)
    if name == "gelu_tanh":
        return torch.nn.functional.gelu(z, approximate="tanh")
    return z


def assert_within(name, got, want, tol):
    """Equal where not finite, within tol elsewhere."""
    got, want = got.to(torch.float64), want.to(torch.float64)
    assert got.shape == want.shape, (name, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine], want[~fine]), f"{name}: infinities differ"
    over = ((got - want).abs() - tol)[fine]
    if over.numel():
        bad = int((~(over <= 0)).sum())     # (NaN counts)
        assert bad == 0, f"{name}: {bad} of {over.numel()} values beyond the bound, worst by {float(over.max()):.3g}"
