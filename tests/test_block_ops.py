"""CPU tests of the transformer-block operators: the float64 forms that the GPU tests compare with,
against autograd, and the refusals that need no GPU."""
import ctypes

import pytest
import torch

import block_ops_ref as ref

D = torch.float64


def _mask(qn, kn, left, right, sinks, end):
    see = torch.zeros(qn, kn, dtype=torch.bool)
    for i in range(qn):
        p = i + (kn - qn if end else 0)
        for j in range(kn):
            see[i, j] = (right < 0 or j <= p + right) and (left < 0 or j < sinks or j >= p - left)
    return see


@pytest.mark.parametrize("H,Hkv,qn,kn,left,right,sinks,end", [
    (2, 1, 9, 9, 3, 0, 2, False), (4, 2, 5, 12, 4, 1, 3, True), (1, 1, 8, 3, 1, 1, 0, False),
    (2, 2, 1, 7, -1, 0, 0, True), (2, 1, 6, 4, 2, 0, 1, True)])
def test_attention_form_against_autograd(H, Hkv, qn, kn, left, right, sinks, end):
    g = torch.Generator().manual_seed(qn * 31 + kn)
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float32)  # noqa: E731
    q, k, v, dO = rnd(H, qn, 64), rnd(Hkv, kn, 64), rnd(Hkv, kn, 64), rnd(H, qn, 64)
    see = _mask(qn, kn, left, right, sinks, end)
    leaves = [t.to(D).requires_grad_(True) for t in (q, k, v)]
    kk, vv = (t.repeat_interleave(H // Hkv, 0) for t in leaves[1:])
    s = (leaves[0] @ kk.transpose(1, 2) * 0.125).masked_fill(~see, -torch.inf)
    some = see.any(1)
    s = torch.where(some[:, None], s, 0.0)
    o = torch.where(some[:, None], torch.softmax(s, -1), 0.0) @ vv
    o.backward(dO.to(D))
    first = ref.attention(q, k, v, 0.125, left, right, sinks, qn, kn, end)
    w = ref.attention(q, k, v, 0.125, left, right, sinks, qn, kn, end, dO, first["o"], first["lse"])
    lse = torch.where(some, torch.logsumexp(s, -1) * ref.LOG2E, -torch.inf)
    assert torch.allclose(w["o"], o.detach(), rtol=1e-12, atol=1e-12)
    assert torch.allclose(w["lse"], lse.detach(), rtol=1e-12, atol=1e-12)
    for n, t in zip(("dq", "dk", "dv"), leaves):
        assert torch.allclose(w[n], t.grad, rtol=1e-10, atol=1e-12), n


def test_layernorm_form_against_autograd():
    g = torch.Generator().manual_seed(3)
    x, dy, gamma, beta = (torch.randn(*s, generator=g, dtype=D) for s in ((5, 33), (5, 33), (33,), (33,)))
    leaves = [t.clone().requires_grad_(True) for t in (x, gamma, beta)]
    y = torch.nn.functional.layer_norm(leaves[0], (33,), leaves[1], leaves[2], 1e-5)
    y.backward(dy)
    w = ref.layernorm(x, gamma, beta, 1e-5, torch.float32, 1)
    b = ref.layernorm_grads(x, dy, gamma, w["mean"], w["rstd"], 1, 1)
    assert torch.allclose(w["y"], y.detach(), rtol=1e-12, atol=1e-12)
    for n, t in zip(("dx", "dgamma", "dbeta"), leaves):
        assert torch.allclose(b[n], t.grad, rtol=1e-10, atol=1e-12), n


def test_sink_attn_refusals():
    import sa3k
    with pytest.raises(sa3k.Sa3kError, match="dtype"):
        sa3k.sink_attn(1, 1, 1, 1, 0.125, dtype="f32")
    for t in (torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(1)):
        with pytest.raises(sa3k.Sa3kError, match="q_len must be"):
            sa3k.sink_attn(1, 1, 1, 1, 0.125, q_len=t)


def test_entry_points_without_a_context(sa3k_lib):
    """No context: an error and a message, not a crash."""
    import sa3k
    L = sa3k_lib
    err = ctypes.create_string_buffer(512)
    p, t = sa3k.sink_attn(1, 1, 1, 1, 0.125), sa3k.Tensor4(None, 64, 64, 64)
    r = ctypes.byref
    calls = (lambda: L.sa3k_layernorm_fwd(None, 1, 8, 0, None, 8, None, None, 1e-5, 0, None, 8, None, None, err, 512),
             lambda: L.sa3k_layernorm_bwd(None, 1, 8, 0, None, 8, None, None, None, 0, None, 8, None, 8, None, None, 0, err, 512),
             lambda: L.sa3k_attention_sink_fwd(None, r(p), r(t), r(t), r(t), r(t), None, err, 512),
             lambda: L.sa3k_attention_sink_bwd(None, r(p), r(t), r(t), r(t), r(t), r(t), None, r(t), None, None, err, 512),
             lambda: L.sa3k_linear_act_fwd(None, None, None, None, 0, 0, None, 1, None, None, None, err, 512),
             lambda: L.sa3k_linear_act_bwd(None, None, None, None, 0, 0, None, 1, None, None, None, None, None, None, None, 0,
                                           err, 512))
    for f in calls:
        err.value = b""
        assert f() != 0 and err.value
