"""CPU tests of what the Python wrappers of the transformer-block operators check before the call.  The context
here is none (no device): a call whose arguments pass ends in "ctx is NULL"."""
import pytest
import torch


@pytest.fixture
def none(sa3k_lib):
    import sa3k
    c = object.__new__(sa3k.Context)
    c.device, c._h = -1, None           # -1: the device of CPU tensors
    return c


class Args:
    """Token-major tensors [B][S][H * 64] of one attention."""

    def __init__(self, B=2, H=4, Hkv=2, Sq=32, Sk=48, dtype=torch.float16):
        self.dims = B, H, Hkv, Sq, Sk
        z = lambda s, h: torch.zeros(B, s, h * 64, dtype=dtype)  # noqa: E731
        self.t = dict(q=z(Sq, H), o=z(Sq, H), dO=z(Sq, H), dq=z(Sq, H), k=z(Sk, Hkv), v=z(Sk, Hkv), dk=z(Sk, Hkv), dv=z(Sk, Hkv))
        self.lse = torch.zeros(B, H, Sq)

    def calls(self, c, p, **other):
        """The forward and the backward, with other Tensor4s in place of some."""
        import sa3k
        h = {n: sa3k.t4(t, t.stride(0), 64, t.stride(1)) for n, t in self.t.items()}
        h.update(other)
        yield lambda: c.attention_sink_fwd(p, h["q"], h["k"], h["v"], h["o"], self.lse)
        yield lambda: c.attention_sink_bwd(p, *(h[n] for n in ("q", "k", "v", "o", "dO")), self.lse, h["dq"], h["dk"], h["dv"])

    def describe(self, **kw):
        import sa3k
        B, H, Hkv, Sq, Sk = self.dims
        return sa3k.sink_attn(**{**dict(B=B, H=H, Sq=Sq, Sk=Sk, scale=0.125, left=8, heads_kv=Hkv), **kw})


def _refuses(f, text):
    import sa3k
    with pytest.raises(sa3k.Sa3kError, match=text):
        f()


@pytest.mark.parametrize("dtype,name", [(torch.float16, "f16"), (torch.bfloat16, "bf16")])
def test_attention_types(none, dtype, name):
    a = Args(dtype=dtype)
    for f in a.calls(none, a.describe(dtype=name)):
        _refuses(f, "ctx is NULL")
    for f in a.calls(none, a.describe(dtype="bf16" if name == "f16" else "f16")):
        _refuses(f, "description's dtype")
    import sa3k
    for n in a.t:
        for wrong in (torch.float32, torch.float16 if name == "bf16" else torch.bfloat16):
            t = a.t[n].to(wrong)
            other = {n: sa3k.t4(t, t.stride(0), 64, t.stride(1))}
            for i, f in enumerate(a.calls(none, a.describe(dtype=name), **other)):
                _refuses(f, "description's dtype" if i == 1 or n in ("q", "k", "v", "o") else "ctx is NULL")


@pytest.mark.parametrize("name", ["q", "k", "v", "o", "dO", "dq", "dk", "dv"])
def test_attention_reach(none, name):
    """Sizes and strides that pass the end of a tensor's storage by a single value, whatever the view."""
    import sa3k
    a = Args()
    B, H, Hkv, Sq, Sk = a.dims
    t = a.t[name]
    h, s = (Hkv, Sk) if name in ("k", "v", "dk", "dv") else (H, Sq)
    i = 0 if name in ("q", "k", "v", "o") else 1          # (the call that takes it)
    n = t.numel()
    store = torch.zeros(n + 16, dtype=torch.float16)
    fits = (t, store[16:], store.view(-1)[16:n].view(-1), store[16:].as_strided((2, 2), (1, 1), 16))
    for u in fits:
        f = list(a.calls(none, a.describe(), **{name: sa3k.t4(u, s * h * 64, 64, h * 64)}))[i]
        _refuses(f, "ctx is NULL")
    short = torch.zeros(n - 1, dtype=torch.float16)
    for u, strides in ((short, (s * h * 64, 64, h * 64)), (store[24:], (s * h * 64, 64, h * 64)), (t, (s * h * 64 + 8, 64, h * 64)),
                       (t, (s * h * 64, 64, h * 64 + 8)), (t, (64, 64 * B, h * 64 * B + 8))):
        f = list(a.calls(none, a.describe(), **{name: sa3k.t4(u, *strides)}))[i]
        _refuses(f, "past a tensor's end")


def test_attention_reach_of_single_entries_and_empty_sizes(none):
    """The stride of a dimension of one entry does not count; without entries nothing is reached."""
    import sa3k
    a = Args(B=1, H=1, Hkv=1, Sq=1, Sk=1)
    big = {n: sa3k.t4(t, 1 << 30, 1 << 30, 1 << 30) for n, t in a.t.items()}
    for f in a.calls(none, a.describe(), **big):
        _refuses(f, "ctx is NULL")
    for kw in (dict(B=0), dict(Sq=0), dict(Sk=0)):
        a = Args(**kw)
        for f in a.calls(none, a.describe()):
            _refuses(f, "ctx is NULL")


def test_attention_devices_come_first(none):
    import sa3k
    a = Args(dtype=torch.bfloat16)
    none.device = 0
    for f in a.calls(none, a.describe(), q=sa3k.t4(a.t["q"], 8192, 64, 256)):
        _refuses(f, "not on the context's device")
    none.device = -1
    # Tensor4s made by hand carry no tensor: they are taken as they are
    raw = sa3k.Tensor4(a.t["q"].data_ptr(), 8192, 64, 256)
    for f in a.calls(none, a.describe(dtype="bf16"), q=raw):
        _refuses(f, "ctx is NULL")


def test_linear_act_adapter_arrays(none):
    """The arrays of an adapter fit the weight that it is used with."""
    import sa3k

    class W:
        _h, inn, out = None, 64, 48

    f = lambda *s: torch.zeros(*s)  # noqa: E731
    x, y, dx = (torch.zeros(4, n, dtype=torch.float16) for n in (64, 48, 64))
    good = dict(A=f(8, 64), B=f(48, 8), m=f(48), bns=f(48))
    grads = dict(dA=f(8, 64), dB=f(48, 8), dm=f(48))
    fwd = lambda a: none.linear_act_fwd(W, x, y, "silu", ad=sa3k.Context.adapter(a["A"], a["B"], 1.0, a["m"], a["bns"]))  # noqa: E731
    bwd = lambda a, g: none.linear_act_bwd(W, x, y, y, dx, "silu", ad=sa3k.Context.adapter(a["A"], a["B"], 1.0, a["m"], a["bns"]), **g)  # noqa: E731
    for call in (lambda: fwd(good), lambda: bwd(good, grads)):
        _refuses(call, "ctx is NULL")
    for n, bad in (("A", f(8, 63)), ("A", f(64, 8).t()), ("B", f(47, 8)), ("B", f(48, 8).half()), ("m", f(47)), ("bns", f(49)),
                   ("A", f(8, 64).numpy())):
        _refuses(lambda: fwd({**good, n: bad}), "linear_act .adapter.")
        _refuses(lambda: bwd({**good, n: bad}, grads), "linear_act .adapter.")
    for n, bad in (("dA", f(7, 64)), ("dB", f(48, 9)), ("dm", f(47)), ("dA", f(8, 64).double())):
        _refuses(lambda: bwd(good, {**grads, n: bad}), "linear_act .adapter.")
    none.device = 0
    for call in (lambda: fwd(good), lambda: bwd(good, grads)):
        _refuses(call, "the context on")
