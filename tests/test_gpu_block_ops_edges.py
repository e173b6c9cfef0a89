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
