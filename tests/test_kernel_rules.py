"""Rules that the kernels keep and no run can show (breaking one could hang the GPU), read off the sources."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sa3.cpp_b200", "csrc")


def _kernels(name):
    """(kernel, body up to the next kernel) of a source file."""
    src = open(os.path.join(CSRC, name)).read()
    starts = [m.start() for m in re.finditer(r"__global__", src)] + [len(src)]
    for a, b in zip(starts, starts[1:]):
        body = src[a:b]
        yield re.search(r"(\w+_kernel)\s*\(", body).group(1), body


def test_attention_kernels_trigger_with_tensor_memory_in_hand():
    """Kernels that may share an SM let the next one start after their tcgen05.alloc, not before it."""
    seen = 0
    for name in ("attention_tc.cu", "attention_sink.cu"):
        for kernel, body in _kernels(name):
            if "tmem_alloc(" not in body:
                continue
            seen += 1
            alloc = body.index("tmem_alloc(")
            barrier = body.index("__syncthreads()", alloc)
            for m in re.finditer(r"pdl_(trigger|prologue)\(\)", body):
                assert m.start() > barrier, f"{name}: {kernel} triggers before it has its tensor memory"
            assert "pdl_trigger()" in body and body.index("pdl_trigger()") < body.index("pdl_wait()"), kernel
    assert seen == 8
