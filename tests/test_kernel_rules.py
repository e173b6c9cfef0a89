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


def test_dkdv_sets_see_every_phase_of_the_barriers_they_wait_on():
    """Two sets of warps take alternate steps; a set that waited on every second phase of a barrier could take an
    older phase for the one it waits for (the parity is the same)."""
    body = dict(_kernels("attention_sink.cu"))["sink_dkdv_kernel"]
    const = {n: int(v) for n, v in re.findall(r"(kDkvSets|kDkvStages|kDkvItems) = (\d+)", open(os.path.join(CSRC, "attention_sink.cu")).read())}
    period, phase = re.search(r"waitw\(&s_full\[t % (\w+)\], \(uint32_t\)\(\(t / (\w+)\) & 1\)", body).groups()
    assert period == phase
    expr = re.search(r"constexpr int " + period + r" = ([^;]+);", body).group(1)
    F = eval(expr, {}, const)
    last = {}
    for t in range(20 * F):
        who = t % const["kDkvSets"], t % F          # the set of step t, the barrier it waits on
        assert t // F == last.get(who, -1) + 1, who
        last[who] = t // F
    assert f"for (int i = 0; i < {expr}; ++i) mbar_init(&s_full[i], 1)" in body
