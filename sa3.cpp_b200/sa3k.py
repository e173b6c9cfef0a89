"""ctypes binding of libsa3k.so (include/sa3k.h) for tests, the benchmark and Python callers.

Device buffers are torch CUDA tensors (torch is only the allocator and stream here: every
computation runs in libsa3k's own kernels).  The library must have been built in-tree
(`python sa3.cpp_b200/build.py`); a missing library raises, there is no fallback.
"""
from __future__ import annotations

import ctypes
import weakref
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "lib", "libsa3k.so")

TYPE_IDS = {"f32": 0, "f16": 1, "q8_0": 8, "q4_k": 12, "bf16": 30}

# every symbol include/sa3k.h declares
ABI_SYMBOLS = (
    "sa3k_version", "sa3k_ctx_create", "sa3k_ctx_destroy", "sa3k_ctx_set_stream", "sa3k_sync", "sa3k_check_bounded_wait",
    "sa3k_weight_upload", "sa3k_weight_free", "sa3k_dequant", "sa3k_row_norms", "sa3k_col_norms", "sa3k_linear_fwd",
    "sa3k_linear_bwd", "sa3k_linear_fwd_bwd", "sa3k_linear_fwd_bwd_host", "sa3k_adamw",
    "sa3k_average_clip_adamw", "sa3k_profile_enable", "sa3k_profile_read", "sa3k_ctx_set_option",
    "sa3k_attention_fwd", "sa3k_attention_bwd", "sa3k_attention_bwd_noalloc", "sa3k_head_prep_fwd", "sa3k_head_prep_bwd",
    "sa3k_dit_create", "sa3k_dit_free", "sa3k_dit_set_tensor", "sa3k_dit_init_adapters", "sa3k_dit_adapter_size",
    "sa3k_dit_adapter_offsets", "sa3k_dit_adapter_buffer", "sa3k_dit_adapter_copy", "sa3k_dit_zero_grads",
    "sa3k_dit_forward_backward", "sa3k_dit_forward_backward_inpaint", "sa3k_dit_apply_adamw", "sa3k_dp_unique_id", "sa3k_dp_comm_create", "sa3k_dp_comm_create_timeout",
    "sa3k_dp_comm_destroy", "sa3k_dp_comm_info", "sa3k_dp_allreduce_sum", "sa3k_dp_allreduce_adamw",
    "sa3k_dit_dp_apply_adamw", "sa3k_dit_save_adapter", "sa3k_dit_load_adapter", "sa3k_dit_save_checkpoint",
    "sa3k_dit_load_checkpoint", "sa3k_adapter_gguf_write", "sa3k_gguf_get_string", "sa3k_gguf_get_u64",
    "sa3k_gguf_get_u64_array", "sa3k_gguf_get_f32", "sa3k_lora_chain_build", "sa3k_lora_chain_free",
    "sa3k_lora_chain_info", "sa3k_linear_fwd_chain", "sa3k_mat_effective_weight", "sa3k_linear_mat_fwd",
    "sa3k_linear_mat_fwd_bwd", "sa3k_dit_adapter_layout", "sa3k_dit_set_xs_bases", "sa3k_layernorm_fwd", "sa3k_layernorm_bwd",
    "sa3k_attention_sink_fwd", "sa3k_attention_sink_bwd", "sa3k_linear_act_fwd", "sa3k_linear_act_bwd",
)
ACTIVATIONS = {"none": 0, "silu": 1, "gelu": 2, "gelu_tanh": 3}
OPT_WEIGHT_F16_CACHE, OPT_SMEM_DEQUANT, OPT_GEMM_TILE_N, OPT_GEMM_PAIR, OPT_ATTN_TC, OPT_PDL = 1, 2, 3, 4, 5, 6
OPT_STEP_GRAPH = 7
OPT_DEQUANT_TMEM = 8
OPT_FUSE_HEAD_PREP = 9


_TYPES = {}


def _torch_types():
    """torch dtype -> SA3K_TYPE_* of the activations (torch is imported on first use)."""
    if not _TYPES:
        import torch
        _TYPES.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 30})
    return _TYPES


class Sa3kError(RuntimeError):
    pass


class Adapter(ctypes.Structure):
    _fields_ = [("A", ctypes.c_void_p), ("B", ctypes.c_void_p), ("magnitude", ctypes.c_void_p),
                ("base_norm_sq", ctypes.c_void_p), ("scale", ctypes.c_float), ("rank", ctypes.c_int)]
    of = None           # A, B, m, bns of Context.adapter()


class Tensor4(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("batch_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64),
                ("row_stride", ctypes.c_int64)]
    of = None           # the tensor that t4() made it of


class SinkAttnC(ctypes.Structure):
    """sa3k_sink_attn: an attention over a sliding window with sink tokens (made by sink_attn())."""
    _fields_ = [("type", ctypes.c_int), ("B", ctypes.c_int), ("H", ctypes.c_int), ("H_kv", ctypes.c_int),
                ("Sq", ctypes.c_int), ("Sk", ctypes.c_int), ("head_dim", ctypes.c_int), ("scale", ctypes.c_float),
                ("left", ctypes.c_int64), ("right", ctypes.c_int64), ("sinks", ctypes.c_int64),
                ("align_end", ctypes.c_int), ("q_len", ctypes.c_void_p), ("kv_len", ctypes.c_void_p)]
    device = None


def sink_attn(B, H, Sq, Sk, scale, left=-1, right=0, sinks=0, heads_kv=None, dtype="f16", align_end=False, q_len=None,
              kv_len=None, head_dim=64):
    """The description of an attention over the window [p - left, p + right] (< 0: no bound) and the first
    `sinks` keys; q_len, kv_len: int32 CUDA tensors [B] or None.  See sa3k_sink_attn in sa3k.h."""
    if dtype not in ("f16", "bf16"):
        raise Sa3kError("sink_attn: dtype must be f16 or bf16")
    p = SinkAttnC(TYPE_IDS[dtype], B, H, H if heads_kv is None else heads_kv, Sq, Sk, head_dim, scale, left, right,
                  sinks, 1 if align_end else 0, None, None)
    p.keep = (q_len, kv_len)     # the tensors live as long as the description
    for name, t in (("q_len", q_len), ("kv_len", kv_len)):
        if t is not None:
            if t.numel() != B or not t.is_cuda or str(t.dtype) != "torch.int32" or not t.is_contiguous():
                raise Sa3kError(f"sink_attn: {name} must be a contiguous int32 CUDA tensor of B values")
            setattr(p, name, t.data_ptr())
            if p.device not in (None, t.get_device()):
                raise Sa3kError("sink_attn: q_len and kv_len must be on one device")
            p.device = t.get_device()
    return p


class HeadSliceC(ctypes.Structure):
    _fields_ = [("col", ctypes.c_int), ("gamma", ctypes.c_void_p), ("rope", ctypes.c_int), ("rstd", ctypes.c_void_p)]


def t4(t, batch_stride, head_stride, row_stride):
    r = Tensor4()
    r.data, r.batch_stride, r.head_stride, r.row_stride = t.data_ptr(), batch_stride, head_stride, row_stride
    r.of = t
    return r


DIT_INT_FIELDS = ("io", "dim", "depth", "heads", "head_dim", "cond_dim", "mem_tokens", "rot", "time_dim",
                  "ff_inner", "differential")
DIT_FLOAT_FIELDS = ("rope_base", "norm_eps", "qk_eps", "time_min_freq", "time_max_freq")


class DitConfigC(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_int) for n in DIT_INT_FIELDS] + [(n, ctypes.c_float) for n in DIT_FLOAT_FIELDS] +
                [("local_dim", ctypes.c_int)])


class ProfileEntry(ctypes.Structure):
    _fields_ = [("name", ctypes.c_char * 48), ("launches", ctypes.c_int64), ("total_ms", ctypes.c_double)]


class ChainTerm(ctypes.Structure):
    """sa3k_chain_term: one adapter of an inference chain (device pointers)."""
    _fields_ = [("A", ctypes.c_void_p), ("B", ctypes.c_void_p), ("magnitude", ctypes.c_void_p), ("rank", ctypes.c_int),
                ("scale", ctypes.c_float)]


class MatAdapter(ctypes.Structure):
    """sa3k_mat_adapter: a materialized adapter of any family ("lora", "dora-rows", "dora-cols",
    "bora", each optionally "-xs"); every array a device pointer."""
    _fields_ = [("adapter_type", ctypes.c_char_p), ("rank", ctypes.c_int), ("scale", ctypes.c_float),
                ("A", ctypes.c_void_p), ("B", ctypes.c_void_p), ("U", ctypes.c_void_p), ("V", ctypes.c_void_p),
                ("M", ctypes.c_void_p), ("m", ctypes.c_void_p), ("m_r", ctypes.c_void_p), ("m_c", ctypes.c_void_p)]


class MatGrads(ctypes.Structure):
    """sa3k_mat_grads: the gradient outputs of sa3k_linear_mat_fwd_bwd (NULL where unused)."""
    _fields_ = [("dA", ctypes.c_void_p), ("dB", ctypes.c_void_p), ("dM", ctypes.c_void_p), ("dm", ctypes.c_void_p),
                ("dm_r", ctypes.c_void_p), ("dm_c", ctypes.c_void_p)]


def _vp(t):
    return None if t is None else t.data_ptr()


class TrainProgress(ctypes.Structure):
    """sa3k_train_progress: the dataset-side progress stored in a trainer-state file."""
    _fields_ = [("epoch", ctypes.c_uint64), ("next_sample", ctypes.c_uint64),
                ("order", ctypes.POINTER(ctypes.c_uint64)), ("n_order", ctypes.c_int64),
                ("compatibility", ctypes.c_char_p), ("rng_shuffle", ctypes.c_char_p), ("rng_crop", ctypes.c_char_p),
                ("rng_cfg", ctypes.c_char_p), ("rng_prompt", ctypes.c_char_p), ("rng_inpaint", ctypes.c_char_p),
                ("rng_diffusion", ctypes.c_char_p)]


class AdamWParams(ctypes.Structure):
    _fields_ = [("learning_rate", ctypes.c_float), ("beta1", ctypes.c_float), ("beta2", ctypes.c_float),
                ("eps", ctypes.c_float), ("weight_decay", ctypes.c_float), ("grad_clip", ctypes.c_float)]


_lib = None


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise Sa3kError(f"{LIB_PATH} is not built (python sa3.cpp_b200/build.py)")
        L = ctypes.CDLL(LIB_PATH)
        P, I, I64, F, E = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_char_p
        L.sa3k_version.restype = ctypes.c_char_p
        L.sa3k_ctx_create.argtypes = [I, ctypes.POINTER(P), E, I]
        L.sa3k_ctx_destroy.argtypes = [P]
        L.sa3k_ctx_destroy.restype = None
        L.sa3k_ctx_set_stream.argtypes = [P, P, E, I]
        L.sa3k_sync.argtypes = [P, E, I]
        L.sa3k_check_bounded_wait.argtypes = [P, I, E, I]
        L.sa3k_weight_upload.argtypes = [P, I, P, I64, I64, ctypes.POINTER(P), E, I]
        L.sa3k_weight_free.argtypes = [P]
        L.sa3k_weight_free.restype = None
        L.sa3k_dequant.argtypes = [P, P, P, E, I]
        L.sa3k_row_norms.argtypes = [P, P, F, P, P, E, I]
        L.sa3k_linear_fwd.argtypes = [P, P, P, P, P, I64, P, E, I]
        L.sa3k_linear_bwd.argtypes = [P, P, P, P, P, P, P, I64, P, P, P, P, I, E, I]
        L.sa3k_linear_fwd_bwd.argtypes = [P, P, P, P, P, P, I64, P, P, P, P, P, E, I]
        L.sa3k_linear_fwd_bwd_host.argtypes = [P, P, P, P, P, P, I64, P, P, P, P, P, E, I]
        L.sa3k_adamw.argtypes = [P, P, P, P, P, I64, ctypes.POINTER(AdamWParams), I, E, I]
        L.sa3k_average_clip_adamw.argtypes = [P, P, P, P, P, I64, I, ctypes.POINTER(AdamWParams), I,
                                              ctypes.POINTER(ctypes.c_double), E, I]
        L.sa3k_profile_enable.argtypes = [P, I, E, I]
        L.sa3k_ctx_set_option.argtypes = [P, I, I64, E, I]
        L.sa3k_dit_create.argtypes = [P, ctypes.POINTER(DitConfigC), ctypes.POINTER(P), E, I]
        L.sa3k_dit_free.argtypes = [P]
        L.sa3k_dit_free.restype = None
        L.sa3k_dit_set_tensor.argtypes = [P, ctypes.c_char_p, I, P, I64, I64, E, I]
        L.sa3k_dit_init_adapters.argtypes = [P, ctypes.c_char_p, I, F, ctypes.POINTER(ctypes.c_char_p), I, E, I]
        L.sa3k_dit_adapter_size.argtypes = [P]
        L.sa3k_dit_adapter_offsets.argtypes = [P, I, ctypes.POINTER(I64), ctypes.POINTER(I64), ctypes.POINTER(I64)]
        L.sa3k_dit_adapter_buffer.argtypes = [P, I, ctypes.POINTER(P), E, I]
        L.sa3k_dit_adapter_layout.argtypes = [P, I, ctypes.POINTER(I64)]
        L.sa3k_dit_set_xs_bases.argtypes = [P, ctypes.c_char_p, P, P, E, I]
        L.sa3k_dit_adapter_copy.argtypes = [P, I, P, I64, I64, I, E, I]
        L.sa3k_dit_zero_grads.argtypes = [P, E, I]
        L.sa3k_dit_forward_backward.argtypes = [P, I, I, I, P, P, P, P, P, P, E, I]
        L.sa3k_dit_apply_adamw.argtypes = [P, I, ctypes.POINTER(AdamWParams), I, ctypes.POINTER(ctypes.c_double), E, I]
        T4 = ctypes.POINTER(Tensor4)
        L.sa3k_attention_fwd.argtypes = [P, I, I, I, I, I, F, I, T4, T4, T4, T4, P, E, I]
        L.sa3k_attention_bwd.argtypes = [P, I, I, I, I, I, F, I, T4, T4, T4, T4, T4, P, T4, T4, T4, E, I]
        L.sa3k_attention_bwd_noalloc.argtypes = [P, I, I, I, I, I, F, I, T4, T4, T4, T4, T4, P, T4, T4, T4, E, I]
        SA = ctypes.POINTER(SinkAttnC)
        L.sa3k_attention_sink_fwd.argtypes = [P, SA, T4, T4, T4, T4, P, E, I]
        L.sa3k_attention_sink_bwd.argtypes = [P, SA, T4, T4, T4, T4, T4, P, T4, T4, T4, E, I]
        L.sa3k_layernorm_fwd.argtypes = [P, I64, I64, I, P, I64, P, P, F, I, P, I64, P, P, E, I]
        L.sa3k_layernorm_bwd.argtypes = [P, I64, I64, I, P, I64, P, P, P, I, P, I64, P, I64, P, P, I, E, I]
        L.sa3k_linear_act_fwd.argtypes = [P, P, P, P, I, I, P, I64, P, P, P, E, I]
        L.sa3k_linear_act_bwd.argtypes = [P, P, P, P, I, I, P, I64, P, P, P, P, P, P, P, I, E, I]
        L.sa3k_head_prep_fwd.argtypes = [P, P, I, I, I, ctypes.POINTER(HeadSliceC), I, I, F, I, F, P, E, I]
        L.sa3k_head_prep_bwd.argtypes = [P, P, I64, P, I, I, I, ctypes.POINTER(HeadSliceC), I, I, F, P, E, I]
        L.sa3k_dp_unique_id.argtypes = [P, I, E, I]
        L.sa3k_dp_comm_create.argtypes = [P, I, I, P, ctypes.POINTER(P), E, I]
        L.sa3k_dp_comm_create_timeout.argtypes = [P, I, I, P, ctypes.c_double, ctypes.POINTER(P), E, I]
        L.sa3k_dp_comm_destroy.argtypes = [P]
        L.sa3k_dp_comm_destroy.restype = None
        L.sa3k_dp_comm_info.argtypes = [P, ctypes.POINTER(I), ctypes.POINTER(I)]
        L.sa3k_dp_allreduce_sum.argtypes = [P, P, P, I64, E, I]
        L.sa3k_dp_allreduce_adamw.argtypes = [P, P, P, P, P, P, I64, I, ctypes.POINTER(AdamWParams), I,
                                              ctypes.POINTER(ctypes.c_double), E, I]
        L.sa3k_dit_dp_apply_adamw.argtypes = [P, P, I, ctypes.POINTER(AdamWParams), I,
                                              ctypes.POINTER(ctypes.c_double), E, I]
        L.sa3k_profile_read.argtypes = [P, ctypes.POINTER(ProfileEntry), I, ctypes.POINTER(I), E, I]
        L.sa3k_lora_chain_build.argtypes = [P, P, ctypes.POINTER(ChainTerm), I, ctypes.POINTER(P), E, I]
        L.sa3k_lora_chain_free.argtypes = [P]
        L.sa3k_lora_chain_free.restype = None
        L.sa3k_lora_chain_info.argtypes = [P, ctypes.POINTER(I), ctypes.POINTER(I)]
        L.sa3k_linear_fwd_chain.argtypes = [P, P, P, P, P, I64, P, E, I]
        L.sa3k_mat_effective_weight.argtypes = [P, P, ctypes.POINTER(MatAdapter), P, E, I]
        L.sa3k_linear_mat_fwd.argtypes = [P, P, ctypes.POINTER(MatAdapter), P, P, I64, P, E, I]
        L.sa3k_linear_mat_fwd_bwd.argtypes = [P, P, ctypes.POINTER(MatAdapter), P, P, P, I64, P, P,
                                              ctypes.POINTER(MatGrads), E, I]
        L.sa3k_dit_save_adapter.argtypes = [P, E, E, I]
        L.sa3k_dit_load_adapter.argtypes = [P, E, E, I]
        L.sa3k_dit_save_checkpoint.argtypes = [P, E, E, I64, ctypes.POINTER(TrainProgress), E, I]
        L.sa3k_dit_load_checkpoint.argtypes = [P, E, E, ctypes.POINTER(I64), E, I]
        PP = ctypes.POINTER(ctypes.c_void_p)
        L.sa3k_adapter_gguf_write.argtypes = [E, E, I, F, I, ctypes.POINTER(ctypes.c_char_p), ctypes.POINTER(I64),
                                              ctypes.POINTER(I64), PP, PP, PP, E, I]
        L.sa3k_gguf_get_string.argtypes = [E, E, E, I64, ctypes.POINTER(I64), E, I]
        L.sa3k_gguf_get_u64.argtypes = [E, E, ctypes.POINTER(ctypes.c_uint64), E, I]
        L.sa3k_gguf_get_u64_array.argtypes = [E, E, ctypes.POINTER(ctypes.c_uint64), I64, ctypes.POINTER(I64), E, I]
        L.sa3k_gguf_get_f32.argtypes = [E, E, P, I64, ctypes.POINTER(I64), ctypes.POINTER(I64), ctypes.POINTER(I), E, I]
        for name in ABI_SYMBOLS:
            if name not in ("sa3k_version", "sa3k_ctx_destroy", "sa3k_weight_free", "sa3k_dit_free",
                            "sa3k_dp_comm_destroy", "sa3k_lora_chain_free"):
                getattr(L, name).restype = I
        L.sa3k_dit_adapter_size.restype = I64
        _lib = L
    return _lib


def _ptr(t):
    if t is None:
        return None
    if hasattr(t, "data_ptr"):
        return ctypes.c_void_p(t.data_ptr())
    if hasattr(t, "ctypes"):
        return t.ctypes.data_as(ctypes.c_void_p)
    return t


def _check(rc, err):
    if rc != 0:
        raise Sa3kError(err.value.decode(errors="replace"))


class Context:
    """A sa3k context bound to one CUDA device (and, by default, torch's current stream)."""

    def __init__(self, device=0, use_torch_stream=True):
        self._h = ctypes.c_void_p()
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_ctx_create(device, ctypes.byref(self._h), err, 512), err)
        self.device = device
        if use_torch_stream:
            import torch
            s = torch.cuda.current_stream(device).cuda_stream
            self.set_stream(s)

    def set_stream(self, stream_handle):
        err = ctypes.create_string_buffer(256)
        _check(lib().sa3k_ctx_set_stream(self._h, ctypes.c_void_p(stream_handle), err, 256), err)

    def set_option(self, option, value):
        err = ctypes.create_string_buffer(256)
        _check(lib().sa3k_ctx_set_option(self._h, option, int(value), err, 256), err)

    def sync(self):
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_sync(self._h, err, 512), err)

    def check_bounded_wait(self, limit_us):
        """Launch the bounded-wait probe (a wait that runs out after limit_us); the next sync()
        raises with the timeout."""
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_check_bounded_wait(self._h, int(limit_us), err, 512), err)

    def _own(self, obj):
        """Objects made on this context (weights, models, communicators) are released before it."""
        if not hasattr(self, "_children"):
            self._children = weakref.WeakSet()
        self._children.add(obj)

    def close(self):
        for obj in list(getattr(self, "_children", ())):
            obj.close()
        if self._h:
            lib().sa3k_ctx_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def profile_enable(self, timing=1):
        """timing 0: count launches only; 1: time each launch class with events (eager);
        2: events captured into a CUDA graph, re-read after each replay."""
        err = ctypes.create_string_buffer(256)
        _check(lib().sa3k_profile_enable(self._h, int(timing), err, 256), err)

    def profile_read(self):
        """{class name: (launches, total_ms)} since the last profile_enable."""
        err = ctypes.create_string_buffer(256)
        n = ctypes.c_int(0)
        _check(lib().sa3k_profile_read(self._h, None, 0, ctypes.byref(n), err, 256), err)
        arr = (ProfileEntry * max(n.value, 1))()
        _check(lib().sa3k_profile_read(self._h, arr, n.value, ctypes.byref(n), err, 256), err)
        return {arr[i].name.decode(): (arr[i].launches, arr[i].total_ms) for i in range(n.value)}

    # -------------------------------------------------------------------- attention
    def attention_fwd(self, B, H, Sq, Sk, scale, window, q, k, v, o, lse):
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_attention_fwd(self._h, B, H, Sq, Sk, 64, scale, window, ctypes.byref(q), ctypes.byref(k),
                                        ctypes.byref(v), ctypes.byref(o), _ptr(lse), err, 512), err)

    def attention_bwd(self, B, H, Sq, Sk, scale, window, q, k, v, o, dO, lse, dq, dk=None, dv=None):
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_attention_bwd(self._h, B, H, Sq, Sk, 64, scale, window, ctypes.byref(q), ctypes.byref(k),
                                        ctypes.byref(v), ctypes.byref(o), ctypes.byref(dO), _ptr(lse), ctypes.byref(dq),
                                        ctypes.byref(dk) if dk else None, ctypes.byref(dv) if dv else None, err, 512),
               err)

    def attention_bwd_noalloc(self, B, H, Sq, Sk, scale, window, q, k, v, o, dO, lse, dq, dk=None, dv=None):
        """attention_bwd with its scratch in a fixed library array (B*H*Sq <= 2**20); see sa3k.h."""
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_attention_bwd_noalloc(self._h, B, H, Sq, Sk, 64, scale, window, ctypes.byref(q),
                                                ctypes.byref(k), ctypes.byref(v), ctypes.byref(o), ctypes.byref(dO),
                                                _ptr(lse), ctypes.byref(dq), ctypes.byref(dk) if dk else None,
                                                ctypes.byref(dv) if dv else None, err, 512), err)

    # ------------------------------------------------------- transformer-block operators
    # (called per token when serving, so the checks are kept cheap)
    def _on_device(self, what, *tensors):
        for t in tensors:
            if t is not None and t.get_device() != self.device:
                raise Sa3kError(f"{what}: a tensor is on {t.device}, the context on cuda:{self.device}")

    @staticmethod
    def _type_id(what, t):
        ids = _torch_types()
        if t.dtype not in ids:
            raise Sa3kError(f"{what}: unsupported type {t.dtype}")
        return ids[t.dtype]

    @staticmethod
    def _f32_vector(what, n, *tensors):
        for t in tensors:
            if t is not None and (t.numel() != n or _torch_types().get(t.dtype) != 0 or not t.is_contiguous()):
                raise Sa3kError(f"{what}: expected a contiguous float32 vector of {n} values")

    @staticmethod
    def _matrix(what, shape, *tensors):
        for t in tensors:
            if t is not None and (t.shape != shape or (shape[1] > 1 and t.stride(1) != 1)):
                raise Sa3kError(f"{what}: expected a [{shape[0]}][{shape[1]}] matrix with contiguous rows")

    def _err_buf(self):
        try:
            return self._err
        except AttributeError:
            self._err = ctypes.create_string_buffer(512)
            return self._err

    def _call(self, fn, *args):
        if fn(self._h, *args, self._err_buf(), 512) != 0:
            raise Sa3kError(self._err.value.decode(errors="replace"))

    def layernorm_fwd(self, x, y, gamma=None, beta=None, eps=1e-5, mean=None, rstd=None):
        """y = layer norm of the rows of x [rows][cols] (f32, f16 or bf16 each); mean, rstd [rows] are kept
        when given."""
        shape = x.shape
        rows, cols = shape
        self._matrix("layernorm", shape, x, y)
        self._f32_vector("layernorm", cols, gamma, beta)
        self._f32_vector("layernorm", rows, mean, rstd)
        self._on_device("layernorm", x, y, gamma, beta, mean, rstd)
        self._call(lib().sa3k_layernorm_fwd, rows, cols, self._type_id("layernorm", x), x.data_ptr(), x.stride(0),
                   _vp(gamma), _vp(beta), eps, self._type_id("layernorm", y), y.data_ptr(), y.stride(0), _vp(mean),
                   _vp(rstd))

    def layernorm_bwd(self, x, dy, dx, mean, rstd, gamma=None, dgamma=None, dbeta=None, accumulate=False):
        """dx (x's type, or None), dgamma and dbeta (f32, or None) for upstream dy."""
        shape = x.shape
        rows, cols = shape
        self._matrix("layernorm", shape, x, dy, dx)
        self._f32_vector("layernorm", cols, gamma, dgamma, dbeta)
        self._f32_vector("layernorm", rows, mean, rstd)
        self._on_device("layernorm", x, dy, dx, mean, rstd, gamma, dgamma, dbeta)
        if dx is not None and dx.dtype != x.dtype:
            raise Sa3kError("layernorm: dx has x's type")
        self._call(lib().sa3k_layernorm_bwd, rows, cols, self._type_id("layernorm", x), x.data_ptr(), x.stride(0),
                   _vp(gamma), _vp(mean), _vp(rstd), self._type_id("layernorm", dy), dy.data_ptr(), dy.stride(0),
                   _vp(dx), 0 if dx is None else dx.stride(0), _vp(dgamma), _vp(dbeta), 1 if accumulate else 0)

    def _sink_args(self, p, lse, queries, keys):
        """Tensors [B][H][Sq] and [B][H_kv][Sk] of the description p: device, type, and that what the sizes and
        strides reach lies in the tensor's storage (Tensor4s that t4() has not made are taken as they are)."""
        dev, kind, B, Sq = self.device, (_TYPES or _torch_types()).get, p.B, p.Sq
        if p.device is not None and p.device != dev:
            raise Sa3kError(f"attention_sink: a tensor is not on the context's device cuda:{dev}")
        want = p.type
        for group, heads, rows in ((queries, p.H, Sq), (keys, p.H_kv, p.Sk)):
            b, h, s = B - 1, heads - 1, rows - 1
            for t in group:
                if t is None or t.of is None:
                    continue
                x = t.of
                if x.get_device() != dev:
                    raise Sa3kError(f"attention_sink: a tensor is not on the context's device cuda:{dev}")
                if kind(x.dtype) != want:
                    raise Sa3kError("attention_sink: a tensor's type is not the description's dtype")
                # (a contiguous tensor's own values first: its storage takes longer to ask for)
                reach = b * t.batch_stride + h * t.head_stride + s * t.row_stride + 64
                if not (x.is_contiguous() and reach <= x.numel()) and reach > x.untyped_storage().nbytes() // 2 - x.storage_offset():
                    self._sink_reach(p, t, heads, rows)
        if lse is not None:
            n = B * p.H * Sq
            if lse.numel() != n or _TYPES.get(lse.dtype) != 0 or not lse.is_contiguous():
                if 0 <= B * p.H <= 65535 and Sq >= 0:     # (other sizes are refused by the call)
                    self._f32_vector("attention_sink (lse)", n, lse)
            if lse.get_device() != dev:
                self._on_device("attention_sink", lse)

    @staticmethod
    def _sink_reach(p, t, heads, rows):
        """Refuse sizes and strides past the end of t's storage, unless the call itself refuses or ignores them."""
        used = [s for n, s in ((p.B, t.batch_stride), (heads, t.head_stride), (rows, t.row_stride)) if n > 1]
        if p.B < 1 or rows < 1 or p.H_kv < 1 or p.H % p.H_kv or p.B * p.H > 65535 or any(s % 8 or s < 0 for s in used):
            return
        raise Sa3kError(f"attention_sink: [{p.B}][{heads}][{rows}][64] at these strides reaches past a tensor's end")

    def attention_sink_fwd(self, p, q, k, v, o, lse=None):
        """Forward of the attention that p (sink_attn()) describes; q, k, v, o are t4() tensors."""
        self._sink_args(p, lse, (q, o), (k, v))
        self._call(lib().sa3k_attention_sink_fwd, p, q, k, v, o, _vp(lse))     # (ctypes takes the structures' addresses)

    def attention_sink_bwd(self, p, q, k, v, o, dO, lse, dq, dk=None, dv=None):
        """dq, and dk, dv (both or neither), for upstream dO, from the forward's o and lse."""
        self._sink_args(p, lse, (q, o, dO, dq), (k, v, dk, dv))
        self._call(lib().sa3k_attention_sink_bwd, p, q, k, v, o, dO, _vp(lse), dq, dk, dv)

    def _act_args(self, w, act, S, ins, outs, vectors):
        if act not in ACTIVATIONS:
            raise Sa3kError(f"linear_act: unknown activation {act!r}")
        kind = None
        for group, shape in ((ins, (S, w.inn)), (outs, (S, w.out))):
            for t in group:
                if t is None:
                    continue
                kind = t.dtype if kind is None else kind
                if t.shape != shape or t.dtype != kind or not t.is_contiguous():
                    raise Sa3kError(f"linear_act: expected contiguous [{S}][{shape[1]}] tensors of one type")
        self._f32_vector("linear_act", w.out, *vectors)
        self._on_device("linear_act", *ins, *outs, *vectors)
        return ACTIVATIONS[act], _torch_types().get(kind, -1)

    def _act_adapter(self, w, ad, *grads):
        """The arrays of an adapter that adapter() made, and its gradients, fit the weight."""
        sizes = ad.rank * w.inn, ad.rank * w.out, w.out, w.out
        for group in (ad.of or (), grads):
            for n, t in zip(sizes, group):
                if t is not None and not hasattr(t, "get_device"):
                    raise Sa3kError("linear_act (adapter): expected CUDA tensors")
                self._f32_vector("linear_act (adapter)", n, t)
            self._on_device("linear_act", *group)

    def linear_act_fwd(self, w, x, y, act="none", bias=None, residual=None, z=None, ad=None):
        """y = act(dit_lin(w, x) + bias) + residual; x, y, residual, z contiguous f16 or f32 (one type)."""
        S = x.shape[0]
        a, t = self._act_args(w, act, S, (x,), (y, residual, z), (bias,))
        if ad:
            self._act_adapter(w, ad)
        self._call(lib().sa3k_linear_act_fwd, w._h, ctypes.byref(ad) if ad else None, _vp(bias), a, t, x.data_ptr(), S,
                   _vp(residual), _vp(z), y.data_ptr())

    def linear_act_bwd(self, w, x, z, dy, dx, act="none", bias=None, dbias=None, ad=None, dA=None, dB=None, dm=None,
                       accumulate=False):
        """dx, dbias and the adapter gradients for upstream dy (x may be None without an adapter)."""
        S = dy.shape[0]
        a, t = self._act_args(w, act, S, (x, dx), (z, dy), (bias, dbias))
        if ad:
            self._act_adapter(w, ad, dA, dB, dm)
        self._call(lib().sa3k_linear_act_bwd, w._h, ctypes.byref(ad) if ad else None, _vp(bias), a, t, _vp(x), S, _vp(z),
                   dy.data_ptr(), _vp(dx), _vp(dbias), _vp(dA), _vp(dB), _vp(dm), 1 if accumulate else 0)

    def head_prep_fwd(self, y, T, ncols, H, slices, tps, eps, rot, base, out):
        err = ctypes.create_string_buffer(512)
        arr = (HeadSliceC * len(slices))(*slices)
        _check(lib().sa3k_head_prep_fwd(self._h, _ptr(y), T, ncols, H, arr, len(slices), tps, eps, rot, base, _ptr(out),
                                        err, 512), err)

    def head_prep_bwd(self, g, g_ld, y, T, ncols, H, sl, tps, rot, base, dy):
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_head_prep_bwd(self._h, _ptr(g), g_ld, _ptr(y), T, ncols, H, ctypes.byref(sl), tps, rot, base,
                                        _ptr(dy), err, 512), err)

    # -------------------------------------------------------------------- weights
    def upload(self, raw_bytes, qtype, inn, out):
        import numpy as np
        raw = np.ascontiguousarray(raw_bytes)
        h = ctypes.c_void_p()
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_weight_upload(self._h, TYPE_IDS[qtype], raw.ctypes.data_as(ctypes.c_void_p),
                                        inn, out, ctypes.byref(h), err, 512), err)
        return Weight(self, h, qtype, inn, out)

    # -------------------------------------------------------------------- ops
    def dequant(self, w, dst):
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_dequant(self._h, w._h, _ptr(dst), err, 512), err)

    def row_norms(self, w, eps, nsq=None, nrm=None):
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_row_norms(self._h, w._h, eps, _ptr(nsq), _ptr(nrm), err, 512), err)

    @staticmethod
    def adapter(A, B, scale, m=None, bns=None):
        rank = A.shape[0]
        ad = Adapter(_ptr(A), _ptr(B), _ptr(m), _ptr(bns), scale, rank)
        ad.of = A, B, m, bns
        return ad

    def linear_fwd(self, w, x, y, ad=None, bias=None):
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_linear_fwd(self._h, w._h, ctypes.byref(ad) if ad else None, _ptr(bias), _ptr(x),
                                     x.shape[0], _ptr(y), err, 512), err)

    def lora_chain(self, w, terms):
        """terms: list of (A [rank][in], B [out][rank], magnitude [out] or None, scale) torch cuda f32 tensors,
        in chain order.  Returns a LoraChain (folded on the device)."""
        arr = (ChainTerm * len(terms))(*[ChainTerm(A.data_ptr(), B.data_ptr(), m.data_ptr() if m is not None else None,
                                                   A.shape[0], s) for A, B, m, s in terms])
        h = ctypes.c_void_p()
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_lora_chain_build(self._h, w._h, arr, len(terms), ctypes.byref(h), err, 512), err)
        return LoraChain(h)

    def linear_fwd_chain(self, w, chain, x, y, bias=None):
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_linear_fwd_chain(self._h, w._h, chain._h, _ptr(bias), _ptr(x), x.shape[0], _ptr(y), err,
                                           512), err)

    @staticmethod
    def mat_adapter(adapter_type, rank, scale, A=None, B=None, U=None, V=None, M=None, m=None, m_r=None, m_c=None):
        """A MatAdapter over device tensors (kept alive by the caller)."""
        return MatAdapter(adapter_type.encode(), rank, scale, _vp(A), _vp(B), _vp(U), _vp(V), _vp(M), _vp(m), _vp(m_r),
                          _vp(m_c))

    def mat_effective_weight(self, w, ad, weff):
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_mat_effective_weight(self._h, w._h, ctypes.byref(ad), _ptr(weff), err, 512), err)

    def linear_mat_fwd(self, w, ad, x, y, bias=None):
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_linear_mat_fwd(self._h, w._h, ctypes.byref(ad), _ptr(bias), _ptr(x), x.shape[0], _ptr(y),
                                         err, 512), err)

    def linear_mat_fwd_bwd(self, w, ad, x, dy, y=None, dx=None, bias=None, dA=None, dB=None, dM=None, dm=None,
                           dm_r=None, dm_c=None):
        err = ctypes.create_string_buffer(512)
        g = MatGrads(_vp(dA), _vp(dB), _vp(dM), _vp(dm), _vp(dm_r), _vp(dm_c))
        _check(lib().sa3k_linear_mat_fwd_bwd(self._h, w._h, ctypes.byref(ad), _ptr(bias), _ptr(x), _ptr(dy),
                                             x.shape[0], _ptr(y), _ptr(dx), ctypes.byref(g), err, 512), err)

    def linear_bwd(self, w, x, y, dy, dx, ad=None, bias=None, dA=None, dB=None, dm=None, accumulate=False):
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_linear_bwd(self._h, w._h, ctypes.byref(ad) if ad else None, _ptr(bias), _ptr(x),
                                     _ptr(y), _ptr(dy), x.shape[0], _ptr(dx), _ptr(dA), _ptr(dB), _ptr(dm),
                                     1 if accumulate else 0, err, 512), err)

    def linear_fwd_bwd(self, w, x, dy, y, dx, ad=None, bias=None, dA=None, dB=None, dm=None):
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_linear_fwd_bwd(self._h, w._h, ctypes.byref(ad) if ad else None, _ptr(bias), _ptr(x),
                                         _ptr(dy), x.shape[0], _ptr(y), _ptr(dx), _ptr(dA), _ptr(dB), _ptr(dm),
                                         err, 512), err)

    def linear_fwd_bwd_host(self, w, x, dy, y, dx, ad=None, bias=None, dA=None, dB=None, dm=None):
        """All arguments are numpy float32 arrays (host memory); ad holds host pointers."""
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_linear_fwd_bwd_host(self._h, w._h, ctypes.byref(ad) if ad else None, _ptr(bias),
                                              _ptr(x), _ptr(dy), x.shape[0], _ptr(y), _ptr(dx), _ptr(dA),
                                              _ptr(dB), _ptr(dm), err, 512), err)

    def adamw(self, p, g, m, v, hp: AdamWParams, step):
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_adamw(self._h, _ptr(p), _ptr(g), _ptr(m), _ptr(v), p.numel(), ctypes.byref(hp),
                                step, err, 512), err)

    def average_clip_adamw(self, p, g, m, v, count, hp: AdamWParams, step, want_norm=False):
        err = ctypes.create_string_buffer(512)
        norm = ctypes.c_double(0.0)
        _check(lib().sa3k_average_clip_adamw(self._h, _ptr(p), _ptr(g), _ptr(m), _ptr(v), p.numel(), count,
                                             ctypes.byref(hp), step, ctypes.byref(norm) if want_norm else None,
                                             err, 512), err)
        return norm.value if want_norm else None


class Weight:
    def __init__(self, ctx, h, qtype, inn, out):
        self.ctx, self._h, self.qtype, self.inn, self.out = ctx, h, qtype, inn, out
        ctx._own(self)

    def free(self):
        if self._h:
            lib().sa3k_weight_free(self._h)
            self._h = ctypes.c_void_p()

    close = free

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class LoraChain:
    def __init__(self, h):
        self._h = h

    def info(self):
        r, f = ctypes.c_int(), ctypes.c_int()
        lib().sa3k_lora_chain_info(self._h, ctypes.byref(r), ctypes.byref(f))
        return r.value, bool(f.value)

    def free(self):
        if self._h:
            lib().sa3k_lora_chain_free(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class Dit:
    """A DiT training model on a context (sa3k_dit_*): tensors by GGUF name, flat adapter state."""

    def __init__(self, ctx, cfg):
        self.ctx = ctx
        c = DitConfigC(**{k: cfg[k] for k in DIT_INT_FIELDS + DIT_FLOAT_FIELDS}, local_dim=cfg.get("local_dim", 0))
        self._h = ctypes.c_void_p()
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_dit_create(ctx._h, ctypes.byref(c), ctypes.byref(self._h), err, 512), err)
        ctx._own(self)

    def close(self):
        if self._h:
            lib().sa3k_dit_free(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def set_tensor(self, name, qtype, host, ne0, ne1=1):
        import numpy as np
        a = np.ascontiguousarray(host)
        if qtype == "f32" and a.nbytes < 4 * ne0 * max(ne1, 1):
            raise Sa3kError(f"{name}: host buffer holds {a.nbytes} bytes, [{ne1}][{ne0}] f32 needs more")
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_dit_set_tensor(self._h, name.encode(), TYPE_IDS[qtype], a.ctypes.data_as(ctypes.c_void_p),
                                         ne0, ne1, err, 512), err)

    def init_adapters(self, adapter_type, rank, alpha, names):
        arr = (ctypes.c_char_p * len(names))(*[n.encode() for n in names])
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_dit_init_adapters(self._h, adapter_type.encode(), rank, alpha, arr, len(names), err, 512), err)

    def size(self):
        return int(lib().sa3k_dit_adapter_size(self._h))

    def offsets(self, idx):
        a, b, m = ctypes.c_int64(), ctypes.c_int64(), ctypes.c_int64()
        if lib().sa3k_dit_adapter_offsets(self._h, idx, ctypes.byref(a), ctypes.byref(b), ctypes.byref(m)):
            raise Sa3kError("bad target index")
        return a.value, b.value, m.value

    def layout(self, idx):
        """(A, B, row magnitude, column magnitude, M_xs) offsets of target idx, -1 where absent."""
        offs = (ctypes.c_int64 * 5)()
        if lib().sa3k_dit_adapter_layout(self._h, idx, offs):
            raise Sa3kError("bad target index")
        return tuple(int(v) for v in offs)

    def set_xs_bases(self, name, U, V):
        import numpy as np
        U = np.ascontiguousarray(U, np.float32)
        V = np.ascontiguousarray(V, np.float32)
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_dit_set_xs_bases(self._h, name.encode(), _ptr(U), _ptr(V), err, 512), err)

    def copy(self, which, buf, offset=0, count=None, to_model=True):
        """which: 0 params, 1 grads, 2 AdamW m, 3 AdamW v; buf: numpy float32 (host) or torch tensor."""
        n = count if count is not None else (buf.size if hasattr(buf, "size") and not callable(buf.size) else buf.numel())
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_dit_adapter_copy(self._h, which, _ptr(buf), offset, n, 1 if to_model else 0, err, 512), err)

    def buffer_ptr(self, which):
        p = ctypes.c_void_p()
        err = ctypes.create_string_buffer(256)
        _check(lib().sa3k_dit_adapter_buffer(self._h, which, ctypes.byref(p), err, 256), err)
        return p.value

    def save_adapter(self, path):
        """The adapters as the reference's adapter GGUF (loads in its generator)."""
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_dit_save_adapter(self._h, path.encode(), err, 512), err)

    def load_adapter(self, path):
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_dit_load_adapter(self._h, path.encode(), err, 512), err)

    def save_checkpoint(self, adapter_path, state_path, step, epoch=0, next_sample=0, order=(0,), compatibility="",
                        rng=None):
        """Immutable adapter + trainer-state pair; rng: dict of the sampler states (shuffle, crop, cfg, prompt,
        inpaint, diffusion) as strings."""
        rng = rng or {}
        order_arr = (ctypes.c_uint64 * len(order))(*order)
        pr = TrainProgress(epoch, next_sample, order_arr, len(order), compatibility.encode(),
                           *[rng.get(k, "").encode() for k in ("shuffle", "crop", "cfg", "prompt", "inpaint",
                                                               "diffusion")])
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_dit_save_checkpoint(self._h, adapter_path.encode(), state_path.encode(), step,
                                              ctypes.byref(pr), err, 512), err)

    def load_checkpoint(self, adapter_path, state_path):
        """Restores parameters and AdamW moments; returns the step (the rest of the progress is read with
        gguf_get_*)."""
        err = ctypes.create_string_buffer(512)
        st = ctypes.c_int64()
        _check(lib().sa3k_dit_load_checkpoint(self._h, adapter_path.encode(), state_path.encode(), ctypes.byref(st),
                                              err, 512), err)
        return st.value

    def zero_grads(self):
        err = ctypes.create_string_buffer(256)
        _check(lib().sa3k_dit_zero_grads(self._h, err, 256), err)

    def forward_backward(self, B, T, ctx_len, x_t, target, t_feat, cross, glob, loss=None):
        err = ctypes.create_string_buffer(1024)
        _check(lib().sa3k_dit_forward_backward(self._h, B, T, ctx_len, _ptr(x_t), _ptr(target), _ptr(t_feat),
                                               _ptr(cross), _ptr(glob), _ptr(loss), err, 1024), err)

    def forward_backward_inpaint(self, B, T, ctx_len, x_t, target, t_feat, cross, glob, local, loss_weight, loss=None):
        """forward_backward with the inpaint local conditioning [B][T][local_dim] and loss weights [B][T][io]."""
        err = ctypes.create_string_buffer(1024)
        _check(lib().sa3k_dit_forward_backward_inpaint(self._h, B, T, ctx_len, _ptr(x_t), _ptr(target), _ptr(t_feat),
                                                       _ptr(cross), _ptr(glob), _ptr(local), _ptr(loss_weight),
                                                       _ptr(loss), err, 1024), err)

    def dp_apply_adamw(self, comm, samples_per_rank, hp, step, want_norm=False):
        """All-reduce the gradients over comm's ranks, then AdamW with count = samples_per_rank x ranks."""
        err = ctypes.create_string_buffer(512)
        norm = ctypes.c_double(0.0)
        _check(lib().sa3k_dit_dp_apply_adamw(self._h, comm._h, samples_per_rank, ctypes.byref(hp), step,
                                             ctypes.byref(norm) if want_norm else None, err, 512), err)
        return norm.value if want_norm else None

    def apply_adamw(self, count, hp, step, want_norm=False):
        err = ctypes.create_string_buffer(512)
        norm = ctypes.c_double(0.0)
        _check(lib().sa3k_dit_apply_adamw(self._h, count, ctypes.byref(hp), step,
                                          ctypes.byref(norm) if want_norm else None, err, 512), err)
        return norm.value if want_norm else None


# ------------------------------------------------------------------------ data parallel
def dp_unique_id():
    """128 bytes identifying a new NCCL clique (make on one rank, hand to all)."""
    buf = ctypes.create_string_buffer(128)
    err = ctypes.create_string_buffer(512)
    _check(lib().sa3k_dp_unique_id(buf, 128, err, 512), err)
    return buf.raw


class DpComm:
    """A data-parallel communicator of nranks processes, one per GPU (sa3k_dp_comm_*)."""

    def __init__(self, ctx, nranks, rank, unique_id, timeout_s=None):
        """timeout_s: bound on the rendezvous (every rank must join within it; default 300 s)."""
        assert len(unique_id) == 128
        self.ctx = ctx
        self._h = ctypes.c_void_p()
        uid = ctypes.create_string_buffer(bytes(unique_id), 128)
        err = ctypes.create_string_buffer(512)
        if timeout_s is None:
            _check(lib().sa3k_dp_comm_create(ctx._h, nranks, rank, uid, ctypes.byref(self._h), err, 512), err)
        else:
            _check(lib().sa3k_dp_comm_create_timeout(ctx._h, nranks, rank, uid, float(timeout_s),
                                                     ctypes.byref(self._h), err, 512), err)
        self.nranks, self.rank = nranks, rank
        ctx._own(self)

    def allreduce_sum(self, buf, n=None):
        n = buf.numel() if n is None else n
        err = ctypes.create_string_buffer(512)
        _check(lib().sa3k_dp_allreduce_sum(self.ctx._h, self._h, _ptr(buf), n, err, 512), err)

    def allreduce_adamw(self, p, g, m, v, samples_per_rank, hp, step, want_norm=False):
        err = ctypes.create_string_buffer(512)
        norm = ctypes.c_double(0.0)
        _check(lib().sa3k_dp_allreduce_adamw(self.ctx._h, self._h, _ptr(p), _ptr(g), _ptr(m), _ptr(v), p.numel(),
                                             samples_per_rank, ctypes.byref(hp), step,
                                             ctypes.byref(norm) if want_norm else None, err, 512), err)
        return norm.value if want_norm else None

    def close(self):
        if self._h:
            lib().sa3k_dp_comm_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ------------------------------------------------------------------ GGUF adapter / trainer-state files
def adapter_gguf_write(path, adapter_type, rank, alpha, targets):
    """targets: list of (stem, A [rank][in], B [out][rank], m [out] or None), numpy float32."""
    import numpy as np
    n = len(targets)
    arrs = [(np.ascontiguousarray(A, np.float32), np.ascontiguousarray(Bm, np.float32),
             None if m is None else np.ascontiguousarray(m, np.float32)) for _, A, Bm, m in targets]
    stems = (ctypes.c_char_p * n)(*[t[0].encode() for t in targets])
    ins = (ctypes.c_int64 * n)(*[a[0].shape[1] for a in arrs])
    outs = (ctypes.c_int64 * n)(*[a[1].shape[0] for a in arrs])
    Ap = (ctypes.c_void_p * n)(*[a[0].ctypes.data for a in arrs])
    Bp = (ctypes.c_void_p * n)(*[a[1].ctypes.data for a in arrs])
    Mp = (ctypes.c_void_p * n)(*[(a[2].ctypes.data if a[2] is not None else None) for a in arrs])
    err = ctypes.create_string_buffer(512)
    _check(lib().sa3k_adapter_gguf_write(path.encode(), adapter_type.encode(), rank, alpha, n, stems, ins, outs, Ap,
                                         Bp, Mp, err, 512), err)


def gguf_get_string(path, key):
    err = ctypes.create_string_buffer(512)
    n = ctypes.c_int64()
    _check(lib().sa3k_gguf_get_string(path.encode(), key.encode(), None, 0, ctypes.byref(n), err, 512), err)
    buf = ctypes.create_string_buffer(n.value + 1)
    _check(lib().sa3k_gguf_get_string(path.encode(), key.encode(), buf, n.value + 1, None, err, 512), err)
    return buf.raw[:n.value].decode()


def gguf_get_u64(path, key):
    err = ctypes.create_string_buffer(512)
    v = ctypes.c_uint64()
    _check(lib().sa3k_gguf_get_u64(path.encode(), key.encode(), ctypes.byref(v), err, 512), err)
    return v.value


def gguf_get_u64_array(path, key):
    err = ctypes.create_string_buffer(512)
    n = ctypes.c_int64()
    _check(lib().sa3k_gguf_get_u64_array(path.encode(), key.encode(), None, 0, ctypes.byref(n), err, 512), err)
    out = (ctypes.c_uint64 * max(n.value, 1))()
    _check(lib().sa3k_gguf_get_u64_array(path.encode(), key.encode(), out, n.value, ctypes.byref(n), err, 512), err)
    return list(out[:n.value])


def gguf_get_f32(path, name):
    """(values as a flat numpy float32 array, ne tuple with ne[0] innermost)."""
    import numpy as np
    err = ctypes.create_string_buffer(512)
    n = ctypes.c_int64()
    ne = (ctypes.c_int64 * 4)()
    nd = ctypes.c_int()
    _check(lib().sa3k_gguf_get_f32(path.encode(), name.encode(), None, 0, ctypes.byref(n), ne, ctypes.byref(nd), err,
                                   512), err)
    out = np.empty(n.value, np.float32)
    _check(lib().sa3k_gguf_get_f32(path.encode(), name.encode(), out.ctypes.data_as(ctypes.c_void_p), n.value,
                                   ctypes.byref(n), ne, ctypes.byref(nd), err, 512), err)
    return out, tuple(ne[:nd.value])
