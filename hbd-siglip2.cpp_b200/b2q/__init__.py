"""Python binding of libb2q.so (include/b2q.h) — the host side used by tests
and benchmarks.  Device buffers are torch CUDA tensors (torch is plumbing
here: memory, streams, process groups); every computation goes through the
C ABI.  There is no fallback: if the library is missing this module raises.
"""
from __future__ import annotations

import ctypes as C
import os
from pathlib import Path

import numpy as np

PKG = Path(__file__).resolve().parents[1]
LIB_PATH = PKG / "lib" / "libb2q.so"

OK = 0
ERR_INVALID, ERR_SHAPE, ERR_ALIGN, ERR_CUDA, ERR_DEVICE, ERR_NOT_INIT, ERR_NOMEM = -1, -2, -3, -4, -5, -6, -7
OPS_I8, OPS_F16 = 0, 1
EPI_NONE, EPI_BIAS, EPI_BIAS_RESIDUAL, EPI_BIAS_GELU_Q8, EPI_BIAS_F16 = 0, 1, 2, 3, 4

#: every symbol include/b2q.h declares (checked by the CPU test suite)
EXPORTS = [
    "b2q_last_error", "b2q_abi_version", "b2q_launch_count", "b2q_graph_launch_count", "b2q_init", "b2q_tune", "b2q_check_device",
    "b2q_weight_register", "b2q_weight_release", "b2q_weight_shape",
    "b2q_act_bytes", "b2q_act_layout", "b2q_quantize_q8_1", "b2q_ln_quantize_q8_1",
    "b2q_mul_mat_q8_0", "b2q_mul_mat_q8_0_f32", "b2q_mul_mat_q8_0_f32_noalloc", "b2q_block_sums",
    "b2q_attention_scratch_bytes", "b2q_attention",
    "b2q_vision_create", "b2q_vision_destroy", "b2q_vision_set_tensor", "b2q_vision_reserve",
    "b2q_vision_encode", "b2q_vision_encode_host", "b2q_vision_submit_host", "b2q_vision_wait",
    "b2q_vision_wait_submitted",
    "b2q_text_create", "b2q_text_destroy", "b2q_text_set_tensor", "b2q_text_reserve", "b2q_text_encode",
    "b2q_text_encode_host", "b2q_score_scratch_bytes", "b2q_score",
    "b2q_kv_plan", "b2q_qk_norm_rope", "b2q_attention_paged_scratch_bytes", "b2q_attention_paged",
    "b2q_weight_q4_register", "b2q_weight_q4_release", "b2q_mul_vec_q4",
    "b2q_gguf_open", "b2q_gguf_close", "b2q_gguf_n_tensors", "b2q_gguf_tensor", "b2q_gguf_scalar_f32",
    "b2q_vision_load_gguf", "b2q_text_load_gguf",
]


class B2QError(RuntimeError):
    def __init__(self, status: int, msg: str):
        super().__init__(f"b2q status {status}: {msg}")
        self.status = status


class VisionConfig(C.Structure):
    _fields_ = [("hidden", C.c_int32), ("ffn", C.c_int32), ("n_head", C.c_int32), ("n_layer", C.c_int32),
                ("patch_dim", C.c_int32), ("pos_side", C.c_int32), ("eps", C.c_float)]


class TextConfig(C.Structure):
    _fields_ = [("hidden", C.c_int32), ("ffn", C.c_int32), ("n_head", C.c_int32), ("n_layer", C.c_int32),
                ("vocab", C.c_int32), ("n_pos", C.c_int32), ("eps", C.c_float)]


POOL_MEAN, POOL_PROBE = 0, 1
GGML_F32, GGML_Q8_0 = 0, 8
GGML_F16, GGML_Q4_0, GGML_Q4_1, GGML_BF16 = 1, 2, 3, 30


class Epilogue(C.Structure):
    _fields_ = [("kind", C.c_int), ("bias", C.c_void_p), ("residual", C.c_void_p),
                ("act_out", C.c_void_p), ("ld_out", C.c_int64)]


class KvCacheDesc(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("dtype", C.c_int32), ("n_pages", C.c_int32),
                ("page_size", C.c_int32), ("n_kv_head", C.c_int32), ("d_head", C.c_int32),
                ("page_stride", C.c_int64), ("head_stride", C.c_int64), ("token_stride", C.c_int64)]


_lib = None
P, I64 = C.c_void_p, C.c_int64
I32P = C.POINTER(C.c_int32)


def lib():
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise RuntimeError(f"{LIB_PATH} is missing: run __graft_entry__.build() (no CPU fallback exists)")
        L = C.CDLL(str(LIB_PATH))
        L.b2q_last_error.restype = C.c_char_p
        L.b2q_abi_version.restype = C.c_int
        L.b2q_launch_count.restype = C.c_uint64
        L.b2q_graph_launch_count.restype = C.c_uint64
        L.b2q_init.argtypes = [C.c_int, C.c_int]
        L.b2q_check_device.argtypes = [P, C.POINTER(C.c_uint32)]
        L.b2q_tune.argtypes = [C.c_int, I64]
        L.b2q_weight_register.argtypes = [P, I64, I64, I64, C.c_int, P, C.POINTER(P)]
        L.b2q_weight_release.argtypes = [P]
        L.b2q_weight_shape.argtypes = [P, C.POINTER(I64), C.POINTER(I64)]
        L.b2q_act_bytes.argtypes = [I64, I64]
        L.b2q_act_bytes.restype = C.c_size_t
        L.b2q_act_layout.argtypes = [I64, I64] + [C.POINTER(I64)] * 4
        L.b2q_quantize_q8_1.argtypes = [P, I64, I64, I64, P, P]
        L.b2q_ln_quantize_q8_1.argtypes = [P, P, P, C.c_float, I64, I64, P, P, P]
        L.b2q_mul_mat_q8_0.argtypes = [P, P, I64, P, C.POINTER(Epilogue), P]
        L.b2q_mul_mat_q8_0_f32.argtypes = [P, P, I64, I64, P, P, P]
        L.b2q_mul_mat_q8_0_f32_noalloc.argtypes = [P, P, I64, I64, P, P]
        L.b2q_block_sums.argtypes = [P, P, I64, P, P]
        L.b2q_attention_scratch_bytes.argtypes = [I32P, C.c_int32]
        L.b2q_attention_scratch_bytes.restype = C.c_size_t
        L.b2q_attention.argtypes = [P, I64, P, I64, P, I64, I32P, I32P, I32P, I32P, I32P, C.c_int32, C.c_int32,
                                    C.c_int32, P, I64, P, P]
        L.b2q_vision_create.argtypes = [C.POINTER(VisionConfig), C.POINTER(P)]
        L.b2q_vision_destroy.argtypes = [P]
        L.b2q_vision_set_tensor.argtypes = [P, C.c_char_p, C.c_int32, P, I64, I64, P]
        L.b2q_vision_reserve.argtypes = [P, I64, C.c_int32]
        L.b2q_vision_encode.argtypes = [P, P, I32P, C.c_int32, C.c_int32, P, P]
        L.b2q_vision_encode_host.argtypes = [P, P, I32P, C.c_int32, C.c_int32, P, P]
        L.b2q_vision_submit_host.argtypes = [P, P, I32P, C.c_int32, C.c_int32, P, P]
        L.b2q_vision_wait.argtypes = [P, P]
        L.b2q_vision_wait_submitted.argtypes = [P, C.c_int32]
        L.b2q_text_create.argtypes = [C.POINTER(TextConfig), C.POINTER(P)]
        L.b2q_text_destroy.argtypes = [P]
        L.b2q_text_set_tensor.argtypes = [P, C.c_char_p, C.c_int32, P, I64, I64, P]
        L.b2q_text_reserve.argtypes = [P, C.c_int32]
        L.b2q_text_encode.argtypes = [P, P, C.c_int32, P, P]
        L.b2q_text_encode_host.argtypes = [P, P, C.c_int32, P, P]
        L.b2q_score_scratch_bytes.argtypes = [C.c_int32, C.c_int32, C.c_int32]
        L.b2q_score_scratch_bytes.restype = C.c_size_t
        L.b2q_score.argtypes = [P, C.c_int32, P, C.c_int32, C.c_int32, C.c_float, C.c_float, P, P, P, P]
        I32 = C.c_int32
        L.b2q_kv_plan.argtypes = [P, P, I32, I32, P, I32, P, I64, I32, I32, P, P, P, P, P, P]
        L.b2q_qk_norm_rope.argtypes = [P, I32, I64, I64, I32, P, P, C.c_float, P, I32, I32, I32, P, P, P, I64, P, P]
        L.b2q_attention_paged_scratch_bytes.argtypes = [I32, I32, I32]
        L.b2q_attention_paged_scratch_bytes.restype = C.c_size_t
        L.b2q_attention_paged.argtypes = [P, I64, I64, I32, P, P, I64, I32, I32, P, P, C.c_float, I32, P, I32, I64, P,
                                          P, P]
        L.b2q_weight_q4_register.argtypes = [P, I32, I64, I64, I64, C.c_int, P, C.POINTER(P)]
        L.b2q_weight_q4_release.argtypes = [P]
        L.b2q_mul_vec_q4.argtypes = [P, P, I32, I64, I64, I64, P, I32, I64, P, P, P]
        L.b2q_gguf_open.argtypes = [C.c_char_p, C.POINTER(P)]
        L.b2q_gguf_close.argtypes = [P]
        L.b2q_gguf_n_tensors.argtypes = [P]
        L.b2q_gguf_n_tensors.restype = I64
        L.b2q_gguf_tensor.argtypes = [P, I64, C.POINTER(C.c_char_p), C.POINTER(C.c_int32), C.POINTER(C.c_int32),
                                      C.POINTER(I64), C.POINTER(P)]
        L.b2q_gguf_scalar_f32.argtypes = [P, C.c_char_p, C.POINTER(C.c_float)]
        L.b2q_vision_load_gguf.argtypes = [P, P, P]
        L.b2q_text_load_gguf.argtypes = [P, P, P]
        for name in EXPORTS:
            fn = getattr(L, name)
            if name not in ("b2q_last_error", "b2q_abi_version", "b2q_act_bytes", "b2q_attention_scratch_bytes",
                            "b2q_attention_paged_scratch_bytes", "b2q_launch_count", "b2q_graph_launch_count"):
                fn.restype = C.c_int
        _lib = L
    return _lib


def launch_count() -> int:
    return int(lib().b2q_launch_count())


def graph_launch_count() -> int:
    """Tower encodes the library launched as one captured CUDA graph."""
    return int(lib().b2q_graph_launch_count())


def check(status: int):
    if status != OK:
        raise B2QError(status, lib().b2q_last_error().decode())


def _ptr(t) -> int | None:
    if t is None:
        return None
    return t.data_ptr()


def _host_ptr(a):
    """Address of a host buffer: a torch CPU tensor or a numpy array."""
    return a.data_ptr() if hasattr(a, "data_ptr") else a.ctypes.data


def _stream(stream=None):
    import torch
    s = stream if stream is not None else torch.cuda.current_stream()
    return C.c_void_p(s.cuda_stream)


def init(device: int = 0, ops_mode: int = -1):
    check(lib().b2q_init(device, ops_mode))


TUNE_GEMM_BN, TUNE_TIMEOUT_NS, TUNE_ATTN_EXACT, TUNE_TEST_STALL, TUNE_ATTN_KERNEL, TUNE_GEMM_CTAS = 1, 2, 3, 4, 5, 6
TUNE_GRAPHS = 7


def tune(key: int, value: int):
    check(lib().b2q_tune(key, value))


def check_device(stream=None) -> int:
    code = C.c_uint32(0)
    check(lib().b2q_check_device(_stream(stream), C.byref(code)))
    return code.value


class Weight:
    """A registered Q8_0 weight (N rows of K; K-padded tensors pass padded K)."""

    def __init__(self, q8_0, n: int, k: int, row_bytes: int | None = None, stream=None):
        import torch
        row_bytes = row_bytes or (k // 32 * 34)
        handle = C.c_void_p()
        if isinstance(q8_0, np.ndarray):
            buf = np.ascontiguousarray(q8_0)
            check(lib().b2q_weight_register(buf.ctypes.data, n, k, row_bytes, 1, _stream(stream), C.byref(handle)))
        else:
            assert isinstance(q8_0, torch.Tensor) and q8_0.is_cuda
            check(lib().b2q_weight_register(q8_0.data_ptr(), n, k, row_bytes, 0, _stream(stream), C.byref(handle)))
        self.handle = handle
        self.n, self.k = n, k

    def release(self):
        if self.handle:
            lib().b2q_weight_release(self.handle)
            self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.release()
        except Exception:
            pass


def act_layout(m: int, k: int):
    kp, es, off, ld = I64(), I64(), I64(), I64()
    check(lib().b2q_act_layout(m, k, C.byref(kp), C.byref(es), C.byref(off), C.byref(ld)))
    return kp.value, es.value, off.value, ld.value


def act_empty(m: int, k: int):
    """Allocate an activation buffer (uint8 torch tensor, 256-byte aligned)."""
    import torch
    nbytes = int(lib().b2q_act_bytes(m, k))
    if nbytes == 0:
        raise B2QError(ERR_SHAPE, "bad activation shape")
    t = torch.empty(nbytes + 256, dtype=torch.uint8, device="cuda")
    off = (-t.data_ptr()) % 256
    return t[off:off + nbytes]


def act_planes(act, m: int, k: int):
    """Decode an activation buffer -> (int8 values [M][Kp], fp32 scales [M][Kb]) as torch tensors."""
    import torch
    kp, es, off, ld = act_layout(m, k)
    if es == 1:
        q = act[: m * kp].view(torch.int8).view(m, kp)
    else:
        q = act[: m * kp * 2].view(torch.float16).view(m, kp).to(torch.int8)
    d = act[off: off + (kp // 32) * ld * 4].view(torch.float32).view(kp // 32, ld)[:, :m].t()
    return q, d


def quantize_q8_1(x, act, m: int, k: int, ldx: int | None = None, stream=None):
    check(lib().b2q_quantize_q8_1(_ptr(x), m, k, ldx or k, _ptr(act), _stream(stream)))


def ln_quantize(x, w, b, eps: float, m: int, h: int, act, y=None, stream=None):
    check(lib().b2q_ln_quantize_q8_1(_ptr(x), _ptr(w), _ptr(b), eps, m, h, _ptr(act), _ptr(y), _stream(stream)))


def mul_mat(w: Weight, act, m: int, y=None, kind: int = EPI_NONE, bias=None, residual=None, act_out=None,
            ld_out: int = 0, stream=None):
    e = Epilogue(kind, _ptr(bias), _ptr(residual), _ptr(act_out), ld_out)
    check(lib().b2q_mul_mat_q8_0(w.handle, _ptr(act), m, _ptr(y), C.byref(e), _stream(stream)))


def mul_mat_f32(w: Weight, x, m: int, x_cols: int, y, scratch, stream=None):
    check(lib().b2q_mul_mat_q8_0_f32(w.handle, _ptr(x), m, x_cols, _ptr(y), _ptr(scratch), _stream(stream)))


def mul_mat_f32_noalloc(w: Weight, x, m: int, x_cols: int, y, stream=None):
    """ggml_mul_mat without caller scratch: uses the library's fixed device
    array (B2Q_NOALLOC_MAX_SCRATCH_BYTES), for callers that cannot allocate."""
    check(lib().b2q_mul_mat_q8_0_f32_noalloc(w.handle, _ptr(x), m, x_cols, _ptr(y), _stream(stream)))


NOALLOC_MAX_SCRATCH_BYTES = 32 << 20


def block_sums(w: Weight, act, m: int, out, stream=None):
    check(lib().b2q_block_sums(w.handle, _ptr(act), m, _ptr(out), _stream(stream)))


def _host_i32(a):
    arr = np.ascontiguousarray(np.asarray(a, dtype=np.int32))
    return arr, arr.ctypes.data_as(C.POINTER(C.c_int32))


def attention(q, ldq, k, ldk, v, ldv, q_off, q_len, k_off, k_len, o_off, n_head, out, ldo, stream=None):
    """Packed-sequence attention (head_dim 72); q/k/v fp16 torch tensors, out fp32."""
    import torch
    keep = [_host_i32(x) for x in (q_off, q_len, k_off, k_len, o_off)]
    n_seq = len(keep[0][0])
    nbytes = int(lib().b2q_attention_scratch_bytes(keep[1][1], n_seq))
    scratch = torch.empty(max(nbytes, 16), dtype=torch.uint8, device="cuda")
    check(lib().b2q_attention(_ptr(q), ldq, _ptr(k), ldk, _ptr(v), ldv, keep[0][1], keep[1][1], keep[2][1],
                              keep[3][1], keep[4][1], n_seq, n_head, 72, _ptr(out), ldo, _ptr(scratch),
                              _stream(stream)))
    return scratch


class VisionTower:
    """Batched SigLIP2 vision tower (the C++ driver behind b2q_vision_*)."""

    def __init__(self, cfg):
        self.cfg = cfg
        c = VisionConfig(cfg.hidden, cfg.ffn, cfg.n_head, cfg.n_layer, cfg.patch_dim, cfg.pos_side, cfg.eps)
        h = C.c_void_p()
        check(lib().b2q_vision_create(C.byref(c), C.byref(h)))
        self.handle = h

    def set_tensor(self, name: str, arr: np.ndarray, q8_shape=None, stream=None):
        arr = np.ascontiguousarray(arr)
        if q8_shape is not None:
            n, _, kp = q8_shape
            check(lib().b2q_vision_set_tensor(self.handle, name.encode(), GGML_Q8_0, arr.ctypes.data, kp, n,
                                              _stream(stream)))
        else:
            a = np.ascontiguousarray(arr, np.float32)
            ne0 = a.shape[-1]
            ne1 = a.size // ne0
            check(lib().b2q_vision_set_tensor(self.handle, name.encode(), GGML_F32, a.ctypes.data, ne0, ne1,
                                              _stream(stream)))

    def load(self, ck, stream=None):
        for name, arr in ck.tensors.items():
            if not name.startswith("v."):
                continue
            self.set_tensor(name, arr, ck.q8_shapes.get(name), stream)

    def reserve(self, max_tokens: int, max_images: int):
        check(lib().b2q_vision_reserve(self.handle, max_tokens, max_images))

    def load_gguf(self, g: "Gguf", stream=None):
        """Every "v." tensor of an open GGUF file (b2q_vision_load_gguf)."""
        check(lib().b2q_vision_load_gguf(self.handle, g.handle, _stream(stream)))

    def encode(self, patches, grids, pooling=POOL_PROBE, out=None, stream=None):
        """patches: torch CUDA fp32 [T][patch_dim] (images back to back); grids: [(h, w), ...]."""
        import torch
        g, gp = _host_i32(np.asarray(grids, np.int32).reshape(-1))
        n = len(grids)
        if out is None:
            out = torch.empty((n, self.cfg.hidden), dtype=torch.float32, device="cuda")
        check(lib().b2q_vision_encode(self.handle, _ptr(patches), gp, n, pooling, _ptr(out), _stream(stream)))
        return out

    def encode_host(self, patches: np.ndarray, grids, pooling=POOL_PROBE, out: np.ndarray | None = None,
                    stream=None):
        """Host in, host out (patch upload and embedding download included)."""
        g, gp = _host_i32(np.asarray(grids, np.int32).reshape(-1))
        n = len(grids)
        if out is None:
            out = np.empty((n, self.cfg.hidden), np.float32)
        check(lib().b2q_vision_encode_host(self.handle, patches.ctypes.data, gp, n, pooling, out.ctypes.data,
                                           _stream(stream)))
        return out

    def submit_host(self, patches, grids, out, pooling=POOL_PROBE, stream=None):
        """Pipelined host entry point (b2q_vision_submit_host): patches and out
        are pinned host tensors (or any host buffers exposing data_ptr / the
        array interface); returns without waiting, see wait()."""
        g, gp = _host_i32(np.asarray(grids, np.int32).reshape(-1))
        # the last two submissions' buffers stay referenced until their copies have run
        self._keep = (getattr(self, "_keep", ((), ()))[-1], (g, patches, out))
        check(lib().b2q_vision_submit_host(self.handle, _host_ptr(patches), gp, len(grids), pooling, _host_ptr(out),
                                           _stream(stream)))

    def wait(self, stream=None):
        check(lib().b2q_vision_wait(self.handle, _stream(stream)))

    def wait_submitted(self, back=0):
        """Wait for one submission's embeddings: back 0 = the latest, 1 = the one before."""
        check(lib().b2q_vision_wait_submitted(self.handle, back))

    def close(self):
        if self.handle:
            lib().b2q_vision_destroy(self.handle)
            self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class TextTower:
    """Batched SigLIP2 text tower (the C++ driver behind b2q_text_*)."""

    def __init__(self, cfg):
        self.cfg = cfg
        c = TextConfig(cfg.hidden, cfg.ffn, cfg.n_head, cfg.n_layer, cfg.vocab, cfg.n_pos, cfg.eps)
        h = C.c_void_p()
        check(lib().b2q_text_create(C.byref(c), C.byref(h)))
        self.handle = h

    def set_tensor(self, name: str, arr: np.ndarray, q8_shape=None, stream=None):
        arr = np.ascontiguousarray(arr)
        if q8_shape is not None:
            n, _, kp = q8_shape
            check(lib().b2q_text_set_tensor(self.handle, name.encode(), GGML_Q8_0, arr.ctypes.data, kp, n,
                                            _stream(stream)))
        else:
            a = np.ascontiguousarray(arr, np.float32)
            ne0 = a.shape[-1]
            check(lib().b2q_text_set_tensor(self.handle, name.encode(), GGML_F32, a.ctypes.data, ne0, a.size // ne0,
                                            _stream(stream)))

    def load(self, ck, stream=None):
        for name, arr in ck.tensors.items():
            if name.startswith("t."):
                self.set_tensor(name, arr, ck.q8_shapes.get(name), stream)

    def reserve(self, max_prompts: int):
        check(lib().b2q_text_reserve(self.handle, max_prompts))

    def load_gguf(self, g: "Gguf", stream=None):
        """Every "t." tensor of an open GGUF file (b2q_text_load_gguf)."""
        check(lib().b2q_text_load_gguf(self.handle, g.handle, _stream(stream)))

    def encode(self, ids, out=None, stream=None):
        """ids: torch CUDA int32 [n_prompts][n_pos]."""
        import torch
        n = ids.shape[0]
        if out is None:
            out = torch.empty((n, self.cfg.hidden), dtype=torch.float32, device="cuda")
        check(lib().b2q_text_encode(self.handle, _ptr(ids), n, _ptr(out), _stream(stream)))
        return out

    def encode_host(self, ids: np.ndarray, stream=None) -> np.ndarray:
        ids = np.ascontiguousarray(ids, np.int32)
        out = np.empty((ids.shape[0], self.cfg.hidden), np.float32)
        check(lib().b2q_text_encode_host(self.handle, ids.ctypes.data, ids.shape[0], out.ctypes.data,
                                         _stream(stream)))
        return out

    def close(self):
        if self.handle:
            lib().b2q_text_destroy(self.handle)
            self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def score(img, txt, logit_scale: float, logit_bias: float, logits=True, probs=True, stream=None):
    """Image-text sigmoid scores on the device (b2q_score); img [I][H], txt [J][H]
    torch CUDA fp32.  Returns (logits, probs), either None if not requested."""
    import torch
    I, H = img.shape
    J = txt.shape[0]
    scratch = torch.empty(int(lib().b2q_score_scratch_bytes(I, J, H)), dtype=torch.uint8, device="cuda")
    lg = torch.empty((I, J), dtype=torch.float32, device="cuda") if logits else None
    pr = torch.empty((I, J), dtype=torch.float32, device="cuda") if probs else None
    check(lib().b2q_score(_ptr(img), I, _ptr(txt), J, H, float(logit_scale), float(logit_bias), _ptr(lg), _ptr(pr),
                          _ptr(scratch), _stream(stream)))
    return lg, pr


# ---- decoding over a paged key-value cache ---------------------------------
# A decode step calls these once per layer on small tensors, so the host's time
# counts.  Valid calls take one native step (csrc/b2q_host.cpp); what it does not
# accept, or every call where it was not built, goes through the checks here, which
# say what is wrong.
_TYPE_IDS: dict = {}
_INT32 = _F32 = None
_device = _raw_stream = None     # torch's cheap forms: current device, stream of a device
_plan = _rope = _paged = _vec = None
HOST_PATH = PKG / "lib" / "b2q_host.so"


def _not_native(*args):
    return None


_native_plan = _native_rope = _native_paged = _native_vec = _not_native


def _setup():
    """What the calls below look up once."""
    global _INT32, _F32, _device, _raw_stream, _plan, _rope, _paged, _vec
    global _native_plan, _native_rope, _native_paged, _native_vec
    import torch
    _INT32, _F32 = torch.int32, torch.float32
    _TYPE_IDS.update({torch.float32: GGML_F32, torch.float16: GGML_F16, torch.bfloat16: GGML_BF16})
    _device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
    L = lib()
    _plan, _rope, _paged, _vec = L.b2q_kv_plan, L.b2q_qk_norm_rope, L.b2q_attention_paged, L.b2q_mul_vec_q4
    if HOST_PATH.exists():
        from importlib import machinery, util
        spec = util.spec_from_file_location("b2q_host", HOST_PATH, loader=machinery.ExtensionFileLoader(
            "b2q_host", str(HOST_PATH)))
        try:
            native = util.module_from_spec(spec)
            spec.loader.exec_module(native)
        except ImportError as e:     # built against another torch or Python than this one
            import warnings
            warnings.warn(f"{HOST_PATH.name} does not load, decode calls take the slower checks in Python: {e}",
                          RuntimeWarning, stacklevel=3)
            return
        native.setup(*(C.cast(f, C.c_void_p).value for f in (_plan, _rope, _paged, L.b2q_attention_paged_scratch_bytes,
                                                             _vec)))
        _native_plan, _native_rope = native.kv_plan, native.qk_norm_rope
        _native_paged, _native_vec = native.attention_paged, native.mul_vec_q4


def _type_of(t) -> int:
    try:
        return _TYPE_IDS[t.dtype]
    except KeyError:
        if _vec is None:
            _setup()
        if t.dtype not in _TYPE_IDS:
            raise B2QError(ERR_INVALID, f"element type {t.dtype} is not one of float32, float16, bfloat16") from None
        return _TYPE_IDS[t.dtype]


def _require(ok: bool, what: str, status: int = ERR_SHAPE):
    if not ok:
        raise B2QError(status, what)


def _rows(t, width: int, name: str) -> int:
    """Row stride of a [rows][width] tensor whose columns are contiguous."""
    shape = t.shape
    if len(shape) != 2 or shape[1] != width:
        raise B2QError(ERR_SHAPE, f"{name} must be [rows][{width}]")
    if t.is_contiguous():
        return width
    ld, step = t.stride()
    if step != 1 and width > 1:
        raise B2QError(ERR_SHAPE, f"{name} must have contiguous columns")
    return ld if shape[0] > 1 else width


def _refuse_device(dev, *tensors):
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise B2QError(ERR_INVALID, f"a tensor on {t.device}, the current device is cuda:{dev}")


def _i32(t, n, name: str) -> int:
    """Address of a contiguous int32 tensor of n entries (None = any number)."""
    if t.dtype is not _INT32:
        raise B2QError(ERR_INVALID, f"{name} must be int32")
    if not t.is_contiguous() or (n is not None and t.numel() != n):
        raise B2QError(ERR_SHAPE, f"{name} must be contiguous with {n} entries")
    return t.data_ptr()


def _f32(t, n: int, name: str):
    """Address of a contiguous fp32 tensor of n entries, None for None."""
    if t is None:
        return None
    if _type_of(t) != GGML_F32 or not t.is_contiguous() or t.numel() != n:
        raise B2QError(ERR_SHAPE, f"{name} must be fp32 with {n} entries")
    return t.data_ptr()


def _table(t):
    """(address, row stride, entries of a row, rows) of a block table."""
    if t.dtype is not _INT32:
        raise B2QError(ERR_INVALID, "block_table must be int32")
    shape = t.shape
    if len(shape) != 2:
        raise B2QError(ERR_SHAPE, "block_table must be [requests][max_blocks]")
    width = shape[1]
    return t.data_ptr(), width if t.is_contiguous() else _rows(t, width, "block_table"), width, shape[0]


class KVCache:
    """A layer's paged keys and values: k, v of shape [n_pages][n_kv_head]
    [page_size][d_head] (fp16 or bf16), in any order of the first three
    dimensions (a permuted view is described by its strides)."""

    def __init__(self, k, v):
        _require(k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype
                 and all(a == b or n == 1 for n, a, b in zip(k.shape, k.stride(), v.stride())),
                 "k and v must be alike, [n_pages][n_kv_head][page_size][d_head]")
        _require(k.device == v.device, f"k on {k.device}, v on {v.device}", ERR_INVALID)
        _require(k.stride(3) == 1 or k.shape[3] == 1, "the elements of a head must be contiguous")
        # (to the library a stride of 0 means the contiguous order)
        _require(all(st or n <= 1 for n, st in zip(k.shape, k.stride())), "k and v must not be expanded")
        self.k, self.v = k, v
        self.n_pages, self.n_kv_head, self.page_size, self.d_head = k.shape
        self.dtype, self.device = k.dtype, k.get_device()
        # a dimension of one entry may have any stride: none is passed on
        strides = [0 if n == 1 else st for n, st in zip(k.shape[:3], k.stride())]
        self.desc = KvCacheDesc(k.data_ptr(), v.data_ptr(), _type_of(k), self.n_pages, self.page_size, self.n_kv_head,
                                self.d_head, *strides)
        self.ref = C.addressof(self.desc)
        self.scratch_bytes: dict[int, int] = {}   # attention_paged scratch by n_head


def kv_plan(ctx_len, new_len, page_size: int, free_pages, block_table, seq_of, pos, slot, kv_len, counts, stream=None):
    """Block tables, positions and cache slots of a step (b2q_kv_plan).
    ctx_len, new_len: int32 [n_seq]; block_table: int32 [n_seq][max_blocks],
    entered in place; seq_of, pos, slot, kv_len: int32 [max_tokens] and counts
    int32 [2], written."""
    status = _native_plan(ctx_len, new_len, page_size, free_pages, block_table, seq_of, pos, slot, kv_len, counts,
                          stream)
    if status is not None:
        return check(status) if status else None
    if _plan is None:
        _setup()
    n, rows, i32, dev = ctx_len.numel(), seq_of.numel(), _INT32, _device()
    table, stride, width, requests = _table(block_table)
    if not (requests == n == new_len.numel() and rows == pos.numel() == slot.numel() == kv_len.numel()
            and counts.numel() == 2 and ctx_len.is_contiguous() and new_len.is_contiguous()
            and free_pages.is_contiguous() and seq_of.is_contiguous() and pos.is_contiguous()
            and slot.is_contiguous() and kv_len.is_contiguous() and counts.is_contiguous()
            and ctx_len.dtype is i32 and new_len.dtype is i32 and free_pages.dtype is i32 and seq_of.dtype is i32
            and pos.dtype is i32 and slot.dtype is i32 and kv_len.dtype is i32 and counts.dtype is i32):
        _require(requests == n, "block_table must be [n_seq][max_blocks]")
        for name, t, k in (("ctx_len", ctx_len, n), ("new_len", new_len, n), ("free_pages", free_pages, None),
                           ("seq_of", seq_of, rows), ("pos", pos, rows), ("slot", slot, rows),
                           ("kv_len", kv_len, rows), ("counts", counts, 2)):
            _i32(t, k, name)
    if not (dev == ctx_len.get_device() == new_len.get_device() == free_pages.get_device() == block_table.get_device()
            == seq_of.get_device() == pos.get_device() == slot.get_device() == kv_len.get_device()
            == counts.get_device()):
        _refuse_device(dev, ctx_len, new_len, free_pages, block_table, seq_of, pos, slot, kv_len, counts)
    status = _plan(ctx_len.data_ptr(), new_len.data_ptr(), n, page_size, free_pages.data_ptr(), free_pages.numel(),
                   table, stride, width, rows, seq_of.data_ptr(), pos.data_ptr(), slot.data_ptr(), kv_len.data_ptr(),
                   counts.data_ptr(), _raw_stream(dev) if stream is None else stream.cuda_stream)
    if status:
        check(status)


def rope_table(n_pos: int, rot_dim: int, theta: float = 10000.0, device="cuda"):
    """The rotation table that qk_norm_rope reads: fp32 [n_pos][rot_dim], the
    cosines of pos * theta^(-2i / rot_dim), then the sines (angles in double)."""
    import torch
    inv = theta ** (-2.0 * torch.arange(rot_dim // 2, dtype=torch.float64, device=device) / max(rot_dim, 1))
    ang = torch.arange(n_pos, dtype=torch.float64, device=device)[:, None] * inv[None]
    return torch.cat([ang.cos(), ang.sin()], 1).float().contiguous()


def qk_norm_rope(qkv, n_head: int, cache: KVCache, q_out, pos, slot, q_weight=None, k_weight=None, eps: float = 1e-6,
                 rope=None, interleaved: bool = False, stream=None):
    """Norm and rotation of the rows' query and key heads, keys and values to
    their cache slots (b2q_qk_norm_rope).  qkv: [rows][(n_head + 2 n_kv_head)
    d_head]; q_out: [rows][n_head d_head] of the cache's type; pos, slot: int32
    [rows]; rope: fp32 [n_pos][rot_dim] (see rope_table)."""
    status = _native_rope(qkv, n_head, cache.ref, cache.device, q_out, pos, slot, q_weight, k_weight, eps, rope,
                          interleaved, stream)
    if status is not None:
        return check(status) if status else None
    if _rope is None:
        _setup()
    d, dev = cache.d_head, _device()
    ld = _rows(qkv, (n_head + 2 * cache.n_kv_head) * d, "qkv")
    ldq = _rows(q_out, n_head * d, "q_out")
    rows = qkv.shape[0]
    if q_out.shape[0] != rows or q_out.dtype is not cache.dtype:
        raise B2QError(ERR_SHAPE, "q_out must have qkv's rows and the cache's type")
    n_pos, rot, table = 0, 0, None
    if rope is not None:
        if rope.dim() != 2 or not rope.is_contiguous() or rope.dtype is not _F32:
            raise B2QError(ERR_SHAPE, "rope must be fp32 [n_pos][rot_dim]")
        n_pos, rot = rope.shape
        if rot:
            table = rope.data_ptr()
    if not (dev == qkv.get_device() == q_out.get_device() == pos.get_device() == slot.get_device() == cache.device
            and (rope is None or rope.get_device() == dev) and (q_weight is None or q_weight.get_device() == dev)
            and (k_weight is None or k_weight.get_device() == dev)):
        _refuse_device(dev, qkv, q_out, pos, slot, cache.k, rope, q_weight, k_weight)
    status = _rope(qkv.data_ptr(), _type_of(qkv), ld, rows, n_head, _f32(q_weight, d, "q_weight"),
                   _f32(k_weight, d, "k_weight"), eps, table, n_pos, rot, interleaved, _i32(pos, rows, "pos"),
                   _i32(slot, rows, "slot"), q_out.data_ptr(), ldq, cache.ref,
                   _raw_stream(dev) if stream is None else stream.cuda_stream)
    if status:
        check(status)


def _paged_scratch_bytes(n_head: int, cache: KVCache) -> int:
    n = cache.scratch_bytes.get(n_head)
    if n is None:
        n = int(lib().b2q_attention_paged_scratch_bytes(n_head, cache.n_kv_head, cache.d_head))
        _require(n > 0, "n_head must be a multiple of n_kv_head")
        cache.scratch_bytes[n_head] = n
    return n


def attention_paged_scratch(n_head: int, cache: KVCache):
    """Zeroed scratch for attention_paged with this cache (one per stream)."""
    import torch
    return torch.zeros(_paged_scratch_bytes(n_head, cache), dtype=torch.uint8, device=cache.k.device)


def attention_paged(q, cache: KVCache, block_table, kv_len, out, scratch, seq_of=None, scale: float | None = None,
                    window: int = 0, lse=None, stream=None):
    """Attention of each row's token over its request's cached keys
    (b2q_attention_paged).  q: [rows][n_head d_head] of the cache's type; out
    the same shape, fp32 or the cache's type; block_table: int32 [requests]
    [max_blocks]; kv_len (and seq_of): int32 [rows]; lse: fp32 [rows][n_head]."""
    status = _native_paged(q, cache.ref, cache.device, block_table, kv_len, out, scratch, seq_of, scale, window, lse,
                           stream)
    if status is not None:
        return check(status) if status else None
    if _paged is None:
        _setup()
    d, dev, shape = cache.d_head, _device(), q.shape
    if len(shape) != 2 or out.shape != shape or q.dtype is not cache.dtype:
        raise B2QError(ERR_SHAPE, "q and out must be [rows][n_head d_head], q of the cache's type")
    rows, width = shape
    n_head = width // d
    ldq, ldo = _rows(q, n_head * d, "q"), _rows(out, width, "out")
    if scratch.numel() < _paged_scratch_bytes(n_head, cache) or not scratch.is_contiguous():
        raise B2QError(ERR_SHAPE, "scratch smaller than attention_paged_scratch, or not contiguous")
    table, stride, blocks, requests = _table(block_table)
    if not (dev == q.get_device() == cache.device == block_table.get_device() == kv_len.get_device()
            == out.get_device() == scratch.get_device() and (seq_of is None or seq_of.get_device() == dev)
            and (lse is None or lse.get_device() == dev)):
        _refuse_device(dev, q, cache.k, block_table, kv_len, out, scratch, seq_of, lse)
    status = _paged(q.data_ptr(), ldq, rows, n_head, cache.ref, table, stride, blocks, requests,
                    None if seq_of is None else _i32(seq_of, rows, "seq_of"), _i32(kv_len, rows, "kv_len"),
                    d ** -0.5 if scale is None else scale, window, out.data_ptr(), _type_of(out), ldo,
                    _f32(lse, rows * n_head, "lse"), scratch.data_ptr(),
                    _raw_stream(dev) if stream is None else stream.cuda_stream)
    if status:
        check(status)


class WeightQ4:
    """A registered ggml Q4_0 / Q4_1 weight (N rows of K): a numpy array or a
    CUDA tensor of its blocks' bytes, rows row_bytes apart."""

    def __init__(self, blocks, n: int, k: int, ggml_type: int = GGML_Q4_0, row_bytes: int | None = None, stream=None):
        self.handle = C.c_void_p()
        row_bytes = row_bytes or k // 32 * (18 if ggml_type == GGML_Q4_0 else 20)
        host = isinstance(blocks, np.ndarray)
        buf = np.ascontiguousarray(blocks) if host else blocks
        size = buf.nbytes if host else buf.numel() * buf.element_size()
        _require(size >= n * row_bytes and (host or (buf.is_cuda and buf.is_contiguous())),
                 "blocks must be contiguous and hold n rows")
        if not host:
            if _device is None:
                _setup()
            _refuse_device(_device(), buf)
        check(lib().b2q_weight_q4_register(buf.ctypes.data if host else buf.data_ptr(), ggml_type, n, k, row_bytes,
                                           int(host), _stream(stream), C.byref(self.handle)))
        self.n, self.k, self.ggml_type = n, k, ggml_type

    def release(self):
        if self.handle:
            lib().b2q_weight_q4_release(self.handle)
            self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.release()
        except Exception:
            pass


def mul_vec_q4(w: WeightQ4, x, m: int, y, bias=None, residual=None, stream=None):
    """y[m][n] = x @ w^T (+ bias) (+ residual) for few rows (b2q_mul_vec_q4).
    x: [m][x_cols] fp32, fp16 or bf16 (x_cols rounds up to the weight's K); y:
    [m][n] fp32 or x's type; bias fp32 [n]; residual fp32 like y."""
    status = _native_vec(w.handle.value, w.n, x, m, y, bias, residual, stream)
    if status is not None:
        return check(status) if status else None
    if _vec is None:
        _setup()
    n, dev, shape = w.n, _device(), x.shape
    if len(shape) != 2:
        raise B2QError(ERR_SHAPE, "x must be [m][x_cols]")
    x_rows, x_cols = shape
    ldx, ldy = _rows(x, x_cols, "x"), _rows(y, n, "y")
    if x_rows < m or y.shape[0] < m:
        raise B2QError(ERR_SHAPE, "x and y need m rows")
    res = None
    if residual is not None:
        if residual.dtype is not _F32 or residual.shape != y.shape or _rows(residual, n, "residual") != ldy:
            raise B2QError(ERR_SHAPE, "residual must be fp32 with y's rows and stride")
        res = residual.data_ptr()
    if not (dev == x.get_device() == y.get_device() and (bias is None or bias.get_device() == dev)
            and (residual is None or residual.get_device() == dev)):
        _refuse_device(dev, x, y, bias, residual)
    status = _vec(w.handle, x.data_ptr(), _type_of(x), m, x_cols, ldx, y.data_ptr(), _type_of(y), ldy,
                  _f32(bias, n, "bias"), res, _raw_stream(dev) if stream is None else stream.cuda_stream)
    if status:
        check(status)


class Gguf:
    """A GGUF checkpoint mapped by the library (b2q_gguf_*)."""

    def __init__(self, path):
        h = C.c_void_p()
        check(lib().b2q_gguf_open(str(path).encode(), C.byref(h)))
        self.handle = h

    def tensors(self):
        """[(name, ggml_type, ne tuple, data address)] in file order."""
        out = []
        for i in range(int(lib().b2q_gguf_n_tensors(self.handle))):
            name, typ, nd = C.c_char_p(), C.c_int32(), C.c_int32()
            ne = (I64 * 4)()
            data = C.c_void_p()
            check(lib().b2q_gguf_tensor(self.handle, i, C.byref(name), C.byref(typ), C.byref(nd), ne, C.byref(data)))
            out.append((name.value.decode(), typ.value, tuple(ne[: nd.value]), data.value))
        return out

    def scalar(self, name: str) -> float:
        v = C.c_float()
        check(lib().b2q_gguf_scalar_f32(self.handle, name.encode(), C.byref(v)))
        return v.value

    def close(self):
        if self.handle:
            lib().b2q_gguf_close(self.handle)
            self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
