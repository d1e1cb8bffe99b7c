"""Python binding of the B200 GPT-2 engine's C ABI (include/gpt2b200.h).

A thin ctypes layer over ``libgpt2b200.so`` (built in-tree by the package
Makefile / ``__graft_entry__.build()``).  The library is mapped on the first
call into it (or by ``load()``), so that importing the package's pure-Python
helpers (``synth``, ``replicas``) maps no engine code.  There is no fallback:
that first call raises ``ImportError`` if the library is missing, and every
call raises ``G2Error`` on a non-zero status.
"""
from __future__ import annotations

import ctypes as C
import os

import numpy as np

PKG_DIR = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
# G2_LIB selects another build of the same ABI, e.g. the bounds-checked
# libgpt2b200_check.so (`make -C gpt2-opencl-1.1_b200 check`).
LIB_PATH = os.environ.get("G2_LIB") or os.path.join(PKG_DIR, "libgpt2b200.so")

G2_F32, G2_F16 = 0, 1
G2_KV_I8, G2_KV_E4M3 = 0, 1
MASKED = -1e30   # G2_MASKED
EOS = 50256
ERRORS = {-1: "ARG", -2: "IO", -3: "FORMAT", -4: "CUDA", -5: "OOM", -6: "RANGE", -7: "STATE", -8: "TIMEOUT"}


class G2Error(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"G2_ERR_{ERRORS.get(code, code)} ({code}): {msg}")
        self.code = code


class Config(C.Structure):
    _fields_ = [("n_layer", C.c_int), ("n_embd", C.c_int), ("n_head", C.c_int), ("n_ctx", C.c_int),
                ("vocab_size", C.c_int), ("ffn_dim", C.c_int), ("padded_vocab", C.c_int), ("dtype", C.c_int),
                ("max_batch", C.c_int), ("device", C.c_int), ("weight_bytes", C.c_size_t),
                ("device_bytes", C.c_size_t), ("persistent", C.c_int)]


class KV8(C.Structure):
    """g2_kv8: a paged cache of 8-bit codes (make one with kv8_cache)."""
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p),
                ("n_pages", C.c_int), ("n_kv_head", C.c_int), ("page_size", C.c_int), ("head_dim", C.c_int),
                ("format", C.c_int)]


class LogitRules(C.Structure):
    """g2_logit_rules (make one with logit_rules)."""
    _fields_ = [("ctx", C.c_void_p), ("ctx_start", C.c_void_p), ("n_prompt", C.c_void_p), ("n_ctx", C.c_int),
                ("rep_penalty", C.c_void_p), ("presence", C.c_void_p), ("frequency", C.c_void_p),
                ("bias_ids", C.c_void_p), ("bias", C.c_void_p), ("bias_start", C.c_void_p), ("n_bias", C.c_int),
                ("mask", C.c_void_p), ("mask_stride", C.c_int)]


def _load():
    if not os.path.exists(LIB_PATH):
        raise ImportError(f"{LIB_PATH} is missing: build it with `make -C {PKG_DIR}` "
                          "or __graft_entry__.build()")
    L = C.CDLL(LIB_PATH)
    vp, ip, fp = C.c_void_p, C.POINTER(C.c_int), C.POINTER(C.c_float)
    L.g2_last_error.restype = C.c_char_p
    L.g2_open.argtypes = [C.c_char_p, C.c_int, C.c_int, C.c_int, C.POINTER(vp)]
    L.g2_close.argtypes = [vp]
    L.g2_get_config.argtypes = [vp, C.POINTER(Config)]
    L.g2_prefill.argtypes = [vp, C.c_int, ip, C.c_int]
    L.g2_decode.argtypes = [vp, C.c_int, C.c_int, C.c_int]
    L.g2_decode_batch.argtypes = [vp, C.c_int, ip, ip, ip]
    L.g2_decode_batch_rows.argtypes = [vp, C.c_int, ip, ip, ip, vp]
    L.g2_lm_head_rows.argtypes = [vp, C.c_int, vp, C.c_int, C.c_int, vp, vp]
    L.g2_logits.argtypes = [vp, C.c_int, fp, C.c_int]
    L.g2_argmax.argtypes = [vp, C.c_int, C.c_int, ip, fp]
    L.g2_topk.argtypes = [vp, C.c_int, C.c_int, fp, ip]
    L.g2_sample.argtypes = [fp, C.c_int, ip, C.c_int, C.c_int, C.c_float, C.c_int, C.c_float, ip]
    L.g2_sample_device.argtypes = [vp, C.c_int, ip, C.c_int, C.c_int, C.c_float, C.c_int, C.c_float, C.c_double, ip]
    L.g2_tokenizer_load.argtypes = [C.c_char_p, C.POINTER(vp)]
    L.g2_tokenizer_free.argtypes = [vp]
    L.g2_tokenizer_free.restype = None
    L.g2_tokenizer_vocab_size.argtypes = [vp]
    L.g2_tok_encode.argtypes = [vp, C.c_char_p, ip, C.c_int]
    L.g2_tok_decode.argtypes = [vp, ip, C.c_int, C.c_char_p, C.c_int]
    L.g2_generate.argtypes = [vp, C.c_int, ip, C.c_int, C.c_int, C.c_int, ip]
    L.g2_generate_batch.argtypes = [vp, C.c_int, ip, ip, ip, C.c_int, ip]
    L.g2_synchronize.argtypes = [vp]
    L.g2_last_timing.argtypes = [vp, fp, fp, ip]
    L.g2_launch_count.argtypes = [vp]
    L.g2_launch_count.restype = C.c_longlong
    L.g2k_matvec_workspace.argtypes = [C.c_int, C.c_int]
    L.g2k_matvec_workspace.restype = C.c_size_t
    L.g2k_matvec.argtypes = [vp, vp, vp, vp, vp, C.c_int, C.c_int, C.c_int, vp, vp, vp, C.c_size_t, vp]
    L.g2k_matvec_noalloc.argtypes = [vp, vp, vp, vp, vp, C.c_int, C.c_int, C.c_int, vp, vp, vp]
    L.g2k_matmul.argtypes = [vp, vp, vp, vp, vp, C.c_int, C.c_int, C.c_int, C.c_int, vp]
    L.g2k_matmul_tc_workspace.argtypes = [C.c_int, C.c_int, C.c_int, C.c_int]
    L.g2k_matmul_tc_workspace.restype = C.c_size_t
    L.g2k_matmul_tc.argtypes = [vp, vp, vp, vp, vp, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, vp, C.c_size_t, vp]
    L.g2k_layernorm.argtypes = [vp, vp, vp, vp, C.c_int, C.c_int, vp]
    L.g2k_attention_workspace.argtypes = [C.c_int, C.c_int]
    L.g2k_attention_workspace.restype = C.c_size_t
    L.g2k_attention.argtypes = [vp, vp, vp, vp, C.c_int, C.c_int, C.c_int, vp, C.c_size_t, vp]
    L.g2k_topk.argtypes = [vp, C.c_int, C.c_int, vp, vp, vp]
    i, ll, sz = C.c_int, C.c_longlong, C.c_size_t
    L.g2k_q4_bytes.argtypes = [i, i, i]
    L.g2k_q4_bytes.restype = sz
    L.g2k_q4_pack.argtypes = [vp, i, i, vp, i, i, i, vp]
    L.g2k_q4_unpack.argtypes = [vp, vp, i, i, i, vp]
    L.g2k_matvec_q4.argtypes = [vp, vp, vp, vp, vp, i, i, i, i, i, i, vp, vp, vp]
    L.g2k_kv8_append.argtypes = [vp, vp, vp, i, ll, i, i, vp, vp, i, vp, i, vp, vp]
    L.g2k_kv8_gather.argtypes = [vp, vp, vp, i, ll, i, i, vp, vp, i, vp, i, vp, vp]
    L.g2k_kv8_attention_workspace.argtypes = [vp, i, i, i]
    L.g2k_kv8_attention_workspace.restype = sz
    L.g2k_kv8_attention.argtypes = [vp, vp, ll, vp, ll, i, i, C.c_float, i, i, vp, vp, i, vp, i, vp, sz, vp, vp]
    L.g2k_process_logits.argtypes = [vp, ll, vp, ll, i, i, vp, vp]
    L.g2_process_logits.argtypes = [vp, i, vp]
    return L


class _Lib:
    """The engine library, mapped on first attribute access."""

    def __init__(self):
        self._L = None

    def __getattr__(self, name):
        if self._L is None:
            self._L = _load()
        f = getattr(self._L, name)
        setattr(self, name, f)   # found without this call from now on
        return f


lib = _Lib()


def load():
    """Map libgpt2b200.so now (raises ImportError if it is missing)."""
    lib.g2_last_error
    return lib._L


def check(rc: int) -> int:
    if rc < 0:
        raise G2Error(rc, lib.g2_last_error().decode(errors="replace"))
    return rc


def _i32(a):
    a = np.ascontiguousarray(a, dtype=np.int32)
    return a, a.ctypes.data_as(C.POINTER(C.c_int))


class Engine:
    """One GPT-2 model on one GPU (g2_open ... g2_close)."""

    def __init__(self, model_dir: str, device: int = 0, max_batch: int = 1, dtype: int = G2_F32):
        self.h = C.c_void_p()
        check(lib.g2_open(model_dir.encode(), device, max_batch, dtype, C.byref(self.h)))
        self.cfg = Config()
        check(lib.g2_get_config(self.h, C.byref(self.cfg)))

    def close(self):
        if self.h:
            check(lib.g2_close(self.h))
            self.h = None

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def prefill(self, ids, slot: int = 0):
        a, p = _i32(ids)
        check(lib.g2_prefill(self.h, slot, p, len(a)))

    def decode(self, token: int, pos: int, slot: int = 0):
        check(lib.g2_decode(self.h, slot, int(token), int(pos)))

    def decode_batch(self, slots, tokens, pos):
        s, sp = _i32(slots)
        t, tp = _i32(tokens)
        q, qp = _i32(pos)
        check(lib.g2_decode_batch(self.h, len(s), sp, tp, qp))

    def logits(self, slot: int = 0, n: int = None) -> np.ndarray:
        n = self.cfg.padded_vocab if n is None else n
        out = np.zeros(n, np.float32)
        check(lib.g2_logits(self.h, slot, out.ctypes.data_as(C.POINTER(C.c_float)), n))
        return out

    def argmax(self, slot: int = 0, forbid_eos: bool = False):
        t, v = C.c_int(), C.c_float()
        check(lib.g2_argmax(self.h, slot, int(forbid_eos), C.byref(t), C.byref(v)))
        return t.value, v.value

    def topk(self, k: int, slot: int = 0):
        """The k largest logits of `slot` (device): (values [k] decreasing,
        token ids [k]), equal values by increasing id."""
        vals, ids = np.zeros(k, np.float32), np.zeros(k, np.int32)
        check(lib.g2_topk(self.h, slot, k, vals.ctypes.data_as(C.POINTER(C.c_float)),
                          ids.ctypes.data_as(C.POINTER(C.c_int))))
        return vals, ids

    def sample_device(self, context, forbid_eos: bool = False, temperature: float = 0.0, top_k: int = 0,
                      rep_penalty: float = 1.0, u: float = 0.0, slot: int = 0) -> int:
        """sample_next_token on the device with the uniform draw `u` in [0, 1)."""
        a, p = _i32(context)
        t = C.c_int()
        check(lib.g2_sample_device(self.h, slot, p, len(a), int(forbid_eos), temperature, top_k, rep_penalty, u,
                                   C.byref(t)))
        return t.value

    def process_logits(self, context=(), n_prompt: int = 0, rep_penalty: float = 1.0, presence: float = 0.0,
                       frequency: float = 0.0, bias=None, allowed=None, slot: int = 0):
        """The rules of g2_process_logits on the logits of `slot`, in place: penalties over the ids of
        `context` (`presence` and `frequency` over those after the first `n_prompt`), `bias` as a dict
        of id -> value, and `allowed` as the ids or a truth value per id that stay possible."""
        V = self.cfg.vocab_size
        ctx = np.ascontiguousarray(context, np.int32)
        ids = np.ascontiguousarray(list(bias or ()), np.int32)
        val = np.ascontiguousarray(list((bias or {}).values()), np.float32)
        one = np.array([rep_penalty, presence, frequency], np.float32)
        n = np.array([n_prompt], np.int32)
        r = LogitRules(ctx=ctx.ctypes.data, n_ctx=ctx.size, n_prompt=n.ctypes.data, rep_penalty=one[0:].ctypes.data,
                       presence=one[1:].ctypes.data, frequency=one[2:].ctypes.data, bias_ids=ids.ctypes.data,
                       bias=val.ctypes.data, n_bias=ids.size)
        if allowed is not None:
            a = np.asarray(allowed)
            ok = np.zeros(-(-V // 32) * 32, bool)
            if a.dtype == bool:
                if a.shape != (V,):
                    raise G2Error(-1, f"allowed has {a.shape} truth values, not one for each of {V} ids")
                ok[:V] = a
            else:
                ok[a.astype(np.int64)[(a >= 0) & (a < V)]] = True
            words = np.packbits(ok, bitorder="little").view("<u4")
            r.mask = words.ctypes.data
        check(lib.g2_process_logits(self.h, slot, C.byref(r)))

    def generate(self, prompt, n_new: int, min_new: int = None, slot: int = 0) -> np.ndarray:
        a, p = _i32(prompt)
        out = np.zeros(n_new, np.int32)
        n = check(lib.g2_generate(self.h, slot, p, len(a), n_new, n_new if min_new is None else min_new,
                                  out.ctypes.data_as(C.POINTER(C.c_int))))
        return out[:n]

    def generate_batch(self, prompts, n_new: int, slots=None) -> np.ndarray:
        slots = list(range(len(prompts))) if slots is None else slots
        s, sp = _i32(slots)
        lens, lp = _i32([len(x) for x in prompts])
        flat, fp_ = _i32(np.concatenate([np.asarray(x, np.int32) for x in prompts]))
        out = np.zeros((len(prompts), n_new), np.int32)
        check(lib.g2_generate_batch(self.h, len(s), sp, fp_, lp, n_new, out.ctypes.data_as(C.POINTER(C.c_int))))
        return out

    def decode_batch_rows(self, slots, tokens, pos, rows):
        """One decode step of several sequences without the LM head; the final
        LayerNorm of each row into `rows` (a device tensor [n, n_embd], fp32)."""
        s, sp = _i32(slots)
        t, tp = _i32(tokens)
        q, qp = _i32(pos)
        check(lib.g2_decode_batch_rows(self.h, len(s), sp, tp, qp, _ptr(rows)))

    def lm_head_rows(self, rows, nrows: int, v0: int, v1: int, best_value, best_index):
        """LM head over vocabulary rows [v0, v1) for `nrows` normalised rows (device
        tensors): each row's first maximum there and its vocabulary index."""
        check(lib.g2_lm_head_rows(self.h, nrows, _ptr(rows), v0, v1, _ptr(best_value), _ptr(best_index)))

    def synchronize(self):
        check(lib.g2_synchronize(self.h))

    def last_timing(self):
        a, b, n = C.c_float(), C.c_float(), C.c_int()
        check(lib.g2_last_timing(self.h, C.byref(a), C.byref(b), C.byref(n)))
        return a.value, b.value, n.value

    def launch_count(self) -> int:
        return lib.g2_launch_count(self.h)


def sample(logits, ctx, forbid_eos=False, temperature=0.0, top_k=40, rep_penalty=1.0, vocab_size=None) -> int:
    """g2_sample: main.c:1872 semantics on host logits."""
    lg = np.ascontiguousarray(logits, dtype=np.float32)
    c, cp = _i32(ctx)
    out = C.c_int()
    check(lib.g2_sample(lg.ctypes.data_as(C.POINTER(C.c_float)), len(lg) if vocab_size is None else vocab_size,
                        cp, len(c), int(forbid_eos), temperature, top_k, rep_penalty, C.byref(out)))
    return out.value


class Tokenizer:
    """GPT-2 byte-level BPE (g2_tokenizer_*; tokenizer.c semantics) from vocab.json + merges.txt."""

    def __init__(self, directory: str):
        self.h = C.c_void_p()
        rc = lib.g2_tokenizer_load(directory.encode(), C.byref(self.h))
        if rc < 0:
            raise G2Error(rc, f"cannot load vocab.json / merges.txt from {directory}")

    def close(self):
        if self.h:
            lib.g2_tokenizer_free(self.h)
            self.h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def vocab_size(self) -> int:
        return lib.g2_tokenizer_vocab_size(self.h)

    def encode(self, text, max_ids: int = None) -> list:
        b = text.encode() if isinstance(text, str) else bytes(text)
        cap = max_ids if max_ids is not None else len(b) + 1
        out = (C.c_int * max(cap, 1))()
        n = check(lib.g2_tok_encode(self.h, b, out, max(cap, 1)))
        return list(out[:n])

    def decode(self, ids, max_bytes: int = None) -> bytes:
        a, p = _i32(ids)
        cap = max_bytes if max_bytes is not None else 16 * len(a) + 1
        buf = C.create_string_buffer(max(cap, 1))
        n = check(lib.g2_tok_decode(self.h, p, len(a), buf, max(cap, 1)))
        return buf.raw[:n]


# ---- single kernels on device pointers (ints = device addresses) ---------------------
def _ptr(t):
    if t is None:
        return None
    return C.c_void_p(t.data_ptr() if hasattr(t, "data_ptr") else int(t))


def matvec_workspace(N: int, K: int) -> int:
    return lib.g2k_matvec_workspace(N, K)


def matvec(x, W, y, N, K, bias=None, residual=None, gelu=False, ln_gamma=None, ln_beta=None, workspace=None,
           workspace_bytes=0, stream=0):
    check(lib.g2k_matvec(_ptr(x), _ptr(W), _ptr(bias), _ptr(residual), _ptr(y), N, K, int(gelu), _ptr(ln_gamma),
                         _ptr(ln_beta), _ptr(workspace), workspace_bytes, C.c_void_p(stream)))


def matvec_noalloc(x, W, y, N, K, bias=None, residual=None, gelu=False, ln_gamma=None, ln_beta=None, stream=0):
    """g2k_matvec with the library's fixed scratch instead of a caller workspace."""
    check(lib.g2k_matvec_noalloc(_ptr(x), _ptr(W), _ptr(bias), _ptr(residual), _ptr(y), N, K, int(gelu),
                                 _ptr(ln_gamma), _ptr(ln_beta), C.c_void_p(stream)))


def matmul(A, B, C_, M, N, K, bias=None, residual=None, gelu=False, stream=0):
    check(lib.g2k_matmul(_ptr(A), _ptr(B), _ptr(bias), _ptr(residual), _ptr(C_), M, N, K, int(gelu),
                         C.c_void_p(stream)))


def matmul_tc_workspace(M: int, N: int, K: int, precision: int = G2_F32) -> int:
    return lib.g2k_matmul_tc_workspace(M, N, K, precision)


def matmul_tc(A, B, C_, M, N, K, bias=None, residual=None, gelu=False, precision=G2_F32, workspace=None,
              workspace_bytes=0, stream=0):
    """Tensor-core matmul (tcgen05): G2_F32 = 3xTF32 split operands, G2_F16 = fp16 operands."""
    check(lib.g2k_matmul_tc(_ptr(A), _ptr(B), _ptr(bias), _ptr(residual), _ptr(C_), M, N, K, int(gelu), precision,
                            _ptr(workspace), workspace_bytes, C.c_void_p(stream)))


def layernorm(x, out, gamma, beta, n_embd, rows, stream=0):
    check(lib.g2k_layernorm(_ptr(x), _ptr(out), _ptr(gamma), _ptr(beta), n_embd, rows, C.c_void_p(stream)))


def topk(logits, n, k, values, ids, stream=0):
    """g2k_topk on device tensors: the k largest of logits[0..n) into values / ids."""
    check(lib.g2k_topk(_ptr(logits), n, k, _ptr(values), _ptr(ids), C.c_void_p(stream)))


def attention_workspace(n_head: int, max_seq: int) -> int:
    return lib.g2k_attention_workspace(n_head, max_seq)


def attention(q, K, V, out, n_head, max_seq, T_kv, workspace, workspace_bytes, stream=0):
    check(lib.g2k_attention(_ptr(q), _ptr(K), _ptr(V), _ptr(out), n_head, max_seq, T_kv, _ptr(workspace),
                            workspace_bytes, C.c_void_p(stream)))


# ---- 4-bit weights, the 8-bit paged cache, rules on logits: kernels on device pointers ----
# Tensors are contiguous but for the row strides that a call takes; only their element types are checked.
def _addr(t):
    """The address of a tensor, or an int (a device address); the library refuses other memory than the current device's."""
    return t if t is None or t.__class__ is int else t.data_ptr()


def _sized(t, size):
    """_addr of a tensor whose elements have `size` bytes: a tensor of another type would be read past its end."""
    if t is None or t.__class__ is int:
        return t
    if t.element_size() != size:
        raise G2Error(-1, f"a tensor has elements of {t.element_size()} bytes, not {size}")
    return t.data_ptr()


_real_types = [None, None]   # torch.float32, torch.float16, once a tensor has been seen


def _real(t, dtype):
    """_addr of a tensor of fp32, or fp16 where `dtype` is G2_F16."""
    if t is None or t.__class__ is int:
        return t
    if t.dtype is not _real_types[1 if dtype else 0]:
        import torch
        _real_types[:] = torch.float32, torch.float16
        if t.dtype is not _real_types[1 if dtype else 0]:
            raise G2Error(-1, f"a tensor is of {t.dtype}, not {_real_types[1 if dtype else 0]}")
    return t.data_ptr()


def q4_bytes(N: int, K: int, group: int) -> int:
    """Bytes of a [K, N] weight matrix packed in 4 bits (0 for a bad shape or group)."""
    return lib.g2k_q4_bytes(N, K, group)


def q4_pack(W, packed, N, K, group, transposed=False, dtype=G2_F32, stream=0):
    """Quantise W ([K, N], or [N, K] if transposed) to 4 bits with a scale for each `group` rows of a column."""
    check(lib.g2k_q4_pack(_real(W, dtype), dtype, int(transposed), _addr(packed), N, K, group, stream))


def q4_unpack(packed, W, N, K, group, stream=0):
    """The values of a packed matrix, fp32 [K, N]."""
    check(lib.g2k_q4_unpack(_addr(packed), _real(W, G2_F32), N, K, group, stream))


def matvec_q4(x, packed, y, M, N, K, group, bias=None, residual=None, gelu=False, ln_gamma=None, ln_beta=None,
              dtype=G2_F32, stream=0):
    """y [M, N] = x' [M, K] times a packed [K, N] matrix; M up to 16 rows; x, residual and y of `dtype`."""
    check(lib.g2k_matvec_q4(_real(x, dtype), _addr(packed), _real(bias, G2_F32), _real(residual, dtype), _real(y, dtype), dtype, M,
                            N, K, group, int(gelu), _real(ln_gamma, G2_F32), _real(ln_beta, G2_F32), stream))


def kv8_cache(k, v, k_scale, v_scale, fmt=G2_KV_I8) -> KV8:
    """A paged 8-bit cache over the caller's tensors: k, v [n_pages, n_kv_head, page_size, head_dim] of one
    byte each, the scales fp32 [n_pages, n_kv_head].  The cache keeps the tensors alive."""
    shape = tuple(k.shape)
    if len(shape) != 4 or tuple(v.shape) != shape or k.element_size() != 1 or v.element_size() != 1:
        raise G2Error(-1, "k and v are one-byte tensors [n_pages, n_kv_head, page_size, head_dim]")
    if tuple(k_scale.shape) != shape[:2] or tuple(v_scale.shape) != shape[:2]:
        raise G2Error(-1, "the scales are fp32 tensors [n_pages, n_kv_head]")
    if not all(t.is_contiguous() for t in (k, v, k_scale, v_scale)):
        raise G2Error(-1, "the cache's tensors are not contiguous")
    c = KV8(_addr(k), _addr(v), _real(k_scale, G2_F32), _real(v_scale, G2_F32), *shape, fmt)
    c.tensors = (k, v, k_scale, v_scale)
    return c


def kv8_append(cache, k, v, n_rows, n_seq, table, table_stride, pos, q_start=None, max_q=1, row_stride=0, dtype=G2_F32,
               status=None, stream=0):
    """Write K and V rows of new tokens into the pages of their sequences (g2k_kv8_append)."""
    check(lib.g2k_kv8_append(C.byref(cache), _real(k, dtype), _real(v, dtype), dtype, row_stride, n_rows, n_seq, _sized(q_start, 4),
                             _sized(pos, 4), max_q, _sized(table, 4), table_stride, _sized(status, 4), stream))


def kv8_gather(cache, k_out, v_out, n_rows, n_seq, table, table_stride, pos, q_start=None, max_q=1, row_stride=0,
               dtype=G2_F32, status=None, stream=0):
    """Read rows of the cache back as values (g2k_kv8_gather)."""
    check(lib.g2k_kv8_gather(C.byref(cache), _real(k_out, dtype), _real(v_out, dtype), dtype, row_stride, n_rows, n_seq,
                             _sized(q_start, 4), _sized(pos, 4), max_q, _sized(table, 4), table_stride, _sized(status, 4), stream))


def kv8_attention_workspace(cache, n_head: int, n_seq: int, max_q: int = 1) -> int:
    return lib.g2k_kv8_attention_workspace(C.byref(cache), n_head, n_seq, max_q)


def kv8_attention(cache, q, out, n_head, n_rows, n_seq, table, table_stride, seq_len, workspace, workspace_bytes,
                  q_start=None, max_q=1, scale=None, q_stride=0, out_stride=0, dtype=G2_F32, status=None, stream=0):
    """Softmax attention of query rows over the cache (g2k_kv8_attention); scale defaults to head_dim ** -0.5."""
    check(lib.g2k_kv8_attention(C.byref(cache), _real(q, dtype), q_stride, _real(out, dtype), out_stride, dtype, n_head,
                                cache.head_dim ** -0.5 if scale is None else scale, n_rows, n_seq, _sized(q_start, 4),
                                _sized(seq_len, 4), max_q, _sized(table, 4), table_stride, _addr(workspace), workspace_bytes,
                                _sized(status, 4), stream))


def logit_rules(ctx=None, ctx_start=None, n_prompt=None, rep_penalty=None, presence=None, frequency=None, bias_ids=None,
                bias=None, bias_start=None, mask=None, mask_stride=0) -> LogitRules:
    """Rules on rows of logits over the caller's device tensors (g2_logit_rules), which it keeps alive."""
    arrays = (ctx, ctx_start, n_prompt, rep_penalty, presence, frequency, bias_ids, bias, bias_start, mask)
    if bias is not None and (bias_ids is None or bias_ids.numel() != bias.numel()):
        raise G2Error(-1, "bias_ids and bias are not of one length")
    if not all(t is None or t.__class__ is int or t.is_contiguous() for t in arrays):
        raise G2Error(-1, "an array of the rules is not contiguous")
    r = LogitRules(_sized(ctx, 4), _sized(ctx_start, 4), _sized(n_prompt, 4), 0 if ctx is None else ctx.numel(),
                   _real(rep_penalty, G2_F32), _real(presence, G2_F32), _real(frequency, G2_F32), _sized(bias_ids, 4),
                   _real(bias, G2_F32), _sized(bias_start, 4), 0 if bias is None else bias.numel(), _sized(mask, 4), mask_stride)
    r.tensors = arrays
    return r


def process_logits(logits, out, rows, vocab_size, rules, ld=0, ld_out=0, stream=0):
    """Apply `rules` to rows of logits (out may be logits); a row stride of 0 means vocab_size."""
    check(lib.g2k_process_logits(_real(logits, G2_F32), ld or vocab_size, _real(out, G2_F32), ld_out or vocab_size, rows, vocab_size,
                                 C.byref(rules), stream))
