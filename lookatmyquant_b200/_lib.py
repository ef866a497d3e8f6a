"""ctypes bindings to liblamq_b200.so (the C ABI declared in include/lamq_b200*.h).

The library is the product's only compute path: if it is missing or cannot load, every entry point raises — there is
no CPU or PyTorch fallback. `torch` tensors are passed as raw device pointers on the current CUDA stream.
"""

from __future__ import annotations

import ctypes
import struct
import threading
from pathlib import Path

_PKG = Path(__file__).resolve().parent
LIB_PATH = _PKG / "liblamq_b200.so"
_lib = None
_lock = threading.Lock()

LAMQ_OK, LAMQ_ERR_INVALID, LAMQ_ERR_CUDA, LAMQ_ERR_NOT_PD, LAMQ_ERR_TIMEOUT, LAMQ_ERR_NOT_PATH = range(6)
LAMQ_F32, LAMQ_BF16, LAMQ_F64 = 0, 1, 2

_c = ctypes
_P, _I64, _I32, _SZ, _D = _c.c_void_p, _c.c_int64, _c.c_int, _c.c_size_t, _c.c_double

# name -> (restype, argtypes): every symbol include/lamq_b200.h, lamq_b200_train.h and lamq_b200_step.h declare
SIGNATURES = {
    "lamq_abi_version": (_I32, []),
    "lamq_kernel_launches": (_c.c_uint64, []),
    "lamq_last_error": (_c.c_char_p, []),
    "lamq_viterbi_workspace_size": (_SZ, [_I64, _I32, _I32, _I32]),
    "lamq_viterbi": (_I32, [_P, _I64, _I32, _P, _I32, _I32, _P, _P, _P, _SZ, _P]),
    "lamq_viterbi_noalloc": (_I32, [_P, _I64, _I32, _P, _I32, _I32, _P, _P, _P]),
    "lamq_ldlq_round_workspace_size": (_SZ, [_I64]),
    "lamq_ldlq_round": (_I32, [_P, _I64, _I64, _I32, _P, _I64, _P, _I32, _I32, _P, _I64, _P, _SZ, _P]),
    "lamq_xtx_accumulate": (_I32, [_P, _I64, _P, _I64, _I64, _I32, _I32, _P, _I64, _I64, _P, _P]),
    "lamq_xtx_accumulate_scaled": (_I32, [_P, _I64, _P, _I64, _I64, _I32, _I32, _c.c_float, _P, _I64, _I64, _P, _P]),
    "lamq_gather_rows": (_I32, [_P, _I64, _P, _I64, _I32, _P, _P]),
    "lamq_weighted_split": (_I32, [_P, _I64, _P, _I64, _P, _P, _I64, _I32, _P, _P, _P]),
    "lamq_hessian_finalize": (_I32, [_P, _P, _I32, _I64, _D, _P, _P, _P]),
    "lamq_rht_rows": (_I32, [_P, _I64, _P, _I64, _I64, _I32, _I32, _P, _P, _P, _P, _D, _P]),
    "lamq_transpose_f64": (_I32, [_P, _I64, _P, _I64, _I32, _I32, _P]),
    "lamq_rht_rows_act": (_I32, [_P, _I32, _I64, _P, _I32, _I64, _I64, _I32, _I32, _P, _P, _P, _P, _D, _P]),
    "lamq_dgemm": (_I32, [_I32, _I32, _I32, _I32, _D, _P, _I64, _P, _I64, _D, _P, _I64, _P]),
    "lamq_factor_workspace_size": (_SZ, [_I32]),
    "lamq_cholesky_inverse_lower": (_I32, [_P, _I64, _I32, _P, _SZ, _P, _P]),
    "lamq_env_factor": (_I32, [_P, _I64, _I32, _D, _P, _I64, _P, _P, _SZ, _P, _P]),
    "lamq_ridge": (_I32, [_P, _I64, _P, _I64, _I32, _D, _P]),
    "lamq_cross_apply_workspace_size": (_SZ, [_I32, _I32]),
    "lamq_cross_apply": (_I32, [_P, _I64, _I32, _I32, _P, _I64, _P, _I64, _D, _P, _I64, _P, _SZ, _P]),
    "lamq_proxy_loss_workspace_size": (_SZ, [_I64, _I32]),
    "lamq_proxy_loss": (_I32, [_P, _I64, _P, _I64, _I64, _I32, _P, _I64, _P, _P, _P, _SZ, _P]),
    "lamq_trellis_words_per_row": (_I64, [_I32, _I32]),
    "lamq_kl_workspace_size": (_SZ, [_I64]),
    "lamq_kl_reference": (_I32, [_P, _I64, _I64, _I32, _P, _I64, _I32, _P, _I64, _P, _P, _P, _P, _SZ, _P, _P]),
    "lamq_kl_head": (_I32, [_P, _I64, _I64, _I32, _P, _I64, _I32, _P, _I64, _P, _P, _P, _P, _P, _P, _P, _SZ, _P, _P]),
    "lamq_ldlq_coltrellis_workspace_size": (_SZ, [_I64, _I32, _I32, _I32, _I32, _I32, _I32]),
    "lamq_ldlq_coltrellis": (_I32, [_P, _I64, _I64, _I32, _P, _I64, _P, _P, _P, _I32, _I32, _I32, _I32, _I32, _P, _P,
                                     _P, _SZ, _P]),
    "lamq_pack_trellis": (_I32, [_P, _I64, _I64, _I32, _I32, _I32, _P, _P, _P]),
    "lamq_unpack_trellis": (_I32, [_P, _I64, _I32, _I32, _I32, _P, _I64, _P]),
    "lamq_decode_trellis": (_I32, [_P, _I64, _I32, _I32, _I32, _P, _P, _P, _P, _I64, _P]),
    "lamq_trellis_product": (_I32, [_P, _I64, _I32, _I32, _I32, _P, _P, _P, _P, _I64, _I32, _P, _I64, _P]),
    "lamq_trellis_product_groups": (_I32, [_P, _I32, _I32, _P, _I64, _I32, _P]),
    "lamq_square_sums_workspace_size": (_SZ, [_I64, _I32]),
    "lamq_square_sums": (_I32, [_P, _I32, _I64, _I32, _I64, _P, _P, _P, _SZ, _P]),
    "lamq_trellis_gemm_workspace_size": (_SZ, [_P, _I32, _I64]),
    "lamq_trellis_gemm": (_I32, [_P, _I32, _I64, _I32, _P, _SZ, _P, _P]),
    "lamq_ldlq_rowtrellis_workspace_size": (_SZ, [_I64, _I32]),
    "lamq_ldlq_rowtrellis": (_I32, [_P, _I64, _I64, _I32, _P, _I64, _P, _P, _P, _P, _I32, _I32, _I32, _I32, _I32,
                                    _P, _P, _P, _SZ, _P]),
    "lamq_embedding_lookup": (_I32, [_P, _I32, _I64, _I64, _I32, _P, _I32, _I64, _c.c_float, _I64, _P, _I64, _P, _P]),
    "lamq_embedding_gradient_workspace_size": (_SZ, [_I64, _I32]),
    "lamq_embedding_gradient": (_I32, [_P, _I32, _I64, _P, _I32, _I64, _I64, _I32, _c.c_float, _I64, _I32, _P, _I64,
                                       _P, _SZ, _P, _P]),
    "lamq_attention_forward": (_I32, [_P, _P, _P]),
    "lamq_attention_backward_workspace_size": (_SZ, [_I64, _I32, _I64]),
    "lamq_attention_backward": (_I32, [_P, _P, _SZ, _P, _P]),
    "lamq_newton_schulz_workspace_size": (_SZ, [_I32, _I32, _I32]),
    "lamq_newton_schulz": (_I32, [_P, _I32, _I64, _I64, _I32, _I32, _I32, _I32, _P, _c.c_float, _P, _P, _SZ, _P, _P]),
    "lamq_norm_forward": (_I32, [_P, _P]),
    "lamq_norm_backward_workspace_size": (_SZ, [_P]),
    "lamq_norm_backward": (_I32, [_P, _P, _SZ, _P]),
    "lamq_gradient_workspace_size": (_SZ, [_I64]),
    "lamq_gradient_norm": (_I32, [_P, _I64, _P, _P, _SZ, _P]),
    "lamq_gradient_clip": (_I32, [_P, _I64, _D, _D, _P, _P, _SZ, _P]),
}

# lamq_attention_args (328 bytes): batch; heads, kv_heads, head_dim, causal; q_len, kv_len; scale, reserved; key_start,
# key_end; q, k, v, o; lse; d_o, dq, dk, dv (a lamq_heads is a pointer and three strides)
ATTENTION_ARGS = struct.Struct("=q4i2qfi2Q16qQ16q")

# lamq_norm_args (264 bytes): rows, gate_span; d, residual_dtype, branch_dtype, weight_dtype, post_dtype, gate_dtype; scale,
# eps, offset, reserved; residual, branch; weight, post, gate; h, y; dh, dy; d_residual, d_branch, d_weight, d_post, d_gate (a
# lamq_rows is a pointer, an inner count and two strides)
NORM_ARGS = struct.Struct("=2q6i3fi8q5Q8q5Q")

# lamq_gradient (32 bytes): data, out; n; dtype, out_dtype
GRADIENT = struct.Struct("=2Qq2i")


class ProductGroup(_c.Structure):
    """lamq_product_group: one packed row group of a grouped product (64 bytes, the header's field order)."""
    _fields_ = [("codes", _P), ("rows", _I64), ("k", _I32), ("L", _I32), ("scales", _P), ("table", _P),
                ("map", _P), ("y", _P), ("ldy", _I64)]


class GemmGroup(_c.Structure):
    """lamq_gemm_group: one row group of a trellis-dequant GEMM and its input (104 bytes, the header's field order)."""
    _fields_ = [("codes", _P), ("states", _P), ("lds", _I64), ("rows", _I64), ("k", _I32), ("L", _I32),
                ("scales", _P), ("table", _P), ("map", _P), ("y", _P), ("ldy", _I64), ("x", _P), ("ldx", _I64),
                ("n", _I32), ("reserved", _I32)]


class LamqError(RuntimeError):
    pass


def load():
    """Loads liblamq_b200.so (raising if it was not built) and declares every exported signature."""
    global _lib
    with _lock:
        if _lib is None:
            if not LIB_PATH.exists():
                raise LamqError(f"{LIB_PATH} is missing: build it with `python -m lookatmyquant_b200.build` "
                                "(the CUDA kernels are the only implementation; there is no fallback)")
            lib = ctypes.CDLL(str(LIB_PATH))
            for name, (res, args) in SIGNATURES.items():
                f = getattr(lib, name)
                f.restype, f.argtypes = res, args
            _lib = lib
    return _lib


def kernel_launches() -> int:
    """Kernels liblamq_b200 has launched in this process (lamq_kernel_launches)."""
    return int(load().lamq_kernel_launches())


def check(status: int, what: str):
    """Raises on a non-zero status."""
    if status != LAMQ_OK:
        msg = load().lamq_last_error().decode(errors="replace")
        if status == LAMQ_ERR_INVALID:
            raise ValueError(f"{what}: {msg}")
        if status == LAMQ_ERR_NOT_PD:
            raise AssertionError("H is not positive definite even with damping")
        if status == LAMQ_ERR_NOT_PATH:
            raise ValueError("the given projection is not a path through this trellis")
        raise LamqError(f"{what} failed (status {status}): {msg}")


def ptr(t) -> int | None:
    """Device pointer of a tensor (None for None)."""
    return None if t is None else t.data_ptr()


def stream_ptr(device=None) -> int:
    import torch
    return torch.cuda.current_stream(device).cuda_stream


class _Here:
    def __enter__(self):
        pass

    def __exit__(self, *exc):
        pass


_HERE = _Here()


def launch_on(device):
    """(a context in which `device` is the current one, its current stream): what a call of a few microseconds needs,
    without torch.cuda.device and torch.cuda.current_stream where they would change nothing (3 us a call)."""
    import torch
    index = device.index
    here = _HERE if torch.cuda.current_device() == index else torch.cuda.device(device)
    return here, torch._C._cuda_getCurrentRawStream(index)


class StatusWord:
    """One device int per GPU that an operator's kernels set on an error (a status argument of the C ABI). Calls only
    pass it on; `check` reads it, which waits for the device. The first call on a device makes it, so that one cannot be
    captured in a CUDA graph."""

    def __init__(self, what: str, invalid: str | None = None):
        self.what, self.invalid = what, invalid  # the operator; what LAMQ_ERR_INVALID says of its inputs
        self.words = {}
        self.lock = threading.Lock()

    def on(self, device):
        """The device's word, made by the first call there (one word, whichever threads come first)."""
        word = self.words.get(device)
        return word if word is not None else self._make(device)

    def _make(self, device):
        import torch
        with self.lock:
            if device not in self.words:
                if torch.cuda.is_current_stream_capturing():  # memory of the graph's would be cleared by every replay
                    raise LamqError("the first call of an operator on a device cannot be captured: make one before")
                with torch.cuda.device(device):
                    word = torch.zeros(1, dtype=torch.int32, device=device)
                    torch.cuda.synchronize(device)  # zero before any stream's kernel can set it
                self.words[device] = word
            return self.words[device]

    def check(self):
        """Raises if a kernel of any call so far, on whatever stream, set a word, and clears it."""
        import torch
        for device, word in list(self.words.items()):
            torch.cuda.synchronize(device)  # .item() would wait for the current stream alone
            st = int(word.item())
            if st:
                word.zero_()
                torch.cuda.synchronize(device)  # cleared before any stream's next kernel can set it
                if st == LAMQ_ERR_INVALID and self.invalid:
                    raise ValueError(self.invalid)
                raise LamqError(f"{self.what}: a kernel gave up on a device wait (status {st}): results since the last "
                                "check may be invalid")
