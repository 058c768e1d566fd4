"""ctypes binding of libdiffphore_train.so (C ABI: include/train/diffphore_train.h).  No fallback: a missing library is an error."""
from __future__ import annotations

import ctypes as C
import os

import torch

from ._lib import DiffPhoreLibraryError

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "csrc", "train", "libdiffphore_train.so")
ABI_VERSION = 1
F32, BF16 = 0, 1
TYPES = {torch.float32: F32, torch.bfloat16: BF16}

i32, i64, f64, P = C.c_int32, C.c_int64, C.c_double, C.c_void_p


class DptAttnArgs(C.Structure):
    _fields_ = ([(n, i32) for n in ("type", "B", "heads", "kv_heads", "dim", "causal", "n_q", "n_k", "max_nq", "max_nk")]
                + [("n_pairs", i64), ("scale", C.c_float), ("splits", i32)]
                + [(n, i64) for n in ("q_row", "q_head", "k_row", "k_head", "v_row", "v_head", "dout_row", "dout_head", "bias_head", "bias_pair")]
                + [(n, P) for n in ("q_ptr", "k_ptr", "pair_ptr", "order", "q", "k", "v", "bias", "out", "stats", "dout", "dq", "dk", "dv", "dbias", "ws")]
                + [("ws_bytes", C.c_size_t)])


class DptAdamWArgs(C.Structure):
    _fields_ = ([(n, i32) for n in ("type", "grad_type", "state_bits", "n_tensors", "block0", "n_blocks", "last")]
                + [(n, f64) for n in ("lr", "beta1", "beta2", "eps", "weight_decay", "ema_decay")]
                + [(n, P) for n in ("lr_dev", "grad_scale", "blocks")] + [("tensor0", i32), ("pad_", i32)]
                + [(n, P) for n in ("master", "ema", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "counter")])


_lib = None


def lib():
    """Load (once) and return the library; raises loudly if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise DiffPhoreLibraryError(f"{LIB_PATH} not found: build it with `python diffphore_amd/csrc/build.py` (there is no CPU / PyTorch fallback)")
        L = C.CDLL(LIB_PATH)
        if L.dpt_abi_version() != ABI_VERSION:
            raise DiffPhoreLibraryError(f"ABI mismatch: library {L.dpt_abi_version()} != binding {ABI_VERSION}")
        sizes = (i32 * 2)()
        L.dpt_struct_sizes(sizes, 2)
        if list(sizes) != [C.sizeof(DptAttnArgs), C.sizeof(DptAdamWArgs)]:
            raise DiffPhoreLibraryError(f"struct layout mismatch: {list(sizes)}")
        L.dpt_layer_norm_fwd.argtypes = [i32, i32, i64, i32, P, i64, P, P, C.c_float, P, i64, P, P, P]
        L.dpt_layer_norm_ws_bytes.argtypes, L.dpt_layer_norm_ws_bytes.restype = [i64, i32], C.c_size_t
        L.dpt_layer_norm_bwd.argtypes = [i32, i32, i64, i32, P, i64, P, i64, P, P, P, P, i64, P, P, P, C.c_size_t, P]
        L.dpt_attn_ws_bytes.argtypes, L.dpt_attn_ws_bytes.restype = [C.POINTER(DptAttnArgs), i32], C.c_size_t
        L.dpt_attn_fwd.argtypes = L.dpt_attn_bwd.argtypes = [C.POINTER(DptAttnArgs), P]
        L.dpt_adamw_step.argtypes = [C.POINTER(DptAdamWArgs), P, P]           # grads: address of a host array of device addresses
        L.dpt_adamw_moments.argtypes = [P, P, P, P, i32, P, P, P]
        _lib = L
    return _lib


_WHY = {-1: "bad argument", -2: "not supported", -3: "too large"}


def check(rc: int, what: str):
    if rc != 0:
        raise DiffPhoreLibraryError(f"{what} failed with code {rc}" + (f" ({_WHY[rc]})" if rc in _WHY else ""))


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def call(what: str, fn, index: int, *args):
    """fn(*args, stream) on the current stream of GPU `index`, with that device current for the launch; a code other than 0 is an error.  (Called for every
    operator: the common case - the tensors' device is the current one - costs half a microsecond beside the launch.)"""
    if torch.cuda.current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        check(rc, what)


class Streams:
    """Memory that an object owns and that its launches read or write on whatever stream is current: the allocator learns of every stream but the one that
    the memory was allocated on, so that dropping the object while such a stream still works does not hand the memory out again."""

    def __init__(self, device: torch.device, tensors):
        self._index, self._tensors = device.index, [t for t in tensors if t is not None]
        self._known = {_raw_stream(self._index)}

    def use(self):
        raw = _raw_stream(self._index)
        if raw not in self._known:
            stream = torch.cuda.current_stream(self._index)
            for t in self._tensors:
                t.record_stream(stream)
            self._known.add(raw)


def need_gpu(t: torch.Tensor, name: str):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: a tensor is wanted, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name} is on {t.device}: the training operators run on the GPU only (there is no CPU fallback)")
    if t.dtype not in TYPES:
        raise TypeError(f"{name} is {t.dtype}: float32 and bfloat16 are supported")
