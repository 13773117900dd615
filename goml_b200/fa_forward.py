"""Host binding of libfa_sm120.so, mirroring goml's backend/cuda/fa_forward.go.

Names and behaviour follow that file: ``FALoad`` (one-time dlopen with the
search order of fa_forward.go:74-115: ``$GOML_FA_LIB``, then
``libs/fa_sm120/libfa_sm120.so``, ``./libfa_sm120.so``,
``/usr/local/lib/libfa_sm120.so`` — this package's own ``libs`` directory is
tried right after the environment override), ``FACreate`` (fa_forward.go:123-142,
including "context returned together with an error is read for its message and
destroyed"), ``FAContext.ForwardTrain`` (fa_forward.go:161-183) and
``FAVersion``.  ``FAContext.Forward`` binds ``fa_forward`` (which the Go file
leaves unbound) and ``FAContext.ForwardEx`` binds the additive struct-pointer
entry.  Pointers are raw device addresses (ints); errors are raised as
``FAError("<entry>: <status text> (<context message>)")``.
"""
from __future__ import annotations

import ctypes as C
import os
import struct
import threading

from . import loader

FA_OK = 0
FA_ERR_INVALID_ARG = 1
FA_ERR_UNSUPPORTED_ARCH = 2
FA_ERR_UNSUPPORTED_HD = 3
FA_ERR_UNSUPPORTED_SHAPE = 4
FA_ERR_CUDA = 5
FA_ERR_OOM = 6
FA_ERR_INTERNAL = 7

FA_KERNEL_NONE = -1
FA_KERNEL_V121R, FA_KERNEL_V121, FA_KERNEL_V118 = 100, 101, 102
FA_KERNEL_V122, FA_KERNEL_V117B, FA_KERNEL_V96B = 103, 104, 105
FA_KERNEL_V89, FA_KERNEL_V80B = 200, 201


class FAError(RuntimeError):
    def __init__(self, entry: str, status: int, msg: str = ""):
        self.status = status
        self.msg = msg
        text = FAStatusString(status)
        super().__init__(f"{entry}: {text} ({msg})" if msg else f"{entry}: {text}")


class ForwardArgs(C.Structure):
    """fa_forward_args_t of include/fa_sm120.h."""
    _fields_ = [
        ("q", C.c_void_p), ("k", C.c_void_p), ("v", C.c_void_p), ("o", C.c_void_p), ("l_out", C.c_void_p),
        ("batch_heads", C.c_int), ("seq_len", C.c_int), ("head_dim", C.c_int),
        ("causal", C.c_int), ("window", C.c_int),
        ("scale", C.c_float), ("v_descale", C.c_float),
        ("scale_q_dev", C.c_void_p), ("scale_k_dev", C.c_void_p), ("scale_v_dev", C.c_void_p),
        ("stream", C.c_void_p),
    ]


class DecodeArgs(C.Structure):
    """fa_decode_args_t (include/fa_sm120.h)."""
    _fields_ = [
        ("q", C.c_void_p), ("k_cache", C.c_void_p), ("v_cache", C.c_void_p), ("o", C.c_void_p), ("l_out", C.c_void_p),
        ("seq_lens", C.c_void_p),
        ("batch", C.c_int), ("q_heads", C.c_int), ("kv_heads", C.c_int), ("head_dim", C.c_int),
        ("s_max", C.c_int), ("seq_len", C.c_int),
        ("scale", C.c_float), ("v_descale", C.c_float),
        ("scale_q_dev", C.c_void_p), ("scale_k_dev", C.c_void_p), ("scale_v_dev", C.c_void_p),
        ("stream", C.c_void_p),
        ("block_table", C.c_void_p), ("page_size", C.c_int), ("max_pages_per_seq", C.c_int), ("num_pages", C.c_int),
    ]


class DecodeFP4Args(C.Structure):
    """fa_decode_fp4_args_t (include/fa_sm120.h)."""
    _fields_ = ([(n, C.c_void_p) for n in ("q", "k_codes", "k_scales", "v_codes", "v_scales", "o", "l_out", "seq_lens", "scale_q_dev", "scale_k_dev", "scale_v_dev",
                                           "block_table", "stream")]
                + [(n, C.c_int) for n in ("batch", "q_heads", "kv_heads", "head_dim", "s_max", "seq_len", "page_size", "max_pages_per_seq", "num_pages", "q_type")]
                + [("scale", C.c_float), ("v_descale", C.c_float)])


# The argument blocks as packed bytes: one struct.pack (native alignment) and a bytes argument cost 1 us of host time
# a call, filling a ctypes structure field by field and passing a reference to it about 4.
_PACK_FORWARD = struct.Struct("@5P5i2f4P").pack
_PACK_DECODE = struct.Struct("@6P6i2f5P3i0P").pack
_PACK_DECODE_FP4 = struct.Struct("@13P10i2f0P").pack
assert struct.calcsize("@5P5i2f4P") == C.sizeof(ForwardArgs) and struct.calcsize("@6P6i2f5P3i0P") == C.sizeof(DecodeArgs)
assert struct.calcsize("@13P10i2f0P") == C.sizeof(DecodeFP4Args)

Q_BF16, Q_FP16, Q_E4M3 = 0, 1, 2   # types of the queries of DecodeFP4


def _pack(pack, block, *args) -> bytes:
    """The argument block's bytes; values that struct.pack has no format for (a c_void_p, a float out of range) go through
    the ctypes structure, which takes or refuses them."""
    try:
        return pack(*args)
    except (struct.error, OverflowError):
        return bytes(block(*args))

_lock = threading.Lock()
_lib = None
_lib_err = None
_forward_ex = None   # fa_forward_ex / fa_decode taking the packed block, set by FALoad
_decode = None
_decode_fp4 = None
_decode_window = None
_decode_shared = None
_forward_sinks = None


def _candidates():
    env = os.environ.get("GOML_FA_LIB", "")
    if env:
        yield env
    yield loader.resolve_lib("libfa_sm120.so")
    yield os.path.join("libs", "fa_sm120", "libfa_sm120.so")
    yield os.path.join(".", "libfa_sm120.so")
    yield "/usr/local/lib/libfa_sm120.so"


def FALoad():
    """One-time dlopen of libfa_sm120.so and symbol registration."""
    global _lib, _lib_err, _forward_ex, _decode, _decode_fp4, _decode_window, _decode_shared, _forward_sinks
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None and _lib_err is None:
            last = None
            for path in _candidates():
                if os.path.sep in path and not os.path.exists(path):
                    continue
                try:
                    lib = loader.dlopen(path)
                except OSError as e:
                    last = e
                    continue
                i, p, f = C.c_int, C.c_void_p, C.c_float
                lib.fa_create.restype = i
                lib.fa_create.argtypes = [C.POINTER(p)]
                lib.fa_destroy.restype = i
                lib.fa_destroy.argtypes = [p]
                lib.fa_version.restype = C.c_char_p
                lib.fa_status_str.restype = C.c_char_p
                lib.fa_status_str.argtypes = [i]
                lib.fa_last_cuda_error.restype = C.c_char_p
                lib.fa_last_cuda_error.argtypes = [p]
                lib.fa_forward.restype = i
                lib.fa_forward.argtypes = [p, p, p, p, p, i, i, i, i, i, f, p]
                lib.fa_forward_train.restype = i
                lib.fa_forward_train.argtypes = [p, p, p, p, p, p, i, i, i, i, i, f, p]
                lib.fa_dispatch_select.restype = i
                lib.fa_dispatch_select.argtypes = [i] * 5
                lib.fa_kernel_name.restype = C.c_char_p
                lib.fa_kernel_name.argtypes = [i]
                lib.fa_forward_ex.restype = i
                lib.fa_forward_ex.argtypes = [p, C.POINTER(ForwardArgs)]
                lib.fa_forward_raise.restype = i
                lib.fa_forward_raise.argtypes = [p, C.POINTER(ForwardArgs), p]
                lib.fa_forward_noalloc.restype = i
                lib.fa_forward_noalloc.argtypes = [C.POINTER(ForwardArgs), C.c_char_p, i]
                lib.fa_decode.restype = i
                lib.fa_decode.argtypes = [p, C.POINTER(DecodeArgs)]
                lib.fa_decode_fp4.restype = i
                lib.fa_decode_fp4.argtypes = [p, C.POINTER(DecodeFP4Args)]
                lib.fa_device_status.restype = i
                lib.fa_device_status.argtypes = [p]
                lib.fa_noalloc_device_status.restype = i
                lib.fa_noalloc_device_status.argtypes = []
                lib.fa_selftest_wait_expiry.restype = i
                lib.fa_selftest_wait_expiry.argtypes = [p, p]
                forward_ex, decode, decode_fp4 = lib["fa_forward_ex"], lib["fa_decode"], lib["fa_decode_fp4"]
                for fn in (forward_ex, decode, decode_fp4):
                    fn.restype = i
                    fn.argtypes = [p, C.c_char_p]
                window, shared, sinks = lib["fa_decode_window"], lib["fa_decode_shared"], lib["fa_forward_sinks"]
                window.restype = shared.restype = sinks.restype = i
                sinks.argtypes = [p, C.c_char_p, i]
                window.argtypes, shared.argtypes = [p, C.c_char_p, i, i], [p, C.c_char_p, p, p, i]
                _forward_ex, _decode, _decode_fp4, _decode_window, _decode_shared, _forward_sinks = forward_ex, decode, decode_fp4, window, shared, sinks
                _lib = lib
                break
            if _lib is None:
                _lib_err = loader.LibraryNotFound(
                    f"fa: dlopen libfa_sm120.so failed ({last}); set GOML_FA_LIB or build with "
                    f"`python -m goml_b200.build`")
    if _lib_err is not None:
        raise _lib_err
    return _lib


def FAStatusString(status: int) -> str:
    try:
        return FALoad().fa_status_str(int(status)).decode()
    except OSError:
        return f"unknown({status})"


def FAVersion() -> str:
    return FALoad().fa_version().decode()


def FADispatchSelect(bh: int, sl: int, hd: int, causal: int, window: int) -> int:
    return FALoad().fa_dispatch_select(bh, sl, hd, causal, window)


def FAKernelName(kid: int) -> str:
    return FALoad().fa_kernel_name(kid).decode()


class FAContext:
    """Opaque handle; one per GPU (the device current when it was created)."""

    def __init__(self, ptr: int):
        self.ptr = ptr

    def _msg(self) -> str:
        return FALoad().fa_last_cuda_error(self.ptr).decode(errors="replace") if self.ptr else ""

    def Destroy(self) -> None:
        if self.ptr:
            FALoad().fa_destroy(self.ptr)
            self.ptr = 0

    def ForwardTrain(self, q, k, v, o, lOut, bh, sl, hd, causal, window, scale, stream=0) -> None:
        if not self.ptr:
            raise FAError("FAContext.ForwardTrain: nil ctx", FA_ERR_INVALID_ARG)
        st = FALoad().fa_forward_train(self.ptr, q, k, v, o, lOut or None, bh, sl, hd, causal, window, scale, stream or None)
        if st != FA_OK:
            raise FAError("fa_forward_train", st, self._msg())

    def Forward(self, q, k, v, o, bh, sl, hd, causal, window, scale, stream=0) -> None:
        if not self.ptr:
            raise FAError("FAContext.Forward: nil ctx", FA_ERR_INVALID_ARG)
        st = FALoad().fa_forward(self.ptr, q, k, v, o, bh, sl, hd, causal, window, scale, stream or None)
        if st != FA_OK:
            raise FAError("fa_forward", st, self._msg())

    def ForwardEx(self, q, k, v, o, lOut, bh, sl, hd, causal, window, scale, v_descale=1.0,
                  scale_q_dev=0, scale_k_dev=0, scale_v_dev=0, stream=0) -> None:
        if not self.ptr:
            raise FAError("FAContext.ForwardEx: nil ctx", FA_ERR_INVALID_ARG)
        st = _forward_ex(self.ptr, _pack(_PACK_FORWARD, ForwardArgs, q or 0, k or 0, v or 0, o or 0, lOut or 0, bh, sl, hd, causal, window,
                                         scale, v_descale, scale_q_dev or 0, scale_k_dev or 0, scale_v_dev or 0, stream or 0))
        if st != FA_OK:
            raise FAError("fa_forward_ex", st, self._msg())

    def ForwardSinks(self, q, k, v, o, lOut, bh, sl, hd, window, sinks, scale, v_descale=1.0, scale_q_dev=0, scale_k_dev=0, scale_v_dev=0, stream=0) -> None:
        """ForwardEx of causal prompts where the first `sinks` tokens stay visible behind the window."""
        if not self.ptr:
            raise FAError("FAContext.ForwardSinks: nil ctx", FA_ERR_INVALID_ARG)
        st = _forward_sinks(self.ptr, _pack(_PACK_FORWARD, ForwardArgs, q or 0, k or 0, v or 0, o or 0, lOut or 0, bh, sl, hd, 1, window, scale, v_descale, scale_q_dev or 0,
                                            scale_k_dev or 0, scale_v_dev or 0, stream or 0), sinks)
        if st != FA_OK:
            raise FAError("fa_forward_sinks", st, self._msg())

    def Decode(self, q, k_cache, v_cache, o, lOut, seq_lens, batch, q_heads, kv_heads, hd, s_max, seq_len, scale, v_descale=1.0,
               scale_q_dev=0, scale_k_dev=0, scale_v_dev=0, stream=0, block_table=0, page_size=0, max_pages_per_seq=0,
               num_pages=0) -> None:
        """One new token per sequence against an e4m3 KV cache [batch, kv_heads, s_max, hd], grouped-query heads;
        seq_lens: device pointer to batch int32 lengths, or 0 to use seq_len for every sequence.  With block_table
        (device pointer to int32 [batch, max_pages_per_seq]) the caches are page pools [num_pages, kv_heads, page_size,
        hd] and s_max is ignored."""
        if not self.ptr:
            raise FAError("FAContext.Decode: nil ctx", FA_ERR_INVALID_ARG)
        st = _decode(self.ptr, _pack(_PACK_DECODE, DecodeArgs, q or 0, k_cache or 0, v_cache or 0, o or 0, lOut or 0, seq_lens or 0, batch, q_heads,
                                     kv_heads, hd, s_max, seq_len, scale, v_descale, scale_q_dev or 0, scale_k_dev or 0, scale_v_dev or 0,
                                     stream or 0, block_table or 0, page_size, max_pages_per_seq, num_pages))
        if st != FA_OK:
            raise FAError("fa_decode", st, self._msg())

    def DecodeFP4(self, q, k_codes, k_scales, v_codes, v_scales, o, lOut, seq_lens, batch, q_heads, kv_heads, hd, s_max, seq_len, scale, v_descale=1.0,
                  q_type=Q_BF16, scale_q_dev=0, scale_k_dev=0, scale_v_dev=0, stream=0, block_table=0, page_size=0, max_pages_per_seq=0, num_pages=0) -> None:
        """One new token per sequence against a KV cache held in 4 bits (e2m1 codes, an e4m3 scale for 16 dims, fp32 scales *scale_k_dev and
        *scale_v_dev): codes [batch, kv_heads, s_max, hd/2], k_scales [batch, kv_heads, s_max, hd/16], v_scales [batch, kv_heads, s_max/16, hd/16, 16],
        or with block_table pools of num_pages pages of page_size keys in the place of the sequences.  q: bf16, fp16 or e4m3 (q_type)."""
        if not self.ptr:
            raise FAError("FAContext.DecodeFP4: nil ctx", FA_ERR_INVALID_ARG)
        st = _decode_fp4(self.ptr, _pack(_PACK_DECODE_FP4, DecodeFP4Args, q or 0, k_codes or 0, k_scales or 0, v_codes or 0, v_scales or 0, o or 0, lOut or 0,
                                         seq_lens or 0, scale_q_dev or 0, scale_k_dev or 0, scale_v_dev or 0, block_table or 0, stream or 0, batch, q_heads, kv_heads, hd,
                                         s_max, seq_len, page_size, max_pages_per_seq, num_pages, q_type, scale, v_descale))
        if st != FA_OK:
            raise FAError("fa_decode_fp4", st, self._msg())

    def DecodeWindow(self, q, k_cache, v_cache, o, lOut, seq_lens, batch, q_heads, kv_heads, hd, s_max, seq_len, window, sinks, scale, v_descale=1.0,
                     scale_q_dev=0, scale_k_dev=0, scale_v_dev=0, stream=0, block_table=0, page_size=0, max_pages_per_seq=0, num_pages=0) -> None:
        """Decode where a sequence of n keys sees keys [0, sinks) and [n - window, n) only (window 0: all)."""
        if not self.ptr:
            raise FAError("FAContext.DecodeWindow: nil ctx", FA_ERR_INVALID_ARG)
        st = _decode_window(self.ptr, _pack(_PACK_DECODE, DecodeArgs, q or 0, k_cache or 0, v_cache or 0, o or 0, lOut or 0, seq_lens or 0, batch, q_heads, kv_heads, hd, s_max, seq_len,
                                            scale, v_descale, scale_q_dev or 0, scale_k_dev or 0, scale_v_dev or 0, stream or 0, block_table or 0, page_size, max_pages_per_seq,
                                            num_pages), window, sinks)
        if st != FA_OK:
            raise FAError("fa_decode_window", st, self._msg())

    def DecodeShared(self, q, k_cache, v_cache, o, lOut, seq_lens, shared_lens, group_starts, groups, batch, q_heads, kv_heads, hd, s_max, scale, v_descale=1.0,
                     scale_q_dev=0, scale_k_dev=0, scale_v_dev=0, stream=0, block_table=0, page_size=0, max_pages_per_seq=0, num_pages=0) -> None:
        """Decode where sequence b begins with shared_lens[b] keys of the first sequence of its group, which are read once for the group; group i has sequences
        [group_starts[i], group_starts[i + 1]).  seq_lens, shared_lens and group_starts (groups + 1): int32 on the device."""
        if not self.ptr:
            raise FAError("FAContext.DecodeShared: nil ctx", FA_ERR_INVALID_ARG)
        st = _decode_shared(self.ptr, _pack(_PACK_DECODE, DecodeArgs, q or 0, k_cache or 0, v_cache or 0, o or 0, lOut or 0, seq_lens or 0, batch, q_heads, kv_heads, hd, s_max, 0,
                                            scale, v_descale, scale_q_dev or 0, scale_k_dev or 0, scale_v_dev or 0, stream or 0, block_table or 0, page_size, max_pages_per_seq,
                                            num_pages), shared_lens or None, group_starts or None, groups)
        if st != FA_OK:
            raise FAError("fa_decode_shared", st, self._msg())

    def DeviceStatus(self) -> None:
        st = FALoad().fa_device_status(self.ptr)
        if st != FA_OK:
            raise FAError("fa_device_status", st, self._msg())

    def SelftestWaitExpiry(self, stream=0) -> None:
        """Launch the one-warp kernel whose bounded wait runs out; the next DeviceStatus() then raises FA_ERR_INTERNAL."""
        st = FALoad().fa_selftest_wait_expiry(self.ptr, stream or None)
        if st != FA_OK:
            raise FAError("fa_selftest_wait_expiry", st, self._msg())

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.Destroy()


NOALLOC_MAX_ELEMS = 16 << 20


def FAForwardNoAlloc(q, k, v, o, lOut, bh, sl, hd, causal, window, scale, v_descale=1.0,
                     scale_q_dev=0, scale_k_dev=0, scale_v_dev=0, stream=0) -> None:
    """Attention forward for callers that may not allocate (frameworks that reserved the whole
    GPU, frozen-memory-map processes): scratch is a fixed 32 MiB array inside the library, so
    bh*sl*hd must not exceed NOALLOC_MAX_ELEMS.  No context is needed.  Calls that overlap on
    the GPU share (and race on) that array; make the first call on a device before any capture."""
    a = ForwardArgs(q, k, v, o, lOut or None, bh, sl, hd, causal, window, scale, v_descale,
                    scale_q_dev or None, scale_k_dev or None, scale_v_dev or None, stream or None)
    buf = C.create_string_buffer(256)
    st = FALoad().fa_forward_noalloc(C.byref(a), buf, len(buf))
    if st != FA_OK:
        raise FAError("fa_forward_noalloc", st, buf.value.decode(errors="replace"))


def FANoAllocDeviceStatus() -> int:
    """fa_device_status without a context (for users of FAForwardNoAlloc): 0, a kernel's wait-expiry code, or
    a negated CUDA error."""
    return FALoad().fa_noalloc_device_status()


def FACreate() -> FAContext:
    """Create an FA context on the current device (fa_forward.go:123-142)."""
    lib = FALoad()
    ptr = C.c_void_p()
    st = lib.fa_create(C.byref(ptr))
    if st != FA_OK:
        if ptr.value:
            msg = lib.fa_last_cuda_error(ptr).decode(errors="replace")
            lib.fa_destroy(ptr)
            raise FAError("fa_create", st, msg)
        raise FAError("fa_create", st)
    return FAContext(ptr.value)
