"""Python mirror of the hardshell-cuda API (crates/hardshell-cuda/src/lib.rs:36-43) over the C ABI
of libhardshell_hip.so (include/hardshell_hip.h): HipDevice, HipModel, HipBatch, HipSession
and the op-level entry points. Errors mirror crates/hardshell-cuda/src/error.rs:9-51.

The native library is required: importing this module never falls back to a CPU path, and
every call fails loudly if libhardshell_hip.so is missing."""

from __future__ import annotations

import ctypes as C
import os
from dataclasses import dataclass
from typing import Iterable, List, NamedTuple, Optional, Sequence, Tuple

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libhardshell_hip.so")

HS_OK, HS_NO_DEVICE, HS_DEVICE_ERROR, HS_UNSUPPORTED, HS_MODEL_ERROR, HS_BAD_SLOT, \
    HS_LENGTH_MISMATCH, HS_INVALID_ARGUMENT = range(8)

MODEL_ERRORS = {
    1: "InvalidShape", 2: "LengthMismatch", 3: "DotTooLong", 4: "BadMagic",
    5: "UnsupportedVersion", 6: "Truncated", 7: "HeaderNotUtf8", 8: "HeaderJson",
    9: "InvalidHeader", 10: "Layout", 11: "NonZeroPadding", 12: "Vocabulary",
    13: "MissingTensor", 14: "UnexpectedTensor", 15: "TensorMismatch", 16: "TokenOutOfRange",
    17: "InvalidOverlap", 18: "BadTruncate", 19: "TooLarge", 20: "Unsupported",
}


class HipError(Exception):
    def __init__(self, status: int, code: int, message: str):
        super().__init__(message)
        self.status, self.code, self.message = status, code, message


class NoDevice(HipError):
    pass


class DeviceError(HipError):
    pass


class Unsupported(HipError):
    pass


class ModelError(HipError):
    @property
    def kind(self) -> str:
        return MODEL_ERRORS.get(self.code, str(self.code))


class BadSlot(HipError):
    pass


class LengthMismatch(HipError):
    pass


_ERRORS = {HS_NO_DEVICE: NoDevice, HS_DEVICE_ERROR: DeviceError, HS_UNSUPPORTED: Unsupported,
           HS_MODEL_ERROR: ModelError, HS_BAD_SLOT: BadSlot, HS_LENGTH_MISMATCH: LengthMismatch,
           HS_INVALID_ARGUMENT: HipError}


class _Input(C.Structure):
    _fields_ = [("slot", C.c_uint32), ("token", C.c_uint32)]


# The mixed coder op of the logs profile (crates/hardshell-cuda/src/mixed.rs).
HS_MIX_NONE = 0xFFFFFFFF   # a mixed table without a prediction
HS_MIX_PLAIN = 0xFFFFFFFE  # the table of GPT-2 alone
HS_TREE_ROOT = 0xFFFFFFFF  # the parent of a tree's node right after the context
HS_NO_TOKEN = 0xFFFFFFFF   # no token to score


class MixStats(C.Structure):
    """MixStats (mixed.rs:36-49): total = sum w, predicted = w[p], top = the largest."""
    _fields_ = [("total", C.c_uint64), ("predicted", C.c_uint64), ("top", C.c_uint32),
                ("pad", C.c_uint32)]


MIXER_FN = C.CFUNCTYPE(C.c_uint32, C.c_void_p, C.c_size_t, C.POINTER(MixStats))


def _mixer(fn):
    """A C callback over fn(input, stats) -> q; an exception gives q = 0 (refused)."""
    def call(_user, i, st):
        try:
            return int(fn(int(i), st.contents))
        except Exception:  # noqa: BLE001 - the library reports the bad q
            return 0
    return MIXER_FN(call)


class _Query(C.Structure):
    _fields_ = [("kind", C.c_uint32), ("value", C.c_uint32)]


class _Interval(C.Structure):
    _fields_ = [("symbol", C.c_uint64), ("start", C.c_uint64), ("freq", C.c_uint64)]


_lib = None


def lib() -> C.CDLL:
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                "taco_amd/libhardshell_hip.so is not built (run `python -c 'import __graft_entry__ as g; "
                "g.build()'`); there is no CPU fallback")
        L = C.CDLL(LIB_PATH)
        P, S, U32, U64 = C.c_void_p, C.c_size_t, C.c_uint32, C.c_uint64
        L.hs_last_error_message.restype = C.c_char_p
        L.hs_last_error_code.restype = C.c_int
        L.hs_version.restype = C.c_char_p
        L.hs_device_open.argtypes = [C.c_int, C.POINTER(P)]
        L.hs_device_close.argtypes = [P]
        L.hs_device_name.argtypes = [P, C.c_char_p, S]
        L.hs_device_memory.argtypes = [P, C.POINTER(S), C.POINTER(S)]
        L.hs_model_load.argtypes = [P, P, S, C.POINTER(P)]
        L.hs_model_free.argtypes = [P]
        L.hs_model_hash.argtypes = [P, P]
        for f in ("vocab", "n_ctx", "eot"):
            getattr(L, "hs_model_" + f).restype = U32
            getattr(L, "hs_model_" + f).argtypes = [P]
        L.hs_model_is_wide.argtypes = [P]
        L.hs_model_weight_bytes.restype = U64
        L.hs_model_weight_bytes.argtypes = [P]
        L.hs_model_cache_bytes_per_slot.restype = U64
        L.hs_model_cache_bytes_per_slot.argtypes = [P]
        L.hs_batch_new.argtypes = [P, S, S, C.POINTER(P)]
        L.hs_batch_free.argtypes = [P]
        L.hs_batch_set_overlap.argtypes = [P, U32]
        for f in ("slots", "max_rows"):
            getattr(L, "hs_batch_" + f).restype = S
            getattr(L, "hs_batch_" + f).argtypes = [P]
        L.hs_batch_gpu_bytes.restype = U64
        L.hs_batch_gpu_bytes.argtypes = [P]
        for f in ("position", "stream_len", "room"):
            getattr(L, "hs_batch_" + f).restype = S
            getattr(L, "hs_batch_" + f).argtypes = [P, S]
        L.hs_batch_reset.argtypes = [P, S]
        L.hs_batch_run_weights.argtypes = [P, P, S, P]
        L.hs_batch_run_coded.argtypes = [P, P, P, S, U32, P]
        L.hs_batch_step.argtypes = [P, P, S]
        L.hs_batch_weights.argtypes = [P, S, P]
        L.hs_batch_truncate.argtypes = [P, S, S]
        L.hs_op_gemm_i8.argtypes = [P, P, P, S, S, S, P]
        L.hs_op_gemm_requant_i8.argtypes = [P, P, P, P, P, C.c_uint8, S, S, S, P]
        L.hs_op_gemm_i8_split.argtypes = [P, P, P, S, S, S, C.c_uint32, P]
        L.hs_op_gemm_i8_i16.argtypes = [P, P, P, S, S, S, C.c_uint32, P]
        L.hs_op_gemm_requant_i8_dev.argtypes = [P, P, P, P, P, C.c_uint8, S, S, S, P, P]
        L.hs_op_gemm_layout.argtypes = [S, S, S, C.POINTER(S), C.POINTER(S), C.POINTER(S)]
        L.hs_op_gemm_layout.restype = None
        L.hs_op_attend_decode_dev.argtypes = [P, P, P, P, P, S, S, S, S, C.c_int32, C.c_uint8,
                                              C.c_int32, C.c_uint8, P, S, C.c_uint8, P, P]
        L.hs_op_attend_decode_dev_noalloc.argtypes = L.hs_op_attend_decode_dev.argtypes
        rows = [P, P, P, P, P, P, P, S, S, S, S, S, C.c_int32, C.c_uint8, C.c_int32, C.c_uint8, P, S,
                C.c_uint8, P, P, S, P]
        L.hs_op_attend_tree_dev.argtypes = rows
        L.hs_op_attend_mass_dev.argtypes = rows
        L.hs_op_attend_rows_workspace.argtypes = [S] * 5
        L.hs_op_attend_rows_workspace.restype = S
        L.hs_op_cache_evict_dev.argtypes = [P, P, P, S, P, P, S, S, S, S, S, S, P, P, P, P]
        L.hs_op_cache_commit_dev.argtypes = [P, P, P, S, P, P, P, S, S, S, S, S, P, P]
        L.hs_op_pages_append_dev.argtypes = [P, P, P, P, U32, S, P, P, P, S, S, S, U32, P, P]
        L.hs_op_attend_paged_dev.argtypes = [P, P, P, S, P, P, P, S, S, S, S, S, C.c_int32, C.c_uint8, C.c_int32,
                                             C.c_uint8, P, S, C.c_uint8, P, P, S, P]
        L.hs_op_attend_paged_workspace.argtypes = [S] * 6
        L.hs_op_attend_paged_workspace.restype = S
        L.hs_op_score_dev.argtypes = [P, P, U32, S, P, P, S, S, S, S, P, P, P, P, P, P]
        L.hs_batch_run_scored.argtypes = [P, P, P, S, S, P, P, P, P, P]
        L.hs_batch_run_tree_scored.argtypes = [P, P, P, P, S, S, P, P, P, P, P]
        L.hs_read_bw.argtypes = [P, S, S, C.POINTER(C.c_uint64)]
        L.hs_probe_issue.argtypes = [P, C.c_uint32, C.c_uint32, C.c_uint32, C.POINTER(C.c_uint64)]
        L.hs_model_load_with.argtypes = [P, P, S, P, C.POINTER(P)]
        L.hs_batch_run_without_readback.argtypes = [P, P, S]
        L.hs_device_kernel_resources.argtypes = [P, P, P, P, P, S, C.POINTER(S)]
        L.hs_device_alloc.argtypes = [P, S, C.POINTER(P)]
        L.hs_device_free.argtypes = [P, P]
        L.hs_device_upload.argtypes = [P, P, P, S]
        L.hs_device_download.argtypes = [P, P, P, S]
        L.hs_device_synchronize.argtypes = [P]
        L.hs_device_copy.argtypes = [P, P, P, S]
        L.hs_op_gemm_requant_gpu_ns.argtypes = [P, P, P, P, P, C.c_uint8, S, S, S, P, S,
                                                C.POINTER(U64)]
        L.hs_op_attend_decode_gpu_ns.argtypes = [P, P, P, P, P, S, S, S, S, C.c_int32,
                                                 C.c_uint8, C.c_int32, C.c_uint8, P, S,
                                                 C.c_uint8, P, S, C.POINTER(U64)]
        L.hs_op_attend_decode_sets_gpu_ns.argtypes = [P, P, P, P, S, P, S, S, S, S, C.c_int32,
                                                      C.c_uint8, C.c_int32, C.c_uint8, P, S,
                                                      C.c_uint8, P, C.POINTER(U64)]
        L.hs_batch_set_profiling.argtypes = [P, C.c_int]
        L.hs_batch_profile.restype = S
        L.hs_batch_profile.argtypes = [P, P, P, P, P, S, C.c_int]
        L.hs_batch_model.restype = P
        L.hs_batch_model.argtypes = [P]
        L.hs_model_validate.argtypes = [P, S, P]
        L.hs_op_coder.argtypes = [P, P, S, S, P, S, P, U32, P]
        L.hs_batch_run_coded_mixed.argtypes = [P, P, P, P, S, U32, MIXER_FN, P, P]
        L.hs_batch_run_coded_dual.argtypes = [P, P, P, P, S, U32, MIXER_FN, P, P, P]
        L.hs_batch_run_tree_weights.argtypes = [P, P, P, S, P]
        L.hs_batch_run_tree_coded.argtypes = [P, P, P, P, S, U32, P]
        L.hs_batch_commit_paths.argtypes = [P, P, P, P, S]
        L.hs_op_mixed_coder.argtypes = [P, P, S, S, P, P, U32, MIXER_FN, P, P, P]
        L.hs_op_mixed_coder_logits.argtypes = [P, P, S, S, P, S, P, P, U32, MIXER_FN, P, P, P]
        _lib = L
    return _lib


def _check(status: int):
    if status != HS_OK:
        L = lib()
        msg = L.hs_last_error_message().decode(errors="replace")
        raise _ERRORS.get(status, HipError)(status, L.hs_last_error_code(), msg)


def _ptr(a: np.ndarray):
    return a.ctypes.data_as(C.c_void_p)


def version() -> str:
    return lib().hs_version().decode()


class HipDevice:
    """CudaDevice (crates/hardshell-cuda/src/device.rs:29-74)."""

    def __init__(self, ordinal: int = 0):
        h = C.c_void_p()
        _check(lib().hs_device_open(ordinal, C.byref(h)))
        self.h = h

    @classmethod
    def open(cls, ordinal: int = 0) -> "HipDevice":
        return cls(ordinal)

    def name(self) -> str:
        buf = C.create_string_buffer(256)
        _check(lib().hs_device_name(self.h, buf, 256))
        return buf.value.decode()

    def memory(self) -> Tuple[int, int]:
        f, t = C.c_size_t(), C.c_size_t()
        _check(lib().hs_device_memory(self.h, C.byref(f), C.byref(t)))
        return f.value, t.value

    def close(self):
        if getattr(self, "h", None):
            lib().hs_device_close(self.h)
            self.h = None

    def __del__(self):
        self.close()


class HipModel:
    """CudaModel (crates/hardshell-cuda/src/model.rs:242-398)."""

    def __init__(self, dev: HipDevice, data: bytes, loaded: Optional["HipModel"] = None):
        self.dev = dev  # the device outlives the model
        buf = np.frombuffer(data, dtype=np.uint8)
        h = C.c_void_p()
        if loaded is None:
            _check(lib().hs_model_load(dev.h, _ptr(buf), len(buf), C.byref(h)))
        else:
            _check(lib().hs_model_load_with(dev.h, _ptr(buf), len(buf), loaded.h, C.byref(h)))
        self.h = h

    @classmethod
    def load(cls, dev: HipDevice, data: bytes) -> "HipModel":
        return cls(dev, data)

    @classmethod
    def load_with(cls, dev: HipDevice, data: bytes, loaded: "HipModel") -> "HipModel":
        """CudaModel::load_with (model.rs:259-349): reuses the parse of `loaded` when the bytes
        are its file."""
        return cls(dev, data, loaded)

    def hash(self) -> bytes:
        out = np.zeros(32, np.uint8)
        lib().hs_model_hash(self.h, _ptr(out))
        return out.tobytes()

    def vocab_size(self) -> int:
        return lib().hs_model_vocab(self.h)

    def n_ctx(self) -> int:
        return lib().hs_model_n_ctx(self.h)

    def eot_token(self) -> int:
        return lib().hs_model_eot(self.h)

    def is_wide(self) -> bool:
        return bool(lib().hs_model_is_wide(self.h))

    def weight_bytes(self) -> int:
        return lib().hs_model_weight_bytes(self.h)

    def cache_bytes_per_slot(self) -> int:
        return lib().hs_model_cache_bytes_per_slot(self.h)

    def free(self):
        if getattr(self, "h", None):
            lib().hs_model_free(self.h)
            self.h = None

    def __del__(self):
        self.free()


@dataclass(frozen=True)
class CoderInterval:
    """CoderInterval (crates/hardshell-cuda/src/batch.rs:49-58)."""
    symbol: int
    start: int
    freq: int
    is_last: bool


ENCODE, DECODE = 0, 1


_U32 = 0xFFFFFFFF


def _u32(x) -> np.ndarray:
    """x as u32. Whole numbers that 32 bits do not hold become 2^32 - 1, which is no slot, token or node (the
    library refuses it), where a cast would bring them round to one."""
    a = np.asarray(x)
    b = np.ascontiguousarray(a, dtype=np.uint32) if a.dtype.kind != "O" else \
        np.array([int(v) if 0 <= int(v) <= _U32 else _U32 for v in a.ravel()], np.uint32).reshape(a.shape)
    if a.dtype.kind in "iu" and a.dtype.itemsize > 4 and not np.array_equal(a, b):
        b = np.where((a < 0) | (a > _U32), _U32, a).astype(np.uint32)
    return b


def _inputs(inputs: Sequence[Tuple[int, int]]) -> np.ndarray:
    return _u32(inputs).reshape(-1, 2)


def _queries(queries) -> np.ndarray:
    a = np.asarray(queries)
    q = _u32(a).reshape(-1, 2)
    if a.dtype != np.uint32 and a.size and not np.array_equal(a.reshape(-1, 2), q):
        raise Unsupported(HS_UNSUPPORTED, 0, "a query that 32 bits do not hold")
    return q


class Scores(NamedTuple):
    """What HipBatch.run_scored gives of each input, as arrays: float32 logprob [n] and u32 rank [n] (None without
    tokens), float32 entropy [n], u32 top_tokens and float32 top_logprob [n, top]."""
    logprob: Optional[np.ndarray]
    rank: Optional[np.ndarray]
    entropy: np.ndarray
    top_tokens: np.ndarray
    top_logprob: np.ndarray


def _whole(tokens, n: int) -> np.ndarray:
    """The n tokens of a scored call as whole numbers: None is -1, and what is no whole number is refused."""
    t = np.asarray(tokens)
    if t.shape not in ((n,), (n, 1)):
        raise LengthMismatch(HS_LENGTH_MISMATCH, 0, f"length mismatch: expected {n}, found {' x '.join(map(str, t.shape)) or 'one'}")
    t = t.reshape(n)
    if t.dtype.kind in "iu":
        return t
    given = [-1 if x is None else x for x in t.tolist()]
    try:
        whole = [int(x) for x in given]
    except (TypeError, ValueError, OverflowError):
        whole = None
    if whole != given:
        raise Unsupported(HS_UNSUPPORTED, 0, "a scored token that is no whole number")
    return np.array(whole, object)


class HipBatch:
    """CudaBatch (crates/hardshell-cuda/src/batch.rs:237-476)."""

    def __init__(self, model: HipModel, slots: int, max_rows: int):
        self.model = model
        h = C.c_void_p()
        _check(lib().hs_batch_new(model.h, slots, max_rows, C.byref(h)))
        self.h = h
        self.vocab = model.vocab_size()

    def set_overlap(self, k: int):
        _check(lib().hs_batch_set_overlap(self.h, k))

    def slots(self) -> int:
        return lib().hs_batch_slots(self.h)

    def max_rows(self) -> int:
        return lib().hs_batch_max_rows(self.h)

    def gpu_bytes(self) -> int:
        return lib().hs_batch_gpu_bytes(self.h)

    def position(self, slot: int) -> int:
        return lib().hs_batch_position(self.h, slot)

    def reset(self, slot: int):
        lib().hs_batch_reset(self.h, slot)

    def run_without_readback(self, inputs) -> None:
        """CudaBatch::run_without_readback (batch.rs:478-484)."""
        a = _inputs(inputs)
        _check(lib().hs_batch_run_without_readback(self.h, _ptr(a), len(a)))

    def run_weights(self, inputs) -> np.ndarray:
        a = _inputs(inputs)
        out = np.zeros((len(a), self.vocab), np.uint64)
        _check(lib().hs_batch_run_weights(self.h, _ptr(a), len(a), _ptr(out)))
        return out

    def run_coded_raw(self, inputs, queries, freq_bits: int = 32) -> np.ndarray:
        """The intervals as an [n, 3] u64 array (symbol, start, freq)."""
        a = _inputs(inputs)
        q = _queries(queries)
        if len(q) != len(a):
            raise LengthMismatch(HS_LENGTH_MISMATCH, 0,
                                 f"length mismatch: expected {len(a)}, found {len(q)}")
        out = np.zeros((len(a), 3), np.uint64)
        _check(lib().hs_batch_run_coded(self.h, _ptr(a), _ptr(q), len(a), freq_bits, _ptr(out)))
        return out

    def run_coded(self, inputs, queries, freq_bits: int = 32) -> List[CoderInterval]:
        raw = self.run_coded_raw(inputs, queries, freq_bits)
        return [CoderInterval(int(s), int(st), int(f), int(s) + 1 == self.vocab) for s, st, f in raw]

    def run_coded_mixed(self, inputs, queries, tables, freq_bits, mixer) -> np.ndarray:
        """CudaBatch::run_coded_mixed: tables[i] is HS_MIX_PLAIN, HS_MIX_NONE or the predicted
        token; mixer(i, stats) -> q. The intervals as an [n, 3] u64 array."""
        a = _inputs(inputs)
        q = _queries(queries)
        t = np.ascontiguousarray(np.asarray(tables, dtype=np.uint32))
        out = np.zeros((len(a), 3), np.uint64)
        cb = _mixer(mixer)
        _check(lib().hs_batch_run_coded_mixed(self.h, _ptr(a), _ptr(q), _ptr(t), len(a), freq_bits,
                                              cb, None, _ptr(out)))
        return out

    def run_coded_dual(self, inputs, tokens, predictions, freq_bits, mixer):
        """CudaBatch::run_coded_dual: (plain, mixed) intervals as two [n, 3] u64 arrays;
        predictions[i] is a token or HS_MIX_NONE."""
        a = _inputs(inputs)
        tk = np.ascontiguousarray(np.asarray(tokens, dtype=np.uint32))
        pr = np.ascontiguousarray(np.asarray(predictions, dtype=np.uint32))
        plain = np.zeros((len(a), 3), np.uint64)
        mixed = np.zeros((len(a), 3), np.uint64)
        cb = _mixer(mixer)
        _check(lib().hs_batch_run_coded_dual(self.h, _ptr(a), _ptr(tk), _ptr(pr), len(a), freq_bits,
                                             cb, None, _ptr(plain), _ptr(mixed)))
        return plain, mixed

    def _parents(self, parents, n: int) -> np.ndarray:
        """The parents for the library: -1 and HS_TREE_ROOT are the root, any other number that is no input of the call
        becomes n, which is none either (the library refuses it)."""
        p = np.asarray(parents)
        if len(p) != n:
            raise LengthMismatch(HS_LENGTH_MISMATCH, 0, f"length mismatch: expected {n}, found {len(p)}")
        if p.dtype.kind not in "iuO":
            p = p.astype(np.int64)
        root = (p == -1) | (p == HS_TREE_ROOT)
        return np.where(root, HS_TREE_ROOT, np.where((p < 0) | (p > n), n, p)).astype(np.uint32)

    def run_tree_weights(self, inputs, parents) -> np.ndarray:
        """The weights of every node of the slots' trees of drafts (hs_batch_run_tree_weights):
        parents[i] is the index of an earlier input of the same slot, or -1. No position changes."""
        a = _inputs(inputs)
        p = self._parents(parents, len(a))
        out = np.zeros((len(a), self.vocab), np.uint64)
        _check(lib().hs_batch_run_tree_weights(self.h, _ptr(a), _ptr(p), len(a), _ptr(out)))
        return out

    def run_tree_coded_raw(self, inputs, parents, queries, freq_bits: int = 32) -> np.ndarray:
        """The intervals of every node's query as an [n, 3] u64 array (hs_batch_run_tree_coded)."""
        a = _inputs(inputs)
        p = self._parents(parents, len(a))
        q = _queries(queries)
        if len(q) != len(a):
            raise LengthMismatch(HS_LENGTH_MISMATCH, 0, f"length mismatch: expected {len(a)}, found {len(q)}")
        out = np.zeros((len(a), 3), np.uint64)
        _check(lib().hs_batch_run_tree_coded(self.h, _ptr(a), _ptr(p), _ptr(q), len(a), freq_bits, _ptr(out)))
        return out

    def _scored(self, n: int, tokens, top: int, call) -> Scores:
        if not 0 <= top <= 64:
            raise Unsupported(HS_UNSUPPORTED, 0, "top is at most 64, and at most the vocabulary")
        t = None
        if tokens is not None:
            t = _whole(tokens, n)
            # other numbers that 32 bits do not hold become the vocabulary's size, which is no symbol either
            none = (t == -1) | (t == HS_NO_TOKEN)
            t = np.where(none, HS_NO_TOKEN, np.where((t < 0) | (t > self.vocab), self.vocab, t)).astype(np.uint32)
        out = Scores(None if t is None else np.zeros(n, np.float32), None if t is None else np.zeros(n, np.uint32),
                     np.zeros(n, np.float32), np.zeros((n, top), np.uint32), np.zeros((n, top), np.float32))
        _check(call(None if t is None else _ptr(t), *[None if x is None else _ptr(x) for x in out]))
        return out

    def run_scored(self, inputs, tokens=None, top: int = 0) -> Scores:
        """Runs the inputs and scores what follows each (hs_batch_run_scored): the log probability and rank of
        tokens[i] (None, -1 or HS_NO_TOKEN: none), the entropy, and the first `top` alternatives."""
        a = _inputs(inputs)
        return self._scored(len(a), tokens, top, lambda t, *out: lib().hs_batch_run_scored(
            self.h, _ptr(a), t, len(a), top, *out))

    def run_tree_scored(self, inputs, parents, tokens=None, top: int = 0) -> Scores:
        """run_scored for every node of the slots' trees of drafts; parents as in run_tree_weights."""
        a = _inputs(inputs)
        p = self._parents(parents, len(a))
        return self._scored(len(a), tokens, top, lambda t, *out: lib().hs_batch_run_tree_scored(
            self.h, _ptr(a), _ptr(p), t, len(a), top, *out))

    def commit_paths(self, paths) -> None:
        """Accepts a path of the last tree of each slot: {slot: node numbers in the slot's tree, from a child
        of the root down} (hs_batch_commit_paths)."""
        slots = _u32(list(paths))
        lengths = np.array([len(p) for p in paths.values()], np.uint32)
        flat = _u32([int(x) for p in paths.values() for x in p])
        _check(lib().hs_batch_commit_paths(self.h, _ptr(slots), _ptr(lengths), _ptr(flat), len(slots)))

    def step(self, inputs):
        a = _inputs(inputs)
        _check(lib().hs_batch_step(self.h, _ptr(a), len(a)))

    def weights(self, slot: int) -> np.ndarray:
        out = np.zeros(self.vocab, np.uint64)
        _check(lib().hs_batch_weights(self.h, slot, _ptr(out)))
        return out

    def stream_len(self, slot: int) -> int:
        return lib().hs_batch_stream_len(self.h, slot)

    def room(self, slot: int) -> int:
        return lib().hs_batch_room(self.h, slot)

    def truncate(self, slot: int, length: int):
        _check(lib().hs_batch_truncate(self.h, slot, length))

    def free(self):
        if getattr(self, "h", None):
            lib().hs_batch_free(self.h)
            self.h = None

    def __del__(self):
        self.free()


class HipSession:
    """CudaSession (crates/hardshell-cuda/src/session.rs:20-91): a batch of one slot with the
    API shape of hardshell::gpt2::Session."""

    def __init__(self, model: HipModel, overlap: int = 0, max_rows: int = 64):
        self.batch = HipBatch(model, 1, max_rows)
        if overlap:
            self.batch.set_overlap(overlap)
        self.eot = model.eot_token()

    def start_block(self) -> np.ndarray:
        self.batch.reset(0)
        return self.batch.run_weights([(0, self.eot)])[0]

    def step(self, token: int) -> np.ndarray:
        return self.batch.run_weights([(0, token)])[0]

    def step_many(self, tokens: Iterable[int]) -> np.ndarray:
        return self.batch.run_weights([(0, t) for t in tokens])

    def position(self) -> int:
        return self.batch.position(0)


def matmul_i8(dev: HipDevice, w: np.ndarray, a: np.ndarray) -> np.ndarray:
    """ops.rs:142-161: out[i][r] = w[r] . a[i], exact i32."""
    w = np.ascontiguousarray(w, dtype=np.int8)
    a = np.ascontiguousarray(a, dtype=np.int8)
    n, k = w.shape
    m = a.shape[0]
    out = np.zeros((m, n), np.int32)
    _check(lib().hs_op_gemm_i8(dev.h, _ptr(w), _ptr(a), m, n, k, _ptr(out)))
    return out


def matmul_i8_split(dev: HipDevice, w: np.ndarray, a: np.ndarray, splits: int) -> np.ndarray:
    """ops.rs:163-184: matmul_i8 with K in `splits` slices whose partials are summed."""
    w = np.ascontiguousarray(w, dtype=np.int8)
    a = np.ascontiguousarray(a, dtype=np.int8)
    n, k = w.shape
    m = a.shape[0]
    out = np.zeros((m, n), np.int32)
    _check(lib().hs_op_gemm_i8_split(dev.h, _ptr(w), _ptr(a), m, n, k, splits, _ptr(out)))
    return out


def matmul_i8_i16(dev: HipDevice, w: np.ndarray, a: np.ndarray, splits: int = 1) -> np.ndarray:
    """ops.rs:220-282: out[i][r] = w[r] . a[i] for i16 activations, exact i64."""
    w = np.ascontiguousarray(w, dtype=np.int8)
    a = np.ascontiguousarray(a, dtype=np.int16)
    n, k = w.shape
    m = a.shape[0]
    out = np.zeros((m, n), np.int64)
    _check(lib().hs_op_gemm_i8_i16(dev.h, _ptr(w), _ptr(a), m, n, k, splits, _ptr(out)))
    return out


def gemm_requant_i8(dev: HipDevice, w, a, bias, mult, shift: int) -> np.ndarray:
    w = np.ascontiguousarray(w, dtype=np.int8)
    a = np.ascontiguousarray(a, dtype=np.int8)
    bias = np.ascontiguousarray(bias, dtype=np.int32)
    mult = np.ascontiguousarray(mult, dtype=np.int32)
    n, k = w.shape
    m = a.shape[0]
    out = np.zeros((m, n), np.int8)
    _check(lib().hs_op_gemm_requant_i8(dev.h, _ptr(w), _ptr(a), _ptr(bias), _ptr(mult), shift,
                                       m, n, k, _ptr(out)))
    return out


def _on_gpu(x) -> bool:
    """Whether x is a tensor, on the GPU (one in host memory is refused)."""
    cuda = getattr(x, "is_cuda", None)
    if cuda is None:
        return hasattr(x, "data_ptr")
    if not cuda:
        raise ValueError("a tensor in host memory where the GPU reads or writes")
    return True


def _dptr(x):
    """The device address of x: a contiguous tensor on the GPU (data_ptr()), an address or a ctypes pointer, or None."""
    cuda = getattr(x, "is_cuda", None)
    if cuda is None and not hasattr(x, "data_ptr"):
        return x
    if cuda is not None and not cuda:
        raise ValueError("a tensor in host memory where the GPU reads or writes")
    if not x.is_contiguous():
        raise ValueError("a tensor with strides of its own: the operators take contiguous ones")
    return x.data_ptr()


_kinds = {}  # a tensor's type: "i" or "f" for integers or floats, and the bytes of an element


def _held(x, kind: str, n: int):
    """_dptr of a tensor that has to hold `n` elements or more of `kind` ("i4": 32-bit integers). Of an address nothing is known."""
    if getattr(x, "is_cuda", False) is not True:
        return _dptr(x)
    own = _kinds.get(x.dtype) or _kind_of(x)
    if own != kind or x.numel() < n:
        raise ValueError(f"a tensor of {x.numel()} {own} where the call reads or writes {n} {kind} "
                         "(integers or floats, bytes of an element)")
    if not x.is_contiguous():
        return _dptr(x)
    return x.data_ptr()


def _kind_of(x) -> str:
    name = str(x.dtype)
    own = _kinds[x.dtype] = ("i" if "int" in name else "f" if "float" in name else "?") + str(x.element_size())
    return own


def _dptrs(xs):
    """The layers' device addresses as a host array, from a list of them or from one contiguous tensor
    whose first axis is the layers."""
    if hasattr(xs, "data_ptr"):
        n, at = xs.shape[0], _dptr(xs)
        step = xs.stride(0) * xs.element_size() if n != 1 else 1  # (the stride of an axis of one may be anything)
        return (C.c_void_p * n)(*range(at, at + n * step, step)) if step else (C.c_void_p * 0)()
    return (C.c_void_p * len(xs))(*[_dptr(x) for x in xs])


class _Rule(NamedTuple):
    score_m: int
    score_s: int
    out_m: int
    out_s: int
    attn_exp: object
    length: int
    softmax_p: int


class AttentionRule(_Rule):
    """The integer rule of an attention layer: score = clamp(rescale(q . k, score_m, score_s), +-2^40),
    weights of softmax_p bits over the device table attn_exp of `length` i32 entries, outputs rescaled
    by (out_m, out_s). Multipliers are 32 bits, shifts and softmax_p 8 (checked here, where a call would cut them)."""
    __slots__ = ()

    def __new__(cls, score_m, score_s, out_m, out_s, attn_exp, length, softmax_p):
        if not (-2 ** 31 <= score_m < 2 ** 31 and -2 ** 31 <= out_m < 2 ** 31 and 0 <= score_s < 256 and
                0 <= out_s < 256 and 0 <= softmax_p < 256 and 0 <= length < 2 ** 64):
            raise Unsupported(HS_UNSUPPORTED, 0, "a rule whose multipliers (i32), shifts (u8) or table do not fit")
        return tuple.__new__(cls, (score_m, score_s, out_m, out_s, attn_exp, length, softmax_p))

    @classmethod
    def _make(cls, fields):
        return cls(*fields)


def attend_tree(dev: HipDevice, q, k_cache, v_cache, ctx, nodes, mask, dims, rule: AttentionRule, out,
                workspace=None, workspace_bytes: int = 0, stream=None) -> None:
    """Attention of each stream's tree of drafted tokens over its cache (hs_op_attend_tree_dev): dims =
    (streams, t, heads, head_dim, ctx_cap); nodes may be None (t each); `tree_mask` builds the mask."""
    m, s, om, os_, table, length, p = rule
    _check(lib().hs_op_attend_tree_dev(dev.h, _dptr(q), _dptr(k_cache), _dptr(v_cache), _dptr(ctx), _dptr(nodes),
                                       _dptr(mask), *dims, m, s, om, os_, _dptr(table), length, p, _dptr(out),
                                       _dptr(workspace), workspace_bytes, stream))


def attend_mass(dev: HipDevice, q, k_cache, v_cache, ctx, rows, mass, dims, rule: AttentionRule, out,
                workspace=None, workspace_bytes: int = 0, stream=None) -> None:
    """Causal attention of the last rows of each stream that adds every key's weights to the u64
    accumulators `mass` (hs_op_attend_mass_dev); dims as in attend_tree, rows may be None (t each)."""
    m, s, om, os_, table, length, p = rule
    _check(lib().hs_op_attend_mass_dev(dev.h, _dptr(q), _dptr(k_cache), _dptr(v_cache), _dptr(ctx), _dptr(rows),
                                       _dptr(mass), *dims, m, s, om, os_, _dptr(table), length, p, _dptr(out),
                                       _dptr(workspace), workspace_bytes, stream))


def attend_rows_workspace(streams: int, t: int, heads: int, head_dim: int, ctx_cap: int) -> int:
    """The bytes of workspace of attend_tree and attend_mass (hs_op_attend_rows_workspace)."""
    return lib().hs_op_attend_rows_workspace(streams, t, heads, head_dim, ctx_cap)


def tree_mask(parents) -> np.ndarray:
    """The ancestor mask [t, ceil(t / 64)] u64 of a tree given as each node's parent (-1: the context's
    end), parents before children."""
    t = len(parents)
    sees = np.zeros((t, (t + 63) // 64 * 64), bool)
    for i, p in enumerate(parents):
        if not -1 <= p < i:
            raise ValueError(f"the parent of node {i} is {p}: parents come before their children")
        if p >= 0:
            sees[i] = sees[p]
        sees[i, i] = True
    return np.packbits(sees, axis=1, bitorder="little").view(np.uint64)


def cache_evict(dev: HipDevice, k_caches, v_caches, mass, ctx, dims, budget: int, recent: int, mass_out, ctx_out,
                kept=None, stream=None) -> None:
    """Cuts the caches (a list of one a layer, or one tensor of all) to `budget` keys by accumulated weight, in
    place (hs_op_cache_evict_dev): dims = (streams, heads, head_dim, ctx_cap)."""
    k, v = _dptrs(k_caches), _dptrs(v_caches)
    if len(k) != len(v):
        raise LengthMismatch(HS_LENGTH_MISMATCH, 0, f"length mismatch: expected {len(k)}, found {len(v)}")
    _check(lib().hs_op_cache_evict_dev(dev.h, k, v, len(k), _dptr(mass), _dptr(ctx), *dims, budget, recent,
                                       _dptr(mass_out), _dptr(ctx_out), _dptr(kept), stream))


def cache_commit(dev: HipDevice, k_caches, v_caches, ctx, path, accepted, dims, ctx_out, stream=None) -> None:
    """Moves the rows of each stream's accepted path behind its context in every layer's cache
    (hs_op_cache_commit_dev): dims = (streams, t, heads, head_dim, ctx_cap)."""
    k, v = _dptrs(k_caches), _dptrs(v_caches)
    if len(k) != len(v):
        raise LengthMismatch(HS_LENGTH_MISMATCH, 0, f"length mismatch: expected {len(k)}, found {len(v)}")
    _check(lib().hs_op_cache_commit_dev(dev.h, k, v, len(k), _dptr(ctx), _dptr(path), _dptr(accepted), *dims,
                                        _dptr(ctx_out), stream))


class _Pages(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p),
                ("pages", C.c_uint32), ("kv_heads", C.c_uint32), ("page", C.c_uint32), ("head_dim", C.c_uint32),
                ("max_scale", C.c_uint32)]


class PagedCache(NamedTuple):
    """One layer's pool of pages (hs_pages): int8 k and v [pages, kv_heads, page, head_dim], 32-bit k_scale and
    v_scale [pages, kv_heads], on the device; scales up to max_scale."""
    k: object
    v: object
    k_scale: object
    v_scale: object
    pages: int
    kv_heads: int
    page: int
    head_dim: int
    max_scale: int

    def _struct(self):
        k, v, ks, vs, pages, heads, page, hd, most = self
        if not (0 <= pages <= _U32 and 0 <= heads <= _U32 and 0 <= page <= _U32 and 0 <= hd <= _U32 and 0 <= most <= _U32):
            raise Unsupported(HS_UNSUPPORTED, 0, "a size that 32 bits do not hold")
        n = pages * heads
        values = n * page * hd
        return _Pages(_held(k, "i1", values), _held(v, "i1", values), _held(ks, "i4", n), _held(vs, "i4", n),
                      pages, heads, page, hd, most)


def _sizes(*numbers):
    """Sizes for the library; a negative one would come round to a large one."""
    if min(numbers) < 0:
        raise Unsupported(HS_UNSUPPORTED, 0, "a negative size")
    return numbers


_types = {}  # the bits of a tensor's type, 0 where it does not hold signed integers


def _bits_of(x) -> int:
    dtype = x.dtype
    bits = _types.get(dtype)
    if bits is None:
        name = str(dtype)
        bits = _types[dtype] = 8 * x.element_size() if "int" in name and "uint" not in name else 0
    return bits


def _rows_of(x, bits: Optional[int], stride: Optional[int], shape):
    """Rows of new tokens as (address, bits of a value, elements from one token to the next): a tensor [streams, t, heads,
    head_dim] on the GPU whose heads of a token lie together and whose tokens at one distance, or an address with
    `bits` and `stride` (None: the rows lie together)."""
    b, t, h, hd = shape
    if getattr(x, "is_cuda", False) is not True and not _on_gpu(x):
        return x, bits or 0, h * hd if stride is None else stride
    st, own = x.stride(), _types.get(x.dtype)
    if own is None:
        own = _bits_of(x)
    if x.shape != shape or own == 0 or (bits is not None and bits != own):
        raise ValueError(f"a tensor that does not hold {tuple(shape)} integers of the operator's types")
    step = st[1] if t > 1 else st[0] if b > 1 else h * hd
    if (h > 1 and st[2] != hd) or (hd > 1 and st[3] != 1) or (b > 1 and st[0] != t * step) or \
            (stride is not None and stride != step):
        raise ValueError("a tensor whose tokens do not lie at one distance, each with its heads together")
    return x.data_ptr(), own, step


def pages_append(dev: HipDevice, cache: PagedCache, k, v, table, ctx, rows, dims, headroom: int = 16, ctx_out=None,
                 bits: Optional[int] = None, stride: Optional[int] = None, stream=None) -> None:
    """Appends rows of keys and values to the streams' pages (hs_op_pages_append_dev): dims = (streams, t, width);
    k and v are tensors [streams, t, kv_heads, head_dim] of int8 or int16, or addresses with `bits` and `stride`."""
    b, t, width = dims
    if b < 0 or t < 0 or width < 0:
        _sizes(b, t, width)
    shape = (b, t, cache.kv_heads, cache.head_dim)
    kp, kb, ks = _rows_of(k, bits, stride, shape)
    vp, vb, vs = _rows_of(v, bits, stride, shape)
    if ks != vs or kb != vb:
        raise ValueError("k and v of different types, or with tokens at different distances")
    if ks < 0:
        _sizes(ks)
    if not 0 <= headroom <= _U32:
        raise Unsupported(HS_UNSUPPORTED, 0, "headroom must be in 16..=64 sixteenths")
    _check(lib().hs_op_pages_append_dev(dev.h, C.byref(cache._struct()), kp, vp, kb, ks, _held(table, "i4", b * width),
                                        _held(ctx, "i4", b), _held(rows, "i4", b), b, t, width, headroom,
                                        _held(ctx_out, "i4", b), stream))


def attend_paged(dev: HipDevice, cache: PagedCache, q, table, ctx, rows, dims, rule: AttentionRule, out,
                 q_stride: Optional[int] = None, workspace=None, workspace_bytes: int = 0, stream=None) -> None:
    """Causal attention over the streams' pages (hs_op_attend_paged_dev): dims = (streams, t, heads, width, keys);
    q is a tensor [streams, t, heads, head_dim] of int8, or an address with `q_stride`; rows may be None (t each)."""
    b, t, heads, width, keys = dims
    if b < 0 or t < 0 or heads < 0 or width < 0 or keys < 0:
        _sizes(*dims)
    qp, bits, step = _rows_of(q, None, q_stride, (b, t, heads, cache.head_dim))
    if bits not in (0, 8):
        raise ValueError("q: [streams, t, heads, head_dim] of int8")
    if step < 0:
        _sizes(step)
    m, s, om, os_, exp, length, p = rule
    space = _dptr(workspace)
    if space is not workspace and workspace.numel() * workspace.element_size() < workspace_bytes:
        raise ValueError("a workspace of fewer bytes than the call says")
    _check(lib().hs_op_attend_paged_dev(dev.h, C.byref(cache._struct()), qp, step, _held(table, "i4", b * width),
                                        _held(ctx, "i4", b), _held(rows, "i4", b), b, t, heads, width, keys, m, s, om, os_,
                                        _held(exp, "i4", length), length, p, _held(out, "i1", b * t * heads * cache.head_dim),
                                        space, workspace_bytes, stream))


def attend_paged_workspace(streams: int, t: int, heads: int, kv_heads: int, head_dim: int, keys: int) -> int:
    """The bytes of workspace of attend_paged (hs_op_attend_paged_workspace)."""
    return lib().hs_op_attend_paged_workspace(*_sizes(streams, t, heads, kv_heads, head_dim, keys))


def score_tokens(dev: HipDevice, logits, tokens, table, dims, top: int, logprob, rank, entropy, top_tokens, top_logprob,
                 bits: Optional[int] = None, stride: Optional[int] = None, stream=None) -> None:
    """The scores of rows of logits on the device (hs_op_score_dev): dims = (rows, vocab, table length); logits is a
    tensor [rows, vocab] of int32 or int64 with its symbols together, or an address with `bits` and `stride`."""
    rows, vocab, length = dims
    if rows < 0 or vocab < 0 or length < 0:
        _sizes(*dims)
    if _on_gpu(logits):
        own, st = _bits_of(logits), logits.stride()
        if logits.shape != (rows, vocab) or own == 0 or (bits is not None and bits != own) or (vocab > 1 and st[1] != 1):
            raise ValueError("logits: [rows, vocab] of int32 or int64, the symbols of a row together")
        bits, stride, logits = own, st[0] if rows > 1 else vocab, logits.data_ptr()
    elif stride is None:
        stride = vocab
    if top < 0 or stride < 0:
        _sizes(top, stride)
    _check(lib().hs_op_score_dev(dev.h, logits, bits or 0, stride, _held(tokens, "i4", rows), _held(table, "i8", length), length,
                                 rows, vocab, top, _held(logprob, "f4", rows), _held(rank, "i4", rows), _held(entropy, "f4", rows),
                                 _held(top_tokens, "i4", rows * top), _held(top_logprob, "f4", rows * top), stream))


def kernel_resources(dev: HipDevice):
    """CudaDevice::kernel_resources (device.rs:65-74): (name, registers, private bytes, static
    LDS bytes) of each main kernel."""
    cap = 64
    names = (C.c_char * (64 * cap))()
    regs, priv, lds = (np.zeros(cap, np.int32) for _ in range(3))
    n = C.c_size_t()
    _check(lib().hs_device_kernel_resources(dev.h, names, _ptr(regs), _ptr(priv), _ptr(lds), cap,
                                            C.byref(n)))
    raw = bytes(names)
    return [(raw[64 * i:64 * i + 64].split(b"\0")[0].decode(), int(regs[i]), int(priv[i]), int(lds[i]))
            for i in range(min(n.value, cap))]


def read_bw(dev: HipDevice, nbytes: int, reps: int) -> float:
    """read_gpu_ns (crates/hardshell-cuda/src/ops.rs:328-335) as bytes per second: a streaming
    kernel reads a device buffer of nbytes, reps times."""
    ns = C.c_uint64()
    _check(lib().hs_read_bw(dev.h, nbytes, reps, C.byref(ns)))
    return nbytes * reps / (ns.value * 1e-9)


def probe_issue(dev: HipDevice, op: int, waves_per_simd: int, iters: int) -> int:
    """hs_probe_issue: the GPU ns of one launch of `iters` rounds of op on every SIMD."""
    ns = C.c_uint64()
    _check(lib().hs_probe_issue(dev.h, op, waves_per_simd, iters, C.byref(ns)))
    return ns.value


def gemm_layout(m: int, n: int, k: int) -> Tuple[int, int, int]:
    a, b, c = C.c_size_t(), C.c_size_t(), C.c_size_t()
    lib().hs_op_gemm_layout(m, n, k, C.byref(a), C.byref(b), C.byref(c))
    return a.value, b.value, c.value


def gemm_pack(x: np.ndarray, rows_pad: int, k_pad: int) -> np.ndarray:
    """An i8 operand [rows, k] in the layout of the _dev GEMM entries: k_pad / 64 panels of
    rows_pad rows x 64 bytes, zero padded (hs_op_gemm_layout)."""
    rows, k = x.shape
    p = np.zeros((rows_pad, k_pad), np.int8)
    p[:rows, :k] = x
    return np.ascontiguousarray(p.reshape(rows_pad, k_pad // 64, 64).transpose(1, 0, 2))


def mixed_intervals_of_weights(dev: HipDevice, weights: np.ndarray, queries, predictions,
                               freq_bits: int, mixer):
    """mixed_intervals_of_weights (mixed.rs:160-233): the statistics [rows, 3] (total,
    predicted, top) and the intervals [rows, 3] of the mixed tables of given weights."""
    w = np.ascontiguousarray(weights, dtype=np.uint64)
    rows, vocab = w.shape
    q = _queries(queries)
    pr = np.ascontiguousarray(np.asarray(predictions, dtype=np.uint32))
    stats = (MixStats * rows)()
    out = np.zeros((rows, 3), np.uint64)
    cb = _mixer(mixer)
    _check(lib().hs_op_mixed_coder(dev.h, _ptr(w), rows, vocab, _ptr(q), _ptr(pr), freq_bits, cb,
                                   None, C.cast(stats, C.c_void_p), _ptr(out)))
    st = np.array([[s.total, s.predicted, s.top] for s in stats], dtype=np.uint64).reshape(rows, 3)
    return st, out


def mixed_coder_logits(dev: HipDevice, logits: np.ndarray, table: np.ndarray, queries, tables,
                       freq_bits: int, mixer):
    """The mixed coder op on given i64 logits [rows, vocab] and a logits table (the compact
    form for tables of at most 16,384 entries): statistics [rows, 3] and intervals [rows, 3]."""
    logits = np.ascontiguousarray(logits, dtype=np.int64)
    table = np.ascontiguousarray(table, dtype=np.uint64)
    rows, vocab = logits.shape
    q = _queries(queries)
    t = np.ascontiguousarray(np.asarray(tables, dtype=np.uint32))
    stats = (MixStats * rows)()
    out = np.zeros((rows, 3), np.uint64)
    cb = _mixer(mixer)
    _check(lib().hs_op_mixed_coder_logits(dev.h, _ptr(logits), rows, vocab, _ptr(table), len(table),
                                          _ptr(q), _ptr(t), freq_bits, cb, None,
                                          C.cast(stats, C.c_void_p), _ptr(out)))
    st = np.array([[s.total, s.predicted, s.top] for s in stats], dtype=np.uint64).reshape(rows, 3)
    return st, out


def coder(dev: HipDevice, logits: np.ndarray, table: np.ndarray, queries, freq_bits: int = 32
          ) -> np.ndarray:
    """The coder op on given i64 logits [rows, vocab]: (symbol, start, freq) per row."""
    logits = np.ascontiguousarray(logits, dtype=np.int64)
    table = np.ascontiguousarray(table, dtype=np.uint64)
    q = _queries(queries)
    rows, vocab = logits.shape
    out = np.zeros((rows, 3), np.uint64)
    _check(lib().hs_op_coder(dev.h, _ptr(logits), rows, vocab, _ptr(table), len(table), _ptr(q),
                             freq_bits, _ptr(out)))
    return out
