"""ctypes binding of include/psx_b200.h.  Device memory comes from torch tensors; every compute
call goes through the C ABI into the CUDA kernels."""
from __future__ import annotations

import array
import ctypes as C
import math
import os
from pathlib import Path

import numpy as np

PACKAGE = Path(__file__).resolve().parent
ROW_OK, ROW_NON_FINITE, ROW_ALL_REMOVED, ROW_TOO_WIDE, ROW_DEVICE_TIMEOUT, ROW_CACHE_FULL, ROW_BAD_OFFSETS, ROW_BAD_TOKEN = 0, 4, 5, 16, 32, 64, 65, 66
OK, ERR_BAD_ARGUMENT, ERR_CUDA, ERR_ROW_FAILED, ERR_UNSUPPORTED = range(5)

EXPORTS = [
    "psx_b200_version", "psx_b200_last_error", "psx_b200_ctx_create", "psx_b200_ctx_destroy", "psx_b200_ctx_stream",
    "psx_b200_sync", "psx_b200_launch_count", "psx_b200_ctx_enable_timing", "psx_b200_ctx_read_timing", "psx_b200_ctx_inputs_are_ready",
    "psx_b200_ctx_set_wait_limit", "psx_b200_test_short_copy", "psx_b200_sample_rows", "psx_b200_sample_rows_host", "psx_b200_row_pass_only", "psx_b200_sample_rows_static", "psx_b200_read_only_pass", "psx_b200_process_logits", "psx_b200_process_logits_host",
    "psx_b200_shard_record_bytes", "psx_b200_shard_scan", "psx_b200_shard_merge", "psx_b200_shard_merge_rows",
    "psx_b200_exchange_handle_bytes", "psx_b200_exchange_create", "psx_b200_exchange_open", "psx_b200_exchange_destroy",
    "psx_b200_exchange_sample", "psx_b200_exchange_results", "psx_b200_exchange_test_wait",
    "psx_b200_top_k_rows", "psx_b200_lm_head_logits", "psx_b200_lm_head_sample_rows", "psx_b200_softmax_rows", "psx_b200_logsumexp_rows", "psx_b200_gather_rows", "psx_b200_decode_attention",
    "psx_b200_beam_select", "psx_b200_reorder_states", "psx_b200_store_cache_8bit", "psx_b200_decode_attention_8bit", "psx_b200_prompt_attention",
    "psx_b200_extend_pages", "psx_b200_fork_pages", "psx_b200_release_pages", "psx_b200_compact_pages", "psx_b200_rotate_heads", "psx_b200_decode_attention_pages",
    "psx_b200_token_log_probs",
    "psx_uniforms_mt19937_64", "psx_uniforms_portable",
]


class PsxError(RuntimeError):
    """A C entry point returned a non-zero psx_status.  `.status` holds it; the text is the
    library's message (the reference's own wording for its std::invalid_argument cases)."""

    def __init__(self, status, message):
        super().__init__(message)
        self.status = status


class SamplingConfig(C.Structure):
    """psx_sampling_config."""

    _fields_ = [
        ("min_new_tokens", C.c_int64),
        ("num_new_tokens", C.c_int64),
        ("eos_token_ids", C.POINTER(C.c_int64)),
        ("num_eos_token_ids", C.c_int64),
        ("do_sample", C.c_int32),
        ("temperature", C.c_float),
        ("top_k", C.c_int64),
        ("top_p", C.c_float),
        ("min_p", C.c_float),
        ("repetition_penalty", C.c_float),
    ]

    @classmethod
    def make(cls, do_sample=False, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, repetition_penalty=1.0,
             min_new_tokens=0, num_new_tokens=0, eos_token_ids=()):
        eos = np.asarray(list(eos_token_ids), dtype=np.int64)
        cfg = cls(min_new_tokens, num_new_tokens, eos.ctypes.data_as(C.POINTER(C.c_int64)), len(eos), int(do_sample),
                  temperature, top_k, top_p, min_p, repetition_penalty)
        cfg._keepalive = eos
        return cfg


class RowDiag(C.Structure):
    """psx_row_diag."""

    _fields_ = [("candidates", C.c_int32), ("survivors", C.c_int32), ("draw_margin", C.c_double),
                ("top_p_margin", C.c_double)]


ROW_DIAG_DTYPE = np.dtype({"names": ["candidates", "survivors", "draw_margin", "top_p_margin"],
                           "formats": ["<i4", "<i4", "<f8", "<f8"], "itemsize": C.sizeof(RowDiag)})


class BeamState(C.Structure):
    """psx_beam_state."""

    _fields_ = [("data", C.c_void_p), ("heads", C.c_int64), ("positions", C.c_int64), ("position_bytes", C.c_int64),
                ("tokens_per_position", C.c_int64)]


class Cache8bitLayout(C.Structure):
    """psx_cache_8bit."""

    _fields_ = [("key_codes", C.c_void_p), ("key_scales", C.c_void_p), ("value_codes", C.c_void_p), ("value_scales", C.c_void_p),
                ("batch", C.c_int64), ("kv_heads", C.c_int64), ("max_len", C.c_int64), ("head_dim", C.c_int64), ("block", C.c_int64)]


class PageTableLayout(C.Structure):
    """psx_page_table."""

    _fields_ = [("pages", C.c_void_p), ("lengths", C.c_void_p), ("references", C.c_void_p), ("rows", C.c_int64), ("max_pages", C.c_int64),
                ("num_pages", C.c_int64), ("page_size", C.c_int64)]


class PagedCacheLayout(C.Structure):
    """psx_paged_cache."""

    _fields_ = [("table", PageTableLayout), ("key_pages", C.c_void_p), ("value_pages", C.c_void_p), ("kv_heads", C.c_int64), ("head_dim", C.c_int64)]


_lib = None
_native = None  # the per-step calls without ctypes (host/python_calls.cpp); bound to the same library


def library_path() -> Path:
    if os.environ.get("PSX_B200_LIBRARY"):  # a variant build (see build.py)
        return Path(os.environ["PSX_B200_LIBRARY"])
    if os.environ.get("PSX_B200_STAGE_CLOCKS") == "1":  # the profiling build (see build.py)
        return PACKAGE / "libpsx_b200_clocks.so"
    return PACKAGE / "libpsx_b200.so"


def library():
    """Loads libpsx_b200.so.  Raises when it has not been built: there is nothing to fall back to."""
    global _lib, _native
    if _lib is None:
        path = library_path()
        if not path.exists():
            raise ImportError(f"{path} is missing: build it with `python -m pulsatrix_b200.build` (needs nvcc)")
        lib = C.CDLL(str(path))
        lib.psx_b200_version.restype = C.c_char_p
        lib.psx_b200_last_error.restype = C.c_char_p
        lib.psx_b200_ctx_stream.restype = C.c_void_p
        lib.psx_b200_ctx_stream.argtypes = [C.c_void_p]
        lib.psx_b200_ctx_destroy.argtypes = [C.c_void_p]
        lib.psx_b200_launch_count.restype = C.c_uint64
        lib.psx_b200_launch_count.argtypes = [C.c_void_p]
        lib.psx_b200_shard_record_bytes.restype = C.c_size_t
        lib.psx_b200_shard_record_bytes.argtypes = [C.c_void_p]
        lib.psx_b200_ctx_create.argtypes = [C.c_int, C.c_void_p]
        lib.psx_b200_sync.argtypes = [C.c_void_p, C.c_void_p]
        lib.psx_b200_ctx_enable_timing.argtypes = [C.c_void_p, C.c_int]
        lib.psx_b200_ctx_inputs_are_ready.argtypes = [C.c_void_p, C.c_int]
        lib.psx_b200_ctx_set_wait_limit.argtypes = [C.c_void_p, C.c_uint64]
        lib.psx_b200_test_short_copy.argtypes = [C.c_void_p, C.c_int]
        lib.psx_b200_ctx_read_timing.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p]
        ptr, i64 = C.c_void_p, C.c_int64
        lib.psx_b200_sample_rows.argtypes = [ptr, ptr, ptr, i64, i64, i64, ptr, ptr, ptr, ptr, ptr, ptr, ptr, ptr]
        lib.psx_b200_sample_rows_static.argtypes = [ptr, ptr, i64, i64, i64, ptr, ptr, ptr, ptr, ptr, ptr, ptr]
        lib.psx_b200_read_only_pass.argtypes = [ptr, ptr, C.c_size_t, ptr]
        lib.psx_b200_process_logits.argtypes = [ptr, ptr, ptr, i64, i64, i64, ptr, ptr, ptr, ptr]
        lib.psx_b200_process_logits_host.argtypes = [ptr, ptr, i64, i64, i64, ptr, ptr, ptr, ptr]
        lib.psx_b200_row_pass_only.argtypes = [ptr, ptr, ptr, i64, i64, i64, ptr, ptr, ptr]
        lib.psx_b200_sample_rows_host.argtypes = [ptr, ptr, i64, i64, i64, ptr, ptr, ptr, ptr, ptr, ptr, ptr, ptr]
        lib.psx_b200_shard_scan.argtypes = [ptr, ptr, ptr, i64, i64, i64, i64, i64, ptr, ptr, ptr, ptr]
        lib.psx_b200_shard_merge.argtypes = [ptr, ptr, ptr, C.c_int32, i64, i64, ptr, ptr, ptr, ptr, ptr, ptr]
        lib.psx_b200_shard_merge_rows.argtypes = [ptr, ptr, ptr, C.c_int32, i64, i64, i64, i64, ptr, ptr, ptr, ptr, ptr, ptr]
        lib.psx_b200_exchange_handle_bytes.restype = C.c_size_t
        lib.psx_b200_exchange_handle_bytes.argtypes = []
        lib.psx_b200_exchange_create.argtypes = [ptr, C.c_int32, C.c_int32, i64, ptr, ptr, ptr]
        lib.psx_b200_exchange_open.argtypes = [ptr, ptr]
        lib.psx_b200_exchange_destroy.argtypes = [ptr]
        lib.psx_b200_exchange_destroy.restype = None
        lib.psx_b200_exchange_sample.argtypes = [ptr, ptr, ptr, i64, i64, i64, i64, ptr, ptr, ptr, ptr]
        lib.psx_b200_exchange_results.argtypes = [ptr, ptr, ptr]
        lib.psx_b200_exchange_test_wait.argtypes = [ptr, C.c_uint64, C.c_uint32]
        lib.psx_b200_top_k_rows.argtypes = [ptr, ptr, ptr, ptr, ptr, C.c_size_t, C.c_size_t, C.c_size_t, C.c_int]
        lib.psx_b200_lm_head_logits.argtypes = [ptr, ptr, ptr, i64, i64, ptr, i64, C.c_int32, ptr, i64]
        lib.psx_b200_lm_head_sample_rows.argtypes = [ptr, ptr, ptr, i64, i64, ptr, i64, C.c_int32, ptr, ptr, ptr, ptr, ptr, ptr,
                                                     ptr, ptr]
        lib.psx_b200_softmax_rows.argtypes = [ptr, ptr, ptr, ptr, C.c_size_t, C.c_size_t]
        lib.psx_b200_logsumexp_rows.argtypes = [ptr, ptr, ptr, ptr, C.c_size_t, C.c_size_t]
        lib.psx_b200_gather_rows.argtypes = [ptr, ptr, ptr, ptr, ptr, C.c_size_t, C.c_size_t]
        lib.psx_b200_decode_attention.argtypes = [ptr, ptr, ptr, ptr, ptr, ptr, ptr, i64, i64, i64, i64, i64, i64, i64, C.c_float, C.c_int32,
                                                  i64, ptr]
        lib.psx_b200_beam_select.argtypes = [ptr, ptr, ptr, i64, i64, i64, i64, ptr, ptr, i64, i64, ptr, ptr, ptr, ptr]
        lib.psx_b200_reorder_states.argtypes = [ptr, ptr, ptr, i64, i64, i64, ptr, ptr]
        lib.psx_b200_store_cache_8bit.argtypes = [ptr, ptr, ptr, ptr, ptr, C.c_int32, i64, i64, i64, ptr, ptr, ptr]
        lib.psx_b200_decode_attention_8bit.argtypes = [ptr, ptr, ptr, C.c_int32, ptr, ptr, ptr, i64, i64, C.c_float, C.c_int32, i64]
        lib.psx_b200_prompt_attention.argtypes = [ptr, ptr, C.c_int32, ptr, ptr, ptr, ptr, i64, i64, i64, i64, i64, ptr, ptr, i64, i64, i64, i64,
                                                  C.c_float, C.c_int32, i64, ptr]
        lib.psx_b200_extend_pages.argtypes = [ptr, ptr, ptr, ptr, ptr, i64, ptr]
        lib.psx_b200_fork_pages.argtypes = [ptr, ptr, ptr, ptr, i64]
        lib.psx_b200_release_pages.argtypes = [ptr, ptr, ptr, ptr]
        lib.psx_b200_compact_pages.argtypes = [ptr, ptr, ptr, ptr, i64, ptr]
        lib.psx_b200_rotate_heads.argtypes = [ptr, ptr, C.c_int32, ptr, ptr, ptr, ptr, ptr, i64, i64, i64, i64, ptr, ptr, i64, i64, i64, i64, ptr, ptr,
                                              C.c_float, ptr, i64, C.c_int32, ptr, ptr]
        lib.psx_b200_decode_attention_pages.argtypes = [ptr, ptr, ptr, C.c_int32, ptr, ptr, i64, i64, C.c_float, C.c_int32, i64]
        lib.psx_b200_token_log_probs.argtypes = [ptr, ptr, C.c_int32, ptr, i64, i64, i64, ptr, ptr, ptr, i64, ptr, ptr, ptr]
        lib.psx_uniforms_mt19937_64.argtypes = [ptr, i64, ptr]
        lib.psx_uniforms_portable.argtypes = [ptr, i64, ptr]
        from . import _native as native
        native.load(str(path))
        _native = native
        _lib = lib
    return _lib


def _stream_of(tensor):
    """The raw handle of torch's current stream on the tensor's device."""
    from torch._C import _cuda_getCurrentRawStream
    device = tensor.get_device()
    if device < 0:
        raise ValueError(f"Expected a cuda tensor, but got one on {tensor.device}")
    return _cuda_getCurrentRawStream(device)


def _zeroed_word(device, stream):
    """A one-element int32 tensor of its own, zeroed on the stream of the call that may set it."""
    import torch
    if stream is None:
        return torch.zeros(1, dtype=torch.int32, device=device)
    with torch.cuda.stream(torch.cuda.ExternalStream(stream, device=device)):
        return torch.zeros(1, dtype=torch.int32, device=device)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _host_array(a):
    """A numpy array as it is (the native calls take its address), any other host array's address."""
    if a is None or (isinstance(a, np.ndarray) and a.ndim > 0):
        return a
    return a.ctypes.data if hasattr(a, "ctypes") else a.data_ptr()


def _check(status):
    if status != OK:
        raise PsxError(status, library().psx_b200_last_error().decode())


def uniforms_mt19937_64(seeds) -> np.ndarray:
    """(std::mt19937_64(seed)() >> 11) * 2^-53 per seed: Generate()'s first draw."""
    seeds = np.ascontiguousarray(seeds, dtype=np.uint64)
    out = np.zeros(seeds.size, dtype=np.float64)
    library().psx_uniforms_mt19937_64(seeds.ctypes.data, seeds.size, out.ctypes.data)
    return out


def uniforms_portable(seeds) -> np.ndarray:
    seeds = np.ascontiguousarray(seeds, dtype=np.uint64)
    out = np.zeros(seeds.size, dtype=np.float64)
    library().psx_uniforms_portable(seeds.ctypes.data, seeds.size, out.ctypes.data)
    return out


def _dptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def read_only_pass(tensor, sink, stream=None):
    """Launches the read-only kernel over a contiguous cuda tensor (benchmark aid)."""
    if stream is None:
        import torch
        stream = torch.cuda.current_stream(tensor.device).cuda_stream
    _check(library().psx_b200_read_only_pass(C.c_void_p(stream), _dptr(tensor), tensor.numel() * tensor.element_size(),
                                             _dptr(sink)))


def sample_rows_static(logits, history_ids, history_offsets, config, uniforms, tokens, log_probs, status, stream=None,
                       vocab=None):
    """psx_b200_sample_rows_static: the sampling step without a context and without any device
    allocation (its scratch is a fixed array inside the library).  All tensors are the caller's:
    cuda inputs as for Context.sample_rows, and preallocated cuda outputs tokens (int64),
    log_probs (float32), status (int32).  Asynchronous on `stream` (default: torch's current)."""
    rows = logits.shape[0]
    vocab = logits.shape[1] if vocab is None else vocab
    if _native is None:
        library()
    status_code = _native.sample_rows_static(
        _stream_of(logits) if stream is None else stream, logits.data_ptr(), rows, vocab, logits.stride(0) if rows else vocab,
        _ptr(history_ids), _ptr(history_offsets), C.addressof(config), _ptr(uniforms), _ptr(tokens), _ptr(log_probs), _ptr(status))
    if status_code:
        _check(status_code)


_torch = None
_DTYPES = {}  # torch dtype -> psx_dtype


def _torch_module():
    """torch, imported by the first call that needs it (and looked up once: a call takes a few microseconds altogether)."""
    global _torch
    if _torch is None:
        import torch
        _DTYPES.update({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2})
        _torch = torch
    return _torch


def _dtype_code(tensor):
    """The psx_dtype of a tensor."""
    code = _DTYPES.get(tensor.dtype)
    if code is None:
        raise TypeError(f"float32, bfloat16 or float16 is expected, got {tensor.dtype}")
    return code


class Cache8bit:
    """A cache of keys and values in 8 bits (psx_cache_8bit) over tensors of the caller's: codes (batch, kv_heads, max_len,
    head_dim), torch.float8_e4m3fn or uint8, and float32 scales (batch, kv_heads, ceil(max_len / block)), all contiguous."""

    def __init__(self, key_codes, key_scales, value_codes, value_scales, block=32):
        torch = _torch or _torch_module()
        shape = key_codes.shape
        if len(shape) != 4 or block <= 0:
            raise ValueError("codes are (batch, kv_heads, max_len, head_dim)")
        batch, kv_heads, max_len, head_dim = shape
        if not (value_codes.shape == shape and key_codes.is_contiguous() and value_codes.is_contiguous() and
                key_codes.dtype in (torch.float8_e4m3fn, torch.uint8) and value_codes.dtype in (torch.float8_e4m3fn, torch.uint8)):
            raise ValueError("codes are contiguous float8_e4m3fn or uint8 tensors of one shape")
        scales = (batch, kv_heads, -(-max_len // block))
        if not (key_scales.shape == scales and value_scales.shape == scales and key_scales.is_contiguous() and value_scales.is_contiguous() and
                key_scales.dtype is torch.float32 and value_scales.dtype is torch.float32):
            raise ValueError("scales are contiguous float32 tensors, one for every `block` positions")
        self.device = device = key_codes.get_device()
        if not device == key_scales.get_device() == value_codes.get_device() == value_scales.get_device():
            raise ValueError("a cache lies on one device")
        self.key_codes, self.key_scales, self.value_codes, self.value_scales = key_codes, key_scales, value_codes, value_scales
        self.batch, self.kv_heads, self.max_len, self.head_dim, self.block = batch, kv_heads, max_len, head_dim, block
        self._layout = Cache8bitLayout(key_codes.data_ptr(), key_scales.data_ptr(), value_codes.data_ptr(), value_scales.data_ptr(), batch,
                                       kv_heads, max_len, head_dim, block)
        self._address = C.addressof(self._layout)

    @classmethod
    def empty(cls, batch, kv_heads, max_len, head_dim, block=32, device="cuda"):
        """One with nothing in it yet."""
        import torch
        codes = [torch.zeros((batch, kv_heads, max_len, head_dim), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2)]
        scales = [torch.zeros((batch, kv_heads, -(-max_len // block)), dtype=torch.float32, device=device) for _ in range(2)]
        return cls(codes[0], scales[0], codes[1], scales[1], block)

    def states(self):
        """Its tensors as Context.reorder_states takes them."""
        return [(self.key_codes, 1), (self.key_scales, self.block), (self.value_codes, 1), (self.value_scales, self.block)]


class PageTable:
    """The table of a cache in pages (psx_page_table) over tensors of the caller's: pages int32 (rows, max_pages), lengths int64 (rows),
    references int32 (num_pages), all contiguous."""

    def __init__(self, pages, lengths, references, page_size=64):
        torch = _torch or _torch_module()
        if pages.dim() != 2 or pages.dtype is not torch.int32 or not pages.is_contiguous():
            raise ValueError("pages are contiguous int32 (rows, max_pages)")
        rows, max_pages = pages.shape
        num_pages = references.numel()
        if not (lengths.dtype is torch.int64 and lengths.numel() == rows and lengths.is_contiguous() and references.dtype is torch.int32 and
                references.is_contiguous()):
            raise ValueError("lengths are int64 (rows), references int32 (num_pages)")
        self.device = device = pages.get_device()
        if not device == lengths.get_device() == references.get_device():
            raise ValueError("a page table lies on one device")
        self.pages, self.lengths, self.references = pages, lengths, references
        self.rows, self.max_pages, self.num_pages, self.page_size = rows, max_pages, num_pages, page_size
        # (PageTableLayout's words: an array is made in a third of the time)
        self._layout = array.array("q", (pages.data_ptr(), lengths.data_ptr(), references.data_ptr(), rows, max_pages, num_pages, page_size))
        self._address = self._layout.buffer_info()[0]

    @classmethod
    def empty(cls, rows, max_pages, num_pages, page_size=64, device="cuda"):
        """One whose rows hold nothing and whose pages are free."""
        import torch
        return cls(torch.full((rows, max_pages), -1, dtype=torch.int32, device=device), torch.zeros(rows, dtype=torch.int64, device=device),
                   torch.zeros(num_pages, dtype=torch.int32, device=device), page_size)


class PagedCache:
    """A layer's cache in pages (psx_paged_cache): a PageTable and two tensors of the caller's, keys and values (num_pages, kv_heads, page_size,
    head_dim), float32, bfloat16 or float16, contiguous."""

    def __init__(self, table, key_pages, value_pages):
        shape = key_pages.shape
        if len(shape) != 4 or shape[0] != table.num_pages or shape[2] != table.page_size:
            raise ValueError("pages are (num_pages, kv_heads, page_size, head_dim)")
        if not (value_pages.shape == shape and key_pages.dtype is value_pages.dtype and key_pages.is_contiguous() and value_pages.is_contiguous()):
            raise ValueError("keys and values are contiguous tensors of one shape and type")
        self.device = device = table.device
        if not device == key_pages.get_device() == value_pages.get_device():
            raise ValueError("a cache lies on one device")
        self.dtype_code = _dtype_code(key_pages)
        self.table, self.key_pages, self.value_pages = table, key_pages, value_pages
        _, self.kv_heads, _, self.head_dim = shape
        self._layout = layout = table._layout[:]  # (PagedCacheLayout's words)
        layout.extend((key_pages.data_ptr(), value_pages.data_ptr(), self.kv_heads, self.head_dim))
        self._address = layout.buffer_info()[0]

    def pools(self):
        """Its tensors as Context.extend_pages and compact_pages take them."""
        return [self.key_pages, self.value_pages]


class Context:
    """A psx_ctx on one CUDA device."""

    def __init__(self, device: int = 0):
        self._lib = library()
        self._ctx = C.c_void_p()
        _check(self._lib.psx_b200_ctx_create(C.c_int(device), C.byref(self._ctx)))
        self._handle = self._ctx.value  # (what the native calls take)
        self.device = device
        self._made = {}  # (shape, dtype) of small outputs -> a tensor like them

    def close(self):
        if self._ctx:
            self._lib.psx_b200_ctx_destroy(self._ctx)
            self._ctx = C.c_void_p()
            self._handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def launches(self) -> int:
        return int(self._lib.psx_b200_launch_count(self._ctx))

    @property
    def stream(self) -> int:
        return int(self._lib.psx_b200_ctx_stream(self._ctx) or 0)

    def inputs_are_ready(self, ready=True):
        """Promise that the inputs of the calls that follow are complete before each call is made
        (see psx_b200_ctx_inputs_are_ready): the row pass then overlaps the kernel before it."""
        _check(self._lib.psx_b200_ctx_inputs_are_ready(self._ctx, int(ready)))

    def set_wait_limit(self, nanoseconds):
        """How long a kernel waits for one of its own copies before the row reports ROW_DEVICE_TIMEOUT."""
        _check(self._lib.psx_b200_ctx_set_wait_limit(self._ctx, int(nanoseconds)))

    def test_short_copy(self, on=True):
        """Test hook (psx_b200_test_short_copy): the row pass's waits for its chunks run out."""
        _check(self._lib.psx_b200_test_short_copy(self._ctx, int(on)))

    def enable_timing(self, on=True):
        _check(self._lib.psx_b200_ctx_enable_timing(self._ctx, int(on)))

    def read_timing(self):
        """(row-pass ms, survivor-stage ms, calls) summed over the calls since the last read."""
        scan, merge, calls = C.c_double(0), C.c_double(0), C.c_uint64(0)
        _check(self._lib.psx_b200_ctx_read_timing(self._ctx, C.addressof(scan), C.addressof(merge),
                                                  C.addressof(calls)))
        return scan.value, merge.value, calls.value

    def sync(self, stream=None):
        _check(self._lib.psx_b200_sync(self._ctx, C.c_void_p(stream) if stream else None))

    # ---- device-resident sampling ------------------------------------------------------------------
    def alloc_outputs(self, rows, with_diag=True):
        import torch
        dev = torch.device("cuda", self.device)
        out = {
            "tokens": torch.empty(rows, dtype=torch.int64, device=dev),
            "log_probs": torch.empty(rows, dtype=torch.float32, device=dev),
            "status": torch.empty(rows, dtype=torch.int32, device=dev),
            "diag": torch.empty(rows * C.sizeof(RowDiag), dtype=torch.uint8, device=dev) if with_diag else None,
        }
        return out

    def sample_rows(self, logits, history_ids, history_offsets, config, uniforms, out=None, stream=None, vocab=None):
        """logits: cuda float32 (rows, >=vocab) with unit column stride; history/uniforms: cuda
        tensors (int64 / float64) or None.  Asynchronous; returns the dict of output tensors."""
        rows, cols = logits.shape
        row_stride, column_stride = logits.stride()
        assert column_stride == 1 or rows == 0
        vocab = cols if vocab is None else vocab
        out = out or self.alloc_outputs(rows)
        status = _native.sample_rows(
            self._handle, _stream_of(logits) if stream is None else stream, logits.data_ptr(), rows, vocab,
            row_stride if rows else vocab, _ptr(history_ids), _ptr(history_offsets), C.addressof(config), _ptr(uniforms),
            out["tokens"].data_ptr(), out["log_probs"].data_ptr(), out["status"].data_ptr(), _ptr(out["diag"]))
        if status:
            _check(status)
        return out

    def bind_sample_rows(self, logits, history_ids, history_offsets, config, uniforms, out=None, stream=None,
                         vocab=None):
        """sample_rows with its arguments converted once: returns a function of no arguments that
        enqueues the same call again (same buffers, same stream) and returns the output dict.  For
        loops over fixed buffers, where building the argument list costs as much as the launches."""
        rows = logits.shape[0]
        vocab = logits.shape[1] if vocab is None else vocab
        assert logits.stride(1) == 1 or rows == 0
        out = out or self.alloc_outputs(rows)
        args = (self._handle, _stream_of(logits) if stream is None else stream, logits.data_ptr(), rows, vocab,
                logits.stride(0) if rows else vocab, _ptr(history_ids), _ptr(history_offsets), C.addressof(config), _ptr(uniforms),
                _ptr(out["tokens"]), _ptr(out["log_probs"]), _ptr(out["status"]), _ptr(out["diag"]))
        fn = _native.sample_rows
        keep = (logits, history_ids, history_offsets, config, uniforms, out)  # the buffers live as long as the call

        def call(fn=fn, args=args, out=out, keep=keep):
            status = fn(*args)
            if status:
                _check(status)
            return out
        return call

    def bind_row_pass_only(self, logits, history_ids, history_offsets, config, stream=None, vocab=None):
        """row_pass_only with its arguments converted once (see bind_sample_rows)."""
        rows = logits.shape[0]
        vocab = logits.shape[1] if vocab is None else vocab
        if stream is None:
            import torch
            stream = torch.cuda.current_stream(logits.device).cuda_stream
        args = (self._ctx, C.c_void_p(stream), _dptr(logits), C.c_int64(rows), C.c_int64(vocab),
                C.c_int64(logits.stride(0) if rows else vocab), _dptr(history_ids), _dptr(history_offsets),
                C.c_void_p(C.addressof(config)))
        fn = self._lib.psx_b200_row_pass_only
        keep = (logits, history_ids, history_offsets, config)

        def call(fn=fn, args=args, keep=keep):
            status = fn(*args)
            if status:
                _check(status)
        return call

    def process_logits_host(self, logits, history_ids, history_offsets, config):
        """ProcessLogits on host rows (numpy float32 (rows, vocab), modified in place).  Returns the
        per-row status array; raises when the device path declines a row."""
        rows, vocab = logits.shape
        status = np.zeros(rows, dtype=np.int32)

        _check(_native.process_logits_host(self._handle, _host_array(logits), rows, vocab, logits.strides[0] // 4, _host_array(history_ids),
                                           _host_array(history_offsets), C.addressof(config), status))
        return status

    def row_pass_only(self, logits, history_ids, history_offsets, config, stream=None, vocab=None):
        """Launches only the kernel that reads the logits (for timing and profiling)."""
        rows = logits.shape[0]
        vocab = logits.shape[1] if vocab is None else vocab
        if stream is None:
            import torch
            stream = torch.cuda.current_stream(logits.device).cuda_stream
        _check(self._lib.psx_b200_row_pass_only(self._ctx, C.c_void_p(stream), _dptr(logits), rows, vocab,
                                                logits.stride(0) if rows else vocab, _dptr(history_ids),
                                                _dptr(history_offsets), C.addressof(config)))

    @staticmethod
    def diag_to_numpy(diag_tensor):
        return diag_tensor.cpu().numpy().view(ROW_DIAG_DTYPE)

    # ---- host-resident sampling (the reference-facing call) ---------------------------------------
    def sample_rows_host(self, logits, history_ids, history_offsets, config, uniforms, row_stride=None, vocab=None,
                         raise_on_row_failure=True):
        """numpy (or pinned torch CPU) inputs; returns (tokens, log_probs, status, diag) as numpy."""
        rows = logits.shape[0]
        vocab = logits.shape[1] if vocab is None else vocab
        row_stride = (logits.strides[0] // 4 if hasattr(logits, "strides") else logits.stride(0)) \
            if row_stride is None else row_stride
        tokens = np.zeros(rows, dtype=np.int64)
        logp = np.zeros(rows, dtype=np.float32)
        status = np.zeros(rows, dtype=np.int32)
        diag = np.zeros(rows, dtype=ROW_DIAG_DTYPE)

        rc = _native.sample_rows_host(self._handle, _host_array(logits), rows, vocab, row_stride, _host_array(history_ids), _host_array(history_offsets),
                                      C.addressof(config), _host_array(uniforms), tokens, logp, status, diag)
        if rc != OK and (rc != ERR_ROW_FAILED or raise_on_row_failure):
            _check(rc)
        return tokens, logp, status, diag

    # ---- top-k ---------------------------------------------------------------------------------------
    def top_k_rows(self, x, k, largest=True, stream=None):
        """x: cuda float32 contiguous (rows, cols).  Returns (values, indices) cuda float32 (rows, k)."""
        import torch
        rows, cols = x.shape
        values = torch.empty((rows, max(k, 0)), dtype=torch.float32, device=x.device)
        indices = torch.empty((rows, max(k, 0)), dtype=torch.float32, device=x.device)
        _check(_native.top_k_rows(self._handle, _stream_of(x) if stream is None else stream, x.data_ptr(), values.data_ptr(),
                                  indices.data_ptr(), rows, cols, k if k >= 0 else 0, int(largest)))
        return values, indices

    # ---- the language-model head -------------------------------------------------------------------------
    def lm_head_logits(self, hidden, weight, vocab_by_d=True, out=None, stream=None):
        """hidden: cuda float32 (rows, d); weight: (vocab, d) when vocab_by_d else (d, vocab).  Returns (rows, vocab)."""
        import torch
        rows, d = hidden.shape
        vocab = weight.shape[0] if vocab_by_d else weight.shape[1]
        out = torch.empty((rows, vocab), dtype=torch.float32, device=hidden.device) if out is None else out
        _check(_native.lm_head_logits(self._handle, _stream_of(hidden) if stream is None else stream, hidden.data_ptr(), rows, d,
                                      weight.data_ptr(), vocab, 0 if vocab_by_d else 1, out.data_ptr(), out.stride(0)))
        return out

    def lm_head_sample_rows(self, hidden, weight, history_ids, history_offsets, config, uniforms, vocab_by_d=True, out=None,
                            stream=None):
        """The head and the sampling step in one call: the logits stay in the context's scratch."""
        rows, d = hidden.shape
        vocab = weight.shape[0] if vocab_by_d else weight.shape[1]
        out = out or self.alloc_outputs(rows)
        _check(_native.lm_head_sample_rows(
            self._handle, _stream_of(hidden) if stream is None else stream, hidden.data_ptr(), rows, d, weight.data_ptr(), vocab,
            0 if vocab_by_d else 1, _ptr(history_ids), _ptr(history_offsets), C.addressof(config), _ptr(uniforms), _ptr(out["tokens"]),
            _ptr(out["log_probs"]), _ptr(out["status"]), _ptr(out["diag"])))
        return out

    # ---- row primitives ---------------------------------------------------------------------------------
    def softmax_rows(self, x, out=None, stream=None):
        """x: cuda float32 contiguous (rows, cols); out may be x itself."""
        import torch
        out = torch.empty_like(x) if out is None else out
        rows, cols = x.shape
        _check(_native.softmax_rows(self._handle, _stream_of(x) if stream is None else stream, x.data_ptr(), out.data_ptr(), rows, cols))
        return out

    def logsumexp_rows(self, x, stream=None):
        import torch
        rows, cols = x.shape
        out = torch.empty(rows, dtype=torch.float32, device=x.device)
        _check(_native.logsumexp_rows(self._handle, _stream_of(x) if stream is None else stream, x.data_ptr(), out.data_ptr(), rows, cols))
        return out

    def gather_rows(self, table, indices, stream=None):
        """table: cuda float32 (n, dim); indices: cuda float32 whole numbers (count,)."""
        import torch
        out = torch.empty((indices.shape[0], table.shape[1]), dtype=torch.float32, device=table.device)
        _check(_native.gather_rows(self._handle, _stream_of(table) if stream is None else stream, table.data_ptr(), indices.data_ptr(),
                                   out.data_ptr(), indices.shape[0], table.shape[1]))
        return out

    def decode_attention(self, q, keys, values, cached, scale=None, causal=True, window=0, key_keep=None, stream=None):
        """Attention of the new positions over the KV cache (psx_b200_decode_attention).  q: cuda float32
        (batch, heads, q_len, head_dim); keys / values: the cache, (batch, kv_heads, max_len, head_dim), with
        positions 0 .. cached + q_len - 1 filled; key_keep: (batch, cached + q_len) or None.  Returns the
        context, (batch, heads, q_len, head_dim), and a one-element int32 status tensor."""
        import torch
        batch, heads, q_len, head_dim = q.shape
        kv_heads, max_len = keys.shape[1], keys.shape[2]
        if scale is None:
            scale = 1.0 / float(np.sqrt(np.float32(head_dim)))
        context = torch.empty_like(q)
        status = _zeroed_word(q.device, stream)
        _check(_native.decode_attention(self._handle, _stream_of(q) if stream is None else stream, q.data_ptr(), keys.data_ptr(),
                                        values.data_ptr(), _ptr(key_keep), context.data_ptr(), batch, heads, kv_heads, q_len, head_dim,
                                        cached, max_len, float(scale), int(bool(causal)), window, status.data_ptr()))
        return context, status

    # ---- beams, states that follow them, the cache in 8 bits, prompts -------------------------------------
    def _empty(self, shape, dtype):
        """torch.empty on the context's device.  Small outputs of one shape come call after call, and like a tensor that is there they are
        made in half the time."""
        like = self._made.get((shape, dtype))
        if like is None:
            if math.prod(shape) > 65536:
                return _torch.empty(shape, dtype=dtype, device=f"cuda:{self.device}")
            if len(self._made) >= 64:
                self._made.clear()
            like = self._made[shape, dtype] = _torch.empty(shape, dtype=dtype, device=f"cuda:{self.device}")
        return _torch.empty_like(like)

    def _elsewhere(self, tensor):
        return ValueError(f"tensors on cuda:{self.device} are expected, got one on {tensor.device}")

    def _here(self, *tensors):
        for t in tensors:
            if t.get_device() != self.device:
                raise self._elsewhere(t)

    def beam_select(self, logits, scores, beams, keep, finished=None, finished_token=0, vocab=None, stream=None):
        """Beam search's selection (psx_b200_beam_select).  logits: cuda float32 (groups * beams, vocab), rows contiguous; scores:
        float32 (groups * beams); finished: bool or uint8 (groups * beams) or None.  Returns {"scores", "parents", "tokens"} of
        shape (groups, keep) and "status" (groups)."""
        torch = _torch or _torch_module()
        rows, columns = logits.shape
        vocab = columns if vocab is None else vocab
        if beams <= 0 or rows % beams or not 0 < vocab <= columns:
            raise ValueError("logits hold `beams` rows per group, of `vocab` columns at least")
        if not (logits.dtype is torch.float32 and scores.dtype is torch.float32 and scores.numel() == rows and scores.is_contiguous()):
            raise ValueError("logits are float32, and so are the scores, one per row")
        row_stride, column_stride = logits.stride()
        if rows == 1:
            row_stride = columns
        if column_stride != 1 and rows:
            raise ValueError("a row's logits are contiguous")
        self._here(logits, scores)
        if finished is not None:
            if not (finished.numel() == rows and finished.is_contiguous() and finished.element_size() == 1):
                raise ValueError("one byte per row says what is finished")
            self._here(finished)
        groups = rows // beams
        stream = _stream_of(logits) if stream is None else stream
        shape = (groups, max(keep, 0))
        out_scores, parents = self._empty(shape, torch.float32), self._empty(shape, torch.int64)
        tokens, status = torch.empty_like(parents), self._empty((groups,), torch.int32)
        code = _native.beam_select(self._handle, stream, logits.data_ptr(), groups, beams, vocab, row_stride, scores.data_ptr(),
                                   None if finished is None else finished.data_ptr(), finished_token, keep, out_scores.data_ptr(),
                                   parents.data_ptr(), tokens.data_ptr(), status.data_ptr())
        if code:
            _check(code)
        return {"scores": out_scores, "parents": parents, "tokens": tokens, "status": status}

    def reorder_states(self, parents, states, lengths=None, stream=None):
        """Rows of states that follow their beams, in place (psx_b200_reorder_states).  parents: int64 (groups, beams), row
        numbers within the group; states: tensors (groups * beams, heads, positions, ...), contiguous, each alone or as (tensor,
        tokens per position); lengths: int64 (groups * beams), the tokens that each row holds before, or None for all positions."""
        torch = _torch or _torch_module()
        if not (parents.dim() == 2 and parents.dtype is torch.int64 and parents.is_contiguous()):
            raise ValueError("parents are contiguous int64 (groups, beams)")
        groups, beams = parents.shape
        rows, here = groups * beams, self.device
        described = []  # (psx_beam_state: five words)
        for state in states:
            tensor, per = state if type(state) in (tuple, list) else (state, 1)
            shape = tensor.shape
            if len(shape) < 3 or shape[0] != rows or not tensor.is_contiguous():
                raise ValueError("a state is a contiguous (groups * beams, heads, positions, ...) tensor")
            if tensor.get_device() != here:
                raise self._elsewhere(tensor)
            heads, positions = shape[1], shape[2]
            size = tensor.element_size() * (shape[3] if len(shape) == 4 else math.prod(shape[3:]))
            described += (tensor.data_ptr(), heads, positions, size, per) if size else (0, 0, 0, 1, 1)  # (nothing to move)
        described = array.array("q", described)
        if lengths is not None:
            if not (lengths.dtype is torch.int64 and lengths.numel() == rows and lengths.is_contiguous()):
                raise ValueError("one int64 length per row")
            self._here(lengths)
        self._here(parents)
        code = _native.reorder_states(self._handle, _stream_of(parents) if stream is None else stream, described.buffer_info()[0], len(states), groups,
                                      beams, parents.data_ptr(), None if lengths is None else lengths.data_ptr())
        if code:
            _check(code)

    def store_cache_8bit(self, cache, keys, values, offsets, cached, stream=None):
        """Appends new positions to a Cache8bit (psx_b200_store_cache_8bit).  keys, values: float32, bfloat16 or float16 (total,
        kv_heads, head_dim), the rows' new positions one row behind the other, heads and dimensions contiguous; offsets: int64
        (batch + 1); cached: int64 (batch), the positions held before.  Returns the rows' statuses, int32 (batch)."""
        torch = _torch or _torch_module()
        shape, kv_heads, head_dim, batch = keys.shape, cache.kv_heads, cache.head_dim, cache.batch
        total = shape[0]
        if not (shape == (total, kv_heads, head_dim) and values.shape == shape and keys.dtype is values.dtype):
            raise ValueError("keys and values are (total, kv_heads, head_dim) of one type")
        key_stride, value_stride = keys.stride(), values.stride()
        if total and not (key_stride[2] == value_stride[2] == 1 and (kv_heads == 1 or key_stride[1] == value_stride[1] == head_dim)):
            raise ValueError("heads and dimensions of a position are contiguous")
        if not (offsets.dtype is torch.int64 and offsets.numel() == batch + 1 and offsets.is_contiguous() and
                cached.dtype is torch.int64 and cached.numel() == batch and cached.is_contiguous()):
            raise ValueError("offsets are int64 (batch + 1), cached is int64 (batch)")
        here = self.device
        if not (cache.device == here == keys.get_device() == values.get_device() == offsets.get_device() == cached.get_device()):
            self._here(cache.key_codes, keys, values, offsets, cached)
        status = self._empty((batch,), torch.int32)
        width = kv_heads * head_dim
        code = _native.store_cache_8bit(self._handle, _stream_of(keys) if stream is None else stream, cache._address, keys.data_ptr(), values.data_ptr(),
                                        _dtype_code(keys), total, key_stride[0] if total > 1 else width, value_stride[0] if total > 1 else width,
                                        offsets.data_ptr(), cached.data_ptr(), status.data_ptr())
        if code:
            _check(code)
        return status

    def decode_attention_8bit(self, q, cache, lengths, scale=None, causal=True, window=0, stream=None):
        """Attention of the new positions over a Cache8bit (psx_b200_decode_attention_8bit).  q: float32, bfloat16 or float16
        (batch, heads, q_len, head_dim); lengths: int64 (batch), the positions that each row sees, the new ones among them.
        Returns the context, like q."""
        torch = _torch or _torch_module()
        batch, heads, q_len, head_dim = q.shape
        if not (batch == cache.batch and head_dim == cache.head_dim and q.is_contiguous()):
            raise ValueError("q is a contiguous (batch, heads, q_len, head_dim) as the cache")
        if not (lengths.dtype is torch.int64 and lengths.numel() == batch and lengths.is_contiguous()):
            raise ValueError("lengths are int64 (batch)")
        if not (cache.device == self.device == q.get_device() == lengths.get_device()):
            self._here(q, cache.key_codes, lengths)
        if scale is None:
            scale = head_dim ** -0.5
        context = torch.empty_like(q)
        code = _native.decode_attention_8bit(self._handle, _stream_of(q) if stream is None else stream, q.data_ptr(), _dtype_code(q), cache._address,
                                             lengths.data_ptr(), context.data_ptr(), heads, q_len, scale, 1 if causal else 0, window)
        if code:
            _check(code)
        return context

    def prompt_attention(self, q, k, v, q_offsets, k_offsets=None, scale=None, causal=True, window=0, out=None, stream=None):
        """Attention of whole prompts, packed one behind the other (psx_b200_prompt_attention).  q: float32, bfloat16 or float16
        (total_q, heads, head_dim); k, v: (total_k, kv_heads, head_dim); heads and dimensions of a position contiguous; q_offsets,
        k_offsets: int64 (batch + 1), the latter the same as q_offsets if None.  Returns the context, (total_q, heads, head_dim)
        (`out` if given: rows of no sequence keep what they hold), and a one-element int32 status tensor."""
        torch = _torch or _torch_module()
        if k_offsets is None:
            k_offsets = q_offsets
        q_shape, k_shape = q.shape, k.shape
        total_q, heads, head_dim = q_shape
        total_k, kv_heads, k_dim = k_shape
        if not (v.shape == k_shape and k_dim == head_dim and q.dtype is k.dtype is v.dtype):
            raise ValueError("q, k and v are of one type and head dimension")
        q_stride, k_stride, v_stride = q.stride(), k.stride(), v.stride()
        if not ((total_q == 0 or (q_stride[2] == 1 and (heads == 1 or q_stride[1] == head_dim))) and
                (total_k == 0 or (k_stride[2] == v_stride[2] == 1 and (kv_heads == 1 or k_stride[1] == v_stride[1] == head_dim)))):
            raise ValueError("heads and dimensions of a position are contiguous")
        batch = q_offsets.numel() - 1
        if not (q_offsets.dtype is k_offsets.dtype is torch.int64 and batch >= 0 and k_offsets.numel() == batch + 1 and q_offsets.is_contiguous() and
                k_offsets.is_contiguous()):
            raise ValueError("offsets are int64 (batch + 1)")
        if out is None:
            out = torch.empty_like(q) if q.is_contiguous() else torch.empty(q_shape, dtype=q.dtype, device=q.device)
        elif not (out.shape == q_shape and out.dtype is q.dtype and out.is_contiguous()):
            raise ValueError("out is contiguous and of q's shape and type")
        here = self.device
        if not (q.get_device() == here == k.get_device() == v.get_device() == q_offsets.get_device() == k_offsets.get_device() == out.get_device()):
            self._here(q, k, v, out, q_offsets, k_offsets)
        if scale is None:
            scale = head_dim ** -0.5
        status = self._empty((1,), torch.int32)
        code = _native.prompt_attention(self._handle, _stream_of(q) if stream is None else stream, _dtype_code(q), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                        out.data_ptr(), total_q, total_k, q_stride[0] if total_q > 1 else heads * head_dim,
                                        k_stride[0] if total_k > 1 else kv_heads * head_dim, v_stride[0] if total_k > 1 else kv_heads * head_dim,
                                        q_offsets.data_ptr(), k_offsets.data_ptr(), batch, heads, kv_heads, head_dim, scale, 1 if causal else 0, window,
                                        status.data_ptr())
        if code:
            _check(code)
        return out, status

    # ---- a cache in pages ---------------------------------------------------------------------------------
    def _pools(self, table, pools):
        """The pools as psx_page_pool (three words each)."""
        described, num_pages, page_size, here = [], table.num_pages, table.page_size, self.device
        for pool in pools:
            shape = pool.shape
            if len(shape) < 3 or shape[0] != num_pages or shape[2] != page_size or not pool.is_contiguous():
                raise ValueError("a pool is a contiguous (num_pages, heads, page_size, ...) tensor")
            if pool.get_device() != here:
                raise self._elsewhere(pool)
            described += (pool.data_ptr(), shape[1], pool.element_size() * (shape[3] if len(shape) == 4 else math.prod(shape[3:])))
        return array.array("q", described)

    def extend_pages(self, table, added, pools=(), stream=None):
        """Room for new positions (psx_b200_extend_pages): the rows of a PageTable hold added (int64, rows) more afterwards.  pools: the tensors
        (num_pages, heads, page_size, ...) of the cache, in which shared last pages are copied.  Returns the rows' statuses, int32."""
        torch = _torch or _torch_module()
        rows = table.rows
        if not (added.dtype is torch.int64 and added.numel() == rows and added.is_contiguous()):
            raise ValueError("one int64 number of new positions per row")
        if not table.device == self.device == added.get_device():
            self._here(table.pages, added)
        described = self._pools(table, pools)
        status = self._empty((rows,), torch.int32)
        code = _native.extend_pages(self._handle, _stream_of(added) if stream is None else stream, table._address, added.data_ptr(),
                                    described.buffer_info()[0], len(pools), status.data_ptr())
        if code:
            _check(code)
        return status

    def fork_pages(self, table, parents, stream=None):
        """Rows of a PageTable that follow their beams by sharing pages (psx_b200_fork_pages).  parents: int64 (groups, beams)."""
        torch = _torch or _torch_module()
        if not (parents.dim() == 2 and parents.dtype is torch.int64 and parents.is_contiguous() and parents.numel() == table.rows):
            raise ValueError("parents are contiguous int64 (groups, beams), one per row")
        if not table.device == self.device == parents.get_device():
            self._here(table.pages, parents)
        code = _native.fork_pages(self._handle, _stream_of(parents) if stream is None else stream, table._address, parents.data_ptr(), parents.shape[1])
        if code:
            _check(code)

    def release_pages(self, table, keep=None, stream=None):
        """Positions given back (psx_b200_release_pages): rows keep their first keep (int64, rows), or none."""
        torch = _torch or _torch_module()
        if keep is not None and not (keep.dtype is torch.int64 and keep.numel() == table.rows and keep.is_contiguous()):
            raise ValueError("one int64 number of positions per row")
        if not table.device == self.device == (self.device if keep is None else keep.get_device()):
            self._here(table.pages, *(() if keep is None else (keep,)))
        code = _native.release_pages(self._handle, _stream_of(table.pages) if stream is None else stream, table._address,
                                     None if keep is None else keep.data_ptr())
        if code:
            _check(code)

    def compact_pages(self, table, pools, stream=None):
        """Brings the pages in use of all pools to their beginning (psx_b200_compact_pages).  Returns how many there are, int64 (1)."""
        torch = _torch or _torch_module()
        if table.device != self.device:
            self._here(table.pages)
        described = self._pools(table, pools)
        used = self._empty((1,), torch.int64)
        code = _native.compact_pages(self._handle, _stream_of(table.pages) if stream is None else stream, table._address, described.buffer_info()[0],
                                     len(pools), used.data_ptr())
        if code:
            _check(code)
        return used

    def _norm_weight(self, weight, kind, head_dim):
        if not (weight.dtype is kind and weight.numel() == head_dim and weight.is_contiguous()):
            raise ValueError("a norm's weight is (head_dim), of q's type")
        if weight.get_device() != self.device:
            self._here(weight)
        return weight.data_ptr()

    def rotate_heads(self, q, k, v=None, *, offsets, first, frequencies=None, q_weight=None, k_weight=None, eps=1e-6, interleaved=False, cache=None,
                     keys_too=None, stream=None):
        """Queries and keys on their way into the attention (psx_b200_rotate_heads): norm per head (q_weight, k_weight: (head_dim)), rotation by the
        position (frequencies: float64, one per pair of dimensions), keys and values into a PagedCache.  q: float32, bfloat16 or float16 (total, heads,
        head_dim); k, v: (total, kv_heads, head_dim); heads and dimensions of a position contiguous; offsets: int64 (batch + 1); first: int64
        (batch), the position of a row's first new one.  Returns q and k as they are then (k only with keys_too, which is so without a cache) and the
        rows' statuses, int32."""
        torch = _torch or _torch_module()
        total, heads, head_dim = q.shape
        k_shape, kind, here = k.shape, q.dtype, self.device
        kv_heads = k_shape[1]
        if not (k_shape == (total, kv_heads, head_dim) and kind is k.dtype):
            raise ValueError("q and k are (total, heads, head_dim) of one type")
        q_stride, q_head, q_dim = q.stride()
        k_stride, k_head, k_dim = k.stride()
        v_stride, v_head, v_dim, v_at, cache_at = k_stride, k_head, 1, None, None
        if cache is not None:
            if v is None or v.shape != k_shape or v.dtype is not kind or kind is not cache.key_pages.dtype:
                raise ValueError("what a cache stores is k and v of one shape and of its type")
            v_stride, v_head, v_dim = v.stride()
            v_at, cache_at = v.data_ptr(), cache._address
            if not cache.device == here == v.get_device():
                self._here(cache.key_pages, v)
        elif keys_too is None:
            keys_too = True
        if total and not (q_dim == k_dim == v_dim == 1 and (heads == 1 or q_head == head_dim) and (kv_heads == 1 or k_head == v_head == head_dim)):
            raise ValueError("heads and dimensions of a position are contiguous")
        batch = offsets.numel() - 1
        if not (offsets.dtype is first.dtype is torch.int64 and batch >= 0 and first.numel() == batch and offsets.is_contiguous() and first.is_contiguous()):
            raise ValueError("offsets are int64 (batch + 1), first is int64 (batch)")
        if not q.get_device() == here == k.get_device() == offsets.get_device() == first.get_device():
            self._here(q, k, offsets, first)
        rotated, frequencies_at, q_weight_at, k_weight_at = 0, None, None, None
        if frequencies is not None:
            if not (frequencies.dtype is torch.float64 and frequencies.is_contiguous()):
                raise ValueError("frequencies are contiguous float64")
            if frequencies.get_device() != here:
                self._here(frequencies)
            rotated, frequencies_at = 2 * frequencies.numel(), frequencies.data_ptr()
        if q_weight is not None:
            q_weight_at = self._norm_weight(q_weight, kind, head_dim)
        if k_weight is not None:
            k_weight_at = self._norm_weight(k_weight, kind, head_dim)
        width, key_width = heads * head_dim, kv_heads * head_dim
        q_out = torch.empty_like(q) if q_stride == width and q.is_contiguous() else self._empty((total, heads, head_dim), kind)
        k_out = self._empty((total, kv_heads, head_dim), kind) if keys_too else None
        status = self._empty((batch,), torch.int32)
        if total <= 1:
            q_stride, k_stride, v_stride = width, key_width, key_width
        code = _native.rotate_heads(self._handle, _stream_of(q) if stream is None else stream, _dtype_code(q), q.data_ptr(), k.data_ptr(), v_at,
                                    q_out.data_ptr(), None if k_out is None else k_out.data_ptr(), total, q_stride, k_stride, v_stride, offsets.data_ptr(),
                                    first.data_ptr(), batch, heads, kv_heads, head_dim, q_weight_at, k_weight_at, eps, frequencies_at, rotated,
                                    1 if interleaved else 0, cache_at, status.data_ptr())
        if code:
            _check(code)
        return q_out, k_out, status

    def decode_attention_pages(self, q, cache, q_len=1, scale=None, causal=True, window=0, stream=None):
        """Attention of the new positions over a PagedCache (psx_b200_decode_attention_pages).  q: of the cache's type, (rows * q_len, heads, head_dim), a
        row's new positions one behind the other; what the rows see is the table's lengths.  Returns the context, like q."""
        torch = _torch or _torch_module()
        total, heads, head_dim = q.shape
        if not (total == cache.table.rows * q_len and head_dim == cache.head_dim and q.dtype is cache.key_pages.dtype and q.is_contiguous()):
            raise ValueError("q is a contiguous (rows * q_len, heads, head_dim) of the cache's type")
        if not cache.device == self.device == q.get_device():
            self._here(q, cache.key_pages)
        if scale is None:
            scale = head_dim ** -0.5
        context = torch.empty_like(q)
        code = _native.decode_attention_pages(self._handle, _stream_of(q) if stream is None else stream, q.data_ptr(), cache.dtype_code, cache._address,
                                              context.data_ptr(), heads, q_len, scale, 1 if causal else 0, window)
        if code:
            _check(code)
        return context

    # ---- log-probabilities of given tokens ----------------------------------------------------------------
    def token_log_probs(self, logits, tokens=None, top=0, entropy=False, vocab=None, stream=None):
        """Log-probabilities of given tokens (psx_b200_token_log_probs).  logits: float32, bfloat16 or float16 (rows, vocab), rows contiguous; tokens:
        int64 (rows) or None.  Returns {"log_probs" (rows), "entropy" (rows), "top_log_probs" and "top_tokens" (rows, top), "status" (rows)}; what is
        not asked for is None."""
        torch = _torch or _torch_module()
        rows, columns = logits.shape
        if vocab is None:
            vocab = columns
        if not 0 < vocab <= columns:
            raise ValueError("a row holds `vocab` logits at least")
        row_stride, column_stride = logits.stride()
        if rows <= 1:
            row_stride = columns
        if column_stride != 1 and rows and vocab > 1:
            raise ValueError("a row's logits are contiguous")
        here = self.device
        if logits.get_device() != here:
            self._here(logits)
        log_probs = entropies = top_log_probs = top_tokens = tokens_at = log_probs_at = entropies_at = top_log_probs_at = top_tokens_at = None
        of_rows = (rows,)
        if tokens is not None:
            if not (tokens.dtype is torch.int64 and tokens.numel() == rows and tokens.is_contiguous()):
                raise ValueError("one int64 token per row")
            if tokens.get_device() != here:
                self._here(tokens)
            log_probs = self._empty(of_rows, torch.float32)
            tokens_at, log_probs_at = tokens.data_ptr(), log_probs.data_ptr()
        if entropy:
            entropies = self._empty(of_rows, torch.float32)
            entropies_at = entropies.data_ptr()
        if top > 0:
            of_top = (rows, top)
            top_log_probs, top_tokens = self._empty(of_top, torch.float32), self._empty(of_top, torch.int64)
            top_log_probs_at, top_tokens_at = top_log_probs.data_ptr(), top_tokens.data_ptr()
        status = self._empty(of_rows, torch.int32)
        code = _native.token_log_probs(self._handle, _stream_of(logits) if stream is None else stream, _dtype_code(logits), logits.data_ptr(), rows, vocab,
                                       row_stride, tokens_at, log_probs_at, entropies_at, top, top_log_probs_at, top_tokens_at, status.data_ptr())
        if code:
            _check(code)
        return {"log_probs": log_probs, "entropy": entropies, "top_log_probs": top_log_probs, "top_tokens": top_tokens, "status": status}

    # ---- vocabulary-sharded -----------------------------------------------------------------------------
    def shard_record_bytes(self, config) -> int:
        return int(self._lib.psx_b200_shard_record_bytes(C.addressof(config)))

    def shard_scan(self, shard_logits, shard_begin, vocab, history_ids, history_offsets, config, records, stream=None):
        rows, cols = shard_logits.shape
        _check(_native.shard_scan(self._handle, _stream_of(shard_logits) if stream is None else stream, shard_logits.data_ptr(), rows,
                                  cols, shard_logits.stride(0), shard_begin, vocab, _ptr(history_ids), _ptr(history_offsets), C.addressof(config),
                                  _ptr(records)))

    def shard_merge(self, gathered, num_shards, rows, vocab, config, uniforms, out=None, stream=None, row_begin=0,
                    row_count=None):
        """Merges rows row_begin .. row_begin + row_count - 1 (all of them by default); `out` holds
        the merged rows only, the first of them at index 0."""
        row_count = rows - row_begin if row_count is None else row_count
        out = out or self.alloc_outputs(row_count)
        _check(_native.shard_merge_rows(self._handle, _stream_of(gathered) if stream is None else stream, gathered.data_ptr(), num_shards,
                                        rows, row_begin, row_count, vocab, C.addressof(config), _ptr(uniforms), _ptr(out["tokens"]),
                                        _ptr(out["log_probs"]), _ptr(out["status"]), _ptr(out.get("diag"))))
        return out

    def exchange(self, world, rank, rows, config):
        """This rank's end of a vocabulary-sharded exchange over peer memory (psx_b200_exchange_*)."""
        return Exchange(self, world, rank, rows, config)


class _DeviceBytes:
    """Device memory that the library owns, as something torch.as_tensor can wrap without a copy."""

    def __init__(self, address, nbytes):
        self.__cuda_array_interface__ = {"shape": (nbytes,), "typestr": "|u1", "data": (address, False), "version": 2}


class Exchange:
    """One rank's end of the vocabulary-sharded step over peer memory (include/psx_b200.h:
    psx_b200_exchange_*).  `handle` (bytes) goes to every rank; open() takes all ranks' handles in
    rank order; sample() is one step; results() are views of the library's own buffer:
    {"tokens", "log_probs", "status"} of shape (world, rows_per_rank), rank r's rows in row r."""

    def __init__(self, ctx, world, rank, rows, config):
        self._lib, self._context = ctx._lib, ctx
        self.world, self.rank, self.rows = world, rank, rows
        self._ex = C.c_void_p()
        handle = C.create_string_buffer(int(self._lib.psx_b200_exchange_handle_bytes()))
        _check(self._lib.psx_b200_exchange_create(ctx._ctx, world, rank, rows, C.addressof(config), C.byref(self._ex), handle))
        self.handle = handle.raw
        self._views = None

    def open(self, handles: bytes):
        if len(handles) != self.world * len(self.handle):
            raise ValueError("open() takes the handles of all ranks, back to back in rank order")
        _check(self._lib.psx_b200_exchange_open(self._ex, handles))

    def sample(self, shard_logits, shard_begin, vocab, history_ids, history_offsets, config, uniforms, stream=None):
        rows, cols = shard_logits.shape
        if rows != self.rows:
            raise ValueError(f"the exchange was created for {self.rows} rows, got {rows}")
        _check(_native.exchange_sample(self._ex.value, _stream_of(shard_logits) if stream is None else stream, shard_logits.data_ptr(),
                                       cols, shard_logits.stride(0), shard_begin, vocab, _ptr(history_ids), _ptr(history_offsets), C.addressof(config),
                                       _ptr(uniforms)))
        return self.results(shard_logits.device)

    def results(self, device):
        """Views of the last step's results (the library keeps two sets and alternates: a step's results
        stay in place until the step after the next one)."""
        import torch
        address, per = C.c_void_p(), C.c_int64()
        _check(self._lib.psx_b200_exchange_results(self._ex, C.byref(address), C.byref(per)))
        if self._views is None:
            self._views = {}
        if address.value not in self._views:
            per = per.value
            raw = torch.as_tensor(_DeviceBytes(address.value, self.world * 16 * per), device=device)
            by_rank = raw.view(self.world, 16 * per)
            self._views[address.value] = {"tokens": by_rank[:, : 8 * per].view(torch.int64),
                                          "log_probs": by_rank[:, 8 * per: 12 * per].view(torch.float32),
                                          "status": by_rank[:, 12 * per:].view(torch.int32)}
        return self._views[address.value]

    def test_wait(self, wait_limit_ns, extra_arrivals):
        _check(self._lib.psx_b200_exchange_test_wait(self._ex, wait_limit_ns, extra_arrivals))

    def close(self):
        """Unmaps and frees.  Across ranks: only after a barrier, so that no rank is still inside a step."""
        if self._ex:
            self._views = None
            self._lib.psx_b200_exchange_destroy(self._ex)
            self._ex = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
