"""ctypes binding of libkascade_b200.so (the C ABI declared in include/kascade_b200.h).

The library is loaded from this package directory.  There is no fallback: if the shared object is
missing or a call is rejected, a ``KascadeNativeError`` is raised.
"""
from __future__ import annotations

import ctypes as C
import functools
import os
import struct
from typing import Optional

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libkascade_b200.so")

HEAD_DIM = 128
GROUP_SIZE = 4
TILE = 32
FP16, BF16, FP8_E4M3, INT4 = 0, 1, 2, 3        # KB200_FP16 / KB200_BF16 / KB200_FP8_E4M3 / KB200_INT4
DTYPES = {torch.float16: FP16, torch.bfloat16: BF16}
FP8_TORCH = (torch.float8_e4m3fn, torch.uint8)   # an FP8 cache may be handed over as raw bytes

EXPORTS = [
    "kb200_init", "kb200_last_error", "kb200_abi_version", "kb200_topk_select", "kb200_topk_select_decode",
    "kb200_decode_workspace_bytes", "kb200_decode_default_splits", "kb200_decode_sparse_paged",
    "kb200_decode_anchor_paged", "kb200_prefill_dense", "kb200_prefill_pool_scores",
    "kb200_prefill_sparse", "kb200_prefill_budgets", "kb200_selftest_umma", "kb200_read_status",
    "kb200_decode_sparse_paged_noalloc", "kb200_prefill_dense_fanout", "kb200_prefill_sparse_fanout",
    "kb200_kv_write", "kb200_prefill_dense_ragged", "kb200_prefill_pool_scores_ragged", "kb200_prefill_sparse_ragged",
    "kb200_prefill_budgets_ragged", "kb200_zero_padding", "kb200_peer_push", "kb200_stream_wait_events", "kb200_selftest_wait_timeout", "kb200_tensor_map_encodes", "kb200_decode_noalloc_splits",
    "kb200_kv_write_at", "kb200_kv_read", "kb200_decode_anchor_paged_mass", "kb200_mass_add_prompt", "kb200_evict",
    "kb200_evict_workspace_bytes", "kb200_kv_layout_bytes",
]


class KascadeNativeError(RuntimeError):
    pass


class KvLayout(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("stride_batch", C.c_int64),
                ("stride_page", C.c_int64), ("stride_token", C.c_int64), ("stride_head", C.c_int64),
                ("block_table", C.c_void_p), ("block_table_stride", C.c_int32),
                ("page_size", C.c_int32), ("dtype", C.c_int32),
                ("k_scale", C.c_void_p), ("v_scale", C.c_void_p), ("scale_stride_batch", C.c_int64),
                ("scale_stride_page", C.c_int64), ("scale_stride_head", C.c_int64),
                ("k_param", C.c_void_p), ("v_param", C.c_void_p), ("param_stride_batch", C.c_int64),
                ("param_stride_page", C.c_int64), ("param_stride_token", C.c_int64), ("param_stride_head", C.c_int64),
                ("act_dtype", C.c_int32)]


_LAYOUT = struct.Struct("PPqqqqPiiiPPqqqPPqqqqi0P")      # the same: packing costs half of what the fields of a KvLayout do
assert _LAYOUT.size == C.sizeof(KvLayout)


class Positions(C.Structure):
    """kb200_positions: rotary positions of new tokens that are not their places in the cache."""
    _fields_ = [("positions", C.c_void_p), ("stride_axis", C.c_int64), ("stride_batch", C.c_int64), ("pair_axis", C.c_void_p),
                ("axes", C.c_int32), ("token_positions", C.c_void_p), ("token_stride", C.c_int64), ("token_rows", C.c_int32)]


class ActLayout(C.Structure):
    _fields_ = [("ptr", C.c_void_p), ("stride_b", C.c_int64), ("stride_t", C.c_int64),
                ("stride_h", C.c_int64), ("dtype", C.c_int32)]


MAX_FANOUT = 8


class OutFanout(C.Structure):
    """kb200_out_fanout: the output rows of a call go into `count` buffers [B, L, total_heads, D]."""
    _fields_ = [("out", C.c_void_p * MAX_FANOUT), ("count", C.c_int32), ("total_heads", C.c_int32),
                ("head_offset", C.c_int32), ("multicast", C.c_int32)]


def out_fanout(pointers, total_heads: int, head_offset: int, multicast: bool = False) -> OutFanout:
    """pointers: device addresses (ints) of the [B, L, total_heads, D] fp16 buffers, own buffer first; with
    `multicast` a single NVLink multicast address that stands for the buffer on every GPU."""
    if not 1 <= len(pointers) <= MAX_FANOUT:
        raise KascadeNativeError(f"fan-out of {len(pointers)} outputs (1..{MAX_FANOUT} supported)")
    f = OutFanout()
    for i, ptr in enumerate(pointers):
        f.out[i] = int(ptr)
    f.count, f.total_heads, f.head_offset = len(pointers), int(total_heads), int(head_offset)
    f.multicast = 1 if multicast else 0
    if multicast and len(pointers) != 1:
        raise KascadeNativeError("a multicast fan-out takes exactly one address")
    return f


class Ragged(C.Structure):
    """kb200_ragged: per-sequence first row and length inside equally sized batch slots."""
    _fields_ = [("seq_start", C.c_void_p), ("seq_len", C.c_void_p)]


def ragged(seq_start: Optional[torch.Tensor], seq_len: torch.Tensor) -> Ragged:
    _want(seq_len, torch.int32, "seq_len")
    _want_opt(seq_start, torch.int32, "seq_start")
    return Ragged(0 if seq_start is None else seq_start.data_ptr(), seq_len.data_ptr())


class PushPlan(C.Structure):
    """kb200_push_plan: peers' buffers with one copy stream and one completion event per peer."""
    _fields_ = [("dst", C.c_void_p * MAX_FANOUT), ("stream", C.c_void_p * MAX_FANOUT),
                ("done_event", C.c_void_p * MAX_FANOUT), ("count", C.c_int32)]


_lib = None
_inited = set()
# Host-side tallies of the kernels of this library launched so far by this process: those that compute, and those that
# clear the padding of a ragged batch's output, one per padded prompt layer, which stand for a memset.
launch_count = 0
clear_count = 0


def _launched(n: int):
    global launch_count
    launch_count += n


def _check_layout(lib):
    """The library and this binding agree on the layout that calls take one or an array of."""
    size = getattr(lib, "kb200_kv_layout_bytes", None)
    if size is not None:
        size.restype = C.c_size_t
    if size is None or size() != C.sizeof(KvLayout):
        raise KascadeNativeError(f"{LIB_PATH} was built from other sources than this binding (its kb200_kv_layout has "
                                 f"{size() if size is not None else 'fewer'} bytes, {C.sizeof(KvLayout)} expected): build it again with "
                                 "`python -m kascade_b200.build`")


def load() -> C.CDLL:
    """dlopen the library (no CUDA call is made)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise KascadeNativeError(
                f"{LIB_PATH} is missing: build it with `python -m kascade_b200.build` "
                "(there is no fallback implementation)")
        lib = C.CDLL(LIB_PATH)
        _check_layout(lib)
        lib.kb200_last_error.restype = C.c_char_p
        lib.kb200_decode_workspace_bytes.restype = C.c_size_t
        lib.kb200_decode_workspace_bytes.argtypes = [C.c_int, C.c_int, C.c_int]
        lib.kb200_decode_default_splits.argtypes = [C.c_int, C.c_int, C.c_int]
        lib.kb200_init.argtypes = [C.c_int]
        vp, i64, i32, f32 = C.c_void_p, C.c_int64, C.c_int, C.c_float
        lib.kb200_topk_select.argtypes = [vp, i64, i32, vp, vp, i32, vp, i64, vp, i64, vp]
        lib.kb200_topk_select_decode.argtypes = [vp, i64, i32, vp, i32, C.c_double, i32, i32, vp, i64, vp, i32, vp]
        lib.kb200_decode_sparse_paged.argtypes = [vp, i64, i64, C.POINTER(KvLayout), vp, i64, i64, vp,
                                                  i32, vp, f32, vp, vp, vp, C.c_size_t, i32, i32, i32,
                                                  i32, vp]
        lib.kb200_decode_sparse_paged_noalloc.argtypes = [vp, i64, i64, C.POINTER(KvLayout), vp, i64, i64, vp,
                                                          i32, vp, f32, vp, vp, i32, i32, i32, i32, vp]
        lib.kb200_decode_anchor_paged.argtypes = [vp, i64, i64, C.POINTER(KvLayout), vp, i32, f32, vp,
                                                  vp, i64, vp, vp, vp, C.c_size_t, i32, i32, i32, i32,
                                                  vp]
        AL = C.POINTER(ActLayout)
        lib.kb200_prefill_dense.argtypes = [AL, AL, AL, f32, vp, vp, i32, i32, i32, i32, vp]
        lib.kb200_prefill_pool_scores.argtypes = [AL, AL, vp, f32, vp, i64, i32, i32, i32, i32, vp]
        lib.kb200_prefill_sparse.argtypes = [AL, AL, AL, vp, i64, vp, vp, f32, vp, vp, i32, i32, i32,
                                             i32, i32, vp]
        FO = C.POINTER(OutFanout)
        lib.kb200_prefill_dense_fanout.argtypes = [AL, AL, AL, f32, FO, vp, i32, i32, i32, i32, vp]
        lib.kb200_prefill_sparse_fanout.argtypes = [AL, AL, AL, vp, i64, vp, vp, f32, FO, vp, i32, i32, i32,
                                                    i32, i32, vp]
        lib.kb200_prefill_budgets.argtypes = [vp, vp, i32, i32, i32, i32, f32, i32, vp]
        RG = C.POINTER(Ragged)
        lib.kb200_prefill_dense_ragged.argtypes = [AL, AL, AL, f32, vp, vp, RG, i32, i32, i32, i32, vp]
        lib.kb200_prefill_pool_scores_ragged.argtypes = [AL, AL, vp, f32, vp, i64, RG, i32, i32, i32, i32, vp]
        lib.kb200_prefill_sparse_ragged.argtypes = [AL, AL, AL, vp, i64, vp, vp, f32, vp, vp, RG, i32, i32, i32,
                                                    i32, i32, vp]
        lib.kb200_prefill_budgets_ragged.argtypes = [vp, vp, vp, i32, i32, i32, i32, f32, i32, vp]
        lib.kb200_zero_padding.argtypes = [vp, RG, i32, i32, i64, vp]
        lib.kb200_kv_write.argtypes = [AL, vp, AL, AL, vp, vp, C.POINTER(KvLayout), vp, vp, f32, vp, f32, i32, i32,
                                       i32, i32, vp]
        lib.kb200_kv_write_at.argtypes = [AL, vp, AL, AL, vp, vp, C.POINTER(KvLayout), vp, vp, f32, vp, f32,
                                          C.POINTER(Positions), i32, i32, i32, i32, vp]
        lib.kb200_kv_read.argtypes = [C.POINTER(KvLayout), vp, vp, vp, i32, i32, i32, vp]
        lib.kb200_decode_anchor_paged_mass.argtypes = [vp, i64, i64, C.POINTER(KvLayout), vp, i32, f32, vp, vp, i64, vp, i64, vp, vp,
                                                       vp, C.c_size_t, i32, i32, i32, i32, vp]
        lib.kb200_mass_add_prompt.argtypes = [vp, i64, vp, vp, vp, i64, i64, i32, i32, i32, i32, vp]
        lib.kb200_evict_workspace_bytes.restype = C.c_size_t
        lib.kb200_evict_workspace_bytes.argtypes = [i32, i32, i32]
        lib.kb200_evict.argtypes = [C.POINTER(KvLayout), i32, vp, vp, i64, vp, i64, i32, i32, i32, vp, vp, vp, i64, vp, C.c_size_t,
                                    i32, i32, i32, vp]
        lib.kb200_selftest_umma.argtypes = [vp, vp, vp, vp, vp]
        lib.kb200_peer_push.argtypes = [C.POINTER(PushPlan), vp, C.c_size_t, C.c_size_t, C.c_size_t, C.c_size_t, vp, vp]
        lib.kb200_stream_wait_events.argtypes = [vp, C.POINTER(C.c_void_p), i32]
        lib.kb200_selftest_wait_timeout.argtypes = [vp, C.c_uint64, i32, vp]
        lib.kb200_tensor_map_encodes.restype = C.c_longlong
        lib.kb200_tensor_map_encodes.argtypes = []
        lib.kb200_decode_noalloc_splits.argtypes = [i32, i32, i32, i32, i32]
        _lib = lib
    return _lib


def _check(rc: int, what: str):
    if rc != 0:
        raise KascadeNativeError(f"{what}: {load().kb200_last_error().decode()}")


def init(device: Optional[int] = None) -> C.CDLL:
    if device in _inited and _lib is not None:      # every call of a step comes through here: nothing but the look-up
        return _lib
    lib = load()
    if not torch.cuda.is_available():
        raise KascadeNativeError("kascade_b200 needs a CUDA device (sm_100a); none is visible")
    dev = torch.cuda.current_device() if device is None else int(device)
    if dev not in _inited:
        _check(lib.kb200_init(dev), "kb200_init")
        _inited.add(dev)
    return lib


def read_status(device=None) -> int:
    """Status word of `device` (default: the current one); 0 = every kernel ran to completion.  Reading
    clears it.  Synchronises the device."""
    dev = torch.cuda.current_device() if device is None else torch.device(device).index
    with torch.cuda.device(dev):
        out = C.c_int(0)
        _check(init(dev).kb200_read_status(C.byref(out)), "kb200_read_status")
    return out.value


def check_status(device=None, where: str = ""):
    """Raise if a kernel of this library gave up a bounded wait on `device` since the last check: its
    outputs (and those of every later tile-prefill launch, which return at entry while the word is set) are
    not valid.  Call it where the host synchronises anyway."""
    st = read_status(device)
    if st != 0:
        raise KascadeNativeError(f"a kernel gave up a bounded device-side wait (code {st}){' ' + where if where else ''}; "
                                 "outputs since the last status check are invalid")


def _on_device_of(arg_index: int):
    """Decorator: run the wrapped call with the GPU of its `arg_index`-th argument (a tensor) current.  The
    library launches on the current device, on the current stream of that device, and keeps its per-device
    state (kernel attributes, the built-in decode scratch) by it; without this a caller whose current device
    differs from the tensors' would launch on the wrong GPU."""
    def deco(fn):
        @functools.wraps(fn)
        def wrapped(*args, **kwargs):
            t = args[arg_index]
            where = t.get_device()                               # (-1: not on a GPU)
            if where < 0:
                raise KascadeNativeError(f"{fn.__name__}: expected CUDA tensors, got one on {t.device}")
            if where == torch._C._cuda_getDevice():              # (a CUDA tensor exists: the runtime is up)
                return fn(*args, **kwargs)
            with torch.cuda.device(t.device):
                return fn(*args, **kwargs)
        return wrapped
    return deco


def _stream() -> int:
    """cudaStream_t of the current device's current stream (read as a handle, without building a torch.cuda.Stream)."""
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())      # (a CUDA tensor exists: the runtime is up)


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _want_opt(t: Optional[torch.Tensor], dtype, name: str):
    if t is not None:
        _want(t, dtype, name)


def _want(t: torch.Tensor, dtype, name: str):
    if t.dtype is not dtype or not t.is_cuda:
        raise KascadeNativeError(f"{name}: expected a CUDA {dtype} tensor, got {t.dtype} on {t.device}")


def _same_device(first: torch.Tensor, **others: Optional[torch.Tensor]):
    where = first.get_device()
    for name, t in others.items():
        if t is not None and t.get_device() != where:
            raise KascadeNativeError(f"{name} is on {t.device}, expected {first.device}")


def _half_code(t: torch.Tensor, name: str) -> int:
    """KB200_FP16 / KB200_BF16 of a CUDA fp16 or bf16 tensor."""
    code = DTYPES.get(t.dtype)
    if code is None or not t.is_cuda:
        raise KascadeNativeError(f"{name}: expected a CUDA fp16 or bf16 tensor, got {t.dtype} on {t.device}")
    return code


# ------------------------------------------------------------------------------------------------
@_on_device_of(0)
def topk_select(scores: torch.Tensor, n_valid: Optional[torch.Tensor], k_row: Optional[torch.Tensor],
                k_max: int, out_idx: torch.Tensor, out_count: Optional[torch.Tensor], n_cols: Optional[int] = None):
    """scores [..., row_stride] fp32 (last dim contiguous, rows equally spaced), out_idx [..., idx_stride]."""
    lib = init(scores.get_device())
    _want(scores, torch.float32, "scores")
    _want(out_idx, torch.int32, "out_idx")
    rows = scores.numel() // scores.shape[-1]
    assert scores.is_contiguous() and out_idx.is_contiguous()
    _check(lib.kb200_topk_select(_ptr(scores), scores.shape[-1], scores.shape[-1] if n_cols is None else n_cols,
                                 _ptr(n_valid), _ptr(k_row), k_max, _ptr(out_idx), out_idx.shape[-1],
                                 _ptr(out_count), rows, _stream()), "kb200_topk_select")
    _launched(1 if rows else 0)


@_on_device_of(0)
def topk_select_decode(scores: torch.Tensor, seq_lens: torch.Tensor, share: float, tile: int, k_max: int,
                       out_idx: torch.Tensor, out_count: torch.Tensor, n_cols: int):
    """topk_select over the pooled scores [B, G, row_stride] of a decode step; every row's number of candidates and
    budget follow from seq_lens [B] int32 inside the kernel."""
    lib = init(scores.get_device())
    _want(scores, torch.float32, "scores")
    _want(seq_lens, torch.int32, "seq_lens")
    _want(out_idx, torch.int32, "out_idx")
    B, G, stride = scores.shape
    assert scores.is_contiguous() and out_idx.is_contiguous() and seq_lens.is_contiguous() and seq_lens.numel() == B
    _check(lib.kb200_topk_select_decode(_ptr(scores), stride, n_cols, _ptr(seq_lens), G, share, tile, k_max,
                                        _ptr(out_idx), out_idx.shape[-1], _ptr(out_count), B, _stream()),
           "kb200_topk_select_decode")
    _launched(1 if B else 0)


@_on_device_of(0)
def prefill_budgets(n_valid, k_row, batch, groups, tiles, k_max, pct, rolling):
    lib = init(n_valid.get_device())
    _check(lib.kb200_prefill_budgets(_ptr(n_valid), _ptr(k_row), batch, groups, tiles, k_max, float(pct),
                                     int(bool(rolling)), _stream()), "kb200_prefill_budgets")
    _launched(1)


@_on_device_of(0)
def prefill_budgets_ragged(n_valid, k_row, seq_len, batch, groups, tiles, k_cap, pct, rolling):
    lib = init(n_valid.get_device())
    _want(seq_len, torch.int32, "seq_len")
    _check(lib.kb200_prefill_budgets_ragged(_ptr(n_valid), _ptr(k_row), _ptr(seq_len), batch, groups, tiles, k_cap,
                                            float(pct), int(bool(rolling)), _stream()), "kb200_prefill_budgets_ragged")
    _launched(1)


def _fp8_scales(k_scale, v_scale, need_v: bool):
    if k_scale is None or (need_v and v_scale is None):
        raise KascadeNativeError("an FP8 cache needs k_scale (and v_scale): one fp32 scale per (page, KV head)")
    _want(k_scale, torch.float32, "k_scale")
    _want_opt(v_scale, torch.float32, "v_scale")
    if v_scale is not None and (v_scale.shape != k_scale.shape or v_scale.stride() != k_scale.stride()):
        raise KascadeNativeError("k_scale and v_scale must have the same shape and strides")


def _holding(layout, *tensors):
    """The layouts carry raw device addresses: keep the tensors alive as long as the layout object is."""
    layout._keep = tuple(t for t in tensors if t is not None)
    return layout


def is_int4(cache: torch.Tensor) -> bool:
    """Whether a cache holds 4-bit codes: uint8 rows of 64 bytes (a raw FP8 row has 128)."""
    return cache.dtype == torch.uint8 and cache.shape[-1] == HEAD_DIM // 2


def _int4_params(k, v, k_param, v_param):
    """The checks of an INT4 cache: codes [..., 64] uint8 and parameters [..., 8] fp16 of the same leading shape.  Returns the
    strides of the codes and of the parameters."""
    where, st = k.get_device(), k.stride()
    if where >= 0 and len(st) == 4 and st[3] == 1 and k_param is not None:
        ps, shape, pshape = k_param.stride(), k.shape, k_param.shape
        if len(ps) == 4 and ps[3] == 1 and k_param.dtype is torch.float16 and k_param.get_device() == where and pshape[:3] == shape[:3] \
                and pshape[-1] == 8:
            if v is None:
                return st, ps
            if v_param is not None and v.shape == shape and v.stride() == st and v.dtype is k.dtype and v.get_device() == where \
                    and v_param.dtype is torch.float16 and v_param.shape == pshape and v_param.stride() == ps \
                    and v_param.get_device() == where:
                return st, ps
    # something is wrong: say what
    if where < 0:
        raise KascadeNativeError(f"k_cache: expected a CUDA uint8 tensor, got one on {k.device}")
    if len(st) != 4 or st[3] != 1:
        raise KascadeNativeError("an INT4 cache holds rows of 64 contiguous bytes: [num_pages, page_size, G, 64]")
    if v is not None and (v.shape != k.shape or v.stride() != st or v.dtype != k.dtype):
        raise KascadeNativeError("k_cache and v_cache must have the same type, shape and strides")
    if k_param is None or (v is not None and v_param is None):
        raise KascadeNativeError("an INT4 cache needs k_scale (and v_scale): eight fp16 per row, four scales and four zeros")
    for name, par in (("k_scale", k_param), ("v_scale", v_param if v is not None else None)):
        if par is None:
            continue
        _want(par, torch.float16, name)
        if par.shape != k.shape[:3] + (8,) or par.stride(3) != 1:
            raise KascadeNativeError(f"{name} of an INT4 cache: expected {tuple(k.shape[:3]) + (8,)}, the last dimension "
                                     f"contiguous, got {tuple(par.shape)}")
    _same_device(k, v_cache=v, k_scale=k_param, v_scale=v_param)
    raise KascadeNativeError("k_scale and v_scale must have the same shape and strides")


def kv_layout_paged(k_cache: torch.Tensor, v_cache: Optional[torch.Tensor], block_table: torch.Tensor,
                    k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
                    act_dtype: torch.dtype = torch.float16) -> KvLayout:
    """vLLM-style cache [num_pages, page_size, G, D] and block table [B, max_pages] int32.  An FP8 cache
    (torch.float8_e4m3fn or raw uint8) comes with k_scale / v_scale [num_pages, G] fp32; an INT4 cache (uint8
    [num_pages, page_size, G, 64]) with k_scale / v_scale [num_pages, page_size, G, 8] fp16 and `act_dtype`, the type of the
    queries, outputs and new rows."""
    if is_int4(k_cache):
        st, ps = _int4_params(k_cache, v_cache, k_scale, v_scale)
        if act_dtype not in DTYPES:
            raise KascadeNativeError(f"act_dtype of an INT4 cache: expected fp16 or bf16, got {act_dtype}")
        ts = block_table.stride()
        if block_table.dtype is not torch.int32 or block_table.get_device() != k_cache.get_device() or len(ts) != 2 or ts[1] != 1:
            _want(block_table, torch.int32, "block_table")
            _same_device(k_cache, block_table=block_table)
            raise KascadeNativeError("block_table: expected [B, max_pages], the last dimension contiguous")
        layout = KvLayout.from_buffer_copy(_LAYOUT.pack(
            k_cache.data_ptr(), 0 if v_cache is None else v_cache.data_ptr(), 0, st[0], st[1], st[2], block_table.data_ptr(), ts[0],
            k_cache.shape[1], INT4, 0, 0, 0, 0, 0, k_scale.data_ptr(), 0 if v_cache is None else v_scale.data_ptr(), 0, ps[0], ps[1],
            ps[2], DTYPES[act_dtype]))
        layout._keep = (k_cache, block_table, k_scale) if v_cache is None else (k_cache, v_cache, block_table, k_scale, v_scale)
        return layout
    if k_cache.dtype in FP8_TORCH:
        assert k_cache.is_cuda and k_cache.dim() == 4 and k_cache.stride(3) == 1
        assert block_table.dtype == torch.int32 and block_table.stride(1) == 1
        if v_cache is not None:
            assert v_cache.shape == k_cache.shape and v_cache.stride() == k_cache.stride() and v_cache.dtype == k_cache.dtype
        _fp8_scales(k_scale, v_scale, v_cache is not None)
        assert k_scale.shape == (k_cache.shape[0], k_cache.shape[2])
        return _holding(KvLayout(k_cache.data_ptr(), 0 if v_cache is None else v_cache.data_ptr(), 0, k_cache.stride(0),
                                 k_cache.stride(1), k_cache.stride(2), block_table.data_ptr(), block_table.stride(0),
                                 k_cache.shape[1], FP8_E4M3, k_scale.data_ptr(),
                                 0 if v_scale is None else v_scale.data_ptr(), 0, k_scale.stride(0), k_scale.stride(1)),
                        k_cache, v_cache, block_table, k_scale, v_scale)
    code = _half_code(k_cache, "k_cache")
    st, ts = k_cache.stride(), block_table.stride()
    assert len(st) == 4 and st[3] == 1
    assert block_table.dtype is torch.int32 and ts[1] == 1
    if v_cache is not None:
        assert v_cache.shape == k_cache.shape and v_cache.stride() == st and v_cache.dtype is k_cache.dtype
    layout = KvLayout.from_buffer_copy(_LAYOUT.pack(
        k_cache.data_ptr(), 0 if v_cache is None else v_cache.data_ptr(), 0, st[0], st[1], st[2], block_table.data_ptr(), ts[0],
        k_cache.shape[1], code, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0))
    layout._keep = (k_cache, block_table) if v_cache is None else (k_cache, v_cache, block_table)
    return layout


def kv_layout_contiguous(k: torch.Tensor, v: Optional[torch.Tensor], page_size: int = 16,
                         k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
                         act_dtype: torch.dtype = torch.float16) -> KvLayout:
    """HF cache view [B, G, L, D] (any batch / head / token strides, D contiguous).  An FP8 cache comes with
    k_scale / v_scale [B, G, ceil(L / page_size)] fp32, an INT4 cache [B, G, L, 64] with [B, G, L, 8] fp16."""
    if is_int4(k):
        st, ps = _int4_params(k, v, k_scale, v_scale)
        if act_dtype not in DTYPES:
            raise KascadeNativeError(f"act_dtype of an INT4 cache: expected fp16 or bf16, got {act_dtype}")
        return _holding(KvLayout(k.data_ptr(), _ptr(v), st[0], st[2] * page_size, st[2], st[1], 0, 0, page_size, INT4, 0, 0, 0, 0,
                                 0, k_scale.data_ptr(), _ptr(v_scale) if v is not None else 0, ps[0], ps[2] * page_size, ps[2],
                                 ps[1], DTYPES[act_dtype]), k, v, k_scale, v_scale)
    if k.dtype in FP8_TORCH:
        assert k.is_cuda and k.dim() == 4 and k.stride(3) == 1
        if v is not None:
            assert v.shape == k.shape and v.stride() == k.stride() and v.dtype == k.dtype
        _fp8_scales(k_scale, v_scale, v is not None)
        assert k_scale.dim() == 3 and k_scale.shape[:2] == k.shape[:2]
        return _holding(KvLayout(k.data_ptr(), 0 if v is None else v.data_ptr(), k.stride(0), k.stride(2) * page_size,
                                 k.stride(2), k.stride(1), 0, 0, page_size, FP8_E4M3, k_scale.data_ptr(),
                                 0 if v_scale is None else v_scale.data_ptr(), k_scale.stride(0), k_scale.stride(2),
                                 k_scale.stride(1)), k, v, k_scale, v_scale)
    code = _half_code(k, "k")
    st = k.stride()
    assert len(st) == 4 and st[3] == 1
    if v is not None:
        assert v.shape == k.shape and v.stride() == st and v.dtype == k.dtype
    return _holding(KvLayout(k.data_ptr(), 0 if v is None else v.data_ptr(), st[0], st[2] * page_size, st[2], st[1], 0, 0,
                             page_size, code), k, v)


def kv_layout_rows(k: torch.Tensor, v: Optional[torch.Tensor], row_table: torch.Tensor) -> KvLayout:
    """HF cache view [B, G, L, D] whose sequences do not start at row 0 (a padded batch): row_table [B, n] int32 gives
    the cache row of every logical position - a block table with one-token pages, which the decode kernels already
    know how to walk."""
    code = _half_code(k, "k")
    assert k.dim() == 4 and k.stride(3) == 1
    assert row_table.dtype == torch.int32 and row_table.dim() == 2 and row_table.stride(1) == 1
    if v is not None:
        assert v.shape == k.shape and v.stride() == k.stride() and v.dtype == k.dtype
    return _holding(KvLayout(k.data_ptr(), 0 if v is None else v.data_ptr(), k.stride(0), k.stride(2), k.stride(2),
                             k.stride(1), row_table.data_ptr(), row_table.stride(0), 1, code), k, v, row_table)


def decode_workspace(batch: int, heads: int, splits: int, device) -> torch.Tensor:
    n = load().kb200_decode_workspace_bytes(batch, heads, splits)
    return torch.empty(max(n, 16), dtype=torch.uint8, device=device)


@functools.lru_cache(maxsize=1024)                    # the layers of a step ask the same; the answer follows from the arguments
def decode_workspace_bytes(batch: int, heads: int, splits: int) -> int:
    return load().kb200_decode_workspace_bytes(batch, heads, splits)


@functools.lru_cache(maxsize=1024)
def _default_splits(batch: int, groups: int, max_keys: int, device: int) -> int:
    with torch.cuda.device(device):
        return init(device).kb200_decode_default_splits(batch, groups, max_keys)


def decode_default_splits(batch: int, groups: int, max_keys: int, device: Optional[int] = None) -> int:
    return _default_splits(batch, groups, max_keys, torch.cuda.current_device() if device is None else int(device))


@functools.lru_cache(maxsize=None)
def sm_count(device: int) -> int:
    return torch.cuda.get_device_properties(device).multi_processor_count


def _check_q(q, kv: KvLayout):
    want = FP16 if kv.dtype == FP8_E4M3 else kv.act_dtype if kv.dtype == INT4 else kv.dtype
    if _half_code(q, "q") != want:
        raise KascadeNativeError(f"q is {q.dtype} but the KV cache has dtype code {kv.dtype} (an FP8 cache takes fp16 q, an INT4 "
                                 "cache the type given as act_dtype)")
    if kv.dtype == INT4 and kv._keep[0].get_device() != q.get_device():
        raise KascadeNativeError(f"q is on {q.device}, the KV cache on {kv._keep[0].device}")


@_on_device_of(0)
def decode_sparse_paged(q, kv: KvLayout, topk_idx, topk_count, k_max, head_map, scale, out, lse2=None,
                        workspace=None, num_splits=0):
    """q [B,H,D] fp16; topk_idx [B,G,kstride] int32; out [B,H,D] fp16 contiguous."""
    lib = init(q.get_device())
    _check_q(q, kv)
    _want(out, q.dtype, "out")
    _want(topk_idx, torch.int32, "topk_idx")
    _want_opt(topk_count, torch.int32, "topk_count")
    _want_opt(head_map, torch.int32, "head_map")
    B, H, D = q.shape
    G = topk_idx.shape[1]
    qs, xs = q.stride(), topk_idx.stride()
    assert D == HEAD_DIM and qs[2] == 1 and out.is_contiguous() and xs[2] == 1
    _check(lib.kb200_decode_sparse_paged(
        q.data_ptr(), qs[0], qs[1], C.byref(kv), topk_idx.data_ptr(), xs[0], xs[1], _ptr(topk_count), k_max, _ptr(head_map),
        float(scale), out.data_ptr(), _ptr(lse2), _ptr(workspace),
        0 if workspace is None else workspace.numel() * workspace.element_size(), B, H, G, num_splits, _stream()),
        "kb200_decode_sparse_paged")
    ns = num_splits if num_splits else lib.kb200_decode_default_splits(B, G, k_max)
    _launched(1 + (ns > 1))


NOALLOC_MAX_SLOTS = 8192


@_on_device_of(0)
def decode_sparse_paged_noalloc(q, kv: KvLayout, topk_idx, topk_count, k_max, head_map, scale, out, lse2=None,
                                num_splits=0):
    """Same result as decode_sparse_paged, for callers that cannot allocate or pass a workspace: the split
    partials live in a fixed array inside the library (batch * heads * splits <= NOALLOC_MAX_SLOTS).
    Calls that overlap on the GPU race on that array; the first call on a device belongs in set-up."""
    lib = init(q.get_device())
    _check_q(q, kv)
    _want(out, q.dtype, "out")
    _want(topk_idx, torch.int32, "topk_idx")
    _want_opt(topk_count, torch.int32, "topk_count")
    _want_opt(head_map, torch.int32, "head_map")
    B, H, D = q.shape
    G = topk_idx.shape[1]
    assert D == HEAD_DIM and q.stride(2) == 1 and out.is_contiguous() and topk_idx.stride(2) == 1
    _check(lib.kb200_decode_sparse_paged_noalloc(
        _ptr(q), q.stride(0), q.stride(1), C.byref(kv), _ptr(topk_idx), topk_idx.stride(0), topk_idx.stride(1),
        _ptr(topk_count), k_max, _ptr(head_map), float(scale), _ptr(out), _ptr(lse2), B, H, G, num_splits,
        _stream()), "kb200_decode_sparse_paged_noalloc")
    _launched(2 if lib.kb200_decode_noalloc_splits(B, H, G, k_max, num_splits) > 1 else 1)


@_on_device_of(0)
def decode_anchor_paged(q, kv: KvLayout, seq_lens, max_seq_len, scale, logits, pooled, out, lse2,
                        workspace=None, num_splits=0, mass=None):
    """q [B,H,D]; logits [B,H,stride] fp32; pooled [B,G,stride] fp32; out [B,H,D] fp16 or None.  `mass` [B, at least max_seq_len] fp32:
    the sum of pooled over the heads is added to it."""
    lib = init(q.get_device())
    _check_q(q, kv)
    _want_opt(out, q.dtype, "out")
    _want(logits, torch.float32, "logits")
    _want(pooled, torch.float32, "pooled")
    B, H, D = q.shape
    G, stride = pooled.shape[1:]
    qs = q.stride()
    assert logits.is_contiguous() and pooled.is_contiguous() and logits.shape[-1] == stride
    before = (q.data_ptr(), qs[0], qs[1], C.byref(kv), seq_lens.data_ptr(), max_seq_len, float(scale), logits.data_ptr(),
              pooled.data_ptr(), stride)
    after = (_ptr(out), _ptr(lse2), _ptr(workspace), 0 if workspace is None else workspace.numel() * workspace.element_size(), B, H, G,
             num_splits, _stream())
    if mass is None:
        _check(lib.kb200_decode_anchor_paged(*before, *after), "kb200_decode_anchor_paged")
    else:
        _want_rows(mass, torch.float32, B, "mass")
        if mass.shape[1] < max_seq_len or mass.get_device() != q.get_device():
            raise KascadeNativeError(f"mass holds {mass.shape[1]} rows on {mass.device}, {max_seq_len} on {q.device} are needed")
        _check(lib.kb200_decode_anchor_paged_mass(*before, mass.data_ptr(), mass.stride(0), *after), "kb200_decode_anchor_paged_mass")
    ns = num_splits if num_splits else lib.kb200_decode_default_splits(B, G, max_seq_len)
    _launched(2 + (ns > 1))


def act_layout(x: torch.Tensor) -> ActLayout:
    """x indexed [B, L, heads, D] (any strides, D contiguous)."""
    b, t, h, d = x.stride()
    assert d == 1 and x.shape[3] == HEAD_DIM
    return ActLayout(x.data_ptr(), b, t, h, _half_code(x, "activation"))


@_on_device_of(0)
def prefill_dense(q, k, v, scale, out, lse2, fanout: Optional[OutFanout] = None, ragged: Optional[Ragged] = None):
    """q [B,L,H,D], k/v [B,L,G,D] (views allowed); out [B,L,H,D] fp16 contiguous or None; lse2 [B,L,H] fp32 or None.
    With `fanout` (see out_fanout) the rows go into several [B,L,total_heads,D] buffers instead of `out`; with
    `ragged` (see ragged()) every sequence has its own first row and length inside its slot of L rows."""
    lib = init(q.get_device())
    B, L, H, _ = q.shape
    G = k.shape[2]
    ql, kl = act_layout(q), act_layout(k)
    vl = act_layout(v) if v is not None else ActLayout(0, 0, 0, 0, 0)
    if ragged is not None:
        if out is not None:
            _want(out, q.dtype, "out")
            assert out.is_contiguous()
        _check(lib.kb200_prefill_dense_ragged(C.byref(ql), C.byref(kl), C.byref(vl), float(scale), _ptr(out), _ptr(lse2),
                                              C.byref(ragged), B, L, H, G, _stream()), "kb200_prefill_dense_ragged")
        _launched(1)
        return
    if fanout is not None:
        _check(lib.kb200_prefill_dense_fanout(C.byref(ql), C.byref(kl), C.byref(vl), float(scale), C.byref(fanout),
                                              _ptr(lse2), B, L, H, G, _stream()), "kb200_prefill_dense_fanout")
        _launched(1)
        return
    if out is not None:
        _want(out, q.dtype, "out")
        assert out.is_contiguous()
    _check(lib.kb200_prefill_dense(C.byref(ql), C.byref(kl), C.byref(vl), float(scale), _ptr(out), _ptr(lse2),
                                   B, L, H, G, _stream()), "kb200_prefill_dense")
    _launched(1)


@_on_device_of(0)
def zero_padding(out: torch.Tensor, ragged: Ragged):
    """Zeros the rows of out [B, L, ...] (contiguous) that lie outside the sequences."""
    global clear_count
    lib = init(out.get_device())
    assert out.is_contiguous()
    B, L = out.shape[:2]
    if out.numel() == 0:
        return
    _check(lib.kb200_zero_padding(_ptr(out), C.byref(ragged), B, L, out.numel() * out.element_size() // (B * L), _stream()),
           "kb200_zero_padding")
    clear_count += 1


@_on_device_of(0)
def prefill_pool_scores(q, k, lse2, scale, pooled, ragged: Optional[Ragged] = None):
    """pooled [B,G,T,row_stride] fp32 contiguous."""
    lib = init(q.get_device())
    B, L, H, _ = q.shape
    G = k.shape[2]
    ql, kl = act_layout(q), act_layout(k)
    _want(pooled, torch.float32, "pooled")
    _want(lse2, torch.float32, "lse2")
    assert pooled.is_contiguous() and lse2.is_contiguous()
    if ragged is not None:
        _check(lib.kb200_prefill_pool_scores_ragged(C.byref(ql), C.byref(kl), _ptr(lse2), float(scale), _ptr(pooled),
                                                    pooled.shape[-1], C.byref(ragged), B, L, H, G, _stream()),
               "kb200_prefill_pool_scores_ragged")
        _launched(1)
        return
    _check(lib.kb200_prefill_pool_scores(C.byref(ql), C.byref(kl), _ptr(lse2), float(scale), _ptr(pooled),
                                         pooled.shape[-1], B, L, H, G, _stream()), "kb200_prefill_pool_scores")
    _launched(1)


@_on_device_of(0)
def prefill_sparse(q, k, v, tile_idx, tile_count, head_map, scale, out, lse2=None, fanout: Optional[OutFanout] = None,
                   ragged: Optional[Ragged] = None):
    """tile_idx [B,G,T,kstride] int32, tile_count [B,G,T] int32, out [B,L,H,D] fp16 contiguous.
    With `fanout` (see out_fanout) the rows go into several [B,L,total_heads,D] buffers instead of `out`."""
    lib = init(q.get_device())
    B, L, H, _ = q.shape
    G = k.shape[2]
    ql, kl, vl = act_layout(q), act_layout(k), act_layout(v)
    _want(tile_idx, torch.int32, "tile_idx")
    _want(tile_count, torch.int32, "tile_count")
    _want_opt(head_map, torch.int32, "head_map")
    assert tile_idx.is_contiguous() and tile_count.is_contiguous()
    if fanout is not None:
        _check(lib.kb200_prefill_sparse_fanout(C.byref(ql), C.byref(kl), C.byref(vl), _ptr(tile_idx),
                                               tile_idx.shape[-1], _ptr(tile_count), _ptr(head_map), float(scale),
                                               C.byref(fanout), _ptr(lse2), B, L, H, G, tile_idx.shape[1],
                                               _stream()), "kb200_prefill_sparse_fanout")
        _launched(1)
        return
    _want(out, q.dtype, "out")
    assert out.is_contiguous()
    if ragged is not None:
        _check(lib.kb200_prefill_sparse_ragged(C.byref(ql), C.byref(kl), C.byref(vl), _ptr(tile_idx), tile_idx.shape[-1],
                                               _ptr(tile_count), _ptr(head_map), float(scale), _ptr(out), _ptr(lse2),
                                               C.byref(ragged), B, L, H, G, tile_idx.shape[1], _stream()),
               "kb200_prefill_sparse_ragged")
        _launched(1)
        return
    _check(lib.kb200_prefill_sparse(C.byref(ql), C.byref(kl), C.byref(vl), _ptr(tile_idx), tile_idx.shape[-1],
                                    _ptr(tile_count), _ptr(head_map), float(scale), _ptr(out), _ptr(lse2), B, L, H,
                                    G, tile_idx.shape[1], _stream()), "kb200_prefill_sparse")
    _launched(1)


@_on_device_of(2)
def kv_write(q_in, q_out, k_new, v_new, start_pos, n_new, kv: KvLayout, q_gain=None, k_gain=None, eps=1e-6,
             inv_freq=None, rope_scale=1.0, positions=None, pair_axis=None, token_positions=None):
    """q_in [B,T,H,D] (or None), k_new / v_new [B,T,G,D] views, all fp16 or all bf16 like the cache and the gains;
    start_pos [B] int32; n_new [B] int32 or None; kv: the cache to append to (kv_layout_paged /
    kv_layout_contiguous); inv_freq [D/2] fp32 or None.  With `positions` [axes, B, T] int32 the tokens have rotary positions of
    their own (kb200_kv_write_at): pair_axis [D/2] int32 or None, token_positions [B, rows] int32 or None."""
    lib = init(k_new.get_device())
    B, T, G, _ = k_new.shape
    kl, vl = act_layout(k_new), act_layout(v_new)
    ql = act_layout(q_in) if q_in is not None else ActLayout(0, 0, 0, 0, 0)
    H = q_in.shape[2] if q_in is not None else 0
    if q_in is not None:
        _want(q_out, k_new.dtype, "q_out")
        assert q_out.is_contiguous() and q_out.shape == q_in.shape
    if kv.dtype == INT4 and kv._keep[0].get_device() != k_new.get_device():
        raise KascadeNativeError(f"the new rows are on {k_new.device}, the KV cache on {kv._keep[0].device}")
    _want(start_pos, torch.int32, "start_pos")
    _want_opt(n_new, torch.int32, "n_new")
    _want_opt(q_gain, k_new.dtype, "q_gain")
    _want_opt(k_gain, k_new.dtype, "k_gain")
    if inv_freq is not None:
        _want(inv_freq, torch.float32, "inv_freq")
        assert inv_freq.is_contiguous() and inv_freq.numel() == HEAD_DIM // 2
    if not B * T:
        return
    if positions is not None:
        where, ps = k_new.get_device(), positions.stride()
        if positions.dtype is not torch.int32 or positions.get_device() != where or len(ps) != 3 or positions.shape[1:] != (B, T) \
                or (T > 1 and ps[2] != 1) or not positions.shape[0]:
            _want(positions, torch.int32, "positions")
            _same_device(k_new, positions=positions)
            raise KascadeNativeError(f"positions: expected [axes, {B}, {T}], the last dimension contiguous, got "
                                     f"{tuple(positions.shape)}")
        if pair_axis is not None and (pair_axis.dtype is not torch.int32 or pair_axis.shape != (HEAD_DIM // 2,)
                                      or not pair_axis.is_contiguous() or pair_axis.get_device() != where):
            raise KascadeNativeError(f"pair_axis: expected [{HEAD_DIM // 2}] int32 contiguous on {k_new.device}, got "
                                     f"{tuple(pair_axis.shape)} {pair_axis.dtype} on {pair_axis.device}")
        if token_positions is not None and (token_positions.dtype is not torch.int32 or token_positions.dim() != 2
                                            or token_positions.shape[0] != B or token_positions.stride(1) != 1
                                            or token_positions.get_device() != where):
            raise KascadeNativeError(f"token_positions: expected [{B}, rows] int32 on {k_new.device}, the last dimension "
                                     f"contiguous, got {tuple(token_positions.shape)} {token_positions.dtype} on {token_positions.device}")
        at = Positions(positions.data_ptr(), ps[0], ps[1], _ptr(pair_axis), positions.shape[0],
                       _ptr(token_positions), 0 if token_positions is None else token_positions.stride(0),
                       0 if token_positions is None else token_positions.shape[1])
        _check(lib.kb200_kv_write_at(C.byref(ql), _ptr(q_out), C.byref(kl), C.byref(vl), _ptr(start_pos), _ptr(n_new),
                                     C.byref(kv), _ptr(q_gain), _ptr(k_gain), float(eps), _ptr(inv_freq), float(rope_scale),
                                     C.byref(at), B, T, H, G, _stream()), "kb200_kv_write_at")
        _launched(1)
        return
    _check(lib.kb200_kv_write(C.byref(ql), _ptr(q_out), C.byref(kl), C.byref(vl), _ptr(start_pos), _ptr(n_new),
                              C.byref(kv), _ptr(q_gain), _ptr(k_gain), float(eps), _ptr(inv_freq), float(rope_scale),
                              B, T, H, G, _stream()), "kb200_kv_write")
    _launched(1)


@_on_device_of(2)
def kv_read(kv: KvLayout, seq_lens, k_out, v_out):
    """Rows 0 .. seq_lens[b] - 1 of an INT4 cache into k_out / v_out [B, max_len, G, D] (contiguous, of the layout's act_dtype);
    rows behind a sequence are written as zeros."""
    where = k_out.get_device()
    lib = init(where)
    B, T, G, D = k_out.shape
    if kv.dtype != INT4:
        raise KascadeNativeError("kv_read: the cache is not INT4: its rows need no conversion")
    if _half_code(k_out, "k_out") != kv.act_dtype or v_out.dtype is not k_out.dtype or v_out.shape != k_out.shape:
        raise KascadeNativeError("kv_read: k_out and v_out must have one shape and the layout's act_dtype")
    if not (k_out.is_contiguous() and v_out.is_contiguous() and seq_lens.is_contiguous()) or seq_lens.shape != (B,) or D != HEAD_DIM \
            or seq_lens.dtype is not torch.int32 or seq_lens.get_device() != where or v_out.get_device() != where:
        raise KascadeNativeError(f"kv_read: expected contiguous k_out / v_out [B, T, G, {HEAD_DIM}] and seq_lens [B] int32 on one device")
    if not k_out.numel():
        return
    _check(lib.kb200_kv_read(C.byref(kv), _ptr(seq_lens), _ptr(k_out), _ptr(v_out), B, T, G, _stream()), "kb200_kv_read")
    _launched(1)


def _want_rows(t: torch.Tensor, dtype, batch: int, name: str):
    """[batch, rows] with the rows of a sequence contiguous."""
    _want(t, dtype, name)
    if t.dim() != 2 or t.shape[0] != batch or (t.shape[1] > 1 and t.stride(1) != 1):
        raise KascadeNativeError(f"{name}: expected [{batch}, rows], the last dimension contiguous, got {tuple(t.shape)} with strides "
                                 f"{t.stride()}")


@_on_device_of(0)
def mass_add_prompt(pooled, mass, out, seq_len=None):
    """out[b, j] = mass[b, j] + the scores of row j over the heads and the later tiles of pooled [B, G, T, row_stride];
    `out` may be `mass`."""
    lib = init(pooled.get_device())
    _want(pooled, torch.float32, "pooled")
    B, G, T, stride = pooled.shape
    _want_rows(mass, torch.float32, B, "mass")
    _want_rows(out, torch.float32, B, "out")
    _want_opt(seq_len, torch.int32, "seq_len")
    if not pooled.is_contiguous() or (seq_len is not None and (seq_len.shape != (B,) or not seq_len.is_contiguous())) \
            or out.shape != mass.shape:
        raise KascadeNativeError("mass_add_prompt: pooled and seq_len [B] must be contiguous, out must have the shape of mass")
    _same_device(pooled, seq_len=seq_len, mass=mass, out=out)
    rows = mass.shape[1]
    if not mass.numel() or not pooled.numel():                # nothing to add to, or nothing to add
        if out is not mass:
            out.copy_(mass)
        return
    _check(lib.kb200_mass_add_prompt(_ptr(pooled), stride, _ptr(seq_len), _ptr(mass), _ptr(out),
                                     mass.stride(0) if B > 1 else rows, out.stride(0) if B > 1 else rows, B, G, T, rows,
                                     _stream()), "kb200_mass_add_prompt")
    _launched(1)


@_on_device_of(0)
def evict(mass, layers, seq_lens, budget: int, recent: int, sinks: int, token_positions, num_kv_heads: int):
    """Shortens the caches of `layers` (KvLayouts that share a block table, a type and strides) in place, see kb200_evict.  Returns
    the new lengths [B], and the rows' weight and token position [B, rows] after the moves."""
    lib = init(mass.get_device())
    if mass.dim() != 2:
        raise KascadeNativeError(f"mass: expected [B, rows], got {tuple(mass.shape)}")
    B, rows = mass.shape
    _want_rows(mass, torch.float32, B, "mass")
    _want(seq_lens, torch.int32, "seq_lens")
    if token_positions is not None:
        _want_rows(token_positions, torch.int32, B, "token_positions")
        if token_positions.shape[1] != rows:
            raise KascadeNativeError(f"token_positions: expected {(B, rows)}, got {tuple(token_positions.shape)}")
    if seq_lens.shape != (B,) or not seq_lens.is_contiguous():
        raise KascadeNativeError("evict: seq_lens [B] must be contiguous")
    _same_device(mass, seq_lens=seq_lens, token_positions=token_positions)
    if B > 1 and mass.stride(0) < rows:                        # the same row for several sequences
        mass = mass.contiguous()
    if B > 1 and token_positions is not None and token_positions.stride(0) < rows:
        token_positions = token_positions.contiguous()
    where, shape = mass.get_device(), layers[0]._keep[0].shape
    for i, layer in enumerate(layers):
        if layer._keep[0].shape != shape:
            raise KascadeNativeError(f"the cache of layer {i} is {tuple(layer._keep[0].shape)}, that of layer 0 {tuple(shape)}")
        for t in layer._keep:
            if t.get_device() != where:
                raise KascadeNativeError(f"the cache of layer {i} is on {t.device}, expected {mass.device}")
    dev = mass.device
    if not mass.numel():
        return torch.zeros_like(seq_lens), torch.empty_like(mass), torch.empty(B, rows, dtype=torch.int32, device=dev)
    lens, mass_out = torch.empty_like(seq_lens), torch.empty_like(mass, memory_format=torch.contiguous_format)
    pos_out = torch.empty(B, rows, dtype=torch.int32, device=dev)
    size = lib.kb200_evict_workspace_bytes(B, rows, budget)
    workspace = torch.empty(max(size, 16), dtype=torch.uint8, device=dev)
    array = (KvLayout * len(layers))(*layers)
    _check(lib.kb200_evict(array, len(layers), seq_lens.data_ptr(), mass.data_ptr(), mass.stride(0), _ptr(token_positions),
                           0 if token_positions is None else token_positions.stride(0), budget, recent, sinks, lens.data_ptr(),
                           mass_out.data_ptr(), pos_out.data_ptr(), rows, workspace.data_ptr(), size, B, num_kv_heads, rows,
                           _stream()), "kb200_evict")
    _launched(3 + (-(-len(layers) // 32) if rows > budget else 0))
    return lens, mass_out, pos_out


@_on_device_of(0)
def selftest_umma(a: torch.Tensor, b: torch.Tensor):
    lib = init(a.get_device())
    out = torch.zeros(4, 128, 128, dtype=torch.float32, device=a.device)
    status = torch.full((4,), -1, dtype=torch.int32, device=a.device)
    _check(lib.kb200_selftest_umma(_ptr(a), _ptr(b), _ptr(out), _ptr(status), _stream()), "kb200_selftest_umma")
    return out, status


def selftest_wait_timeout(device, limit_ns: int = 1_000_000, code: int = 77) -> torch.Tensor:
    """Runs the wait-that-runs-out selftest on `device`; returns [code, threads that gave up, elapsed ns].
    The device status word then holds `code` until read_status() / check_status() clears it."""
    result = torch.zeros(3, dtype=torch.int32, device=device)
    with torch.cuda.device(result.device):
        lib = init(result.get_device())
        _check(lib.kb200_selftest_wait_timeout(_ptr(result), int(limit_ns), int(code), _stream()),
               "kb200_selftest_wait_timeout")
    _launched(1)
    return result


def tensor_map_encodes() -> int:
    return int(load().kb200_tensor_map_encodes())


def _cuda_event(ev: torch.cuda.Event) -> int:
    """cudaEvent_t of a torch event (torch creates it lazily, at the first record)."""
    if not ev.cuda_event:
        ev.record()
    return int(ev.cuda_event)


def push_plan(dst_pointers, streams, done_events) -> PushPlan:
    """One entry per peer: device address of its buffer, a torch stream for the copy, a torch event."""
    if not (len(dst_pointers) == len(streams) == len(done_events)) or len(dst_pointers) > MAX_FANOUT:
        raise KascadeNativeError("push_plan: one stream and one event per peer, at most %d peers" % MAX_FANOUT)
    plan = PushPlan()
    for i, (ptr, st, ev) in enumerate(zip(dst_pointers, streams, done_events)):
        plan.dst[i], plan.stream[i], plan.done_event[i] = int(ptr), int(st.cuda_stream), _cuda_event(ev)
    plan.count = len(dst_pointers)
    return plan


def peer_push(plan: PushPlan, src: torch.Tensor, offset_bytes: int, pitch_bytes: int, width_bytes: int, rows: int,
              ready_event: torch.cuda.Event):
    """Copy the row slice [offset, offset + width) of every `pitch`-byte row of `src` into the peers' buffers with
    the copy engines, after everything queued on the current stream (see kb200_peer_push)."""
    with torch.cuda.device(src.device):
        _check(load().kb200_peer_push(C.byref(plan), _ptr(src), offset_bytes, pitch_bytes, width_bytes, rows,
                                      C.c_void_p(_cuda_event(ready_event)), _stream()), "kb200_peer_push")


def stream_wait_events(events):
    """Make the current stream wait for the given torch events (those already recorded)."""
    handles = [int(e.cuda_event) for e in events if e.cuda_event]
    if handles:
        arr = (C.c_void_p * len(handles))(*handles)
        _check(load().kb200_stream_wait_events(_stream(), arr, len(handles)), "kb200_stream_wait_events")
