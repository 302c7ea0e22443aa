"""ctypes binding of libcacheslide_sm100.so (the C ABI in include/cacheslide_b200.h).

Loading is strict: if the shared library is missing or cannot be loaded, every
operator raises ``RuntimeError``.  There is no CPU fallback anywhere in this
package; operators also reject CPU tensors.
"""

from __future__ import annotations

import ctypes
import threading
from pathlib import Path

import torch

LIB_PATH = Path(__file__).resolve().parent / "_lib" / "libcacheslide_sm100.so"

CS_OK, CS_ERR_INVALID, CS_ERR_CUDA, CS_ERR_UNSUPPORTED, CS_ERR_TOO_LARGE = 0, 1, 2, 3, 4
CS_F32, CS_F16, CS_BF16, CS_F64 = 0, 1, 2, 3

ST_SLOT_RANGE = 1 << 0
ST_NONFINITE = 1 << 1
ST_LOGIT_NONFINITE = 1 << 2
ST_POS_RANGE = 1 << 3
ST_PATH_NEG = 1 << 4
ST_PATH_AVAIL = 1 << 5
ST_PATH_INCR = 1 << 6
ST_PATH_GAP = 1 << 7
ST_TIMEOUT = 1 << 8
ST_INPUT_NONFINITE = 1 << 9
ST_CAPACITY = 1 << 10

POS_CONTEXTUAL, POS_FIXED, POS_TABLE, POS_CHUNK = 0, 1, 2, 3
LAUNCH_OVERLAP_PREV = 1

DTYPES = {
    torch.float32: CS_F32,
    torch.float16: CS_F16,
    torch.bfloat16: CS_BF16,
    torch.float64: CS_F64,
}

_p = ctypes.c_void_p
_i64 = ctypes.c_int64
_i32 = ctypes.c_int32
_f64 = ctypes.c_double


class PagedKV(ctypes.Structure):
    device = None  # index of the cache's device, where paged_view made the view
    _fields_ = [
        ("cache", _p),
        ("num_blocks", _i64), ("kv_heads", _i64), ("block_size", _i64), ("head_dim", _i64),
        ("stride_block", _i64), ("stride_head", _i64), ("stride_offset", _i64),
        ("stride_elem", _i64),
        ("side_k", _p), ("side_v", _p), ("side_capacity", _i64),
        ("side_stride_row", _i64), ("side_stride_head", _i64), ("side_stride_elem", _i64),
        ("dtype", _i32),
    ]


class AttnParams(ctypes.Structure):
    _fields_ = [
        ("q", _p), ("q_stride_tok", _i64), ("q_stride_head", _i64),
        ("nq", _i32), ("hq", _i32), ("d", _i32),
        ("qpos", _p),
        ("k", _p), ("v", _p),
        ("k_stride_tok", _i64), ("k_stride_head", _i64),
        ("v_stride_tok", _i64), ("v_stride_head", _i64),
        ("paged", PagedKV),
        ("kv_slots", _p),
        ("nk", _i32), ("hkv", _i32), ("dv", _i32),
        ("kpos", _p),
        ("E", _p), ("e_stride_d", _i64), ("e_stride_p", _i64), ("npos", _i32),
        ("scale", _f64),
        ("pos_mode", _i32),
        ("fixed_pos", _p), ("fp_stride_h", _i64), ("fp_stride_q", _i64), ("fp_stride_k", _i64),
        ("table", _p), ("tb_stride_h", _i64), ("tb_stride_r", _i64), ("tb_stride_c", _i64),
        ("q_row", _p), ("k_ord", _p),
        ("key_chunk", _p), ("chunk_off", _p), ("co_stride_h", _i64), ("co_stride_q", _i64),
        ("nchunks", _i32),
        ("gate_mask", _p), ("gm_stride_h", _i64), ("gm_stride_q", _i64),
        ("vis_mask", _p), ("vm_stride_h", _i64), ("vm_stride_q", _i64),
        ("q_selected", _p), ("k_fixed", _p),
        ("strict", _i32), ("atol", _f64), ("positions_only", _i32),
        ("out_positions", _p), ("op_stride_h", _i64), ("op_stride_q", _i64),
        ("out", _p), ("o_stride_tok", _i64), ("o_stride_head", _i64),
        ("in_dtype", _i32), ("out_dtype", _i32),
        ("status", _p),
        ("launch_flags", _i32),
        ("nq_dev", _p),
    ]


class ScatterItem(ctypes.Structure):
    """cs_slide_scatter_item: one request of cs_slide_scatter_batch."""
    _fields_ = [
        ("slots", _p), ("rows", _p), ("n", _i64), ("k", _p), ("v", _p),
        ("in_stride_row", _i64), ("in_stride_head", _i64), ("status", _p),
    ]


class InitializeItem(ctypes.Structure):
    """cs_wca_initialize_item: one request of cs_wca_initialize_batch."""
    _fields_ = [
        ("cached", _p), ("c_stride_row", _i64), ("c_stride_head", _i64),
        ("fresh", _p), ("f_stride_row", _i64), ("f_stride_head", _i64),
        ("n", _i64), ("reused", _p), ("dev_out", _p), ("alpha_out", _p), ("candidate", _p),
        ("selected", _p), ("removed", _p), ("counts_out", _p), ("status", _p),
    ]


class UpdateItem(ctypes.Structure):
    """cs_wca_update_item: one request of cs_wca_update_batch."""
    _fields_ = [
        ("cached_k", _p), ("cached_v", _p), ("c_stride_row", _i64), ("c_stride_head", _i64),
        ("fresh_k", _p), ("fresh_v", _p), ("f_stride_row", _i64), ("f_stride_head", _i64),
        ("indices", _p), ("a", _i64), ("alpha", _p), ("mandatory", _p),
        ("fused_k", _p), ("fused_v", _p), ("next_alpha_out", _p), ("used_alpha_out", _p),
        ("cos_out", _p), ("slots", _p), ("status", _p), ("a_dev", _p),
    ]


class CommitItem(ctypes.Structure):
    """cs_wca_commit_item: one request of cs_wca_commit_batch."""
    _fields_ = [
        ("indices", _p), ("a", _i64), ("next_alpha", _p), ("cos", _p), ("n", _i64),
        ("budget", _i64), ("initial_dev", _p), ("alpha", _p), ("candidate", _p),
        ("selected", _p), ("removed", _p), ("removed_out", _p), ("promoted_out", _p),
        ("counts_out", _p), ("status", _p), ("a_dev", _p),
    ]


class QKVParams(ctypes.Structure):
    """cs_qkv_params: the selective-layer QKV projection (cs_qkv_gather_lora)."""
    _fields_ = [
        ("src0", _p), ("src0_stride", _i64), ("src0_rows", _i64),
        ("src1", _p), ("src1_stride", _i64), ("src1_rows", _i64),
        ("row_src", _p), ("row_idx", _p), ("a", _i64), ("hidden", _i64), ("n_out", _i64),
        ("w", _p), ("lora_a", _p), ("lora_b", _p), ("rank", _i32),
        ("out", _p), ("out_stride", _i64), ("dtype", _i32), ("status", _p), ("a_dev", _p),
    ]


class RotaryParams(ctypes.Structure):
    """cs_rotary_params: head norms and position rotation of queries and keys."""
    _fields_ = [
        ("cos", _p), ("sin", _p), ("table_rows", _i64), ("table_stride", _i64),
        ("positions", _p), ("tokens", _i64),
        ("head_dim", _i32), ("rot", _i32), ("interleaved", _i32), ("dtype", _i32),
        ("weight_dtype", _i32), ("eps", _f64),
        ("q", _p), ("q_stride_tok", _i64), ("q_stride_head", _i64), ("q_heads", _i32),
        ("q_weight", _p), ("q_out", _p), ("qo_stride_tok", _i64), ("qo_stride_head", _i64),
        ("k", _p), ("k_stride_tok", _i64), ("k_stride_head", _i64), ("k_heads", _i32),
        ("k_weight", _p), ("k_out", _p), ("ko_stride_tok", _i64), ("ko_stride_head", _i64),
        ("status", _p),
    ]


class PrefixShape(ctypes.Structure):
    """cs_prefix_shape: the lengths of a batch behind shared prefixes."""
    _fields_ = [
        ("q_heads", _i32), ("kv_heads", _i32), ("head_dim", _i32), ("dtype", _i32),
        ("groups", _i32), ("requests", _i32),
        ("prefix_lens", _p), ("group_sizes", _p), ("query_lens", _p), ("suffix_lens", _p),
    ]


class PrefixPlanInfo(ctypes.Structure):
    """cs_prefix_plan_info: where a plan's parts lie and what a call needs."""
    _fields_ = [
        ("words", _i64), ("workspace", _i64), ("tokens", _i64), ("n_prefix", _i64),
        ("n_suffix", _i64), ("item_off", _i64), ("n_items", _i64), ("join_off", _i64),
        ("n_join", _i64), ("list_off", _i64), ("part_tokens", _i64), ("variant", _i32),
        ("group", _i32),
    ]


class PrefixParams(ctypes.Structure):
    """cs_prefix_params: one call of the attention behind shared prefixes."""
    _fields_ = [
        ("q", _p), ("q_stride_tok", _i64), ("q_stride_head", _i64), ("paged", PagedKV),
        ("prefix_slots", _p), ("suffix_slots", _p), ("q_heads", _i32), ("scale", _f64),
        ("out", _p), ("o_stride_tok", _i64), ("o_stride_head", _i64), ("lse", _p),
        ("status", _p),
    ]


class StepMapsParams(ctypes.Structure):
    """cs_step_maps_params: block tables and slot maps of a step."""
    _fields_ = [
        ("lengths", _p), ("new_tokens", _p), ("requests", _i32), ("block_size", _i32),
        ("num_blocks", _i64), ("tables", _p), ("table_stride", _i64), ("table_width", _i32),
        ("position_offset", _i32), ("free_blocks", _p), ("free_count", _p), ("free_left", _p),
        ("free_size", _i64),
        ("tokens", _i64), ("keys", _i64), ("starts", _p), ("positions", _p), ("slots", _p),
        ("key_starts", _p), ("key_slots", _p), ("status", _p),
    ]


class KV4Pool(ctypes.Structure):
    """cs_kv4_pool: a paged pool held in 4 bits."""
    _fields_ = [
        ("storage", _p), ("num_blocks", _i64), ("kv_heads", _i32), ("block_size", _i32),
        ("head_dim", _i32), ("group", _i32), ("dtype", _i32),
    ]


class KV4AttnParams(ctypes.Structure):
    """cs_kv4_attn_params: attention over a pool held in 4 bits."""
    _fields_ = [
        ("q", _p), ("q_stride_tok", _i64), ("q_stride_head", _i64), ("tokens", _i64),
        ("q_heads", _i32), ("requests", _i32), ("pool", KV4Pool), ("tables", _p),
        ("table_stride", _i64), ("table_width", _i32), ("zero_rest", _i32), ("lengths", _p),
        ("starts", _p), ("scale", _f64), ("out", _p), ("o_stride_tok", _i64),
        ("o_stride_head", _i64), ("lse", _p), ("status", _p),
    ]


_SIGNATURES = {
    "cs_step_maps": [ctypes.POINTER(StepMapsParams), _p],
    "cs_kv4_append": [ctypes.POINTER(KV4Pool), _p, _i64, _p, _i64, _i64, _p, _i64, _i64, _p, _p],
    "cs_kv4_gather": [ctypes.POINTER(KV4Pool), _p, _i64, _p, _i64, _i64, _p, _i64, _i64, _p, _p],
    "cs_kv4_attn_workspace": [ctypes.POINTER(KV4AttnParams)],
    "cs_kv4_attn": [ctypes.POINTER(KV4AttnParams), _p, _p],
    "cs_prefix_plan": [ctypes.POINTER(PrefixShape), ctypes.POINTER(PrefixPlanInfo), _p, _i64],
    "cs_prefix_attn": [ctypes.POINTER(PrefixParams), ctypes.POINTER(PrefixPlanInfo), _p, _p, _p],
    "cs_qk_norm_rope": [ctypes.POINTER(RotaryParams), _p],
    "cs_qk_norm_rope_grad_workspace": [ctypes.POINTER(RotaryParams)],
    "cs_qk_norm_rope_grad": [ctypes.POINTER(RotaryParams), _p, _p, _p, _p, _p, _p],
    "cs_kv_append_rotated": [ctypes.POINTER(RotaryParams), ctypes.POINTER(PagedKV), _p, _p, _i64,
                             _i64, _p],
    "cs_slide_gather": [ctypes.POINTER(PagedKV), _p, _i64, _p, _p, _i64, _i64, _p, _p],
    "cs_slide_scatter": [ctypes.POINTER(PagedKV), _p, _p, _i64, _p, _p, _i64, _i64, _p, _p],
    "cs_slide_relocate": [ctypes.POINTER(PagedKV), _p, _p, _i64, _p, _p],
    "cs_slide_pack_pages": [ctypes.POINTER(PagedKV), _p, _i64, _p, _p, _p],
    "cs_slide_unpack_pages": [ctypes.POINTER(PagedKV), _p, _i64, _p, _p, _p],
    "cs_slide_scatter_batch": [ctypes.POINTER(PagedKV), ctypes.POINTER(ScatterItem), _i32, _p],
    "cs_wca_initialize_batch": [ctypes.POINTER(InitializeItem), _i32, _i64, _i64, _i32, _f64,
                                _i32, _p],
    "cs_wca_update_batch": [ctypes.POINTER(UpdateItem), _i32, _i64, _i64, _i32, _i32, _f64,
                            _i32, ctypes.POINTER(PagedKV), _p],
    "cs_wca_commit_batch": [ctypes.POINTER(CommitItem), _i32, _f64, _i32, _p],
    "cs_wca_deviation": [_p, _i64, _i64, _p, _p, _i64, _i64, _i64, _i64, _i64, _i32, _f64,
                         _i32, _p, _p, _p, _p],
    "cs_wca_cosine": [_p, _i64, _i64, _p, _i64, _i64, _p, _i64, _i64, _i64, _i32, _f64, _p,
                      _p, _p],
    "cs_wca_row_sums": [_p, _i64, _i64, _p, _p, _i64, _i64, _i64, _i64, _i64, _i32, _i64, _p,
                        _p, _p, _p, _p],
    "cs_wca_weights": [_p, _p, _i64, _f64, _i32, _p, _p, _p, _p, _p, _p],
    "cs_wca_select_topk": [_p, _p, _i64, _i64, _p, _p, _p, _p, _p],
    "cs_wca_active_rows": [_p, _p, _i64, _i64, _p, _p, _p, _p, _p],
    "cs_wca_initialize": [_p, _i64, _i64, _p, _i64, _i64, _i64, _i64, _i64, _i32, _p, _f64,
                          _i32, _p, _p, _p, _p, _p, _p, _p, _p],
    "cs_wca_update": [_p, _p, _i64, _i64, _p, _p, _i64, _i64, _p, _i64, _i64, _i64, _i32, _p,
                      _p, _i32, _f64, _i32, _p, _p, _p, _p, _p, ctypes.POINTER(PagedKV), _p,
                      _p, _p],
    "cs_wca_commit": [_p, _i64, _p, _p, _f64, _i32, _i64, _i64, _p, _p, _p, _p, _p, _p, _p,
                      _p, _p, _p],
    "cs_qkv_gather_lora": [ctypes.POINTER(QKVParams), _p],
    "cs_cope_attn": [ctypes.POINTER(AttnParams), _p],
    "cs_cope_attn_prefill": [ctypes.POINTER(AttnParams), _p],
    "cs_cope_attn_prefill_batch": [ctypes.POINTER(AttnParams), _i32, _p],
    "cs_cope_attn_decode_workspace": [ctypes.POINTER(AttnParams)],
    "cs_cope_attn_decode": [ctypes.POINTER(AttnParams), _p, _p],
    "cs_cope_attn_decode_noalloc": [ctypes.POINTER(AttnParams), _p],
    "cs_cope_attn_decode_batch_workspace": [ctypes.POINTER(AttnParams), _i32],
    "cs_cope_attn_decode_batch": [ctypes.POINTER(AttnParams), _i32, _p, _p],
    "cs_cope_positions": [_p, _i64, _i64, _p, _i64, _i64, _i32, _i64, _i64, _i32, _i32, _p,
                          _i64, _i64, _p, _p],
    "cs_cope_bias": [_p, _i64, _i64, _p, _i64, _i64, _i32, _i32, _p, _i64, _i64, _i32, _i64,
                     _i64, _i32, _p, _i64, _i64, _p, _p],
    "cs_cope_chunk_offsets": [_p, _i64, _i64, _i32, _i32, _i32, _p, _p, _p, _p, _i64, _i64,
                              _i32, _p, _p, _p, _i32, _p, _i64, _i64, _i64, _i32, _i32, _i32,
                              _p, _i64, _i64, _i32, _p, _p],
    "cs_cope_validate_path": [_p, _i64, _i64, _p, _p, _p, _i64, _i64, _i32, _i64, _i64, _f64,
                              _i32, _p, _p],
    "cs_build_info": [],
    "cs_abi_version": [],
}
_RESTYPES = {"cs_build_info": ctypes.c_char_p, "cs_abi_version": _i32,
             "cs_cope_attn_decode_workspace": _i64,
             "cs_qk_norm_rope_grad_workspace": _i64,
             "cs_kv4_attn_workspace": _i64,
             "cs_cope_attn_decode_batch_workspace": _i64}

EXPORTED = tuple(_SIGNATURES)

_lib = None
_lock = threading.Lock()


def load() -> ctypes.CDLL:
    """Load the CUDA library once; raise RuntimeError when it is unavailable."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not LIB_PATH.exists():
                raise RuntimeError(
                    f"{LIB_PATH.name} is not built; run `python -m cacheslide_b200.build`"
                )
            lib = ctypes.CDLL(str(LIB_PATH))
            for name, args in _SIGNATURES.items():
                fn = getattr(lib, name)
                fn.argtypes = args
                fn.restype = _RESTYPES.get(name, ctypes.c_int)
            _lib = lib
    return _lib


def check(rc: int, name: str) -> None:
    if rc == CS_OK:
        return
    if rc == CS_ERR_INVALID:
        raise ValueError(f"{name}: invalid arguments for the CUDA kernel")
    if rc == CS_ERR_UNSUPPORTED:
        raise ValueError(f"{name}: shape/dtype combination is not supported on device")
    raise RuntimeError(f"{name}: CUDA launch failed (status {rc})")


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


# the current stream's handle without a Stream object around it, where this
# torch has that (a decode step calls this a few hundred times)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream_of(device: torch.device) -> int:
    if _raw_stream is not None and device.index is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def launch(name: str, device: torch.device, *args) -> None:
    """Call an entry point whose last argument is the stream, on ``device``'s
    current stream and with ``device`` current, and check its status."""
    fn = getattr(load(), name)
    if torch.cuda.current_device() == device.index:
        rc = fn(*args, stream_of(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, stream_of(device))
    check(rc, name)


def require_cuda(*tensors: torch.Tensor) -> torch.device:
    device = None
    for t in tensors:
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or t.device.type != "cuda":
            raise ValueError(
                "cacheslide_b200 operators run on CUDA tensors only (no CPU fallback)"
            )
        if device is None:
            device = t.device
        elif t.device != device:
            raise ValueError("all tensors must be on the same CUDA device")
    if device is None:
        raise ValueError("cacheslide_b200 operators need at least one CUDA tensor")
    return device


class Status:
    """A device int32 status word per call; read after the stream drains."""

    def __init__(self, device: torch.device):
        self.word = torch.zeros(1, dtype=torch.int32, device=device)

    @property
    def ptr(self) -> int:
        return self.word.data_ptr()

    def read(self) -> int:
        return int(self.word.item())


def status_ptr(status: Status | None, device: int) -> int | None:
    """The status word's address for a launch on the device of that index."""
    if status is None:
        return None
    if status.word.get_device() != device:
        raise ValueError("the status must be on the same CUDA device as the tensors")
    return status.ptr


def require_pool_on(kv: PagedKV, device: int) -> None:
    """Raise if the pool behind a view is known to lie on another device."""
    if kv.device is not None and kv.device != device:
        raise ValueError("the pool must be on the same CUDA device as the tensors")


def paged_view(
    cache: torch.Tensor,
    side_k: torch.Tensor | None = None,
    side_v: torch.Tensor | None = None,
) -> PagedKV:
    """Describe a [blocks, kv_heads, block_size, 2*D] view (any strides)."""
    if cache.ndim != 4 or cache.shape[-1] % 2:
        raise ValueError("cache must be [blocks, kv_heads, block_size, 2*D]")
    if cache.dtype not in DTYPES:
        raise ValueError("cache dtype must be float16/bfloat16/float32/float64")
    blocks, heads, block_size, width = cache.shape
    kv = PagedKV(cache.data_ptr(), blocks, heads, block_size, width // 2, *cache.stride(),
                 None, None, 0, 0, 0, 0, DTYPES[cache.dtype])
    kv.device = cache.get_device()
    if side_k is not None and side_v is not None:
        if side_k.stride() != side_v.stride() or side_k.shape != side_v.shape:
            raise ValueError("sidecar K and V must share shape and strides")
        kv.side_k, kv.side_v = side_k.data_ptr(), side_v.data_ptr()
        kv.side_capacity = side_k.shape[0]
        kv.side_stride_row, kv.side_stride_head, kv.side_stride_elem = side_k.stride()
    return kv
