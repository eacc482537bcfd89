"""ctypes binding of the C ABI in ``include/fftsparse_amd.h``.

The shared library is built in-tree (``python -m fftsparse_amd.build``).  torch
is imported first so that the library's HIP runtime dependency resolves to the
runtime torch already loaded: device pointers and streams are shared.
Loading fails loudly when the library is missing -- there is no fallback.
"""
from __future__ import annotations

import ctypes
import os
from ctypes import POINTER, c_float, c_int, c_int32, c_int64, c_size_t, c_uint8, c_uint16, c_void_p
from pathlib import Path

import torch  # noqa: F401  (must precede the library load, see module docstring)

# FFTSPARSE_AMD_LIB may name another build of the same library (e.g. one built
# with different compile-time options); by default the in-tree build is used.
LIB_PATH = Path(os.environ.get("FFTSPARSE_AMD_LIB") or Path(__file__).resolve().with_name("libfftsparse_amd.so"))

FS_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ABI_VERSION = 15


class PoolArgs(ctypes.Structure):
    _fields_ = [("q", c_void_p), ("q_sh", c_int64), ("q_sl", c_int64),
                ("k", c_void_p), ("k_sh", c_int64), ("k_sl", c_int64),
                ("dtype", c_int), ("Hq", c_int), ("Hk", c_int), ("L", c_int), ("D", c_int), ("bs", c_int),
                ("q_b", c_void_p), ("k_b", c_void_p)]


class RopePoolArgs(ctypes.Structure):
    _fields_ = [("q", c_void_p), ("q_sh", c_int64), ("q_sl", c_int64),
                ("k", c_void_p), ("k_sh", c_int64), ("k_sl", c_int64),
                ("cos", c_void_p), ("sin", c_void_p), ("cs_sl", c_int64),
                ("q_out", c_void_p), ("qo_sh", c_int64), ("qo_sl", c_int64),
                ("k_out", c_void_p), ("ko_sh", c_int64), ("ko_sl", c_int64),
                ("dtype", c_int), ("Hq", c_int), ("Hk", c_int), ("L", c_int), ("D", c_int), ("bs", c_int),
                ("q_b", c_void_p), ("k_b", c_void_p)]


class XattnArgs(ctypes.Structure):
    _fields_ = [("q", c_void_p), ("q_sh", c_int64), ("q_sl", c_int64),
                ("k", c_void_p), ("k_sh", c_int64), ("k_sl", c_int64),
                ("dtype", c_int), ("Hq", c_int), ("Hk", c_int), ("L", c_int), ("D", c_int), ("stride", c_int),
                ("bs", c_int), ("norm", c_float), ("threshold", c_void_p), ("keep_sink", c_int),
                ("sums", c_void_p), ("blk_cnt", c_void_p), ("blk_bits", c_void_p), ("work", c_void_p),
                ("non_causal", c_int), ("torch_path", c_int), ("select_mode", c_int), ("perm", c_int * 16),
                ("kdb", c_int), ("no_softmax", c_int), ("chunk", c_int), ("keep_recent", c_int),
                ("head_group", c_int)]


class FlexArgs(ctypes.Structure):
    _fields_ = [("q", c_void_p), ("q_sh", c_int64), ("q_sl", c_int64),
                ("k", c_void_p), ("k_sh", c_int64), ("k_sl", c_int64),
                ("dtype", c_int), ("Hq", c_int), ("Hk", c_int), ("L", c_int), ("D", c_int), ("bs", c_int),
                ("gamma", c_float), ("tau", c_float), ("min_blocks", c_int), ("max_blocks", c_int),
                ("gqa_interleave", c_int), ("blk_cnt", c_void_p), ("blk_bits", c_void_p),
                ("head_info", c_void_p), ("head_js", c_void_p), ("vertical", c_void_p), ("slash", c_void_p),
                ("work", c_void_p)]


class CorrArgs(ctypes.Structure):
    _fields_ = [("q_b", c_void_p), ("k_b", c_void_p),
                ("dtype", c_int), ("Hq", c_int), ("Hk", c_int), ("N", c_int), ("D", c_int),
                ("local_window", c_int), ("keep_sink", c_int), ("remote_start", c_int),
                ("corr_threshold", c_float), ("corr_mode", c_int), ("corr_quantile", c_float),
                ("work", c_void_p), ("corr", c_void_p), ("corr_sum", c_void_p), ("keep_tau", c_void_p)]


class StatsArgs(ctypes.Structure):
    _fields_ = [("q_b", c_void_p), ("k_b", c_void_p),
                ("dtype", c_int), ("Hq", c_int), ("Hk", c_int), ("N", c_int), ("D", c_int),
                ("sample_taus", c_void_p), ("n_samples", c_int),
                ("col_start", c_int), ("col_end", c_int), ("n_cols", c_int),
                ("last_k", c_int),
                ("diag_var", c_void_p), ("col_mean", c_void_p), ("col_sel", c_void_p),
                ("last_scores", c_void_p), ("last_sel", c_void_p)]


class ScoresArgs(ctypes.Structure):
    _fields_ = [("q_b", c_void_p), ("k_b", c_void_p),
                ("dtype", c_int), ("Hq", c_int), ("Hk", c_int), ("N", c_int), ("D", c_int),
                ("local_window", c_int), ("keep_sink", c_int), ("remote_start", c_int),
                ("corr_threshold", c_float), ("corr_mode", c_int), ("corr_quantile", c_float),
                ("corr", c_void_p), ("corr_sum", c_void_p), ("keep_tau", c_void_p),
                ("sample_taus", c_void_p), ("n_samples", c_int),
                ("col_start", c_int), ("col_end", c_int), ("n_cols", c_int),
                ("last_k", c_int),
                ("diag_var", c_void_p), ("col_mean", c_void_p), ("col_sel", c_void_p),
                ("last_scores", c_void_p), ("last_sel", c_void_p),
                ("work", c_void_p)]


class SelectArgs(ctypes.Structure):
    _fields_ = [("q_b", c_void_p), ("k_b", c_void_p),
                ("dtype", c_int), ("Hq", c_int), ("Hk", c_int), ("N", c_int), ("Nk", c_int), ("D", c_int),
                ("mask_causal", c_int),
                ("keep_sink", c_int), ("keep_recent", c_int), ("local_window", c_int), ("remote_start", c_int),
                ("dyn_mode", c_int), ("stripe_all_diffuse", c_int),
                ("diag_var", c_void_p), ("n_samples", c_int), ("stripe_threshold", c_float),
                ("keep_tau", c_void_p),
                ("qk_topk_ratio", c_float),
                ("col_mode", c_int), ("col_sel", c_void_p), ("last_sel", c_void_p),
                ("mean_var", c_void_p), ("is_stripe", c_void_p),
                ("blk_cnt", c_void_p), ("blk_bits", c_void_p)]


class AttnArgs(ctypes.Structure):
    _fields_ = [("q", c_void_p), ("q_sb", c_int64), ("q_sh", c_int64), ("q_sl", c_int64),
                ("k", c_void_p), ("k_sb", c_int64), ("k_sh", c_int64), ("k_sl", c_int64),
                ("v", c_void_p), ("v_sb", c_int64), ("v_sh", c_int64), ("v_sl", c_int64),
                ("out", c_void_p), ("o_sb", c_int64), ("o_sh", c_int64), ("o_sl", c_int64),
                ("dtype", c_int), ("B", c_int), ("Hq", c_int), ("Hk", c_int), ("Lq", c_int), ("Lk", c_int),
                ("D", c_int), ("bs", c_int),
                ("is_causal", c_int), ("softmax_scale", c_float), ("gqa_interleave", c_int),
                ("blk_cnt", c_void_p), ("blk_bits", c_void_p), ("work", c_void_p)]


class PlanArgs(ctypes.Structure):
    _fields_ = [("block_table", c_void_p), ("t_sb", c_int64), ("seq_lens", c_void_p), ("new_lens", c_void_p),
                ("free_pages", c_void_p), ("free_count", c_void_p),
                ("B", c_int), ("P", c_int), ("F", c_int), ("page_size", c_int), ("T", c_int),
                ("cu_lens", c_void_p), ("seq_lens_out", c_void_p), ("positions", c_void_p), ("slots", c_void_p),
                ("free_count_out", c_void_p), ("lacking", c_void_p)]


class RopeArgs(ctypes.Structure):
    _fields_ = [("q", c_void_p), ("q_st", c_int64), ("q_sh", c_int64),
                ("k", c_void_p), ("k_st", c_int64), ("k_sh", c_int64),
                ("v", c_void_p), ("v_st", c_int64), ("v_sh", c_int64),
                ("positions", c_void_p), ("inv_freq", c_void_p), ("attention_factor", c_float),
                ("pos_bytes", c_int), ("half", c_int), ("interleaved", c_int),
                ("dtype", c_int), ("T", c_int), ("Hq", c_int), ("Hk", c_int), ("D", c_int),
                ("q_out", c_void_p), ("qo_st", c_int64), ("qo_sh", c_int64),
                ("k_out", c_void_p), ("ko_st", c_int64), ("ko_sh", c_int64),
                ("slots", c_void_p),
                ("k_cache", c_void_p), ("kc_sp", c_int64), ("kc_ss", c_int64), ("kc_sh", c_int64),
                ("v_cache", c_void_p), ("vc_sp", c_int64), ("vc_ss", c_int64), ("vc_sh", c_int64),
                ("num_pages", c_int64), ("page_size", c_int), ("k_scale", c_void_p), ("v_scale", c_void_p)]


class PagedAttnArgs(ctypes.Structure):
    _fields_ = [("q", c_void_p), ("q_st", c_int64), ("q_sh", c_int64),
                ("out", c_void_p), ("o_st", c_int64), ("o_sh", c_int64),
                ("k_cache", c_void_p), ("k_sp", c_int64), ("k_ss", c_int64), ("k_sh", c_int64),
                ("v_cache", c_void_p), ("v_sp", c_int64), ("v_ss", c_int64), ("v_sh", c_int64),
                ("block_table", c_void_p), ("t_sb", c_int64), ("cu_lens", c_void_p), ("seq_lens", c_void_p),
                ("dtype", c_int), ("B", c_int), ("T", c_int), ("Hq", c_int), ("Hk", c_int), ("D", c_int),
                ("P", c_int), ("page_size", c_int), ("num_pages", c_int64),
                ("max_new", c_int), ("window", c_int), ("sinks", c_int), ("softmax_scale", c_float),
                ("work", c_void_p), ("k_scale", c_void_p), ("v_scale", c_void_p),
                ("mask", c_void_p), ("mask_words", c_int), ("positions", c_void_p)]


class WindowAttnArgs(ctypes.Structure):
    _fields_ = [("q", c_void_p), ("q_sb", c_int64), ("q_sh", c_int64), ("q_sl", c_int64),
                ("k", c_void_p), ("k_sb", c_int64), ("k_sh", c_int64), ("k_sl", c_int64),
                ("v", c_void_p), ("v_sb", c_int64), ("v_sh", c_int64), ("v_sl", c_int64),
                ("out", c_void_p), ("o_sb", c_int64), ("o_sh", c_int64), ("o_sl", c_int64),
                ("dtype", c_int), ("B", c_int), ("Hq", c_int), ("Hk", c_int), ("Lq", c_int), ("Lk", c_int),
                ("D", c_int), ("window", c_int), ("sinks", c_int), ("softmax_scale", c_float), ("work", c_void_p)]


class TreePlanArgs(ctypes.Structure):
    _fields_ = [("parents", c_void_p), ("cu_lens", c_void_p), ("seq_lens", c_void_p),
                ("B", c_int), ("T", c_int), ("words", c_int), ("window", c_int), ("sinks", c_int),
                ("positions", c_void_p), ("mask", c_void_p)]


class TreeAcceptArgs(ctypes.Structure):
    _fields_ = [("parents", c_void_p), ("tokens", c_void_p), ("chosen", c_void_p), ("cu_lens", c_void_p),
                ("token_bytes", c_int), ("B", c_int), ("T", c_int), ("most", c_int),
                ("kept", c_void_p), ("kept_lens", c_void_p), ("dropped", c_void_p), ("next_tokens", c_void_p)]


class CacheMoveArgs(ctypes.Structure):
    _fields_ = [("k_caches", POINTER(c_void_p)), ("v_caches", POINTER(c_void_p)),
                ("k_cache", c_void_p), ("k_sl", c_int64), ("k_sp", c_int64), ("k_ss", c_int64), ("k_sh", c_int64),
                ("v_cache", c_void_p), ("v_sl", c_int64), ("v_sp", c_int64), ("v_ss", c_int64), ("v_sh", c_int64),
                ("block_table", c_void_p), ("t_sb", c_int64), ("cu_lens", c_void_p), ("seq_lens", c_void_p),
                ("kept", c_void_p), ("layers", c_int), ("B", c_int), ("T", c_int), ("Hk", c_int), ("D", c_int),
                ("P", c_int), ("page_size", c_int), ("elem_bytes", c_int), ("num_pages", c_int64)]


STRUCTS = [PoolArgs, CorrArgs, StatsArgs, SelectArgs, AttnArgs, ScoresArgs, RopePoolArgs, XattnArgs, FlexArgs,
           PlanArgs, RopeArgs, PagedAttnArgs, WindowAttnArgs, TreePlanArgs, TreeAcceptArgs, CacheMoveArgs]

ENTRY_POINTS = ["fs_pool", "fs_rope_pool", "fs_corr_work_bytes", "fs_corr", "fs_stats", "fs_scores_work_bytes",
                "fs_scores", "fs_scores_noalloc", "fs_select", "fs_bsattn_work_bytes",
                "fs_bsattn", "fs_bsattn_prepare", "fs_bsattn_run", "fs_xattn_work_bytes", "fs_xattn",
                "fs_flex_work_bytes", "fs_flex", "fs_plan", "fs_rope", "fs_paged_attn_work_bytes", "fs_paged_attn",
                "fs_window_attn_work_bytes", "fs_window_attn", "fs_tree_plan", "fs_tree_accept", "fs_cache_move",
                "fs_last_error", "fs_abi_version", "fs_sizeof_args"]

_lib = None


def load() -> ctypes.CDLL:
    """Load the in-tree library once; raise if it is missing or stale."""
    global _lib
    if _lib is not None:
        return _lib
    if not LIB_PATH.exists():
        raise RuntimeError(
            f"fftsparse_amd native library not found at {LIB_PATH}; build it with "
            "`python -m fftsparse_amd.build` (no CPU fallback exists)")
    lib = ctypes.CDLL(str(LIB_PATH))
    lib.fs_last_error.restype = ctypes.c_char_p
    lib.fs_abi_version.restype = c_int
    lib.fs_sizeof_args.restype = c_size_t
    lib.fs_sizeof_args.argtypes = [c_int]
    lib.fs_corr_work_bytes.restype = c_size_t
    lib.fs_corr_work_bytes.argtypes = [c_int, c_int, c_int]
    lib.fs_scores_work_bytes.restype = c_size_t
    lib.fs_scores_work_bytes.argtypes = [c_int, c_int, c_int]
    lib.fs_flex_work_bytes.restype = c_size_t
    lib.fs_flex_work_bytes.argtypes = [c_int, c_int, c_int, c_int, c_float]
    lib.fs_xattn_work_bytes.restype = c_size_t
    lib.fs_xattn_work_bytes.argtypes = [ctypes.POINTER(XattnArgs)]
    lib.fs_bsattn_work_bytes.restype = c_size_t
    lib.fs_bsattn_work_bytes.argtypes = [POINTER(AttnArgs)]
    lib.fs_paged_attn_work_bytes.restype = c_size_t
    lib.fs_paged_attn_work_bytes.argtypes = [POINTER(PagedAttnArgs)]
    lib.fs_window_attn_work_bytes.restype = c_size_t
    lib.fs_window_attn_work_bytes.argtypes = [POINTER(WindowAttnArgs)]
    for name, st in [("fs_pool", PoolArgs), ("fs_rope_pool", RopePoolArgs), ("fs_corr", CorrArgs),
                     ("fs_stats", StatsArgs), ("fs_scores", ScoresArgs), ("fs_scores_noalloc", ScoresArgs),
                     ("fs_select", SelectArgs), ("fs_bsattn", AttnArgs), ("fs_bsattn_prepare", AttnArgs),
                     ("fs_bsattn_run", AttnArgs), ("fs_xattn", XattnArgs),
                     ("fs_flex", FlexArgs), ("fs_plan", PlanArgs), ("fs_rope", RopeArgs),
                     ("fs_paged_attn", PagedAttnArgs), ("fs_window_attn", WindowAttnArgs),
                     ("fs_tree_plan", TreePlanArgs), ("fs_tree_accept", TreeAcceptArgs),
                     ("fs_cache_move", CacheMoveArgs)]:
        fn = getattr(lib, name)
        fn.restype = c_int
        fn.argtypes = [POINTER(st), c_void_p]
    if lib.fs_abi_version() != ABI_VERSION:
        raise RuntimeError("fftsparse_amd: library ABI version mismatch; rebuild it")
    for i, st in enumerate(STRUCTS):
        if lib.fs_sizeof_args(i) != ctypes.sizeof(st):
            raise RuntimeError(f"fftsparse_amd: {st.__name__} layout differs from the library; rebuild it")
    _lib = lib
    return lib


def same_device(*tensors) -> torch.device:
    """The one GPU that every given tensor (None entries skipped) lives on.
    The kernels dereference the tensors' pointers on that GPU, so a host
    tensor, or tensors on two GPUs, raise ValueError before any launch."""
    first = index = None
    for t in tensors:
        if t is None:
            continue
        if t.get_device() != index:                        # -1: on the host
            if not t.is_cuda:
                raise ValueError(f"tensors must be on the GPU, got one on {t.device}")
            if first is not None:
                raise ValueError(f"tensors on different devices: {first.device} and {t.device}")
            first, index = t, t.get_device()
    if first is None:
        raise ValueError("no tensor given")
    return first.device


def _raw_stream(index: int) -> int:
    """hipStream_t of torch's current stream of a device (the device and Stream objects that
    torch.cuda.current_stream() makes on the way cost 2-3 us of a call)."""
    return torch._C._cuda_getCurrentRawStream(index)


def call(name: str, args, device: torch.device | None = None) -> None:
    """Invoke an entry point on torch's current stream of ``device`` (default:
    the current device), with that device current; raise on a non-zero status."""
    lib = load()
    current = torch.cuda.current_device()
    if device is None or device.index is None or device.index == current:
        rc = getattr(lib, name)(ctypes.byref(args), _raw_stream(current))
    else:
        with torch.cuda.device(device):
            rc = getattr(lib, name)(ctypes.byref(args), _raw_stream(device.index))
    if rc != 0:
        msg = lib.fs_last_error().decode(errors="replace")
        if rc == -1:
            raise ValueError(msg)
        raise RuntimeError(msg)


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()
