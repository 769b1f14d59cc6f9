"""ferry_amd -- MI355X-native per-GPU sparse KV miss-stream executor.

Python mirror of the C-ABI in include/ferry_amd.h, loaded with ctypes.  The
compute path is libferry_amd.so (hand-written gfx950 HIP kernels); there is no
CPU fallback: importing this package without the built library raises.

torch supplies device memory and streams only.  It is imported before the
library so that one HIP runtime serves both.

Reference interfaces mirrored (clearleo126/ferry, paths relative to its tree):
  Executor.fetch_step      run_miss_workload mode C / exec_step C engine
                           (src/workloads/kv_exec.cuh:188-292,
                           src/runtime/wla_multigpu.cuh:2527-2604)
  Executor.sparse_decode   attn_kernel / wla_attn_kernel (real attention here)
  Pages, rope_freqs        (none: a paged cache of whole contexts; its pages are
                           block records of the host tier)
  queue_selftest           bench_queue (src/benches/bench_queue.cu:62-123)
  SelGen / refgen_selections  replay_miss_stream (src/workloads/missstream.cuh:104)
  arrivals / Sched         request arrivals and the per-GPU tick loop
                           (src/runtime/wla_multigpu.cuh:497-501, 829-864,
                           2610-2665)
"""
import ctypes as C
import os
import struct

import numpy as np
import torch  # noqa: F401  (HIP runtime + device memory; load before the library)

__all__ = [
    "FerryError", "Executor", "SelGen", "Sched", "queue_selftest", "refgen_selections",
    "ctx_uniform", "arrivals", "lib", "LIB_PATH", "F32", "F16", "BF16", "FP8", "LRU_STEP",
    "LRU_SERIAL", "ASSIGN_SPREAD", "ASSIGN_AFFINITY", "ATTN_AUTO", "ATTN_VALU", "ATTN_MFMA",
    "ATTN_GROUP", "MISS_DTYPE", "EMPTY", "ARRIVAL_STEADY", "ARRIVAL_BURSTY", "ARRIVAL_POISSON", "ARRIVAL_MMPP",
    "SCHED_FIFO", "SCHED_PINNED", "trace_load", "TOPK_PER_HEAD", "TOPK_LAYER_MAX", "CAP_GROUP",
    "CAP_PER_MEMBER", "Pages", "rope_freqs", "ROPE_PLAIN", "ROPE_LINEAR", "ROPE_BASE", "ROPE_PARTS",
]

LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libferry_amd.so")
if not os.path.exists(LIB_PATH):
    raise ImportError(f"{LIB_PATH} is not built: run `make -C ferry_amd` "
                      "(or __graft_entry__.build()); there is no fallback path")
lib = C.CDLL(LIB_PATH)

F32, F16, BF16, FP8 = 0, 1, 2, 3
LRU_STEP, LRU_SERIAL = 0, 1
ASSIGN_SPREAD, ASSIGN_AFFINITY = 0, 1
ATTN_AUTO, ATTN_VALU, ATTN_MFMA, ATTN_GROUP = 0, 1, 2, 3
CAP_GROUP, CAP_PER_MEMBER = 0, 1
PROBE_HBM_GATHER, PROBE_HOST_READ, PROBE_HOST_DMA, PROBE_HBM_COPY, PROBE_KTAB_READ = 0, 1, 2, 3, 4
PROBE_SUMS_READ = 5
ARRIVAL_STEADY, ARRIVAL_BURSTY, ARRIVAL_POISSON, ARRIVAL_MMPP = 0, 1, 2, 3
EMPTY = 0xFFFFFFFF  # selection id of an empty position (and its slot)
SCHED_FIFO, SCHED_PINNED = 0, 1
TOPK_PER_HEAD, TOPK_LAYER_MAX = 0, 1
ROPE_PLAIN, ROPE_LINEAR, ROPE_BASE, ROPE_PARTS = 0, 1, 2, 3
ESIZE = {F32: 4, F16: 2, BF16: 2, FP8: 1}
MISS_DTYPE = np.dtype([("block", "<u4"), ("slot", "<u4"), ("evicted", "<u4"), ("set", "<u4")])

_ERRORS = {-1: "EINVAL", -2: "EHIP", -3: "ERANGE", -4: "ECAPACITY", -5: "ENOMEM",
           -6: "ESPIN", -7: "ESTATE"}


class FerryError(RuntimeError):
    def __init__(self, code, where, msg=None):
        self.code = code
        if msg is None:  # the library's last refusal on the host
            msg = lib.ferry_last_error().decode()
        super().__init__(f"{where}: {_ERRORS.get(code, code)} ({code}) {msg}")


class Config(C.Structure):
    _fields_ = [
        ("n_req", C.c_int32), ("group", C.c_int32), ("n_layers", C.c_int32),
        ("kv_heads", C.c_int32), ("q_heads", C.c_int32), ("head_dim", C.c_int32),
        ("block_tokens", C.c_int32), ("k", C.c_int32), ("slots_per_set", C.c_int32),
        ("max_blocks", C.c_int32), ("dtype", C.c_int32), ("lru_mode", C.c_int32),
        ("host_blocks", C.c_uint64), ("host_seed", C.c_uint64), ("value_std", C.c_float),
        ("fetch_workers", C.c_int32), ("steal", C.c_int32), ("assign", C.c_int32),
        ("attn", C.c_int32), ("cap_mode", C.c_int32),
    ]


class Stats(C.Structure):
    _fields_ = [
        ("steps", C.c_uint64), ("selections", C.c_uint64), ("misses", C.c_uint64),
        ("fetched_bytes", C.c_uint64), ("steals", C.c_uint64), ("stolen", C.c_uint64),
        ("last_misses", C.c_uint64), ("device_error", C.c_int32), ("pad", C.c_int32),
    ]


class SelGenConfig(C.Structure):
    _fields_ = [
        ("n_req", C.c_int32), ("group", C.c_int32), ("n_layers", C.c_int32),
        ("kv_heads", C.c_int32), ("k", C.c_int32), ("dist", C.c_int32),
        ("zipf_s", C.c_double), ("reuse", C.c_double), ("prefix_blocks", C.c_int32),
        ("pad", C.c_int32), ("seed", C.c_uint64),
    ]


class TraceInfo(C.Structure):
    _fields_ = [
        ("requests", C.c_uint32), ("steps", C.c_uint32), ("layers", C.c_uint32),
        ("page_tokens", C.c_uint32), ("block_tokens", C.c_uint32), ("kv_heads", C.c_uint32),
        ("head_dim", C.c_uint32), ("sel_pages", C.c_uint32), ("sel_blocks", C.c_uint32),
        ("short_records", C.c_uint32), ("unique_blocks", C.c_uint64),
        ("max_blocks_per_req", C.c_uint64),
    ]


_vp = C.c_void_p
_i32 = C.c_int32
_i64x2 = C.c_int64 * 2


class PagesDesc(C.Structure):
    _fields_ = [
        ("n_layers", _i32), ("kv_heads", _i32), ("head_dim", _i32), ("block_tokens", _i32),
        ("dtype", _i32), ("n_pages", _i32), ("n_lanes", _i32), ("max_pages", _i32),
        ("device", _i32), ("pad", _i32), ("pool", _vp), ("scales", _vp), ("table", _vp),
        ("len", _vp), ("refs", _vp), ("error", _vp), ("work", _vp), ("work_bytes", C.c_uint64),
    ]


class AppendArgs(C.Structure):
    _fields_ = [
        ("n_tokens", _i32), ("q_heads", _i32), ("x_dtype", _i32), ("q_out_dtype", _i32),
        ("rot_dim", _i32), ("pairs", _i32), ("factor", C.c_float), ("pad", _i32),
        ("lane", _vp), ("pos", _vp), ("inv_freq", _vp), ("kv_scale", _vp), ("q", _vp), ("k", _vp),
        ("v", _vp), ("q_out", _vp), ("q_stride", _i64x2), ("k_stride", _i64x2),
        ("v_stride", _i64x2), ("q_out_stride", _i64x2),
    ]


class AttendArgs(C.Structure):
    _fields_ = [
        ("n_req", _i32), ("n_tokens", _i32), ("n_groups", _i32), ("q_heads", _i32),
        ("scale", C.c_float), ("pad", _i32), ("lanes", _vp), ("q_start", _vp), ("group_start", _vp),
        ("shared", _vp), ("q", _vp), ("out", _vp), ("lse", _vp), ("q_stride", _i64x2),
        ("out_stride", _i64x2), ("work", _vp), ("work_bytes", C.c_uint64),
    ]


_PROTOS = {
    "ferry_last_error": (C.c_char_p, []),
    "ferry_version": (C.c_char_p, []),
    "ferry_ctx_create": (C.c_int, [C.POINTER(Config), C.c_int, C.POINTER(_vp)]),
    "ferry_ctx_destroy": (C.c_int, [_vp]),
    "ferry_ctx_config": (C.c_int, [_vp, C.POINTER(Config)]),
    "ferry_ctx_sizes": (C.c_int, [_vp, C.POINTER(C.c_uint32), C.POINTER(C.c_uint32),
                                  C.POINTER(C.c_uint64), C.POINTER(C.c_uint64)]),
    "ferry_hosttier_fill": (C.c_int, [_vp, _vp]),
    "ferry_hosttier_view": (C.c_int, [_vp, C.POINTER(_vp), C.POINTER(_vp)]),
    "ferry_hosttier_register": (C.c_int, [_vp, _vp, C.c_uint64, _vp, C.c_uint64]),
    "ferry_pool_view": (C.c_int, [_vp, C.POINTER(_vp), C.POINTER(_vp)]),
    "ferry_sets_reset": (C.c_int, [_vp, _vp]),
    "ferry_sets_state": (C.c_int, [_vp, _vp, _vp, _vp]),
    "ferry_sets_reset_owners": (C.c_int, [_vp, _vp, C.c_uint32, _vp]),
    "ferry_members_leave": (C.c_int, [_vp, _vp, C.c_uint32, _vp]),
    "ferry_members_join": (C.c_int, [_vp, _vp, C.c_uint32, _vp]),
    "ferry_members_get": (C.c_int, [_vp, _vp]),
    "ferry_selgen_admit": (C.c_int, [_vp, _i32, _i32, _i32, _i32]),
    "ferry_selgen_retire": (C.c_int, [_vp, _i32]),
    "ferry_arrivals": (C.c_int, [C.c_int, C.c_uint32, C.c_double, C.c_double, C.c_double,
                                 C.c_uint64, _vp]),
    "ferry_sched_create": (C.c_int, [_i32, _i32, C.c_uint32, _vp, _vp, C.POINTER(_vp)]),
    "ferry_trace_load": (C.c_int, [C.c_char_p, C.c_int, C.POINTER(TraceInfo), _vp, C.c_uint64]),
    "ferry_summaries_build": (C.c_int, [_vp, C.c_uint64, _vp]),
    "ferry_set_batch_policy": (C.c_int, [_vp, C.c_double, C.c_double, C.c_double]),
    "ferry_owner_image_bytes": (C.c_int, [_vp, C.POINTER(C.c_uint64)]),
    "ferry_owner_export": (C.c_int, [_vp, C.c_uint32, _vp, C.c_uint64, _vp]),
    "ferry_owner_import": (C.c_int, [_vp, C.c_uint32, _vp, C.c_uint64, _vp]),
    "ferry_owner_export_member": (C.c_int, [_vp, C.c_uint32, _vp, C.c_uint64, _vp]),
    "ferry_owner_import_member": (C.c_int, [_vp, C.c_uint32, _vp, C.c_uint64, _vp]),
    "ferry_sets_own": (C.c_int, [_vp, _vp]),
    "ferry_decode_chunks": (C.c_int, [_vp, C.c_uint64, C.POINTER(_i32)]),
    "ferry_attn_kernel": (C.c_int, [_vp, C.POINTER(_i32), C.POINTER(_i32)]),
    "ferry_summaries_view": (C.c_int, [_vp, C.POINTER(_vp), C.POINTER(_vp), C.POINTER(C.c_uint64)]),
    "ferry_select_topk": (C.c_int, [_vp, _vp, _vp, C.c_int, _vp, _vp]),
    "ferry_select_topk_layers": (C.c_int, [_vp, _i32, _i32, _vp, _vp, C.c_int, _vp, _vp]),
    "ferry_ktiles_build": (C.c_int, [_vp, C.c_uint64, _vp]),
    "ferry_ktiles_view": (C.c_int, [_vp, C.POINTER(_vp), C.POINTER(_vp), C.POINTER(C.c_uint64)]),
    "ferry_select_mass": (C.c_int, [_vp, _vp, _vp, _vp, _vp]),
    "ferry_select_mass_layers": (C.c_int, [_vp, _i32, _i32, _vp, _vp, _vp, _vp]),
    "ferry_select_mass_noalloc": (C.c_int, [_vp, _vp, _vp, _vp, _vp]),
    "ferry_sched_destroy": (C.c_int, [_vp]),
    "ferry_sched_tick": (C.c_int, [_vp, C.c_double, _vp, _vp, _vp, C.POINTER(_i32), _vp,
                                   C.POINTER(_i32), C.POINTER(_i32), C.POINTER(_i32)]),
    "ferry_sched_next_arrival": (C.c_int, [_vp, C.POINTER(C.c_double)]),
    "ferry_sched_request_ticks": (C.c_int, [_vp, _vp, _vp]),
    "ferry_fetch_step": (C.c_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp]),
    "ferry_bookkeep_step": (C.c_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp]),
    "ferry_bookkeep_layers": (C.c_int, [_vp, _i32, _i32, _vp, _vp, _vp, _vp, _vp, _vp]),
    "ferry_sparse_decode_layers": (C.c_int, [_vp, _i32, _i32, _vp, _vp, _vp, _vp]),
    "ferry_decode_step": (C.c_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i32, _vp, _vp]),
    "ferry_selgen_set_reuse": (C.c_int, [_vp, _vp]),
    "ferry_missq_push": (C.c_int, [_vp, _vp, C.c_uint32, _vp]),
    "ferry_missq_drain": (C.c_int, [_vp, _vp]),
    "ferry_sparse_decode": (C.c_int, [_vp, _vp, _vp, _vp, _vp]),
    "ferry_stats_get": (C.c_int, [_vp, C.POINTER(Stats)]),
    "ferry_bw_probe": (C.c_int, [_vp, C.c_int, _vp, C.c_uint64, C.c_int,
                                 C.POINTER(C.c_uint64), C.POINTER(C.c_float), _vp]),
    "ferry_stats_reset": (C.c_int, [_vp]),
    "ferry_queue_ticket_probe": (C.c_int, [C.c_int, C.c_int, C.c_int, C.c_int, C.POINTER(C.c_uint64),
                                          C.POINTER(C.c_float)]),
    "ferry_queue_selftest": (C.c_int, [C.c_int, C.c_uint64, C.c_uint64, C.c_int, C.c_int,
                                       C.c_int, C.POINTER(C.c_uint64), C.POINTER(C.c_uint64),
                                       C.POINTER(C.c_float)]),
    "ferry_selgen_create": (C.c_int, [C.POINTER(SelGenConfig), _vp, C.POINTER(_vp)]),
    "ferry_selgen_destroy": (C.c_int, [_vp]),
    "ferry_selgen_max_blocks": (C.c_int, [_vp, C.POINTER(_i32)]),
    "ferry_selgen_set_private_ranges": (C.c_int, [_vp, _i32]),
    "ferry_selgen_admit_member": (C.c_int, [_vp, _i32, _i32, _i32, _i32, _i32]),
    "ferry_selgen_step": (C.c_int, [_vp, _i32, _vp]),
    "ferry_ctx_uniform": (C.c_int, [C.c_uint64, _i32, _i32, _i32, _vp]),
    "ferry_pages_work_bytes": (C.c_int, [C.POINTER(PagesDesc), C.POINTER(C.c_uint64)]),
    "ferry_pages_reserve": (C.c_int, [C.POINTER(PagesDesc), _vp, _vp, _i32, _vp]),
    "ferry_pages_fork": (C.c_int, [C.POINTER(PagesDesc), _vp, _vp, _vp, _i32, _vp]),
    "ferry_pages_trim": (C.c_int, [C.POINTER(PagesDesc), _vp, _vp, _i32, _vp]),
    "ferry_pages_compact": (C.c_int, [C.POINTER(PagesDesc), _vp, _vp]),
    # (args: AppendArgs / AttendArgs by reference, or packed as below)
    "ferry_pages_append": (C.c_int, [C.POINTER(PagesDesc), _i32, _vp, _vp]),
    "ferry_pages_attend_work_bytes": (C.c_int, [C.POINTER(PagesDesc), _vp, C.POINTER(C.c_uint64)]),
    "ferry_pages_attend": (C.c_int, [C.POINTER(PagesDesc), _i32, _vp, _vp]),
    "ferry_rope_freqs": (C.c_int, [C.c_int, _i32, C.c_double, C.c_double, C.c_double, C.c_double,
                                   C.c_double, _vp]),
    "ferry_refgen_selections": (C.c_int, [_i32, _i32, _i32, _i32, C.c_uint64, _vp]),
}
for _name, (_res, _args) in _PROTOS.items():
    _f = getattr(lib, _name)
    _f.restype = _res
    _f.argtypes = _args


def _check(rc, where):
    if rc != 0:
        raise FerryError(rc, where)


def _ptr(t):
    """Device/host pointer of a tensor or ndarray (None -> NULL)."""
    if t is None:
        return None
    if isinstance(t, torch.Tensor):
        return t.data_ptr()
    return t.ctypes.data


def _dev(t, name, numel, dtypes, device):
    """Pointer of a contiguous tensor on CUDA device `device` holding at least
    `numel` elements of one of `dtypes`: the kernels read and write exactly
    that many through the raw pointer, so anything else is refused here
    instead of reaching the device."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name}: expected a CUDA tensor, got {type(t).__name__}"
                         f"{'' if not isinstance(t, torch.Tensor) else ' on ' + str(t.device)}")
    if t.device.index != device:
        raise ValueError(f"{name}: on {t.device}, the executor is on cuda:{device}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name}: dtype {t.dtype}, expected {' or '.join(map(str, dtypes))}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")
    if t.numel() < numel:
        raise ValueError(f"{name}: {t.numel()} elements, the geometry needs {numel}")
    return t.data_ptr()


_I32 = (torch.int32,)
_F32 = (torch.float32,)
_U8 = (torch.uint8,)


def _stream(stream):
    if stream is None:
        return torch.cuda.current_stream().cuda_stream
    return getattr(stream, "cuda_stream", stream)


class Executor:
    """One executor (HBM slot pool + LRU sets + miss ring + pinned host tier)."""

    def __init__(self, n_req, n_layers, kv_heads, k, slots_per_set, max_blocks,
                 q_heads=None, group=1, head_dim=128, block_tokens=16, dtype=F16,
                 lru_mode=LRU_STEP, host_blocks=1 << 16, host_seed=7, value_std=0.5,
                 fetch_workers=0, steal=1, assign=ASSIGN_SPREAD, attn=ATTN_AUTO, device=0,
                 cap_mode=CAP_GROUP):
        cfg = Config(n_req, group, n_layers, kv_heads, q_heads or kv_heads, head_dim,
                     block_tokens, k, slots_per_set, max_blocks, dtype, lru_mode,
                     host_blocks, host_seed, value_std, fetch_workers, steal, assign, attn,
                     cap_mode)
        self.device = device
        torch.cuda.set_device(device)
        h = _vp()
        _check(lib.ferry_ctx_create(C.byref(cfg), device, C.byref(h)), "ferry_ctx_create")
        self._h = h
        full = Config()
        _check(lib.ferry_ctx_config(h, C.byref(full)), "ferry_ctx_config")
        self.cfg = full
        ns, ms, bb, ps = C.c_uint32(), C.c_uint32(), C.c_uint64(), C.c_uint64()
        _check(lib.ferry_ctx_sizes(h, C.byref(ns), C.byref(ms), C.byref(bb), C.byref(ps)),
               "ferry_ctx_sizes")
        self.n_sets, self.max_sel = ns.value, ms.value
        self.block_bytes, self.pool_slots = bb.value, ps.value
        self.sel_shape = (n_req, n_layers, kv_heads, k)

    def close(self):
        h, self._h = getattr(self, "_h", None), None
        if h and lib is not None:
            lib.ferry_ctx_destroy(h)

    def __del__(self):
        self.close()

    # ---- buffers --------------------------------------------------------
    # ---- argument checks (shapes the kernels index) ---------------------------
    def _sel(self, t, name="sel"):
        return _dev(t, name, int(np.prod(self.sel_shape)), _I32, self.device)

    def _q(self, t, name="q"):
        B, L = self.sel_shape[0], self.sel_shape[1]
        return _dev(t, name, B * L * self.cfg.q_heads * self.cfg.head_dim, _F32, self.device)

    def _ctx(self, t):
        return _dev(t, "ctx_blocks", self.sel_shape[0], _I32, self.device)

    def _bufs(self, bufs, flags=True):
        n = int(np.prod(self.sel_shape))
        return (_dev(bufs["slots"], "slots", n, _I32, self.device),
                _dev(bufs["miss_count"], "miss_count", self.n_sets, _I32, self.device),
                _dev(bufs["misses"], "misses", self.n_sets * self.max_sel * 4, _I32, self.device),
                _dev(bufs["miss_flag"], "miss_flag", n, _U8, self.device) if flags else None)

    def alloc_step_buffers(self):
        dev = torch.device("cuda", self.device)
        return dict(
            slots=torch.empty(self.sel_shape, dtype=torch.int32, device=dev),
            miss_count=torch.empty(self.n_sets, dtype=torch.int32, device=dev),
            misses=torch.empty((self.n_sets, self.max_sel, 4), dtype=torch.int32, device=dev),
            miss_flag=torch.empty(self.sel_shape, dtype=torch.uint8, device=dev),
        )

    # ---- path -------------------------------------------------------------
    def hosttier_fill(self, stream=None):
        _check(lib.ferry_hosttier_fill(self._h, _stream(stream)), "ferry_hosttier_fill")

    def fetch_step(self, sel, bufs, stream=None, flags=True):
        _check(lib.ferry_fetch_step(self._h, self._sel(sel), *self._bufs(bufs, flags),
                                    _stream(stream)), "ferry_fetch_step")

    def bookkeep_step(self, sel, bufs, stream=None, flags=True):
        _check(lib.ferry_bookkeep_step(self._h, self._sel(sel), *self._bufs(bufs, flags),
                                       _stream(stream)), "ferry_bookkeep_step")

    def bookkeep_layers(self, l0, nl, sel, bufs, stream=None, flags=True):
        _check(lib.ferry_bookkeep_layers(self._h, l0, nl, self._sel(sel), *self._bufs(bufs, flags),
                                         _stream(stream)), "ferry_bookkeep_layers")

    def sparse_decode_layers(self, l0, nl, q, slots, out, stream=None):
        _check(lib.ferry_sparse_decode_layers(self._h, l0, nl, self._q(q), self._sel(slots, "slots"),
                                              self._q(out, "out"), _stream(stream)),
               "ferry_sparse_decode_layers")

    def owner_image_bytes(self):
        n = C.c_uint64()
        _check(lib.ferry_owner_image_bytes(self._h, C.byref(n)), "ferry_owner_image_bytes")
        return n.value

    def alloc_owner_image(self):
        """A device buffer for one owner image (uint8 tensor)."""
        return torch.empty(self.owner_image_bytes(), dtype=torch.uint8,
                           device=torch.device("cuda", self.device))

    def owner_export(self, owner, image, stream=None):
        _check(lib.ferry_owner_export(self._h, owner, _dev(image, "image", 0, _U8, self.device),
                                      image.numel(), _stream(stream)), "ferry_owner_export")

    def owner_import(self, owner, image, stream=None):
        _check(lib.ferry_owner_import(self._h, owner, _dev(image, "image", 0, _U8, self.device),
                                      image.numel(), _stream(stream)), "ferry_owner_import")

    def owner_export_member(self, lane, image, stream=None):
        """Image of the blocks only `lane`'s member of its prefix group touched
        (kv_handoff_owned's carry, src/runtime/wla_multigpu.cuh:1996-2016)."""
        _check(lib.ferry_owner_export_member(self._h, lane,
                                             _dev(image, "image", 0, _U8, self.device),
                                             image.numel(), _stream(stream)),
               "ferry_owner_export_member")

    def owner_import_member(self, lane, image, stream=None):
        """Merge a member image into `lane`'s owner (join the lane first)."""
        _check(lib.ferry_owner_import_member(self._h, lane,
                                             _dev(image, "image", 0, _U8, self.device),
                                             image.numel(), _stream(stream)),
               "ferry_owner_import_member")

    def set_batch_policy(self, min_mb=32.0, max_mb=512.0, target_batches=8.0):
        _check(lib.ferry_set_batch_policy(self._h, min_mb, max_mb, target_batches),
               "ferry_set_batch_policy")

    def decode_chunks(self, pending_blocks):
        """Layer chunks the adaptive policy picks for a step fetching this many blocks."""
        n = _i32()
        _check(lib.ferry_decode_chunks(self._h, pending_blocks, C.byref(n)), "ferry_decode_chunks")
        return n.value

    def decode_step(self, sel, q, bufs, out, chunks=0, stream=None, side_stream=None):
        """Whole step; fetch of layer chunk c+1 (side stream) overlaps attention
        of chunk c (stream).  side_stream None runs everything on one stream.
        chunks 0 = adaptive (from the last step's fetched bytes)."""
        slots, miss_count, misses, _ = self._bufs(bufs, flags=False)
        _check(lib.ferry_decode_step(self._h, self._sel(sel), self._q(q), slots, self._q(out, "out"),
                                     miss_count, misses, chunks,
                                     _stream(stream),
                                     None if side_stream is None else _stream(side_stream)),
               "ferry_decode_step")

    def missq_push(self, misses, n, stream=None):
        _check(lib.ferry_missq_push(self._h, _dev(misses, "misses", 4 * n, _I32, self.device), n,
                                    _stream(stream)), "ferry_missq_push")

    def missq_drain(self, stream=None):
        _check(lib.ferry_missq_drain(self._h, _stream(stream)), "ferry_missq_drain")

    def attn_kernel(self):
        """(kind, waves) of the attention kernel sparse_decode runs: kind is
        ATTN_VALU, ATTN_MFMA (per request row) or ATTN_GROUP (per group set);
        waves per workgroup of that launch (the group kernel runs 8 on a launch
        of no more group sets than CUs where its LDS allows, else 4)."""
        kind, waves = _i32(), _i32()
        _check(lib.ferry_attn_kernel(self._h, C.byref(kind), C.byref(waves)), "ferry_attn_kernel")
        return kind.value, waves.value

    def sparse_decode(self, q, slots, out, stream=None):
        _check(lib.ferry_sparse_decode(self._h, self._q(q), self._sel(slots, "slots"),
                                       self._q(out, "out"), _stream(stream)), "ferry_sparse_decode")

    def summaries_build(self, n_records=0, stream=None):
        """K min/max summaries for select_topk: n_records records (a multiple of
        the host tier's blocks; 0 = one per host-tier block)."""
        _check(lib.ferry_summaries_build(self._h, n_records, _stream(stream)),
               "ferry_summaries_build")

    def summaries_array(self):
        """Device summaries copied to host: uint8 [records, 2*128*esize] and
        fp8 K scales [records] (or None)."""
        p, sc, n = _vp(), _vp(), C.c_uint64()
        _check(lib.ferry_summaries_view(self._h, C.byref(p), C.byref(sc), C.byref(n)),
               "ferry_summaries_view")
        hb = n.value
        rec = 2 * 128 * ESIZE[self.cfg.dtype]
        sums = _gather_d2h(p.value, hb * rec, [0]).reshape(hb, rec)
        scales = None
        if sc.value:
            scales = _gather_d2h(sc.value, hb * 4, [0]).view(np.float32).reshape(hb)
        return sums, scales

    def select_topk(self, q, ctx_blocks, sel, mode=TOPK_PER_HEAD, stream=None, layers=None):
        """Top-k blocks of every (request, layer, kv head) from q (device
        tensors: q [B,L,Hq,128] fp32, ctx_blocks [B] int32, sel out [B,L,Hkv,k])."""
        if layers is None:
            _check(lib.ferry_select_topk(self._h, self._q(q), self._ctx(ctx_blocks), mode,
                                         self._sel(sel), _stream(stream)), "ferry_select_topk")
        else:
            l0, nl = layers
            _check(lib.ferry_select_topk_layers(self._h, l0, nl, self._q(q), self._ctx(ctx_blocks),
                                                mode, self._sel(sel), _stream(stream)),
                   "ferry_select_topk_layers")

    def ktiles_build(self, n_records=0, stream=None):
        """Dense K table for select_mass: n_records records (a multiple of the
        host tier's blocks; 0 = one per host-tier block)."""
        _check(lib.ferry_ktiles_build(self._h, n_records, _stream(stream)), "ferry_ktiles_build")

    def ktiles_array(self):
        """The K table copied to host: uint8 [records, block_bytes / 2] (fp32
        row-major; 16-bit and fp8 lane-transposed: 16-byte word c of token row
        t at word 64 (c // 4) + 16 (c % 4) + t) and fp8 K scales [records] (or
        None)."""
        p, sc, n = _vp(), _vp(), C.c_uint64()
        _check(lib.ferry_ktiles_view(self._h, C.byref(p), C.byref(sc), C.byref(n)),
               "ferry_ktiles_view")
        rec = self.block_bytes // 2
        kt = _gather_d2h(p.value, n.value * rec, [0]).reshape(n.value, rec)
        scales = None
        if sc.value:
            scales = _gather_d2h(sc.value, n.value * 4, [0]).view(np.float32).reshape(n.value)
        return kt, scales

    def select_mass(self, q, ctx_blocks, sel, stream=None, layers=None):
        """The softmax-mass top-k of every (request, layer), written to every kv
        head's row of sel [B,L,Hkv,k] (device tensors as for select_topk)."""
        if layers is None:
            _check(lib.ferry_select_mass(self._h, self._q(q), self._ctx(ctx_blocks), self._sel(sel),
                                         _stream(stream)), "ferry_select_mass")
        else:
            l0, nl = layers
            _check(lib.ferry_select_mass_layers(self._h, l0, nl, self._q(q), self._ctx(ctx_blocks),
                                                self._sel(sel), _stream(stream)),
                   "ferry_select_mass_layers")

    def select_mass_noalloc(self, q, ctx_blocks, sel, stream=None):
        """select_mass over every layer with the library's static per-GPU
        workspace instead of the context's: allocates nothing.  Calls that
        overlap on one GPU race for that workspace."""
        _check(lib.ferry_select_mass_noalloc(self._h, self._q(q), self._ctx(ctx_blocks),
                                             self._sel(sel), _stream(stream)),
               "ferry_select_mass_noalloc")

    def sets_reset(self, stream=None):
        _check(lib.ferry_sets_reset(self._h, _stream(stream)), "ferry_sets_reset")

    def reset_owners(self, owners, stream=None):
        """Empty the sets of the owners in `owners` (int32 device tensor)."""
        _check(lib.ferry_sets_reset_owners(self._h, _dev(owners, "owners", 0, _I32, self.device),
                                           int(owners.numel()), _stream(stream)),
               "ferry_sets_reset_owners")

    # ---- inspection (synchronous) ---------------------------------------
    def members_leave(self, lanes, stream=None):
        """The requests of these lanes (int32 device tensor) leave their owners;
        under CAP_PER_MEMBER the owners' sets are trimmed to the new capacity."""
        n = int(lanes.numel())
        _check(lib.ferry_members_leave(self._h, _dev(lanes, "lanes", n, _I32, self.device), n,
                                       _stream(stream)), "ferry_members_leave")

    def members_join(self, lanes, stream=None):
        """New requests of the owners' groups take these lanes (resident again)."""
        n = int(lanes.numel())
        _check(lib.ferry_members_join(self._h, _dev(lanes, "lanes", n, _I32, self.device), n,
                                      _stream(stream)), "ferry_members_join")

    def members(self):
        """Resident members of every owner (synchronises)."""
        out = np.zeros((self.sel_shape[0] + self.cfg.group - 1) // self.cfg.group, np.uint32)
        _check(lib.ferry_members_get(self._h, out.ctypes.data), "ferry_members_get")
        return out

    def stats(self):
        s = Stats()
        _check(lib.ferry_stats_get(self._h, C.byref(s)), "ferry_stats_get")
        return {f: getattr(s, f) for f, _ in Stats._fields_ if f != "pad"}

    def bw_probe(self, kind, n, slots=None, iters=5, stream=None):
        """Plain-read bandwidth ceiling (ferry_bw_probe): returns (bytes per
        launch, mean ms per launch, GB/s)."""
        b, ms = C.c_uint64(), C.c_float()
        if kind == PROBE_HBM_GATHER:  # n rows of the slot table
            slots_p = _dev(slots, "slots", n * self.cfg.k, _I32, self.device)
        else:
            slots_p = None
        _check(lib.ferry_bw_probe(self._h, kind, slots_p, n, iters, C.byref(b), C.byref(ms),
                                  _stream(stream)), "ferry_bw_probe")
        return b.value, ms.value, b.value / (ms.value * 1e-3) / 1e9

    def stats_reset(self):
        _check(lib.ferry_stats_reset(self._h), "ferry_stats_reset")

    def sets_state(self):
        cap = self.cfg.slots_per_set
        fill = np.zeros(self.n_sets, np.uint32)
        ord_ = np.zeros((self.n_sets, cap), np.uint32)
        tag = np.zeros((self.n_sets, cap), np.uint32)
        _check(lib.ferry_sets_state(self._h, fill.ctypes.data, ord_.ctypes.data, tag.ctypes.data),
               "ferry_sets_state")
        return fill, ord_, tag

    def sets_own(self):
        """Per-slot member masks [n_sets, slots] of prefix groups (synchronises)."""
        own = np.zeros((self.n_sets, self.cfg.slots_per_set), np.uint32)
        _check(lib.ferry_sets_own(self._h, own.ctypes.data), "ferry_sets_own")
        return own

    def hosttier_register(self, host, scales=None):
        """Use the caller's pinned host memory (a pin_memory uint8 CPU tensor of
        host_blocks * block_bytes, plus float32 scales for fp8) as the host tier.
        The tensors are kept alive by the executor."""
        sb = 0 if scales is None else scales.numel() * scales.element_size()
        _check(lib.ferry_hosttier_register(self._h, _ptr(host), host.numel() * host.element_size(),
                                           _ptr(scales), sb), "ferry_hosttier_register")
        self._registered = (host, scales)

    def hosttier_array(self):
        """numpy view of the pinned host tier (bytes) and fp8 scales (or None)."""
        b, s = _vp(), _vp()
        _check(lib.ferry_hosttier_view(self._h, C.byref(b), C.byref(s)), "ferry_hosttier_view")
        n = self.cfg.host_blocks * self.block_bytes
        arr = np.ctypeslib.as_array(C.cast(b, C.POINTER(C.c_uint8)), shape=(n,))
        sc = None
        if s.value:
            sc = np.ctypeslib.as_array(C.cast(s, C.POINTER(C.c_float)),
                                       shape=(self.cfg.host_blocks * 2,))
        return arr, sc

    def pool_ptrs(self):
        p, s = _vp(), _vp()
        _check(lib.ferry_pool_view(self._h, C.byref(p), C.byref(s)), "ferry_pool_view")
        return p.value, s.value

    def pool_slots_bytes(self, slot_ids):
        """Copy the given pool slots (global ids) to host: [n, block_bytes] uint8."""
        p, _ = self.pool_ptrs()
        return _gather_d2h(p, self.block_bytes, slot_ids)

    def pool_slot_scales(self, slot_ids):
        """fp8 scales (k, v) of the given pool slots, or None."""
        _, s = self.pool_ptrs()
        if not s:
            return None
        return _gather_d2h(s, 8, slot_ids).view(np.float32).reshape(-1, 2)


def rope_freqs(kind, rot_dim, base=10000.0, stretch=1.0, trained_ctx=0.0, slow=1.0, fast=32.0):
    """Radians per token of the rot_dim / 2 rotary pairs (float64 array), plain or
    in one of the forms for contexts `stretch` times the trained one."""
    if not 2 <= rot_dim <= 128:
        raise ValueError("rot_dim must be even, 2..128")
    out = np.zeros(rot_dim // 2, np.float64)
    _check(lib.ferry_rope_freqs(kind, rot_dim, base, stretch, trained_ctx, slow, fast,
                                out.ctypes.data), "ferry_rope_freqs")
    return out


_X_DTYPE = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
_APPEND = struct.Struct("@6ifi8P8q")  # AppendArgs, AttendArgs: packing them takes a tenth of
_ATTEND = struct.Struct("@4ifi7P4qPQ")  # the time of filling a ctypes structure
assert _APPEND.size == C.sizeof(AppendArgs) and _ATTEND.size == C.sizeof(AttendArgs)
_PAGE_TORCH = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16,
               FP8: torch.float8_e4m3fn}


class Pages:
    """A paged KV cache (ferry_pages_*): whole contexts of lanes in pages of 16
    tokens, next to the executor's cache of selected blocks.  It is made over the
    caller's tensors and keeps them:

      pool    [layers, pages, kv heads, 2 (K, V), 16, 128], float32, float16,
              bfloat16 or float8_e4m3fn (or uint8 with dtype=FP8)
      scales  [layers, pages, kv heads, 2] float32, fp8 pages only
      table   [lanes, pages per lane] int32, -1 (EMPTY) where unused
      length  [lanes] int32, tokens
      refs    [pages] int32, table entries that name each page; None where the
              program hands out the pages itself

    Pages.empty() allocates an empty one.  Errors found on the device are kept in
    `error` (an int32 tensor); check() reads it and raises."""

    def __init__(self, pool, table, length, refs=None, scales=None, dtype=None, error=None):
        if not isinstance(pool, torch.Tensor) or not pool.is_cuda:
            raise ValueError("pool: expected a CUDA tensor")
        if pool.dim() != 6 or tuple(pool.shape[3:]) != (2, 16, 128):
            raise ValueError("pool: expected [layers, pages, kv heads, 2, 16, 128]")
        if dtype is None:
            dtype = {v: k for k, v in _PAGE_TORCH.items()}.get(pool.dtype)
        if dtype not in _PAGE_TORCH:
            raise ValueError(f"pool: dtype {pool.dtype} holds no KV element type")
        L, P, H = pool.shape[:3]
        if table.dim() != 2 or length.dim() != 1 or length.shape[0] != table.shape[0]:
            raise ValueError("table and length: expected [lanes, pages per lane] and [lanes]")
        dev = self.device = pool.device.index
        ok = (_PAGE_TORCH[dtype], torch.uint8) if dtype == FP8 else (_PAGE_TORCH[dtype],)
        d = PagesDesc(L, H, 128, 16, dtype, P, table.shape[0], table.shape[1], dev, 0)
        d.pool = _dev(pool, "pool", 1, ok, dev)
        d.table = _dev(table, "table", 1, _I32, dev)
        d.len = _dev(length, "length", 1, _I32, dev)
        if (scales is None) != (dtype != FP8):
            raise ValueError("scales go with fp8 pages")
        if scales is not None:
            if tuple(scales.shape) != (L, P, H, 2):
                raise ValueError("scales: expected [layers, pages, kv heads, 2]")
            d.scales = _dev(scales, "scales", 1, _F32, dev)
        if error is None:
            error = torch.zeros(1, dtype=torch.int32, device=pool.device)
        d.error = _dev(error, "error", 1, _I32, dev)
        work = None
        if refs is not None:
            if tuple(refs.shape) != (P,):
                raise ValueError("refs: expected [pages]")
            d.refs = _dev(refs, "refs", 1, _I32, dev)
            n = C.c_uint64()
            _check(lib.ferry_pages_work_bytes(C.byref(d), C.byref(n)), "ferry_pages_work_bytes")
            work = torch.empty(n.value, dtype=torch.uint8, device=pool.device)
            d.work, d.work_bytes = work.data_ptr(), n.value
        self.pool, self.table, self.length, self.refs = pool, table, length, refs
        self.scales, self.error, self.dtype, self._work = scales, error, dtype, work
        self.q_dtype = torch.bfloat16 if dtype == FP8 else _PAGE_TORCH[dtype]
        self._d, self._r, self._attend_bytes = d, C.byref(d), {}

    @classmethod
    def empty(cls, n_layers, kv_heads, n_pages, n_lanes, max_pages, dtype=BF16, device=0):
        dev = torch.device("cuda", device)

        def ints(shape, v):
            return torch.full(shape, v, dtype=torch.int32, device=dev)

        return cls(torch.empty((n_layers, n_pages, kv_heads, 2, 16, 128), dtype=_PAGE_TORCH[dtype],
                               device=dev),
                   ints((n_lanes, max_pages), -1), ints((n_lanes,), 0), refs=ints((n_pages,), 0),
                   scales=torch.ones((n_layers, n_pages, kv_heads, 2), device=dev)
                   if dtype == FP8 else None)

    def _s(self, stream):
        if stream is None:
            return torch._C._cuda_getCurrentRawStream(self.device)
        return getattr(stream, "cuda_stream", stream)

    def _list(self, t, name, n):
        if t is None:
            return None
        if t.dtype is torch.int32 and t.get_device() == self.device and t.is_contiguous() \
                and t.numel() >= n:
            return t.data_ptr()
        return _dev(t, name, n, _I32, self.device)  # says what is wrong

    def check(self):
        """Raise the first error that calls on any stream found since the last check
        (waits for the device)."""
        torch.cuda.synchronize(self.device)
        code = int(self.error.item())
        if code:
            self.error.zero_()
            torch.cuda.synchronize(self.device)  # before a call on another stream finds one
            raise FerryError(code, "pages", "found on the device")

    # ---- managing pages ---------------------------------------------------------
    def reserve(self, lanes, tokens, stream=None):
        """lanes[i] grows by tokens[i]; a shared last page that is begun is copied."""
        n = lanes.numel()
        _check(lib.ferry_pages_reserve(self._r, self._list(lanes, "lanes", n),
                                       self._list(tokens, "tokens", n), n, self._s(stream)),
               "ferry_pages_reserve")

    def fork(self, src, dst, keep=None, stream=None):
        """The empty lanes dst[i] share the first keep[i] tokens (all) of src[i]."""
        n = dst.numel()
        _check(lib.ferry_pages_fork(self._r, self._list(src, "src", n), self._list(dst, "dst", n),
                                    self._list(keep, "keep", n), n, self._s(stream)),
               "ferry_pages_fork")

    def trim(self, lanes, keep=None, stream=None):
        """lanes[i] keeps its first keep[i] tokens (none: the lane ends)."""
        n = lanes.numel()
        _check(lib.ferry_pages_trim(self._r, self._list(lanes, "lanes", n),
                                    self._list(keep, "keep", n), n, self._s(stream)),
               "ferry_pages_trim")

    def compact(self, live=None, stream=None):
        """Pages in use move into the lowest ids; live[0] gets their number."""
        _check(lib.ferry_pages_compact(self._r, self._list(live, "live", 1), self._s(stream)),
               "ferry_pages_compact")

    # ---- tokens -----------------------------------------------------------------
    def _rows(self, t, name, rows, heads, dtypes):
        """Pointer and strides between tokens and heads of a [rows, heads, 128] tensor."""
        if not isinstance(t, torch.Tensor) or t.get_device() != self.device:
            raise ValueError(f"{name}: expected a CUDA tensor on cuda:{self.device}")
        if t.dtype not in dtypes:
            raise ValueError(f"{name}: dtype {t.dtype}, expected {' or '.join(map(str, dtypes))}")
        if t.dim() != 3 or t.shape != (rows, heads or t.shape[1], 128):
            raise ValueError(f"{name}: shape {tuple(t.shape)}, expected [{rows}, {heads or 'heads'}, 128]")
        a, b, c = t.stride()
        if c != 1:
            raise ValueError(f"{name}: a head's 128 values must be contiguous")
        return t.data_ptr(), a, b

    def append(self, layer, lane, pos, k=None, v=None, q=None, q_out=None, inv_freq=None, factor=1.0,
               pairs=False, kv_scale=None, stream=None):
        """Rotary positions of q (into q_out) and k, and k and v into the pages:
        token t is at place pos[t] of lane[t] (int32 tensors).  inv_freq is a
        float64 tensor of rot_dim / 2 radians per token."""
        n = pos.numel()
        x = q if q is not None else k
        if x is None:
            raise ValueError("neither q nor k")
        if inv_freq is None:
            raise ValueError("inv_freq: expected a CUDA tensor")
        heads, out_type = 0, 0
        qp = op = kp = vp = sp = (0, 0, 0)
        if q is not None:
            heads = q.shape[1]
            qp = self._rows(q, "q", n, 0, _X_DTYPE)
            op = self._rows(q_out, "q_out", n, heads, _X_DTYPE)
            out_type = _X_DTYPE[q_out.dtype]
        if k is not None or v is not None:
            H = self._d.kv_heads
            kp = self._rows(k, "k", n, H, (x.dtype,))
            vp = self._rows(v, "v", n, H, (x.dtype,))
            if self.dtype == FP8:
                sp = (_dev(kv_scale, "kv_scale", 2 * H, _F32, self.device),)
        a = _APPEND.pack(n, heads, _X_DTYPE.get(x.dtype, -1), out_type, 2 * inv_freq.numel(), bool(pairs),
                         factor, 0, self._list(lane, "lane", n) or 0, self._list(pos, "pos", n),
                         _dev(inv_freq, "inv_freq", 1, (torch.float64,), self.device), sp[0],
                         qp[0], kp[0], vp[0], op[0], qp[1], qp[2], kp[1], kp[2], vp[1], vp[2], op[1], op[2])
        if n == 0 and 0 <= layer < self._d.n_layers:
            return  # empty tensors have no address
        _check(lib.ferry_pages_append(self._r, layer, a, self._s(stream)), "ferry_pages_append")

    def attend(self, layer, q, out, lanes, q_start=None, group_start=None, shared=None, scale=0.0,
               lse=None, stream=None):
        """Attention of the new query rows q [rows, q heads, 128] of lanes (all rows
        of request r are [q_start[r], q_start[r+1]); None: one row each), into
        out; requests [group_start[g], group_start[g+1]) share their first
        shared[g] pages."""
        n, rows, heads, groups, sp = lanes.numel(), q.shape[0], q.shape[1], 0, None
        dt = (self.q_dtype,)
        qp, qa, qb = self._rows(q, "q", rows, 0, dt)
        op, oa, ob = self._rows(out, "out", rows, heads, dt)
        if group_start is not None:
            groups = group_start.numel() - 1
            sp = _dev(shared, "shared", groups, _I32, self.device)
        ep = None if lse is None else _dev(lse, "lse", rows * heads, _F32, self.device)
        # the scratch's size follows from these, the same in every call on this cache
        shape = (n, rows, groups, heads, q_start is None)
        need = self._attend_bytes.get(shape)
        if need is None:
            b = C.c_uint64()
            a = AttendArgs(n, rows, groups, heads, scale, q_start=None if q_start is None else 1)
            _check(lib.ferry_pages_attend_work_bytes(self._r, C.byref(a), C.byref(b)),
                   "ferry_pages_attend_work_bytes")
            if len(self._attend_bytes) >= 4096:
                self._attend_bytes.clear()
            need = self._attend_bytes[shape] = b.value
        s = self._s(stream)
        if stream is None or s == self._s(None):
            work = torch.empty(need, dtype=torch.uint8, device=self.pool.device)
        else:  # of the stream that uses it: what the current one frees it may still use
            with torch.cuda.stream(torch.cuda.ExternalStream(s, self.device) if s
                                   else torch.cuda.default_stream(self.device)):
                work = torch.empty(need, dtype=torch.uint8, device=self.pool.device)
        a = _ATTEND.pack(n, rows, groups, heads, scale, 0, self._list(lanes, "lanes", n),
                         self._list(q_start, "q_start", n + 1) or 0,
                         self._list(group_start, "group_start", 1) or 0, sp or 0, qp, op, ep or 0,
                         qa, qb, oa, ob, work.data_ptr(), need)
        _check(lib.ferry_pages_attend(self._r, layer, a, s), "ferry_pages_attend")


_hip = None


def _gather_d2h(base, row_bytes, ids):
    """rows base[ids[i] * row_bytes : +row_bytes] of device memory -> host array."""
    global _hip
    if _hip is None:
        _hip = C.CDLL("libamdhip64.so.7")  # the runtime already loaded with torch
        _hip.hipMemcpy.restype = C.c_int
        _hip.hipMemcpy.argtypes = [_vp, _vp, C.c_size_t, C.c_int]
        _hip.hipDeviceSynchronize.restype = C.c_int
    ids = np.asarray(ids, np.int64).reshape(-1)
    out = np.zeros((ids.size, row_bytes), np.uint8)
    if _hip.hipDeviceSynchronize() != 0:
        raise RuntimeError("hipDeviceSynchronize failed")
    order = np.argsort(ids, kind="stable")
    i = 0
    while i < ids.size:  # copy runs of consecutive ids in one call
        j = i + 1
        while j < ids.size and ids[order[j]] == ids[order[j - 1]] + 1 and \
                order[j] == order[j - 1] + 1:
            j += 1
        rc = _hip.hipMemcpy(out[order[i]:].ctypes.data, base + int(ids[order[i]]) * row_bytes,
                            (j - i) * row_bytes, 2)
        if rc != 0:
            raise RuntimeError(f"hipMemcpy D2H failed ({rc})")
        i = j
    return out


class SelGen:
    """Synthetic top-k selection stream (host).  Steps must be drawn in order."""

    def __init__(self, n_req, n_layers, kv_heads, k, ctx_blocks, dist=1, zipf_s=1.1,
                 reuse=0.66, group=1, prefix_blocks=0, seed=1):
        self.cfg = SelGenConfig(n_req, group, n_layers, kv_heads, k, dist, zipf_s, reuse,
                                prefix_blocks, 0, seed)
        ctx = np.ascontiguousarray(ctx_blocks, np.int32)
        h = _vp()
        _check(lib.ferry_selgen_create(C.byref(self.cfg), ctx.ctypes.data, C.byref(h)),
               "ferry_selgen_create")
        self._h = h
        mb = _i32()
        _check(lib.ferry_selgen_max_blocks(h, C.byref(mb)), "ferry_selgen_max_blocks")
        self.max_blocks = mb.value
        self.shape = (n_req, n_layers, kv_heads, k)

    def set_reuse(self, reuse):
        """Per-request reuse probabilities (None: the configured one for all)."""
        self._reuse = None if reuse is None else np.ascontiguousarray(reuse, np.float64)
        _check(lib.ferry_selgen_set_reuse(self._h, None if self._reuse is None
                                          else self._reuse.ctypes.data), "ferry_selgen_set_reuse")

    def step(self, step):
        out = np.zeros(self.shape, np.uint32)
        _check(lib.ferry_selgen_step(self._h, step, out.ctypes.data), "ferry_selgen_step")
        return out

    def admit(self, lane, request_id, ctx_blocks, step):
        """Request `request_id` (context ctx_blocks) takes `lane` from `step` on."""
        _check(lib.ferry_selgen_admit(self._h, lane, request_id, ctx_blocks, step),
               "ferry_selgen_admit")

    def retire(self, lane):
        """`lane` produces empty rows until its next admission."""
        _check(lib.ferry_selgen_retire(self._h, lane), "ferry_selgen_retire")

    def set_private_ranges(self, ranges):
        """`ranges` (>= group) private id ranges per prefix-group owner, for
        members that turn over; updates max_blocks."""
        _check(lib.ferry_selgen_set_private_ranges(self._h, ranges),
               "ferry_selgen_set_private_ranges")
        mb = _i32()
        _check(lib.ferry_selgen_max_blocks(self._h, C.byref(mb)), "ferry_selgen_max_blocks")
        self.max_blocks = mb.value

    def admit_member(self, lane, request_id, ctx_blocks, step, private_range):
        """A request of the lane's prefix group takes `lane` from `step` on,
        its private blocks in id range `private_range`."""
        _check(lib.ferry_selgen_admit_member(self._h, lane, request_id, ctx_blocks, step,
                                             private_range), "ferry_selgen_admit_member")

    def __del__(self):
        h, self._h = getattr(self, "_h", None), None
        if h and lib is not None:
            lib.ferry_selgen_destroy(h)


def ctx_uniform(seed, n_req, lo, hi):
    out = np.zeros(n_req, np.int32)
    _check(lib.ferry_ctx_uniform(seed, n_req, lo, hi, out.ctypes.data), "ferry_ctx_uniform")
    return out


def arrivals(kind, n, gap_ms, period_ms=50.0, ratio=10.0, seed=0):
    """Arrival times (ms) of n requests (ferry_arrivals)."""
    out = np.zeros(n, np.float64)
    _check(lib.ferry_arrivals(kind, n, gap_ms, period_ms, ratio, seed, out.ctypes.data),
           "ferry_arrivals")
    return out


class Sched:
    """Tick scheduler of one executor (ferry_sched_*): `lanes` batch lanes
    serve requests that arrive at arrive_ms and decode len_steps steps."""

    def __init__(self, lanes, arrive_ms, len_steps, pinned=False):
        self.lanes = lanes
        self._arr = np.ascontiguousarray(arrive_ms, np.float64)
        self._len = np.ascontiguousarray(len_steps, np.int32)
        self.n = self._arr.size
        h = _vp()
        _check(lib.ferry_sched_create(lanes, SCHED_PINNED if pinned else SCHED_FIFO, self.n,
                                      self._arr.ctypes.data, self._len.ctypes.data, C.byref(h)),
               "ferry_sched_create")
        self._h = h

    def tick(self, now_ms):
        """One tick: returns dict(lane_req, lane_step, admitted, retired,
        resident, done)."""
        lr = np.zeros(self.lanes, np.int32)
        ls = np.zeros(self.lanes, np.int32)
        ad = np.zeros(self.lanes, np.int32)
        rt = np.zeros(self.lanes, np.int32)
        na, nr, nres, done = _i32(), _i32(), _i32(), _i32()
        _check(lib.ferry_sched_tick(self._h, now_ms, lr.ctypes.data, ls.ctypes.data,
                                    ad.ctypes.data, C.byref(na), rt.ctypes.data, C.byref(nr),
                                    C.byref(nres), C.byref(done)), "ferry_sched_tick")
        return dict(lane_req=lr, lane_step=ls, admitted=ad[:na.value].copy(),
                    retired=rt[:nr.value].copy(), resident=nres.value, done=bool(done.value))

    def next_arrival(self):
        v = C.c_double()
        _check(lib.ferry_sched_next_arrival(self._h, C.byref(v)), "ferry_sched_next_arrival")
        return v.value

    def request_ticks(self):
        a = np.zeros(self.n, np.int32)
        d = np.zeros(self.n, np.int32)
        _check(lib.ferry_sched_request_ticks(self._h, a.ctypes.data, d.ctypes.data),
               "ferry_sched_request_ticks")
        return a, d

    def __del__(self):
        h, self._h = getattr(self, "_h", None), None
        if h and lib is not None:
            lib.ferry_sched_destroy(h)


def trace_load(path, strict=True):
    """Read an FMT1 selection trace: (info dict, dense ids [R, S, L, sel_blocks])."""
    info = TraceInfo()
    p = os.fsencode(path)
    _check(lib.ferry_trace_load(p, int(strict), C.byref(info), None, 0), "ferry_trace_load")
    ids = np.zeros((info.requests, info.steps, info.layers, info.sel_blocks), np.uint32)
    _check(lib.ferry_trace_load(p, int(strict), C.byref(info), ids.ctypes.data, ids.size),
           "ferry_trace_load")
    return {f: getattr(info, f) for f, _ in TraceInfo._fields_}, ids


def refgen_selections(R, L, S, sel, seed=42):
    """replay_miss_stream's selections, (r, s, l, k) order -> array [R, S, L, sel]."""
    out = np.zeros((R, S, L, sel), np.uint32)
    _check(lib.ferry_refgen_selections(R, L, S, sel, seed, out.ctypes.data),
           "ferry_refgen_selections")
    return out


def queue_selftest(capacity=1 << 20, n_tasks=1 << 22, producers=512, consumers=512, mode=1,
                   device=0):
    """Exactly-once run of the device MPMC ring.  Returns (popped, dups, ms)."""
    p, d, ms = C.c_uint64(), C.c_uint64(), C.c_float()
    _check(lib.ferry_queue_selftest(device, capacity, n_tasks, producers, consumers, mode,
                                    C.byref(p), C.byref(d), C.byref(ms)), "ferry_queue_selftest")
    return p.value, d.value, ms.value


def queue_ticket_probe(threads=512, iters=4096, kind=1, device=0):
    """Tickets taken from one shared word by `threads` threads, `iters` each:
    kind 0 fetch-add per thread, kind 1 a load + compare-and-swap retry per
    thread, kind 2 that retry once per wavefront for its 64 lanes.
    Returns (tickets, ms)."""
    t, ms = C.c_uint64(), C.c_float()
    _check(lib.ferry_queue_ticket_probe(device, threads, iters, kind, C.byref(t), C.byref(ms)),
           "ferry_queue_ticket_probe")
    return t.value, ms.value
