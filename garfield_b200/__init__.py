"""garfield_b200: the Garfield GMG query path on NVIDIA B200 (sm_100a).

Python host mirror of the C ABI declared in include/garfield.h.  The compute runs in
libgarfield_b200.so (hand-written CUDA); this module only marshals arrays.  Device
arrays are torch CUDA tensors (used as plain device memory); host arrays are numpy.

The reference (ZJU-DAILY/Garfield) exposes its query path as host functions inside one
CUDA translation unit; the mapping is:
  Index(...)                 real_dataset_test_multiD loading block (realdataset_search.cu:2118-2393)
  Index.plan(...)            intersection_area_mark_little_seg_V2 (real_dataset_adapter.cuh:390)
                             + get_partitions_access_order_V2 (gpu_graph.cu:11742)
  Index.search(...)          batch_graph_search_gpu_with_prefilter_and_postfilter (gpu_graph.cu:12464)
  Index.bruteforce(...)      naive_brute_force_with_filter (gpu_graph.cu:10782)
  quantize_fp4, dequantize_fp4, product_fp4   rows held in 4-bit block floating point (no counterpart)
  read_* / write_*           loaders of tools.cuh / real_dataset_adapter.cuh (formats: Appendix of the docs)
If the shared library is missing the import still succeeds, but every call that needs
it raises: there is no CPU fallback.
"""
from __future__ import annotations

import ctypes as C
import os
from dataclasses import dataclass
from pathlib import Path

import numpy as np

__all__ = [
    "GarfieldError", "lib", "lib_path", "SearchParams", "Index", "Plan", "NO_ID", "schedule_batches",
    "read_fvecs", "write_fvecs", "read_attrs", "write_attrs", "read_u32mat", "write_u32mat",
    "read_ranges", "write_ranges", "read_labels", "read_grid",
    "Fp4Rows", "quantize_fp4", "dequantize_fp4", "product_fp4", "product_fp4_timeouts", "quantize_fp4_host",
    "dequantize_fp4_host",
]

NO_ID = 0xFFFFFFFF
_PKG = Path(__file__).resolve().parent
lib_path = _PKG / "libgarfield_b200.so"


class GarfieldError(RuntimeError):
    def __init__(self, status: int, what: str, msg: str):
        super().__init__(f"{what}: status {status} ({msg})")
        self.status = status


class _IndexDesc(C.Structure):
    _fields_ = [
        ("n", C.c_uint32), ("dim", C.c_uint32), ("n_attr", C.c_uint32),
        ("vectors", C.c_void_p), ("attrs", C.c_void_p), ("grid", C.c_void_p),
        ("l_quant", C.c_void_p), ("r_quant", C.c_void_p), ("cell_of", C.c_void_p),
        ("degree", C.c_uint32), ("graphs", C.c_void_p), ("cross_e", C.c_uint32),
        ("cross", C.c_void_p), ("n_clusters", C.c_uint32), ("labels", C.c_void_p),
        ("f2h_factor", C.c_float), ("keep_fp32", C.c_uint32), ("host_graph", C.c_uint32),
        ("shard_cells", C.c_void_p), ("n_shard_cells", C.c_uint32),
        ("codec", C.c_uint32), ("codes", C.c_void_p), ("code_scales", C.c_void_p),
        ("code_zero_points", C.c_void_p), ("cross_spokesman", C.c_uint32),
    ]


class _IndexFiles(C.Structure):
    _fields_ = [
        ("data_path", C.c_char_p), ("cagra_prefix", C.c_char_p), ("cagra_suffix", C.c_char_p),
        ("global_graph", C.c_char_p), ("grid", C.c_char_p), ("attrs", C.c_char_p),
        ("cluster", C.c_char_p), ("degree", C.c_uint32), ("f2h_factor", C.c_float),
        ("keep_fp32", C.c_uint32), ("host_graph", C.c_uint32), ("codec", C.c_uint32),
        ("quantized", C.c_char_p), ("uniform_dims", C.c_uint32),
        ("uniform_shape", C.c_void_p),
        ("uniform_lo", C.c_float), ("uniform_hi", C.c_float),
    ]


class _SearchParams(C.Structure):
    _fields_ = [(n, C.c_uint32) for n in
                ("L", "k", "width", "max_iter", "n_entry", "postfilter", "hash_slots", "test_wait", "exact_tc",
                 "route")]


class _BfParams(C.Structure):
    _fields_ = [("path", C.c_uint32), ("test_fallback_every", C.c_uint32), ("test_wait", C.c_uint32),
                ("stats_out", C.c_void_p)]


class _SearchStats(C.Structure):
    _fields_ = [(n, C.c_uint64) for n in ("n_dist", "n_exp", "n_cross", "n_hops", "n_exact", "n_queries",
                                          "n_timeouts", "n_plan_fallbacks", "n_plan_reranked")]


class _IndexInfo(C.Structure):
    _fields_ = [(n, C.c_uint32) for n in
                ("n", "dim", "n_attr", "n_cells", "degree", "cross_e", "n_clusters", "d_stored",
                 "min_cell_size", "cross_rows")] + [("device_bytes", C.c_uint64)]


_LIB = None
_P = C.c_void_p
_U32 = C.c_uint32
_PTR = C.POINTER


def lib() -> C.CDLL:
    """Load libgarfield_b200.so (raises if it has not been built)."""
    global _LIB
    if _LIB is not None:
        return _LIB
    if not lib_path.exists():
        raise GarfieldError(-1, "load", f"{lib_path} not built; run python -m garfield_b200.build")
    L = C.CDLL(str(lib_path))
    sig = {
        "gf_status_string": (C.c_char_p, [C.c_int]),
        "gf_last_error": (C.c_char_p, []),
        "gf_version": (C.c_char_p, []),
        "gf_search_defaults": (None, [_PTR(_SearchParams)]),
        "gf_index_create": (C.c_int, [_PTR(_IndexDesc), C.c_int, _PTR(_P)]),
        "gf_index_open": (C.c_int, [_PTR(_IndexFiles), C.c_int, _PTR(_P)]),
        "gf_index_info_get": (C.c_int, [_P, _PTR(_IndexInfo)]),
        "gf_index_entry_points": (C.c_int, [_P, _U32, _P]),
        "gf_index_destroy": (C.c_int, [_P]),
        "gf_plan_create": (C.c_int, [_P, _U32, _PTR(_P)]),
        "gf_plan_destroy": (C.c_int, [_P]),
        "gf_plan_queries": (C.c_int, [_P, _P, _P, _P, _P, _U32, C.c_float, _P]),
        "gf_plan_read": (C.c_int, [_P, _P, _P, _P, C.c_uint64, _P, _P]),
        "gf_search": (C.c_int, [_P, _P, _PTR(_SearchParams), _P, _P, _P]),
        "gf_search_stats_read": (C.c_int, [_P, _PTR(_SearchStats)]),
        "gf_search_host": (C.c_int, [_P, _P, _PTR(_SearchParams), _P, _P, _P, _U32, C.c_float, _P, _P, _P]),
        "gf_search_batched": (C.c_int, [_P, _P, _PTR(_SearchParams), _P, _P, _U32, _P, _P, _P]),
        "gf_search_keys": (C.c_int, [_P, _P, _PTR(_SearchParams), _P, _P]),
        "gf_merge_keys": (C.c_int, [_P, _P, _U32, _U32, _U32, _P, _P, _P]),
        "gf_schedule_batches": (C.c_int, [_P, _U32, _P, _P, _PTR(_U32), _PTR(C.c_uint64)]),
        "gf_schedule_batches_host": (C.c_int, [_U32, _U32, _P, _P, _P, _U32, _P, _P, _PTR(_U32),
                                               _PTR(C.c_uint64)]),
        "gf_bruteforce": (C.c_int, [_P, _P, _P, _P, _U32, _U32, _P, _P, _P]),
        "gf_bruteforce_ex": (C.c_int, [_P, _P, _P, _P, _U32, _U32, _P, _P, _PTR(_BfParams), _P]),
        "gf_index_assemble": (C.c_int, [_P, _U32]),
        "gf_search_fullgraph": (C.c_int, [_P, _P, _PTR(_SearchParams), _P, _P, _P]),
        "gf_free": (None, [_P]),
        "gf_read_fvecs": (C.c_int, [C.c_char_p, _PTR(_P), _PTR(_U32), _PTR(_U32)]),
        "gf_write_fvecs": (C.c_int, [C.c_char_p, _P, _U32, _U32]),
        "gf_read_u8bin": (C.c_int, [C.c_char_p, _PTR(_P), _PTR(_U32), _PTR(_U32)]),
        "gf_read_attrs": (C.c_int, [C.c_char_p, _PTR(_P), _PTR(_U32), _PTR(_U32)]),
        "gf_read_q": (C.c_int, [C.c_char_p, _PTR(_P), _PTR(_P), _PTR(_P), _PTR(_U32), _PTR(_U32)]),
        "gf_write_q": (C.c_int, [C.c_char_p, _P, _P, _P, _U32, _U32]),
        "gf_quantize_i8": (C.c_int, [_P, _U32, _U32, C.c_float, _P, _P, _P, _P]),
        "gf_quantize_i8_host": (C.c_int, [_P, _U32, _U32, C.c_float, _P, _P, _P]),
        "gf_fp4_bytes": (C.c_uint64, [_U32, _U32, _U32]),
        "gf_quantize_fp4": (C.c_int, [_P, _U32, C.c_uint64, _U32, _U32, C.c_float, _U32, _P, _P]),
        "gf_dequantize_fp4": (C.c_int, [_P, _U32, _U32, _U32, C.c_float, _P, _U32, C.c_uint64, _P]),
        "gf_product_fp4": (C.c_int, [_P, _U32, _P, _U32, _U32, _U32, C.c_float, _P, _U32, C.c_uint64, _U32, _P]),
        "gf_product_fp4_raw": (C.c_int, [_P, _U32, C.c_uint64, _U32, C.c_float, _P, _U32, _U32, _U32, C.c_float, _P, _U32,
                                         C.c_uint64, _P, _U32, _P]),
        "gf_product_fp4_timeouts": (C.c_int, [_PTR(C.c_uint64)]),
        "gf_quantize_fp4_host": (C.c_int, [_P, _U32, _U32, C.c_float, _U32, _P]),
        "gf_dequantize_fp4_host": (C.c_int, [_P, _U32, _U32, _U32, C.c_float, _P]),
        "gf_write_attrs": (C.c_int, [C.c_char_p, _P, _U32, _U32]),
        "gf_read_u32mat": (C.c_int, [C.c_char_p, _PTR(_P), _PTR(_U32), _PTR(_U32)]),
        "gf_write_u32mat": (C.c_int, [C.c_char_p, _P, _U32, _U32]),
        "gf_read_ranges": (C.c_int, [C.c_char_p, _U32, _U32, _P, _P]),
        "gf_write_ranges": (C.c_int, [C.c_char_p, _P, _P, _U32, _U32]),
        "gf_read_labels": (C.c_int, [C.c_char_p, _PTR(_P), _PTR(_U32)]),
        "gf_read_grid": (C.c_int, [C.c_char_p, _PTR(_U32), _PTR(_U32), _PTR(_P), _PTR(_P), _PTR(_P), _PTR(_P)]),
        "gf_spokesman_host": (C.c_int, [_U32, _U32, _P, _U32, _P, _P, _P, _PTR(_U32)]),
        "gf_write_spokesman_graph": (C.c_int, [C.c_char_p, _U32, _U32, _U32, _P, _P, _P, _P]),
        "gf_read_spokesman_graph": (C.c_int, [C.c_char_p, _PTR(_U32), _PTR(_U32), _PTR(_U32), _PTR(_P), _PTR(_P),
                                              _PTR(_P), _PTR(_P)]),
    }
    for name, (res, args) in sig.items():
        f = getattr(L, name)
        f.restype = res
        f.argtypes = args
    _LIB = L
    return L


def _check(status: int, what: str) -> None:
    if status != 0:
        L = lib()
        raise GarfieldError(status, what, L.gf_last_error().decode(errors="replace"))


def _np_ptr(a: np.ndarray | None):
    if a is None:
        return None
    assert a.flags["C_CONTIGUOUS"], "array must be C-contiguous"
    return a.ctypes.data_as(C.c_void_p)


def _dev_ptr(t):
    if t is None:
        return None
    import torch
    assert isinstance(t, torch.Tensor) and t.is_cuda and t.is_contiguous(), "expected a contiguous CUDA tensor"
    return C.c_void_p(t.data_ptr())


def _stream_ptr(stream):
    if stream is None:
        import torch
        return C.c_void_p(torch.cuda.current_stream().cuda_stream)
    return C.c_void_p(stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream))


# ------------------------------------------------------------------ params

@dataclass
class SearchParams:
    """Search knobs; defaults are the reference's values (gpu_graph.cu:39, realdataset_search.cu:2495)."""
    L: int = 64
    k: int = 10
    width: int = 1
    max_iter: int = 10000
    n_entry: int = 0          # 0 = graph degree
    postfilter: int = 0xFFFFFFFF
    hash_slots: int = 0       # 0 = automatic
    test_wait: int = 0        # test hook: staging waits give up after this many polls and never complete
    exact_tc: int = 0         # 1: exact-route queries go to the tensor-core exact scan (fp32 rows)
    route: int = 0            # 1: also route by cost (box count vs cells x (L + 64)); needs exact_tc

    def _c(self) -> _SearchParams:
        return _SearchParams(self.L, self.k, self.width, self.max_iter, self.n_entry, self.postfilter,
                             self.hash_slots, self.test_wait, self.exact_tc, self.route)


# ------------------------------------------------------------------ index

class Index:
    """Device-resident GMG index (gf_index)."""

    def __init__(self, handle: C.c_void_p, keep: tuple = ()):
        self._h = handle
        self._keep = keep
        info = _IndexInfo()
        _check(lib().gf_index_info_get(self._h, C.byref(info)), "gf_index_info_get")
        self.n, self.dim, self.n_attr = info.n, info.dim, info.n_attr
        self.n_cells, self.degree, self.cross_e = info.n_cells, info.degree, info.cross_e
        self.n_clusters, self.min_cell_size = info.n_clusters, info.min_cell_size
        self.device_bytes = info.device_bytes
        self.cross_rows = info.cross_rows

    @classmethod
    def create(cls, *, vectors, attrs, grid, l_quant, r_quant, cell_of, graphs, degree, cross=None,
               cross_e=0, labels=None, f2h_factor=1.0, keep_fp32=True, host_graph=False, shard_cells=None,
               codec=0, codes=None, code_scales=None, code_zero_points=None, cross_spokesman=False,
               device=0) -> "Index":
        """Build from host arrays in the reference's layout (see gf_index_desc).  With
        host_graph the graphs and cross edges stay in pinned host memory (search with
        Plan.search_batched); with shard_cells the device holds only those cells (a shard
        of a cell-sharded index: Plan.search_keys + Index.merge_keys)."""
        vectors = np.ascontiguousarray(vectors, dtype=np.float32)
        attrs = np.ascontiguousarray(attrs, dtype=np.float32)
        grid = np.ascontiguousarray(grid, dtype=np.uint32)
        lq = np.ascontiguousarray(l_quant, dtype=np.float32)
        rq = np.ascontiguousarray(r_quant, dtype=np.float32)
        cell_of = np.ascontiguousarray(cell_of, dtype=np.uint32)
        graphs = np.ascontiguousarray(graphs, dtype=np.uint32)
        cross = None if cross is None else np.ascontiguousarray(cross, dtype=np.uint32)
        labels = None if labels is None else np.ascontiguousarray(labels, dtype=np.int32)
        n, dim = vectors.shape
        d = _IndexDesc()
        d.n, d.dim, d.n_attr = n, dim, attrs.shape[1]
        d.vectors, d.attrs, d.grid = _np_ptr(vectors), _np_ptr(attrs), _np_ptr(grid)
        d.l_quant, d.r_quant, d.cell_of = _np_ptr(lq), _np_ptr(rq), _np_ptr(cell_of)
        d.degree, d.graphs = degree, _np_ptr(graphs)
        d.cross_e, d.cross = (cross_e if cross is not None else 0), _np_ptr(cross)
        d.n_clusters, d.labels = (1 if labels is not None else 0), _np_ptr(labels)
        d.f2h_factor, d.keep_fp32 = f2h_factor, 1 if keep_fp32 else 0
        d.host_graph = 1 if host_graph else 0
        shard = None
        if shard_cells is not None:
            shard = np.ascontiguousarray(shard_cells, dtype=np.uint32)
            d.shard_cells, d.n_shard_cells = _np_ptr(shard), len(shard)
            d.keep_fp32 = 0
        d.codec = codec
        d.cross_spokesman = 1 if cross_spokesman else 0
        keep = []
        if codes is not None:
            codes = np.ascontiguousarray(codes).view(np.uint8)
            keep.append(codes)
            d.codes = _np_ptr(codes)
        if code_scales is not None:
            code_scales = np.ascontiguousarray(code_scales, dtype=np.float32)
            keep.append(code_scales)
            d.code_scales = _np_ptr(code_scales)
        if code_zero_points is not None:
            code_zero_points = np.ascontiguousarray(code_zero_points, dtype=np.int32)
            keep.append(code_zero_points)
            d.code_zero_points = _np_ptr(code_zero_points)
        h = C.c_void_p()
        _check(lib().gf_index_create(C.byref(d), device, C.byref(h)), "gf_index_create")
        return cls(h)

    @classmethod
    def open(cls, *, data_path, cagra_prefix, cagra_suffix, global_graph, grid=None, attrs, cluster=None,
             degree=32, f2h_factor=1.0, keep_fp32=False, device=0, uniform_shape=None, uniform_lo=0.0,
             uniform_hi=1e6, host_graph=False, codec=0, quantized=None) -> "Index":
        """Load the reference's index files (realdataset_search flags).  Without a grid file,
        `uniform_shape` gives the uniform grid of normaldataset_search."""
        f = _IndexFiles()
        f.data_path, f.cagra_prefix, f.cagra_suffix = (str(data_path).encode(), str(cagra_prefix).encode(),
                                                       str(cagra_suffix).encode())
        f.global_graph, f.attrs = str(global_graph).encode(), str(attrs).encode()
        f.grid = None if grid is None else str(grid).encode()
        f.cluster = None if cluster is None else str(cluster).encode()
        f.degree, f.f2h_factor, f.keep_fp32 = degree, f2h_factor, 1 if keep_fp32 else 0
        f.host_graph = 1 if host_graph else 0
        f.codec = codec
        f.quantized = None if quantized is None else str(quantized).encode()
        shape = None
        if uniform_shape is not None:
            shape = np.ascontiguousarray(uniform_shape, dtype=np.uint32)
            f.uniform_dims, f.uniform_shape = len(shape), _np_ptr(shape)
            f.uniform_lo, f.uniform_hi = uniform_lo, uniform_hi
        h = C.c_void_p()
        _check(lib().gf_index_open(C.byref(f), device, C.byref(h)), "gf_index_open")
        return cls(h)

    def close(self) -> None:
        if self._h:
            lib().gf_index_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def entry_points(self, n: int) -> np.ndarray:
        out = np.zeros(n, np.uint32)
        _check(lib().gf_index_entry_points(self._h, n, _np_ptr(out)), "gf_index_entry_points")
        return out

    def assemble(self, reserve: int = 2) -> None:
        """gf_index_assemble: the full-graph ablation's graph (assemble_edges) on the device."""
        _check(lib().gf_index_assemble(self._h, reserve), "gf_index_assemble")

    def plan(self, max_queries: int) -> "Plan":
        return Plan(self, max_queries)

    def merge_keys(self, keys, k: int, stream=None):
        """gf_merge_keys: keys (lists, qnum, k) int64 CUDA tensor -> (ids int32, dists)."""
        import torch
        lists, q = keys.shape[0], keys.shape[1]
        ids = torch.empty((q, k), dtype=torch.int32, device=keys.device)
        dist = torch.empty((q, k), dtype=torch.float32, device=keys.device)
        _check(lib().gf_merge_keys(self._h, _dev_ptr(keys), lists, q, k, _dev_ptr(ids), _dev_ptr(dist),
                                   _stream_ptr(stream)), "gf_merge_keys")
        return ids, dist

    def bruteforce(self, queries, lb, rb, k: int, stream=None, path: int = 0, test_fallback_every: int = 0,
                   stats=None, test_wait: int = 0):
        """Exact filtered k-NN on the device; returns (ids, dists) CUDA tensors.

        path: 0 automatic (tensor cores when available), 1 CUDA cores, 2 tensor cores.
        stats: optional int32 CUDA tensor of 3 words (queries answered by the CUDA-core
        kernel after the tensor-core pass, waits that ran out, 128 x 128 tile products)."""
        import torch
        q = queries.shape[0]
        ids = torch.empty((q, k), dtype=torch.int32, device=queries.device)
        dist = torch.empty((q, k), dtype=torch.float32, device=queries.device)
        if path == 0 and test_fallback_every == 0 and stats is None and test_wait == 0:
            _check(lib().gf_bruteforce(self._h, _dev_ptr(queries), _dev_ptr(lb), _dev_ptr(rb), q, k,
                                       _dev_ptr(ids), _dev_ptr(dist), _stream_ptr(stream)), "gf_bruteforce")
        else:
            prm = _BfParams(path, test_fallback_every, test_wait, _dev_ptr(stats).value if stats is not None else None)
            _check(lib().gf_bruteforce_ex(self._h, _dev_ptr(queries), _dev_ptr(lb), _dev_ptr(rb), q, k,
                                          _dev_ptr(ids), _dev_ptr(dist), C.byref(prm), _stream_ptr(stream)),
                   "gf_bruteforce_ex")
        return ids, dist

    def search(self, queries, lb, rb, params: SearchParams | None = None, prefilter: float = 0.0,
               plan: "Plan | None" = None, stream=None):
        """Plan + search on the device; returns (ids int32, dists) CUDA tensors (ids: global, NO_ID = -1)."""
        params = params or SearchParams()
        own = plan is None
        plan = plan or Plan(self, queries.shape[0])
        try:
            plan.build(queries, lb, rb, prefilter, stream)
            return plan.search(params, stream)
        finally:
            if own:
                plan.close()

    def search_host(self, queries: np.ndarray, lb: np.ndarray, rb: np.ndarray, plan: "Plan",
                    params: SearchParams | None = None, prefilter: float = 0.0, with_dist: bool = False,
                    stream=None):
        """End-to-end call from host memory (gf_search_host): H2D, plan, search, D2H."""
        params = params or SearchParams()
        q = queries.shape[0]
        ids = np.empty((q, params.k), np.uint32)
        dist = np.empty((q, params.k), np.float32) if with_dist else None
        cp = params._c()
        _check(lib().gf_search_host(self._h, plan._h, C.byref(cp), _np_ptr(queries), _np_ptr(lb), _np_ptr(rb),
                                    q, prefilter, _np_ptr(ids), _np_ptr(dist), _stream_ptr(stream)),
               "gf_search_host")
        return ids, dist


class Plan:
    """Planned query batch (gf_plan): cell lists in cluster-guided order."""

    def __init__(self, index: Index, max_queries: int):
        self.index = index
        self.max_queries = max_queries
        h = C.c_void_p()
        _check(lib().gf_plan_create(index._h, max_queries, C.byref(h)), "gf_plan_create")
        self._h = h
        self.qnum = 0

    def close(self) -> None:
        if self._h:
            lib().gf_plan_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def build(self, queries, lb, rb, prefilter: float = 0.0, stream=None) -> None:
        self.qnum = queries.shape[0]
        _check(lib().gf_plan_queries(self.index._h, self._h, _dev_ptr(queries), _dev_ptr(lb), _dev_ptr(rb),
                                     self.qnum, prefilter, _stream_ptr(stream)), "gf_plan_queries")

    def read(self):
        """(counts, offsets, cells, top4, box_counts) as numpy (synchronises)."""
        q = self.qnum
        counts = np.zeros(q, np.uint32)
        offsets = np.zeros(q, np.uint32)
        top4 = np.zeros((q, 4), np.uint32)
        box = np.zeros(q, np.uint32)
        cap = q * max(self.index.n_cells, 1)
        cells = np.zeros(cap, np.uint32)
        _check(lib().gf_plan_read(self._h, _np_ptr(counts), _np_ptr(offsets), _np_ptr(cells), cap,
                                  _np_ptr(top4), _np_ptr(box)), "gf_plan_read")
        total = int(counts.sum())
        return counts, offsets, cells[:total], top4, box

    def search(self, params: SearchParams | None = None, stream=None, ids=None, dist=None):
        import torch
        params = params or SearchParams()
        dev = torch.device("cuda", torch.cuda.current_device())
        if ids is None:
            ids = torch.empty((self.qnum, params.k), dtype=torch.int32, device=dev)
        if dist is None:
            dist = torch.empty((self.qnum, params.k), dtype=torch.float32, device=dev)
        cp = params._c()
        _check(lib().gf_search(self.index._h, self._h, C.byref(cp), _dev_ptr(ids), _dev_ptr(dist),
                               _stream_ptr(stream)), "gf_search")
        return ids, dist

    def search_fullgraph(self, params: SearchParams | None = None, stream=None, ids=None, dist=None):
        """gf_search_fullgraph: the full-graph post-filter ablation over the index's assembled
        graph (Index.assemble first)."""
        import torch
        params = params or SearchParams()
        dev = torch.device("cuda", torch.cuda.current_device())
        if ids is None:
            ids = torch.empty((self.qnum, params.k), dtype=torch.int32, device=dev)
        if dist is None:
            dist = torch.empty((self.qnum, params.k), dtype=torch.float32, device=dev)
        cp = params._c()
        _check(lib().gf_search_fullgraph(self.index._h, self._h, C.byref(cp), _dev_ptr(ids), _dev_ptr(dist),
                                         _stream_ptr(stream)), "gf_search_fullgraph")
        return ids, dist

    def search_batched(self, batches, params: SearchParams | None = None, stream=None, ids=None, dist=None):
        """gf_search_batched: `batches` is a list of cell-id lists (each cell in at most one)."""
        import torch
        params = params or SearchParams()
        dev = torch.device("cuda", torch.cuda.current_device())
        if ids is None:
            ids = torch.empty((self.qnum, params.k), dtype=torch.int32, device=dev)
        if dist is None:
            dist = torch.empty((self.qnum, params.k), dtype=torch.float32, device=dev)
        sizes = np.array([len(b) for b in batches], np.uint32)
        cells = np.ascontiguousarray(np.concatenate([np.asarray(b, np.uint32) for b in batches])
                                     if len(batches) else np.zeros(0, np.uint32), dtype=np.uint32)
        cp = params._c()
        _check(lib().gf_search_batched(self.index._h, self._h, C.byref(cp), _np_ptr(cells), _np_ptr(sizes),
                                       len(batches), _dev_ptr(ids), _dev_ptr(dist), _stream_ptr(stream)),
               "gf_search_batched")
        return ids, dist

    def search_keys(self, params: SearchParams | None = None, stream=None, keys=None):
        """gf_search_keys: (qnum, k) int64 CUDA tensor of merge keys."""
        import torch
        params = params or SearchParams()
        if keys is None:
            keys = torch.empty((self.qnum, params.k), dtype=torch.int64,
                               device=torch.device("cuda", torch.cuda.current_device()))
        cp = params._c()
        _check(lib().gf_search_keys(self.index._h, self._h, C.byref(cp), _dev_ptr(keys), _stream_ptr(stream)),
               "gf_search_keys")
        return keys

    def schedule(self, max_cells: int):
        """gf_schedule_batches: (list of cell lists, splits) for search_batched."""
        n = self.index.n_cells
        cells, sizes = np.zeros(n, np.uint32), np.zeros(n, np.uint32)
        nb, splits = _U32(), C.c_uint64()
        _check(lib().gf_schedule_batches(self._h, max_cells, _np_ptr(cells), _np_ptr(sizes), C.byref(nb),
                                         C.byref(splits)), "gf_schedule_batches")
        return _unpack_batches(cells, sizes, nb.value), int(splits.value)

    def stats(self) -> dict:
        s = _SearchStats()
        _check(lib().gf_search_stats_read(self._h, C.byref(s)), "gf_search_stats_read")
        return {n: getattr(s, n) for n, _ in _SearchStats._fields_}


# ------------------------------------------------------------------ file formats

def _unpack_batches(cells, sizes, nb):
    out, o = [], 0
    for b in range(nb):
        out.append(cells[o:o + int(sizes[b])].tolist())
        o += int(sizes[b])
    return out


def schedule_batches(ncells: int, counts, offsets, cells, max_cells: int):
    """gf_schedule_batches_host on host plan arrays: (list of cell lists, splits)."""
    counts = np.ascontiguousarray(counts, np.uint32)
    offsets = np.ascontiguousarray(offsets, np.uint32)
    cells = np.ascontiguousarray(cells, np.uint32)
    bc, bs = np.zeros(max(ncells, 1), np.uint32), np.zeros(max(ncells, 1), np.uint32)
    nb, splits = _U32(), C.c_uint64()
    _check(lib().gf_schedule_batches_host(ncells, len(counts), _np_ptr(counts), _np_ptr(offsets), _np_ptr(cells),
                                          max_cells, _np_ptr(bc), _np_ptr(bs), C.byref(nb), C.byref(splits)),
           "gf_schedule_batches_host")
    return _unpack_batches(bc, bs, nb.value), int(splits.value)


def quantize_i8_host(data: np.ndarray, alpha: float = 1.0):
    """gf_quantize_i8_host: (codes int8 n x dim, scales, zero points)."""
    data = np.ascontiguousarray(data, dtype=np.float32)
    n, dim = data.shape
    q = np.zeros((n, dim), np.int8)
    sc, zp = np.zeros(dim, np.float32), np.zeros(dim, np.int32)
    _check(lib().gf_quantize_i8_host(_np_ptr(data), n, dim, alpha, _np_ptr(q), _np_ptr(sc), _np_ptr(zp)),
           "gf_quantize_i8_host")
    return q, sc, zp


def quantize_i8(data, alpha: float = 1.0, stream=None):
    """gf_quantize_i8 on a CUDA tensor: (codes int8, scales, zero points) CUDA tensors."""
    import torch
    n, dim = data.shape
    q = torch.empty((n, dim), dtype=torch.int8, device=data.device)
    sc = torch.empty(dim, dtype=torch.float32, device=data.device)
    zp = torch.empty(dim, dtype=torch.int32, device=data.device)
    _check(lib().gf_quantize_i8(_dev_ptr(data), n, dim, alpha, _dev_ptr(q), _dev_ptr(sc), _dev_ptr(zp),
                                _stream_ptr(stream)), "gf_quantize_i8")
    return q, sc, zp


# ------------------------------------------------- 4-bit block floating point

@dataclass
class Fp4Rows:
    """n x dim rows held in 4 bits (the packed form that include/garfield.h describes): codes with one
    scale per `block` elements of a row, standing for the data multiplied by alpha (an fp32 number: what is
    given is rounded to one).  packed is a uint8 CUDA tensor, or a numpy array from quantize_fp4_host."""
    packed: object
    n: int
    dim: int
    block: int
    alpha: float

    def __post_init__(self):
        self.alpha = C.c_float(self.alpha).value


def _fp4_need(ok: bool, what: str, msg: str) -> None:
    if not ok:
        raise GarfieldError(1, what, msg)


_FP4_DTYPES = {}


def _fp4_dtype(dtype, what: str) -> int:
    if not _FP4_DTYPES:
        import torch
        _FP4_DTYPES.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
    dt = _FP4_DTYPES.get(dtype)
    if dt is None:
        raise GarfieldError(1, what, f"dtype {dtype} is not float32, float16 or bfloat16")
    return dt


def _fp4_float32():
    import torch
    return torch.float32


def _fp4_matrix(t, what: str, name: str):
    """(rows, columns, row stride) of a CUDA tensor, which has to be a matrix whose rows are each without gaps."""
    shape = t.shape
    if len(shape) != 2:
        raise GarfieldError(1, what, f"{name}: expected a 2-D CUDA tensor")
    n, dim = shape
    ld, step = t.stride()
    if n <= 1:
        ld = dim
    if not (0 < dim < 2 ** 32 and n < 2 ** 32):
        raise GarfieldError(1, what, f"{name}: shape {(n, dim)} out of range")
    if step != 1 and dim > 1 and n > 0:
        raise GarfieldError(1, what, f"{name}: the elements of a row must be adjacent")
    if ld < dim:
        raise GarfieldError(1, what, f"{name}: rows overlap (stride {ld} below {dim})")
    return n, dim, ld


def _fp4_size(n: int, dim: int, block: int) -> int:
    """gf_fp4_bytes: panels of 128 rows, in each the scales of every 128 elements, then columns of 32."""
    rows = 128 if n >= 128 else -(-n // 16) * 16
    return -(-n // 128) * (-(-dim // 128) * (16384 // block) + -(-dim // 32) * rows * 16)


def _fp4_shape(rows, what: str) -> int:
    """The size of rows, whose shape has to be one that the library takes."""
    n, dim, block = rows.n, rows.dim, rows.block
    if block not in (16, 32) or not (0 < dim < 2 ** 32 and 0 <= n < 2 ** 32):
        raise GarfieldError(1, what, f"n {n}, dim {dim}, block {block}")
    return _fp4_size(n, dim, block)


def _fp4_rows(rows, what: str):
    p = getattr(rows, "packed", None)
    if not isinstance(rows, Fp4Rows) or not getattr(p, "is_cuda", False):
        raise GarfieldError(1, what, "expected Fp4Rows on a GPU")
    size = _fp4_shape(rows, what)
    if p.numel() < size or p.element_size() != 1 or not p.is_contiguous():
        raise GarfieldError(1, what, f"Fp4Rows.packed: expected {size} contiguous bytes")
    return p


class _on_stream:
    """Makes a device current, and the given stream of it (None: the device's current one), so that
    what is allocated inside belongs to the stream that the kernels run on."""

    def __init__(self, device, stream):
        import torch
        if stream is not None and not hasattr(stream, "cuda_stream"):
            stream = torch.cuda.ExternalStream(int(stream), device=device)
        self.stream = stream if stream is not None else torch.cuda.current_stream(device)
        self.device, self.ctx = torch.cuda.device(device), torch.cuda.stream(self.stream)

    def __enter__(self):
        self.device.__enter__()
        self.ctx.__enter__()
        return self.stream.cuda_stream

    def __exit__(self, *exc):
        self.ctx.__exit__(*exc)
        self.device.__exit__(*exc)


def _fp4_run(what, device, stream, f, *args):
    """f(raw stream, *args) with the device and the stream current.  The usual case, the current stream
    of the current device, reads torch's raw handle: entering contexts costs more than a small call.
    On another stream than the current one, the allocator is told that the call's tensors are used there,
    and its result here: either may be dropped while the other stream has still to read it."""
    import torch
    if stream is None and device.index == torch._C._cuda_getDevice():
        return f(torch._C._cuda_getCurrentRawStream(device.index), *args)
    other = getattr(stream, "device", device)
    if isinstance(other, torch.device) and other != device:
        raise GarfieldError(1, what, f"a stream of {other}, data on {device}")
    here, on = torch.cuda.current_stream(device), _on_stream(device, stream)
    with on as s:
        result = f(s, *args)
    if on.stream.cuda_stream != here.cuda_stream:
        for t in args:
            t = t.packed if isinstance(t, Fp4Rows) else t
            if isinstance(t, torch.Tensor):
                t.record_stream(on.stream)
        (result.packed if isinstance(result, Fp4Rows) else result).record_stream(here)
    return result


def _fp4_quantize(s, data, alpha, block):
    import torch
    what = "gf_quantize_fp4"
    n, dim, ld = _fp4_matrix(data, what, "data")
    dt = _fp4_dtype(data.dtype, what)
    if block != 32 and block != 16:
        raise GarfieldError(1, what, f"block {block} is not 16 or 32")
    packed = torch.empty(_fp4_size(n, dim, block), dtype=torch.uint8, device=data.device)
    st = lib().gf_quantize_fp4(data.data_ptr(), dt, ld, n, dim, alpha, block, packed.data_ptr(), s)
    if st:
        _check(st, what)
    return Fp4Rows(packed, n, dim, block, alpha)


def quantize_fp4(data, alpha: float = 1.0, block: int = 32, stream=None) -> Fp4Rows:
    """gf_quantize_fp4: the rows of a float32, float16 or bfloat16 CUDA matrix, held in 4 bits.
    stream: where the kernels run (None: the current stream).  As with torch's own streams, the caller orders
    another stream after the work that makes the inputs and before the work that reads the result; the
    tensors need not be kept meanwhile."""
    if not getattr(data, "is_cuda", False):
        raise GarfieldError(1, "gf_quantize_fp4", "data: expected a 2-D CUDA tensor")
    return _fp4_run("gf_quantize_fp4", data.device, stream, _fp4_quantize, data, alpha, block)


def _fp4_out(out, m: int, n: int, dtype, device, what: str):
    """(out, its row stride): a new m x n tensor, or the caller's, checked."""
    import torch
    if out is None:
        return torch.empty((m, n), dtype=dtype, device=device), n
    if not getattr(out, "is_cuda", False) or tuple(out.shape) != (m, n) or out.dtype != dtype or out.device != device:
        raise GarfieldError(1, what, f"out: expected a {dtype} tensor of shape {(m, n)} on {device}")
    return out, (_fp4_matrix(out, what, "out")[2] if m and n else n)


def _fp4_dequantize(s, p, rows, dtype, out):
    what = "gf_dequantize_fp4"
    dt = _fp4_dtype(dtype, what)
    out, ld = _fp4_out(out, rows.n, rows.dim, dtype, p.device, what)
    st = lib().gf_dequantize_fp4(p.data_ptr(), rows.n, rows.dim, rows.block, rows.alpha, out.data_ptr(), dt, ld, s)
    if st:
        _check(st, what)
    return out


def dequantize_fp4(rows: Fp4Rows, dtype=None, out=None, stream=None):
    """gf_dequantize_fp4: the values that rows are held as (n x dim, float32 unless dtype or out say
    otherwise).  out does not overlap rows; stream is as in quantize_fp4."""
    p = _fp4_rows(rows, "gf_dequantize_fp4")
    if dtype is None:
        dtype = _fp4_float32() if out is None else out.dtype
    return _fp4_run("gf_dequantize_fp4", p.device, stream, _fp4_dequantize, p, rows, dtype, out)


def _fp4_scale(query_alpha: float, alpha: float, what: str) -> float:
    """What the products of the held values are multiplied by.  Outside fp32's normal range it would be rounded
    to few bits, or to none."""
    both = query_alpha * alpha
    if not 2.0 ** -127 <= both <= 2.0 ** 126:
        raise GarfieldError(1, what, f"query_alpha {query_alpha} * alpha {alpha} must lie in [2^-127, 2^126]")
    return 1.0 / both


def _fp4_product(s, queries, p, rows, dtype, out, query_alpha, test_wait):
    what = "gf_product_fp4"
    dt = _fp4_dtype(dtype, what)
    device, dim, block = p.device, rows.dim, rows.block
    if isinstance(queries, Fp4Rows):
        qp = _fp4_rows(queries, what)
        m, qdim = queries.n, queries.dim
        if queries.block != block:
            raise GarfieldError(1, what, f"queries of block {queries.block}, rows of block {block}")
    else:
        qp = queries
        m, qdim, qld = _fp4_matrix(queries, what, "queries")
        qdt = _fp4_dtype(queries.dtype, what)
    if qp.device != device or qdim != dim:
        raise GarfieldError(1, what, f"queries of dim {qdim} on {qp.device}, rows of dim {dim} on {device}")
    out, ld = _fp4_out(out, m, rows.n, dtype, device, what)
    if qp is queries:
        # (what the call quantises in passing needs no room)
        ws = None
        if not (m <= 16 and dim <= 8192 and m * dim <= 32768):
            import torch
            ws = torch.empty(_fp4_size(m, dim, block), dtype=torch.uint8, device=device)
        st = lib().gf_product_fp4_raw(qp.data_ptr(), qdt, qld, m, query_alpha, p.data_ptr(), rows.n, dim, block,
                                      _fp4_scale(C.c_float(query_alpha).value, rows.alpha, what), out.data_ptr(), dt, ld,
                                      None if ws is None else ws.data_ptr(), test_wait, s)
    else:
        st = lib().gf_product_fp4(qp.data_ptr(), m, p.data_ptr(), rows.n, dim, block,
                                  _fp4_scale(queries.alpha, rows.alpha, what), out.data_ptr(), dt, ld, test_wait, s)
    if st:
        _check(st, what)
    return out


def product_fp4(queries, rows: Fp4Rows, dtype=None, out=None, query_alpha: float = 1.0, stream=None,
                test_wait: int = 0):
    """gf_product_fp4: the inner products of every query with every row (m x n, float32 unless dtype or
    out say otherwise).  queries: Fp4Rows of the same dim and block, or a float32, float16 or
    bfloat16 CUDA matrix, which is held in 4 bits (quantize_fp4 with query_alpha and the rows'
    block) for the call (gf_product_fp4_raw).  The product of both alphas lies in [2^-127, 2^126].
    out overlaps neither input; stream is as in quantize_fp4; test_wait is a test hook (0 in normal use).
    product_fp4_timeouts tells outputs that a wait which ran out left as NaN from those of NaN data."""
    p = _fp4_rows(rows, "gf_product_fp4")
    if not isinstance(queries, Fp4Rows) and not getattr(queries, "is_cuda", False):
        raise GarfieldError(1, "gf_product_fp4", "queries: expected Fp4Rows or a 2-D CUDA tensor")
    if dtype is None:
        dtype = _fp4_float32() if out is None else out.dtype
    return _fp4_run("gf_product_fp4", p.device, stream, _fp4_product, queries, p, rows, dtype, out, query_alpha, test_wait)


def product_fp4_timeouts(device=None) -> int:
    """gf_product_fp4_timeouts: how many thread blocks of product_fp4 stopped on a device (None: the current one)
    because a wait ran out, each leaving NaN in its outputs.  0 on a sound GPU.  Waits for the device."""
    import torch
    with torch.cuda.device(device):
        torch.cuda.synchronize()
        count = C.c_uint64()
        _check(lib().gf_product_fp4_timeouts(C.byref(count)), "gf_product_fp4_timeouts")
    return count.value


def quantize_fp4_host(data: np.ndarray, alpha: float = 1.0, block: int = 32) -> Fp4Rows:
    """gf_quantize_fp4_host on a float32 array: the same bytes as quantize_fp4."""
    data = np.ascontiguousarray(data, dtype=np.float32)
    _fp4_need(data.ndim == 2, "gf_quantize_fp4_host", "data: expected a 2-D array")
    n, dim = data.shape
    _fp4_need(dim > 0 and block in (16, 32), "gf_quantize_fp4_host", f"dim {dim}, block {block}")
    packed = np.empty(_fp4_size(n, dim, block), np.uint8)
    _check(lib().gf_quantize_fp4_host(_np_ptr(data), n, dim, alpha, block, _np_ptr(packed)), "gf_quantize_fp4_host")
    return Fp4Rows(packed, n, dim, block, alpha)


def dequantize_fp4_host(rows: Fp4Rows) -> np.ndarray:
    """gf_dequantize_fp4_host: the float32 values that rows with a host array are held as."""
    what = "gf_dequantize_fp4_host"
    _fp4_need(isinstance(rows, Fp4Rows), what, "expected Fp4Rows")
    size = _fp4_shape(rows, what)
    p = rows.packed
    _fp4_need(isinstance(p, np.ndarray) and p.dtype == np.uint8 and p.flags["C_CONTIGUOUS"], what,
              "Fp4Rows.packed: expected a contiguous uint8 array")
    _fp4_need(p.size >= size, what, "Fp4Rows.packed is too short")
    out = np.empty((rows.n, rows.dim), np.float32)
    _check(lib().gf_dequantize_fp4_host(_np_ptr(p), rows.n, rows.dim, rows.block, rows.alpha, _np_ptr(out)), what)
    return out


def read_q(path):
    """.q file -> (codes int8 n x dim, scales, zero points)."""
    q, sc, zp = _P(), _P(), _P()
    n, d = _U32(), _U32()
    _check(lib().gf_read_q(str(path).encode(), C.byref(q), C.byref(sc), C.byref(zp), C.byref(n), C.byref(d)),
           "gf_read_q")
    codes = _take(q, n.value * d.value, np.int8).reshape(n.value, d.value)
    return codes, _take(sc, d.value, np.float32), _take(zp, d.value, np.int32)


def write_q(path, codes, scales, zero_points) -> None:
    codes = np.ascontiguousarray(codes, dtype=np.int8)
    sc = np.ascontiguousarray(scales, dtype=np.float32)
    zp = np.ascontiguousarray(zero_points, dtype=np.int32)
    _check(lib().gf_write_q(str(path).encode(), _np_ptr(codes), _np_ptr(sc), _np_ptr(zp), codes.shape[0],
                            codes.shape[1]), "gf_write_q")


def _take(ptr: C.c_void_p, count: int, dtype) -> np.ndarray:
    arr = np.ctypeslib.as_array(C.cast(ptr, C.POINTER(np.ctypeslib.as_ctypes_type(dtype))), shape=(count,)).copy()
    lib().gf_free(ptr)
    return arr


def read_fvecs(path) -> np.ndarray:
    p, n, d = C.c_void_p(), C.c_uint32(), C.c_uint32()
    _check(lib().gf_read_fvecs(str(path).encode(), C.byref(p), C.byref(n), C.byref(d)), "gf_read_fvecs")
    return _take(p, n.value * d.value, np.float32).reshape(n.value, d.value)


def write_fvecs(path, data: np.ndarray) -> None:
    a = np.ascontiguousarray(data, np.float32)
    _check(lib().gf_write_fvecs(str(path).encode(), _np_ptr(a), a.shape[0], a.shape[1]), "gf_write_fvecs")


def read_attrs(path) -> np.ndarray:
    p, n, a = C.c_void_p(), C.c_uint32(), C.c_uint32()
    _check(lib().gf_read_attrs(str(path).encode(), C.byref(p), C.byref(n), C.byref(a)), "gf_read_attrs")
    return _take(p, n.value * a.value, np.int32).reshape(n.value, a.value)


def write_attrs(path, attrs: np.ndarray) -> None:
    a = np.ascontiguousarray(attrs, np.int32)
    _check(lib().gf_write_attrs(str(path).encode(), _np_ptr(a), a.shape[0], a.shape[1]), "gf_write_attrs")


def read_u32mat(path) -> np.ndarray:
    p, n, k = C.c_void_p(), C.c_uint32(), C.c_uint32()
    _check(lib().gf_read_u32mat(str(path).encode(), C.byref(p), C.byref(n), C.byref(k)), "gf_read_u32mat")
    return _take(p, n.value * k.value, np.uint32).reshape(n.value, k.value)


def write_u32mat(path, m: np.ndarray) -> None:
    a = np.ascontiguousarray(m, np.uint32)
    _check(lib().gf_write_u32mat(str(path).encode(), _np_ptr(a), a.shape[0], a.shape[1]), "gf_write_u32mat")


def read_ranges(path, qnum: int, a: int):
    lo = np.zeros((qnum, a), np.int32)
    hi = np.zeros((qnum, a), np.int32)
    _check(lib().gf_read_ranges(str(path).encode(), qnum, a, _np_ptr(lo), _np_ptr(hi)), "gf_read_ranges")
    return lo, hi


def write_ranges(path, lo: np.ndarray, hi: np.ndarray) -> None:
    lo = np.ascontiguousarray(lo, np.int32)
    hi = np.ascontiguousarray(hi, np.int32)
    _check(lib().gf_write_ranges(str(path).encode(), _np_ptr(lo), _np_ptr(hi), lo.shape[0], lo.shape[1]),
           "gf_write_ranges")


def read_labels(path) -> np.ndarray:
    p, n = C.c_void_p(), C.c_uint32()
    _check(lib().gf_read_labels(str(path).encode(), C.byref(p), C.byref(n)), "gf_read_labels")
    return _take(p, n.value, np.int32)


def read_grid(path):
    """(grid, l_quant, r_quant, cell_of) of a grid_info file."""
    n, a = C.c_uint32(), C.c_uint32()
    g, lq, rq, co = C.c_void_p(), C.c_void_p(), C.c_void_p(), C.c_void_p()
    _check(lib().gf_read_grid(str(path).encode(), C.byref(n), C.byref(a), C.byref(g), C.byref(lq), C.byref(rq),
                              C.byref(co)), "gf_read_grid")
    grid = _take(g, a.value, np.uint32)
    tot = int(grid.sum())
    return grid, _take(lq, tot, np.int32), _take(rq, tot, np.int32), _take(co, n.value, np.uint32)


def spokesman(cell_sizes, graphs):
    """gf_spokesman_host: (spokesman position, spokesman rank, number of spokesmen) of every
    position (cell order) from the per-cell graphs (n x R local ids, rows in cell order)."""
    sizes = np.ascontiguousarray(cell_sizes, np.uint32)
    g = np.ascontiguousarray(graphs, np.uint32)
    n = g.shape[0]
    spk = np.zeros(n, np.uint32)
    rank = np.zeros(n, np.uint32)
    ns = C.c_uint32()
    _check(lib().gf_spokesman_host(n, len(sizes), _np_ptr(sizes), g.shape[1], _np_ptr(g), _np_ptr(spk), _np_ptr(rank),
                                   C.byref(ns)), "gf_spokesman_host")
    return spk, rank, ns.value


def compress_cross(cell_of, graphs, cross, cross_e: int):
    """The reference's compressed cross graph (compress_global_graph_extreme, tools.cuh:917-1010)
    from index arrays in the reference layout (global order): returns (center_num, col_offset,
    center_pos, edges) with center_pos indexed by position (cell order) and edges
    n_cells x n_spokesmen x E local ids, as gf_write_spokesman_graph writes them."""
    cell_of = np.asarray(cell_of, np.uint32)
    P = int(cell_of.max()) + 1
    order = np.argsort(cell_of, kind="stable")                    # position -> global id
    sizes = np.bincount(cell_of, minlength=P).astype(np.uint32)
    spk, rank, ns = spokesman(sizes, np.asarray(graphs, np.uint32))
    heads = np.nonzero(spk == np.arange(len(spk)))[0]              # spokesman positions, rank order
    seg = np.concatenate([[0], np.cumsum(sizes)])
    center_num = np.array([((heads >= seg[c]) & (heads < seg[c + 1])).sum() for c in range(P)], np.uint32)
    col_offset = np.concatenate([[0], np.cumsum(center_num)[:-1]]).astype(np.uint32)
    x = np.asarray(cross, np.uint32).reshape(len(cell_of), P, cross_e)[order[heads]]  # ns x P x E
    edges = np.ascontiguousarray(x.transpose(1, 0, 2))
    return center_num, col_offset, rank.astype(np.uint32), edges


def write_spokesman_graph(path, center_num, col_offset, center_pos, edges) -> None:
    cn = np.ascontiguousarray(center_num, np.uint32)
    co = np.ascontiguousarray(col_offset, np.uint32)
    cp = np.ascontiguousarray(center_pos, np.uint32)
    e = np.ascontiguousarray(edges, np.uint32)
    _check(lib().gf_write_spokesman_graph(str(path).encode(), len(cp), len(cn), e.shape[2], _np_ptr(cn), _np_ptr(co),
                                          _np_ptr(cp), _np_ptr(e)), "gf_write_spokesman_graph")


def read_spokesman_graph(path):
    n, P, E = C.c_uint32(), C.c_uint32(), C.c_uint32()
    a, b, c, d = C.c_void_p(), C.c_void_p(), C.c_void_p(), C.c_void_p()
    _check(lib().gf_read_spokesman_graph(str(path).encode(), C.byref(n), C.byref(P), C.byref(E), C.byref(a),
                                         C.byref(b), C.byref(c), C.byref(d)), "gf_read_spokesman_graph")
    cn = _take(a, P.value, np.uint32)
    total = int(cn.sum())
    return (cn, _take(b, P.value, np.uint32), _take(c, n.value, np.uint32),
            _take(d, P.value * total * E.value, np.uint32).reshape(P.value, total, E.value))


def recall(res: np.ndarray, gt: np.ndarray) -> float:
    """Mean over queries of |res ∩ gt| / |gt| (cal_recall_show_partition_multi_attrs,
    tools.cuh:456-544); an empty ground-truth row counts as 1; NO_ID entries are ignored."""
    res = np.asarray(res, np.uint32)
    gt = np.asarray(gt, np.uint32)
    total = 0.0
    for r, g in zip(res, gt):
        g = g[g != NO_ID]
        total += 1.0 if g.size == 0 else np.isin(g, r[r != NO_ID]).sum() / g.size
    return total / max(1, res.shape[0])


def version() -> str:
    return lib().gf_version().decode()


if os.environ.get("GARFIELD_B200_EAGER_LOAD"):
    lib()
