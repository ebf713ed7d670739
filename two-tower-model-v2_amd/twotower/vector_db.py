"""VectorDatabase on MI355X: drop-in for the reference's FAISS-backed class.

Reference: src/inference/vector_db.py (class VectorDatabase :10).  Same constructor,
methods, attributes, return types and error messages; the faiss.IndexFlatIP it wraps
(:48, :54, :160, :197) is replaced by ``FlatIPIndex``, a device-resident catalog whose
search is the fused HIP scan + top-k kernel (csrc/tt_scan.hip).

Numerics: build_index normalises rows on the GPU with numpy's exact float32 algorithm
(bit-identical to the reference's ``embeddings / (norms + 1e-8)``, :44-45); queries get the
same treatment (:152-153, :189-190); scores are exact float32 inner products (canonical
fma order), sorted descending, ties to the lower row.
"""
from __future__ import annotations

import collections
import ctypes
import json
import struct
import threading
from pathlib import Path
from typing import List, Optional, Tuple

import numpy as np
import torch

from . import _lib, kernels


class FlatIPIndex:
    """Device-resident exact inner-product index (the faiss.IndexFlatIP surface used by the
    reference: ``d``, ``ntotal``, ``add``, ``search``).

    Layout in HBM: ``xb`` = [capacity, tt_padded_dim(d)] float32, row-major, zero padded,
    rows L2-normalised by ``add`` exactly as the reference does before ``index.add``.
    """

    def __init__(self, d: int, device=None, row_base: int = 0, int8_image: bool = True):
        self.d = int(d)
        self.row_base = int(row_base)  # global id of local row 0 (catalog row shard)
        self.ep = _lib.padded_dim(self.d)
        self.scan_dim = _lib.scan_kernel_dim(self.d)  # d <= 768: the scan / bf16 filter
        self.device = device or _lib.device()
        self.xb = torch.zeros((0, self.ep), dtype=torch.float32, device=self.device)
        self.xb16 = torch.zeros((0, self.ep), dtype=torch.bfloat16, device=self.device)
        # (max ||x_r||, max ||x_r - bf16(x_r)||): the bf16 filter's error-bound inputs
        self._bounds_dev = torch.zeros(2, dtype=torch.float32, device=self.device)
        self.bounds = (0.0, 0.0)
        self.ntotal = 0
        # int8 image (codes, tile scales, bounds) for nq <= 8 searches (and a large batch's
        # sample level) at padded dim 384 / 768: built lazily, on the first search after an
        # add() (one O(n) pass per burst of adds, not per add); int8_image=False: never
        self.int8_image = bool(int8_image)
        self._i8 = None
        self._i8_stale = False
        self.version = 0  # bumped by every catalog / int8-image change (serving-slot caches)
        self._ws = _lib.StreamWorkspaces(4)  # search_device's workspace, one per HIP stream
        # host searches (the /retrieve path, FlatIPIndex.search_host): serving slots, each with
        # its own HIP stream, device query / output buffers, pinned host staging and filter
        # workspace, checked out by ONE call at a time and grown only when a call needs more,
        # so any k in 1..1000 per request (server.py:46) reuses them, and concurrent callers
        # run on separate streams; pooled per nq bucket (power of two), least recently used out
        self._slots = collections.OrderedDict()  # nq bucket -> [free _ServingSlot, ...]
        self.max_slots = 16
        self.allocations = 0  # serving-slot buffer (re)allocations: a test / ops counter
        # the slot pool and the catalog state are guarded by one lock, held only to check a
        # slot out / in and to read the catalog state: faiss' search is re-entrant, and the
        # reference's /retrieve may be called from several threads (server.py:212-244)
        self._lock = threading.RLock()
        self.coalesce = True  # batch concurrent single-query host searches (search_host)
        self._qlock = threading.Lock()
        self._queue = []
        self._leading = False
        self.coalesce_stats = [0, 0]  # [batches run, requests served] by the coalescing path

    def _append(self, rows: torch.Tensor, rows16: torch.Tensor) -> None:
        # bounds first: they only grow (max-combined), so a search snapshot taken between the
        # two updates pairs larger bounds with the old rows -- conservative, still exact
        if rows.shape[0]:  # build-time statistic over the new rows (max-combined)
            kernels.bf16_image_bounds(rows, rows16, self.d, out2=self._bounds_dev)
            self.bounds = tuple(self._bounds_dev.tolist())
        if self.ntotal:
            rows = torch.cat([self.xb[: self.ntotal], rows])
            rows16 = torch.cat([self.xb16[: self.ntotal], rows16])
        with self._lock:  # searches read (xb, xb16, ntotal, bounds, i8) as one snapshot
            self.xb, self.xb16 = rows, rows16
            self.ntotal = rows.shape[0]
            self._i8 = None
            self._i8_stale = self.int8_image and self.ep in kernels.I8_DIMS and self.ntotal > 0
            self.version += 1

    @property
    def i8(self):
        """The int8 image (codes, tile scales, (X, R, S)) of the current rows, or None; built
        here on first use after the rows changed."""
        if self._i8_stale:
            with self._lock:
                if self._i8_stale:
                    self._i8 = self._i8_image(self.xb[: self.ntotal])
                    self._i8_stale = False
                    self.version += 1
        return self._i8

    @i8.setter
    def i8(self, value) -> None:
        with self._lock:
            self._i8, self._i8_stale = value, False
            self.version += 1

    def _snapshot(self):
        """One consistent catalog state for a search: (xb, xb16, ntotal, bounds, i8, version)."""
        with self._lock:
            i8 = self.i8
            return (self.xb, self.xb16, self.ntotal, self.bounds, i8, self.version)

    def _i8_image(self, rows: torch.Tensor):
        """(codes, tile scales, bounds, tiled) of the int8 single pass for one-buyer searches
        (kernels.i8_image; padded dims 384 / 768), or None.  tiled = the MFMA-ordered copy of
        the codes (kernels.i8_tile) the register-fed stream reads at padded dim 384, else None."""
        if self.ep not in kernels.I8_DIMS or rows.shape[0] == 0:
            return None
        n = rows.shape[0]
        codes, scales, b3 = kernels.i8_image(rows, self.d)
        tiled = kernels.i8_tile(codes, n, self.d) if self.ep in kernels.I8T_DIMS else None
        return codes, scales, tuple(b3.tolist()), tiled

    def build_i8(self) -> None:
        """(Re)build the int8 image of the current rows (for an index whose xb was set
        directly rather than through add)."""
        self.i8 = self._i8_image(self.xb[: self.ntotal])

    # faiss-style add of ALREADY-normalised float32 rows (host or device)
    def add(self, x) -> None:
        if isinstance(x, np.ndarray) and not x.flags.writeable:
            x = np.array(x)  # torch refuses read-only numpy buffers (e.g. np.load mmap)
        x = torch.as_tensor(x, dtype=torch.float32)
        if x.dim() != 2 or x.shape[1] != self.d:
            raise ValueError(f"add: expected [n, {self.d}] float32")
        rows = torch.zeros((x.shape[0], self.ep), dtype=torch.float32, device=self.device)
        rows[:, : self.d].copy_(x, non_blocking=False)
        self._append(rows, rows.to(torch.bfloat16))

    def add_normalized_from(self, x) -> None:
        """Copy raw rows to the device and normalise there (x / (||x|| + 1e-8))."""
        x = torch.as_tensor(x)
        if x.dim() != 2 or x.shape[1] != self.d:
            raise ValueError(f"add: expected [n, {self.d}]")
        raw = torch.zeros((x.shape[0], self.ep), dtype=torch.float32, device=self.device)
        raw[:, : self.d].copy_(x.to(torch.float32))
        raw16 = torch.empty((x.shape[0], self.ep), dtype=torch.bfloat16, device=self.device)
        kernels.l2norm_rows(raw, self.d, _lib.TT_NORM_ADD_EPS, out=raw, out_bf16=raw16)
        self._append(raw, raw16)

    def search_device(self, q: torch.Tensor, k: int, method: str = "auto"):
        """q: [nq, ep] normalised device rows -> (scores [nq,k], labels [nq,k]) on device.

        method "auto": bf16 filter + exact f32 re-rank for k <= 128 (nq <= 8 at padded dim 384 /
        768: the int8 single pass), else exact f32 scores + radix select (k <= 1024); "f32" /
        "bf16" force the f32 scan / the bf16 filter.  All give bit-identical results."""
        if k < 1:
            raise RuntimeError("Error: 'k > 0' failed")  # faiss' own assertion text
        use_bf16 = method == "bf16" or (method == "auto" and k <= kernels.FILTER_KMAX)
        if k > kernels.SCAN_KMAX or not self.scan_dim:
            # faiss takes any k and any d: the generic exact path (GEMM scores + key top-k)
            return kernels.scan_topk_large(self.xb, self.ntotal, self.d, q, k,
                                           row_base=self.row_base)
        use_select = method == "auto" and k > kernels.FILTER_KMAX
        if use_bf16:
            need = kernels.filter_workspace_bytes(self.ntotal, self.d, q.shape[0], k)
        elif use_select:
            need = kernels.select_workspace_bytes(self.ntotal, q.shape[0], k)
        else:
            need = kernels.scan_workspace_bytes(self.ntotal, self.d, q.shape[0], k)
        with self._lock:  # the workspace cache is shared; the outputs are fresh per call
            ws = self._ws.get(need, self.device)
            i8 = self.i8 if use_bf16 and method == "auto" else None
            if kernels.i8_pass_ok(self.ntotal, self.d, q.shape[0], k, i8):
                codes, scales, b3, tiled = i8  # one-buyer calls: the int8 single pass
                return kernels.scan_topk_i8(self.xb, codes, scales, self.ntotal, self.d, q, k, b3,
                                            row_base=self.row_base, workspace=ws, tiled=tiled)
            if use_bf16:  # (a large batch runs its sample level on the int8 image, if any)
                return kernels.scan_topk_bf16(self.xb, self.xb16, self.ntotal, self.d, q, k,
                                              self.bounds, row_base=self.row_base, workspace=ws,
                                              i8=i8)
            if use_select:
                return kernels.scan_topk_select(self.xb, self.ntotal, self.d, q, k,
                                                row_base=self.row_base, workspace=ws)
            return kernels.scan_topk(self.xb, self.ntotal, self.d, q, k,
                                     row_base=self.row_base, workspace=ws)

    def _checkout(self, nq: int) -> "_ServingSlot":
        bucket = 1 << max(0, (nq - 1).bit_length())
        with self._lock:
            free = self._slots.get(bucket)
            if free:
                self._slots.move_to_end(bucket)
                return free.pop()
        return _ServingSlot(self, bucket)

    def _checkin(self, slot: "_ServingSlot") -> None:
        with self._lock:
            self._slots.setdefault(slot.bucket, []).append(slot)
            self._slots.move_to_end(slot.bucket)
            while sum(len(v) for v in self._slots.values()) > self.max_slots:
                b, v = next(iter(self._slots.items()))
                v.pop(0)
                if not v:
                    del self._slots[b]

    def search_host(self, x: np.ndarray, k: int, normalize: bool = False):
        """Host float32 [nq, d] queries -> host (D [nq,k] f32, I [nq,k] i64).  normalize=True
        first applies the reference's q/(||q||+1e-8) on the device (vector_db.py:152-153,
        189-190).  The serving path of VectorDatabase.retrieve / retrieve_batch: one H2D copy,
        the device normalisation, the search, one D2H copy, on a serving slot's own stream; the
        index lock is held only to check the slot out and to read the catalog state, not across
        the kernels or the stream synchronisation."""
        x = np.ascontiguousarray(x, dtype=np.float32)
        if x.ndim != 2 or x.shape[1] != self.d:
            raise ValueError(f"search: expected [nq, {self.d}] float32 queries")
        nq = x.shape[0]
        state = self._snapshot()  # one consistent catalog state for this call
        if nq == 0 or not (1 <= k <= state[2]):
            q = torch.zeros((nq, self.ep), dtype=torch.float32, device=self.device)
            q[:, : self.d] = torch.from_numpy(x).to(self.device)
            if normalize:
                kernels.l2norm_rows(q, self.d, _lib.TT_NORM_ADD_EPS, out=q)
            s, i = self.search_device(q, k)
            torch.cuda.current_stream().synchronize()
            return s.cpu().numpy(), i.cpu().numpy()
        if nq == 1 and self.coalesce:
            return self._coalesced(x, k, normalize)
        return self._run_batch(x, k, normalize, state)

    def _run_batch(self, x: np.ndarray, k: int, normalize: bool, state=None):
        if state is None:
            state = self._snapshot()
        slot = self._checkout(x.shape[0])
        try:
            return slot.run(x, k, normalize, state)
        finally:
            self._checkin(slot)

    # ---- request coalescing (concurrent one-query callers, e.g. /retrieve under a threaded
    # server): while one search is in flight, arriving single-query requests queue up; the
    # thread that leads runs the queue's requests as ONE batched search (up to COALESCE_MAX
    # queries of the same search path -- k <= 128: the bf16 filter, k <= 1024: scores + select
    # -- at the batch's largest k; a request gets the first k entries of its row, which are its
    # own exact top k: the lists are sorted by (score desc, row asc)), then hands the lead to
    # the next waiting thread.  One caller alone is a batch of one.
    COALESCE_MAX = 8
    # a leader whose own request is answered may go on serving the queue for up to LEAD_EXTRA
    # more batches before handing the lead over (no thread wake-up between two batches); 0:
    # measured slower at 2 and 4 (tools/bench_api.py: 4 threads 7.7k calls/s at 0, 7.2-7.4k
    # at 2 / 4 -- fewer requests per batch while the leader's own caller waits)
    LEAD_EXTRA = 0

    def _path(self, k: int) -> int:
        return 0 if k <= kernels.FILTER_KMAX else 1 if k <= kernels.SCAN_KMAX else 2

    def _coalesced(self, x: np.ndarray, k: int, normalize: bool):
        req = _Request(x, k, normalize)
        with self._qlock:
            self._queue.append(req)
            lead = not self._leading
            if lead:
                self._leading = True
        if not lead:
            req.event.wait()
            if not req.finished:  # handed the lead: this thread serves the queue now
                self._serve(req)
        else:
            self._serve(req)
        if req.error is not None:
            raise req.error
        return req.result

    def _serve(self, me: "_Request") -> None:
        extra = 0
        released = False  # the lead was cleared or handed over
        batch = []
        try:
            while True:
                with self._qlock:
                    head = self._queue[0]
                    cls = (head.normalize, self._path(head.k))
                    batch, rest = [], []
                    for r in self._queue:
                        if len(batch) < self.COALESCE_MAX and (r.normalize, self._path(r.k)) == cls:
                            batch.append(r)
                        else:
                            rest.append(r)
                    self._queue[:] = rest
                kk = max(r.k for r in batch)
                self.coalesce_stats[0] += 1
                self.coalesce_stats[1] += len(batch)
                try:
                    state = self._snapshot()
                    kk = min(kk, state[2])
                    xs = np.concatenate([r.x for r in batch]) if len(batch) > 1 else batch[0].x
                    s, i = self._run_batch(xs, kk, head.normalize, state)
                    for j, r in enumerate(batch):
                        r.result = (s[j:j + 1, :r.k], i[j:j + 1, :r.k])
                except Exception as e:  # every request of the failed batch sees the error
                    for r in batch:
                        r.error = e
                except BaseException:  # e.g. KeyboardInterrupt / SystemExit in this thread:
                    for r in batch:  # the batch's other callers fail, this one re-raises
                        if r is not me:
                            r.error = RuntimeError("search aborted: the thread running this "
                                                   "coalesced batch was interrupted")
                    raise
                finally:
                    for r in batch:
                        r.finished = True
                        if r is not me:
                            r.event.set()
                    batch = []
                with self._qlock:
                    if me.finished:
                        if not self._queue:
                            self._leading = False
                            released = True
                            return
                        if extra >= self.LEAD_EXTRA:  # hand the lead to the oldest waiting thread
                            self._queue[0].event.set()
                            released = True
                            return
                        extra += 1
        finally:
            if not released:  # left by an exception: never leave the lead held (later
                with self._qlock:  # single-query callers would wait for it forever)
                    me.finished = True
                    if self._queue:
                        self._queue[0].event.set()
                    else:
                        self._leading = False

    def search(self, x: np.ndarray, k: int):
        """faiss signature: float32 [nq, d] host queries -> (D [nq,k] f32, I [nq,k] i64) host."""
        return self.search_host(x, k, normalize=False)

    def reconstruct(self, i: int) -> np.ndarray:
        return self.xb[i, : self.d].cpu().numpy()


_HIP = None


def _hip():
    """The HIP runtime torch already loaded (ctypes): the serving slot's async copies."""
    global _HIP
    if _HIP is None:
        h = ctypes.CDLL("libamdhip64.so")
        h.hipMemcpyAsync.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t,
                                     ctypes.c_int, ctypes.c_void_p]
        h.hipMemcpy2DAsync.argtypes = [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p,
                                       ctypes.c_size_t, ctypes.c_size_t, ctypes.c_size_t,
                                       ctypes.c_int, ctypes.c_void_p]
        h.hipStreamSynchronize.argtypes = [ctypes.c_void_p]
        _HIP = h
    return _HIP


class _Request:
    """One queued single-query host search (FlatIPIndex._coalesced)."""

    __slots__ = ("x", "k", "normalize", "event", "result", "error", "finished")

    def __init__(self, x, k, normalize):
        self.x, self.k, self.normalize = x, k, normalize
        self.event = threading.Event()
        self.result = self.error = None
        self.finished = False


def _align256(nbytes: int) -> int:
    return (nbytes + 255) // 256 * 256


class _ServingSlot:
    """One in-flight host search's device state (FlatIPIndex.search_host): a HIP stream, the
    device query rows [bucket, ep], flat device / pinned host outputs, pinned query staging and
    one workspace for the bf16 filter (k <= 128) and the radix-select path (k <= 1024).  Every
    buffer grows to the largest (nq, k) it has served and is then reused, so a client mixing k
    values causes no allocation after warm-up.  Used by one call at a time (checked out)."""

    KCAP = 1024  # outputs sized for the /retrieve cap (k <= 1000, server.py:46) up front

    def __init__(self, index: FlatIPIndex, bucket: int):
        self.ix, self.bucket = index, bucket
        dev = index.device
        self.stream = torch.cuda.Stream(device=dev)
        pin = torch.cuda.is_available()
        self.q = torch.zeros((bucket, index.ep), dtype=torch.float32, device=dev)
        self.qh = torch.empty((bucket, index.d), dtype=torch.float32, pin_memory=pin)
        kc = self.KCAP if bucket <= 256 else 128
        self._outs(kc, pin)
        self.ws = torch.empty(0, dtype=torch.uint8, device=dev)
        self.ws_need = {}  # (n, nq, k, kind) -> workspace bytes (memoised size queries)
        self.synced = None  # catalog state this slot's stream is ordered after
        self.fn = _lib.lib().tt_scan_topk_bf16f32
        self.norm_fn = _lib.lib().tt_l2norm_rows_f32
        self.qh_np = self.qh.numpy()
        self.args = None  # (self.bound / self.args_key: _outs, akey -> bound C arguments)
        index.allocations += 1

    def _outs(self, kc: int, pin: bool) -> None:
        # scores and ids share one device and one pinned host buffer: the fast path lays a
        # call's [nq, k] scores and ids out back to back and copies them in ONE transfer
        dev = self.ix.device
        self.kc = kc
        self.bound = collections.OrderedDict()  # bound C arguments name the old buffers
        self.args_key = None
        m = self.bucket * kc
        o = _align256(4 * m)
        self.dout = torch.empty(o + 8 * m, dtype=torch.uint8, device=dev)
        self.hout = torch.empty(o + 8 * m, dtype=torch.uint8, pin_memory=pin)
        self.s, self.i = self.dout[:4 * m].view(torch.float32), self.dout[o:].view(torch.int64)
        self.sh, self.ih = self.hout[:4 * m].view(torch.float32), self.hout[o:].view(torch.int64)
        self.hout_np = self.hout.numpy()

    def _workspace(self, n: int, nq: int, k: int, kind: str) -> torch.Tensor:
        key = (n, nq, k, kind)
        need = self.ws_need.get(key)
        if need is None:
            need = (kernels.filter_workspace_bytes(n, self.ix.d, nq, k) if kind == "bf16"
                    else kernels.select_workspace_bytes(n, nq, k))
            if len(self.ws_need) > 256:
                self.ws_need.clear()
            self.ws_need[key] = need
        if self.ws.numel() < need:
            self.ws = torch.empty(need, dtype=torch.uint8, device=self.ix.device)
            self.ix.allocations += 1
            self.bound.clear()  # bound C arguments name the old workspace
            self.args_key = None
        return self.ws

    def _fast(self, x: np.ndarray, k: int, normalize: bool, state, skey):
        """The bf16-filter search (k <= 128, d <= 768) with no torch op per call: the staging
        copies, the normalisation, the search and the result copies are C calls on this slot's
        stream (hipMemcpy*Async, tt_l2norm_rows_f32, tt_scan_topk_bf16f32), the arguments bound
        once per (catalog state, nq, k); the stream synchronisation releases the GIL (ctypes),
        so other serving threads run their host work meanwhile.  ~25% less host time per call
        than the torch-op form."""
        ix = self.ix
        xb, xb16, n, bounds, i8, _ = state
        nq, d = x.shape
        ws = self._workspace(n, nq, k, "bf16")
        use8 = kernels.i8_pass_ok(n, d, nq, k, i8)
        # skey = the catalog state's version (rows, bounds and int8 image); the workspace and
        # output buffers are fixed while an entry lives (their reallocation clears self.bound)
        akey = (skey, nq, k, normalize, use8)
        o8 = _align256(nq * k * 4)  # this call's ids follow its scores
        if akey != self.args_key and akey in self.bound:  # coalesced batches vary nq
            self.fn, self.args, self.h2d, self.norm, self.d2h = self.bound[akey]
            self.bound.move_to_end(akey)
            self.args_key = akey
        if akey != self.args_key:  # the C arguments, bound once per (state, nq, k)
            vp = ctypes.c_void_p
            qp, st = vp(self.q.data_ptr()), vp(self.stream.cuda_stream)
            sp, ip = vp(self.dout.data_ptr()), vp(self.dout.data_ptr() + o8)
            if use8:  # the int8 single pass (one-buyer /retrieve calls, nq <= 8)
                codes, scales, (X, R, S), tiled = i8
                if tiled is not None:  # padded dim 384: the register-fed stream, tiled image
                    self.fn = _lib.lib().tt_scan_topk_i8t_f32
                    self.args = (
                        vp(xb.data_ptr()), vp(tiled.data_ptr()), vp(scales.data_ptr()), n, d,
                        xb.stride(0), ix.row_base, qp, nq, self.q.stride(0), k,
                        ctypes.c_float(X), ctypes.c_float(R), ctypes.c_float(S), sp, ip,
                        vp(ws.data_ptr()), ws.numel(), st, None, None)
                else:
                    self.fn = _lib.lib().tt_scan_topk_i8f32
                    self.args = (
                        vp(xb.data_ptr()), vp(codes.data_ptr()), vp(scales.data_ptr()), n, d,
                        xb.stride(0), codes.stride(0), ix.row_base, qp, nq, self.q.stride(0), k,
                        ctypes.c_float(X), ctypes.c_float(R), ctypes.c_float(S), sp, ip,
                        vp(ws.data_ptr()), ws.numel(), st, None, None)
            elif i8 is not None:  # a large batch's sample level on the int8 image (same results)
                codes, scales = i8[0], i8[1]
                self.fn = _lib.lib().tt_scan_topk_bf16f32_i8s
                self.args = (
                    vp(xb.data_ptr()), vp(xb16.data_ptr()), vp(codes.data_ptr()),
                    vp(scales.data_ptr()), n, d, xb.stride(0), codes.stride(0), ix.row_base, qp,
                    nq, self.q.stride(0), k, ctypes.c_float(bounds[0]),
                    ctypes.c_float(bounds[1]), sp, ip, vp(ws.data_ptr()), ws.numel(), st, None,
                    None)
            else:
                self.fn = _lib.lib().tt_scan_topk_bf16f32
                self.args = (
                    vp(xb.data_ptr()), vp(xb16.data_ptr()), n, d, xb.stride(0), ix.row_base, qp,
                    nq, self.q.stride(0), k, ctypes.c_float(bounds[0]),
                    ctypes.c_float(bounds[1]), sp, ip, vp(ws.data_ptr()), ws.numel(), st, None,
                    None)
            self.h2d = (qp, ctypes.c_size_t(self.q.stride(0) * 4), vp(self.qh.data_ptr()),
                        ctypes.c_size_t(d * 4), ctypes.c_size_t(d * 4), ctypes.c_size_t(nq), 1, st)
            self.norm = ((qp, nq, d, self.q.stride(0), qp, self.q.stride(0), None,
                          _lib.TT_NORM_ADD_EPS, st) if normalize else None)
            self.d2h = (vp(self.hout.data_ptr()), sp, ctypes.c_size_t(o8 + nq * k * 8), 2, st)
            self.args_key = akey
            self.bound[akey] = (self.fn, self.args, self.h2d, self.norm, self.d2h)
            if len(self.bound) > 8:
                self.bound.popitem(last=False)
        self.qh_np[:nq] = x
        hip = _hip()
        if hip.hipMemcpy2DAsync(*self.h2d):
            raise RuntimeError("hipMemcpy2DAsync (queries) failed")
        if self.norm is not None:
            _lib.check(self.norm_fn(*self.norm), "tt_l2norm_rows_f32")
        rc = self.fn(*self.args)
        if rc:
            _lib.check(rc, "tt_scan_topk_i8f32" if use8 else "tt_scan_topk_bf16f32[_i8s]")
        if hip.hipMemcpyAsync(*self.d2h):
            raise RuntimeError("hipMemcpyAsync (results) failed")
        if hip.hipStreamSynchronize(self.args[-3]):
            raise RuntimeError("hipStreamSynchronize failed")
        h = self.hout_np
        return (h[: nq * k * 4].view(np.float32).reshape(nq, k).copy(),
                h[o8:o8 + nq * k * 8].view(np.int64).reshape(nq, k).copy())

    def run(self, x: np.ndarray, k: int, normalize: bool, state):
        ix = self.ix
        xb, xb16, n, _, _, version = state
        nq, d = x.shape
        if k > self.kc:
            self._outs(k, torch.cuda.is_available())
            ix.allocations += 1
        q = self.q[:nq]
        # ordered after the caller's stream once per catalog state (an add() whose kernels may
        # still run there); later calls on the same state need no cross-stream wait
        skey = version
        if skey != self.synced:
            self.stream.wait_stream(torch.cuda.current_stream())
            self.synced = skey
        if ix.scan_dim and k <= kernels.FILTER_KMAX and k <= self.kc:
            return self._fast(x, k, normalize, state, skey)
        with torch.cuda.stream(self.stream):
            self.qh[:nq].numpy()[...] = x
            q[:, :d].copy_(self.qh[:nq], non_blocking=True)
            if normalize:
                kernels.l2norm_rows(q, d, _lib.TT_NORM_ADD_EPS, out=q)
            s, i = self.s[: nq * k].view(nq, k), self.i[: nq * k].view(nq, k)
            # (k <= 128 at a scan dim always took _fast above: outputs grow to k first)
            if ix.scan_dim and k <= kernels.SCAN_KMAX:
                ws = self._workspace(n, nq, k, "select")
                kernels.scan_topk_select(xb, n, d, q, k, row_base=ix.row_base, workspace=ws,
                                         out=(s, i))
            else:  # k > 1024 or d > 768: the generic exact path (allocates; not the serving k)
                s2, i2 = kernels.scan_topk_large(xb, n, d, q, k, row_base=ix.row_base)
                s.copy_(s2)
                i.copy_(i2)
            sh, ih = self.sh[: nq * k], self.ih[: nq * k]
            sh.copy_(s.view(-1), non_blocking=True)
            ih.copy_(i.view(-1), non_blocking=True)
        self.stream.synchronize()
        return sh.numpy().reshape(nq, k).copy(), ih.numpy().reshape(nq, k).copy()


# ------------------------------------------------------------------ index file format
# Best-effort faiss IndexFlatIP layout (fourcc "IxFI", header, codes).  The real faiss
# reader is absent offline, so compatibility with faiss.read_index is UNPINNED;
# our own load_index reads exactly what save_index writes.
_FOURCC = b"IxFI"


def write_flat_ip(index: FlatIPIndex, path: str) -> None:
    xb = index.xb[: index.ntotal, : index.d].contiguous().cpu().numpy().astype("<f4")
    with open(path, "wb") as f:
        f.write(_FOURCC)
        f.write(struct.pack("<iqqqBi", index.d, index.ntotal, 1 << 20, 1 << 20, 1, 0))
        f.write(struct.pack("<Q", xb.size))
        f.write(xb.tobytes())


def read_flat_ip(path: str, device=None) -> FlatIPIndex:
    with open(path, "rb") as f:
        if f.read(4) != _FOURCC:
            raise RuntimeError(f"{path}: not an IndexFlatIP file")
        d, ntotal, _, _, _, _ = struct.unpack("<iqqqBi", f.read(struct.calcsize("<iqqqBi")))
        (size,) = struct.unpack("<Q", f.read(8))
        xb = np.frombuffer(f.read(size * 4), dtype="<f4").reshape(ntotal, d)
    index = FlatIPIndex(d, device)
    index.add(xb)
    return index


class VectorDatabase:
    """Mirror of reference ``VectorDatabase`` (src/inference/vector_db.py:10-233)."""

    def __init__(self, embedding_dim: int = 384):
        self.embedding_dim = embedding_dim
        self.index: Optional[FlatIPIndex] = None
        self.product_ids = None
        self.id_to_index = None
        self.index_to_id = None

    def build_index(self, embeddings: np.ndarray, product_ids: List[str]):
        """reference :25-61"""
        n_products, dim = embeddings.shape
        if dim != self.embedding_dim:
            raise ValueError(
                f"Embedding dimension mismatch: expected {self.embedding_dim}, got {dim}")
        index = FlatIPIndex(self.embedding_dim)
        # reference normalises in the input dtype (:44-45) then casts to f32 (:51); for the
        # float32 inputs the pipeline produces this is the GPU numpy-exact normalisation.
        if np.asarray(embeddings).dtype == np.float32:
            index.add_normalized_from(torch.from_numpy(np.ascontiguousarray(embeddings)))
        else:
            norms = np.linalg.norm(embeddings, axis=1, keepdims=True)
            index.add((embeddings / (norms + 1e-8)).astype(np.float32))
        self.index = index
        self.product_ids = product_ids
        self.id_to_index = {pid: idx for idx, pid in enumerate(product_ids)}
        self.index_to_id = {idx: pid for idx, pid in enumerate(product_ids)}
        print(f"Built FAISS index with {n_products} products")

    def load_index(self, index_path: str, product_ids_path: Optional[str] = None,
                   mapping_path: Optional[str] = None):
        """reference :63-98"""
        self.index = read_flat_ip(index_path)
        if product_ids_path:
            product_ids_array = np.load(product_ids_path, allow_pickle=False)
            self.product_ids = product_ids_array.tolist()
        else:
            n_products = self.index.ntotal
            self.product_ids = [f"product_{i}" for i in range(n_products)]
        if mapping_path and Path(mapping_path).exists():
            with open(mapping_path, "r", encoding="utf-8") as f:
                self.id_to_index = json.load(f)
            self.index_to_id = {v: k for k, v in self.id_to_index.items()}
        else:
            self.id_to_index = {pid: idx for idx, pid in enumerate(self.product_ids)}
            self.index_to_id = {idx: pid for idx, pid in enumerate(self.product_ids)}
        print(f"Loaded FAISS index with {len(self.product_ids)} products")

    def save_index(self, index_path: str, product_ids_path: Optional[str] = None,
                   mapping_path: Optional[str] = None):
        """reference :100-128"""
        if self.index is None:
            raise ValueError("Index not built. Call build_index() first.")
        write_flat_ip(self.index, index_path)
        if product_ids_path:
            np.save(product_ids_path, np.array(self.product_ids))
        if mapping_path and self.id_to_index:
            with open(mapping_path, "w", encoding="utf-8") as f:
                json.dump(self.id_to_index, f, ensure_ascii=False, indent=2)
        print(f"Saved FAISS index to {index_path}")

    # -------------------------------------------------------------- device fast path
    def normalize_queries(self, q: torch.Tensor) -> torch.Tensor:
        """Device queries [nq, >=d] -> [nq, ep] rows q/(||q||+1e-8) (reference :152-153)."""
        out = torch.empty((q.shape[0], self.index.ep), dtype=torch.float32, device=q.device)
        return kernels.l2norm_rows(q, self.embedding_dim, _lib.TT_NORM_ADD_EPS, out=out)

    def search(self, query_embeddings: torch.Tensor, k: int = 10, normalized: bool = False):
        """Device-level retrieve_batch: returns (scores [nq,k], rows [nq,k]) device tensors.
        ``normalized=True`` skips the q/(||q||+1e-8) step (rows already [nq, ep], padded)."""
        if self.index is None:
            raise ValueError("Index not built. Call build_index() or load_index() first.")
        k = min(k, self.index.ntotal)
        q = query_embeddings if normalized else self.normalize_queries(query_embeddings)
        return self.index.search_device(q, k)

    def _search_host(self, query_embeddings: np.ndarray, k: int):
        """Host queries -> host (scores, rows) through the index's prepared serving path
        (FlatIPIndex.search_host: one H2D copy, the device normalisation, the search, one D2H
        copy per call)."""
        x = np.ascontiguousarray(query_embeddings)
        k = min(k, self.index.ntotal)  # reference :159 / :196
        if x.dtype != np.float32:
            # reference normalises in the input dtype, then casts (:189-193): do the same
            norms = np.linalg.norm(x, axis=1, keepdims=True)
            return self.index.search_host((x / (norms + 1e-8)).astype(np.float32), k)
        return self.index.search_host(x, k, normalize=True)

    def _to_results(self, scores: np.ndarray, indices: np.ndarray):
        out = []
        n = len(self.product_ids)
        ids = self.product_ids
        # Python ints / floats first (.tolist()): per-element numpy scalars made a k = 1000
        # response cost ~0.25 ms of host time; float(np.float32 x) == the list's float of x
        for query_scores, query_indices in zip(scores.tolist(), indices.tolist()):
            if query_indices and max(query_indices) < n:  # the common case: one C-level pass
                out.append(list(zip(map(ids.__getitem__, query_indices), query_scores)))
            else:
                out.append([(ids[idx], score) for idx, score in zip(query_indices, query_scores)
                            if idx < n])  # reference :165 (-1 would pass, as in the reference)
        return out

    def retrieve(self, query_embedding: np.ndarray, k: int = 10) -> List[Tuple[str, float]]:
        """reference :130-169"""
        if self.index is None:
            raise ValueError("Index not built. Call build_index() or load_index() first.")
        if query_embedding.ndim == 1:
            query_embedding = query_embedding.reshape(1, -1)
        return self._to_results(*self._search_host(query_embedding, k))[0]

    def retrieve_batch(self, query_embeddings: np.ndarray,
                       k: int = 10) -> List[List[Tuple[str, float]]]:
        """reference :171-209"""
        if self.index is None:
            raise ValueError("Index not built. Call build_index() or load_index() first.")
        return self._to_results(*self._search_host(query_embeddings, k))

    # -------------------------------------------------------------- additions
    def log_probs(self, query_embeddings: np.ndarray, product_ids: Optional[List[str]] = None,
                  temperature: float = 0.07, top: int = 0):
        """Log-probabilities under softmax over the whole catalog of cosine / temperature (the
        distribution InfoNCE trains towards): for queries [nq, d] and one product id each
        (None: none) -> (log_prob [nq] float32, NaN for an id that is not in the catalog; entropy
        [nq] float32; per query the ``top`` (<= 32) most probable products as (id, log_prob))."""
        if self.index is None:
            raise ValueError("Index not built. Call build_index() or load_index() first.")
        q = np.asarray(query_embeddings)
        q = q.reshape(1, -1) if q.ndim == 1 else q
        if q.shape[1] != self.embedding_dim:
            raise ValueError(f"Embedding dimension mismatch: expected {self.embedding_dim}, got "
                             f"{q.shape[1]}")
        if product_ids is not None and len(product_ids) != len(q):
            raise ValueError(f"log_probs: {len(q)} queries, {len(product_ids)} product ids")
        if len(q) == 0:
            none = np.zeros(0, np.float32)
            return none if product_ids is not None else None, none, []
        from .losses import catalog_log_probs

        index, rows_of = self.index, self.id_to_index
        with index._lock:  # one state of the catalog
            xb, n = index.xb, index.ntotal
        with _lib.on_device(xb):
            dev = xb.device
            rows = self.normalize_queries(
                torch.from_numpy(np.ascontiguousarray(q, dtype=np.float32)).to(dev))
            ids = None
            if product_ids is not None:
                at = [rows_of.get(p, -1) for p in product_ids]
                ids = torch.tensor([i if 0 <= i < n else -1 for i in at], dtype=torch.int64,
                                   device=dev)
            r = catalog_log_probs(rows, xb[:n], ids, temperature, entropy=True, top=min(top, n))
            lp = None
            if ids is not None:
                lp = torch.where(ids >= 0, r.log_prob,
                                 torch.full_like(r.log_prob, float("nan"))).cpu().numpy()
            alt = [[] for _ in range(len(q))]
            if top:
                alt = self._to_results(r.top_log_probs.cpu().numpy(), r.top_ids.cpu().numpy())
            return lp, r.entropy.cpu().numpy(), alt

    def get_embedding(self, product_id: str) -> Optional[np.ndarray]:
        """reference :211-231 (always None there: FAISS cannot reconstruct in that code)."""
        if self.index is None or self.id_to_index is None:
            return None
        if product_id not in self.id_to_index:
            return None
        return None
