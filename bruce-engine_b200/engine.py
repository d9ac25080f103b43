"""Host-side mirror of the reference engine's attention call surface, over the C ABI.

Method names follow the reference's launches (engine/src/bruce.cu): `qkv_prep_store` is the
quantise-and-store half of k_qkv_prep / k_qkv_prep_fast / k_qkv_prep_fast_ms (:644, :1732, :1835),
`launch_attn_m` is launch_attn_m + the merge (:3942, :928, :1999), `launch_attn_ms` is
launch_attn_ms + the merge (:4158), `attn_combine` is k_attn_combine (:992).  Arguments keep the
reference's meaning: device buffers owned by the caller, device-resident positions, `part` scratch.

torch is used only for device memory and streams; every computation is a call into libbattn.so.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import capi
from .layout import F16, Geom


def _ptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


class AttnEngine:
    """One attention context (geometry + device), the replacement of the reference's lazily-set
    kernel attributes and its g_kv_nctx symbol (bruce.cu:65, 3948-3955, 5482)."""

    def __init__(self, geom: Geom, device: int = 0):
        if not torch.cuda.is_available():
            raise RuntimeError("AttnEngine needs a CUDA device (sm_100a); there is no CPU path")
        self.lib = capi.load()
        self.geom = geom
        self.device = torch.device("cuda", device)
        cg = capi.CGeom(geom.n_head, geom.n_kv, geom.head_dim, geom.window, geom.slot_ctx,
                        geom.n_slots, geom.q_dtype, geom.out_dtype, geom.softmax_scale)
        h = C.c_void_p()
        rc = self.lib.battn_init(C.byref(cg), device, C.byref(h))
        if rc:
            raise capi.BattnError("battn_init", rc, self.lib.battn_last_cuda_error(None))
        self.h = h
        self._ws_need = {}
        self.q_torch = torch.float16 if geom.q_dtype == F16 else torch.float32
        self.out_torch = torch.float16 if geom.out_dtype == F16 else torch.float32

    def close(self):
        if getattr(self, "h", None):
            self.lib.battn_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # ---- sizes and allocation (alloc_buffers, bruce.cu:5460-5507, 5564) --------------------------
    def _check(self, fn: str, rc: int):
        if rc:
            raise capi.BattnError(fn, rc, self.lib.battn_last_cuda_error(self.h))

    def kv_layer_bytes(self, is_swa: bool) -> int:
        n = C.c_size_t()
        self._check("battn_kv_layer_bytes", self.lib.battn_kv_layer_bytes(self.h, int(is_swa), C.byref(n)))
        return n.value

    def alloc_kv_layer(self, is_swa: bool, fill: int | None = None):
        """One layer's K and V buffers for all slots."""
        n = self.kv_layer_bytes(is_swa)
        mk = (lambda: torch.empty(n, dtype=torch.uint8, device=self.device)) if fill is None else \
             (lambda: torch.full((n,), fill, dtype=torch.uint8, device=self.device))
        return mk(), mk()

    def workspace_bytes(self, n_seq: int, rows: int) -> int:
        n = C.c_size_t()
        self._check("battn_workspace_bytes", self.lib.battn_workspace_bytes(self.h, n_seq, rows, C.byref(n)))
        return n.value

    def exact_workspace_bytes(self, n_seq: int, rows: int, nsplit: int) -> int:
        n = C.c_size_t()
        self._check("battn_exact_workspace_bytes",
                    self.lib.battn_exact_workspace_bytes(self.h, n_seq, rows, nsplit, C.byref(n)))
        return n.value

    def alloc_part(self, n_seq: int, rows: int) -> torch.Tensor:
        """The split-K scratch (`part`, bruce.cu:5564)."""
        return torch.empty(self.workspace_bytes(n_seq, rows), dtype=torch.uint8, device=self.device)

    @staticmethod
    def _stream():
        return C.c_void_p(torch.cuda.current_stream().cuda_stream)

    # ---- KV append ---------------------------------------------------------------------------------
    def qkv_prep_store(self, k, v, kvk, kvv, pos, kslot=None, act=None, rows: int = 1, is_swa: bool = False):
        """k, v: fp32 [n_seq][rows][n_kv][head_dim]; pos/kslot/act: int32 device tensors."""
        n_seq = pos.numel()
        self._check("battn_kv_append", self.lib.battn_kv_append(
            self.h, _ptr(k), _ptr(v), _ptr(kvk), _ptr(kvv), _ptr(pos), _ptr(kslot), _ptr(act),
            n_seq, rows, int(is_swa), self._stream()))

    def kv_copy_prefix(self, kvk, kvv, src_slot: int, dst_slot: int, n_pos: int, is_swa: bool = False, sinks=None, score=None):
        """Prefix sharing between slots: the first n_pos cached positions of src_slot copied into dst_slot, and with them what
        the layer keeps beside its records: a window layer's sink buffers (`sinks`, a descriptor over buffers of all slots) or a
        full layer's accumulated scores (`score` [slot][n_kv][slot_ctx])."""
        g = self.geom
        if sinks is not None and (not is_swa or getattr(sinks, "slots", 0) < g.n_slots):
            raise ValueError("kv_copy_prefix: sinks are a window layer's, over buffers of all slots made by sinks() or alloc_sinks()")
        if score is not None:
            if is_swa:
                raise ValueError("kv_copy_prefix: scores are a full layer's")
            self._dev("score", score, torch.float32, g.n_slots * g.n_kv * g.slot_ctx)
        self._check("battn_kv_copy_prefix", self.lib.battn_kv_copy_prefix(
            self.h, _ptr(kvk), _ptr(kvv), src_slot, dst_slot, n_pos, int(is_swa), self._stream()))
        beside = [] if score is None else [(score, (g.slot_ctx,), n_pos)]
        if sinks is not None:
            beside += [(b, (sinks.cap, g.rec), min(n_pos, sinks.cap)) for b in sinks.bufs]
        for buf, shape, n in beside:
            x = buf.reshape(-1)[:g.n_slots * g.n_kv * math.prod(shape)].view(g.n_slots, g.n_kv, *shape)
            x[dst_slot, :, :n].copy_(x[src_slot, :, :n])

    def qkv_prep(self, q_out, q, k, v, sqk, cs, sn, kvk, kvv, pos, kslot=None, act=None, rows: int = 1,
                 is_swa: bool = False, theta_sel: int = 1):
        """The whole k_qkv_prep_fast / k_qkv_prep_fast_ms step (bruce.cu:1732-1812, 1835-1918): L2 scale + RoPE
        (+ sqk on q) and the quantised append, one launch.  q_out: the geometry's q dtype (fp32 may be q itself)."""
        n_seq = pos.numel()
        self._check("battn_qkv_prep", self.lib.battn_qkv_prep(
            self.h, _ptr(q_out), _ptr(q), _ptr(k), _ptr(v), _ptr(sqk), _ptr(cs), _ptr(sn), int(theta_sel),
            _ptr(kvk), _ptr(kvv), _ptr(pos), _ptr(kslot), _ptr(act), n_seq, rows, int(is_swa), self._stream()))

    def rope_tables(self, cs, sn, pos, rows: int = 1):
        """k_rope_tables_rows / _ms (bruce.cu:1641-1654, 1821-1833): cs, sn fp32 [n_seq*rows][head_dim]."""
        self._check("battn_rope_tables", self.lib.battn_rope_tables(
            self.h, _ptr(cs), _ptr(sn), _ptr(pos), pos.numel(), rows, self._stream()))

    # ---- attention ---------------------------------------------------------------------------------
    def launch_attn_m(self, out, q, kvk, kvv, pos, part, rows: int, is_swa: bool = False):
        """Single-sequence attention: rows == 1 decode, 2..8 speculative verify, > 8 prompt chunk
        (the dispatch of launch_attn_m, bruce.cu:3942-4122), merge included."""
        st = self._stream()
        if rows == 1:
            rc = self.lib.battn_decode(self.h, _ptr(out), _ptr(q), _ptr(kvk), _ptr(kvv), _ptr(pos), None, None,
                                       _ptr(part), 1, int(is_swa), st)
            self._check("battn_decode", rc)
        elif rows <= 8 and rows * self.geom.group <= 32:
            rc = self.lib.battn_verify(self.h, _ptr(out), _ptr(q), _ptr(kvk), _ptr(kvv), _ptr(pos), None, None,
                                       _ptr(part), rows, 1, int(is_swa), st)
            self._check("battn_verify", rc)
        else:
            rc = self.lib.battn_prefill(self.h, _ptr(out), _ptr(q), _ptr(kvk), _ptr(kvv), _ptr(pos), _ptr(part),
                                        rows, int(is_swa), st)
            self._check("battn_prefill", rc)

    def launch_attn_ms(self, out, q, kvk, kvv, pos, kslot, act, part, rows: int, is_swa: bool = False,
                       rows_per_seq: int = 1):
        """Multi-slot attention: `rows` independent sequences (launch_attn_ms, bruce.cu:4158-4177);
        rows_per_seq > 1 runs a batched speculative verify."""
        st = self._stream()
        if rows_per_seq == 1:
            rc = self.lib.battn_decode(self.h, _ptr(out), _ptr(q), _ptr(kvk), _ptr(kvv), _ptr(pos), _ptr(kslot),
                                       _ptr(act), _ptr(part), rows, int(is_swa), st)
            self._check("battn_decode", rc)
        else:
            rc = self.lib.battn_verify(self.h, _ptr(out), _ptr(q), _ptr(kvk), _ptr(kvv), _ptr(pos), _ptr(kslot),
                                       _ptr(act), _ptr(part), rows_per_seq, rows, int(is_swa), st)
            self._check("battn_verify", rc)

    def decode_append(self, out, q, k, v, kvk, kvv, pos, part, kslot=None, act=None, is_swa: bool = False):
        """One row per sequence: append k, v ([n_seq][n_kv][head_dim] fp32) at pos[i] and attend, the append done by
        the decode kernel itself (battn_decode_append)."""
        rc = self.lib.battn_decode_append(self.h, _ptr(out), _ptr(q), _ptr(k), _ptr(v), _ptr(kvk), _ptr(kvv), _ptr(pos),
                                          _ptr(kslot), _ptr(act), _ptr(part), pos.numel(), int(is_swa), self._stream())
        self._check("battn_decode_append", rc)

    def qkv_decode(self, out, q, k, v, sqk, cs, sn, kvk, kvv, pos, part, kslot=None, act=None, is_swa: bool = False,
                   theta_sel: int = 1):
        """One row per sequence: the QKV prologue (as qkv_prep), the append and the attention in one call whose decode
        kernel does all three (battn_qkv_decode); q, k, v are the raw fp32 rows."""
        rc = self.lib.battn_qkv_decode(self.h, _ptr(out), _ptr(q), _ptr(k), _ptr(v), _ptr(sqk), _ptr(cs), _ptr(sn),
                                       int(theta_sel), _ptr(kvk), _ptr(kvv), _ptr(pos), _ptr(kslot), _ptr(act),
                                       _ptr(part), pos.numel(), int(is_swa), self._stream())
        self._check("battn_qkv_decode", rc)

    def decode_append_paged(self, out, q, k, v, pages, pos, part, ktab=None, act=None):
        rc = self.lib.battn_decode_append_paged(self.h, _ptr(out), _ptr(q), _ptr(k), _ptr(v), C.byref(pages), _ptr(pos),
                                                _ptr(ktab), _ptr(act), _ptr(part), pos.numel(), self._stream())
        self._check("battn_decode_append_paged", rc)

    def qkv_decode_paged(self, out, q, k, v, sqk, cs, sn, pages, pos, part, ktab=None, act=None, theta_sel: int = 1):
        rc = self.lib.battn_qkv_decode_paged(self.h, _ptr(out), _ptr(q), _ptr(k), _ptr(v), _ptr(sqk), _ptr(cs), _ptr(sn),
                                             int(theta_sel), C.byref(pages), _ptr(pos), _ptr(ktab), _ptr(act), _ptr(part),
                                             pos.numel(), self._stream())
        self._check("battn_qkv_decode_paged", rc)

    def set_early_kv_stream(self, enable: bool):
        """Whether decode calls stream the cache tiles below their first position before the preceding kernel of
        the stream has finished (battn_set_early_kv_stream; off by default: the host must not let a kernel that
        writes positions or older cache rows directly precede an attention call)."""
        self._check("battn_set_early_kv_stream", self.lib.battn_set_early_kv_stream(self.h, int(enable)))

    def decode_noalloc(self, out, q, kvk, kvv, pos, kslot=None, act=None, is_swa: bool = False):
        """Decode attention without a caller-provided `part` buffer: the scratch is a fixed array
        inside the library (for hosts that cannot allocate device memory while serving)."""
        rc = self.lib.battn_decode_noalloc(self.h, _ptr(out), _ptr(q), _ptr(kvk), _ptr(kvv), _ptr(pos),
                                           _ptr(kslot), _ptr(act), pos.numel(), int(is_swa), self._stream())
        self._check("battn_decode_noalloc", rc)

    def attn_exact(self, out, q, kvk, kvv, pos, part, n_seq: int, rows: int, nsplit: int, is_swa: bool = False,
                   kslot=None, act=None):
        """The exact fp32 path (k_attn / k_attn_rows / k_attn_m + k_attn_combine_rows)."""
        rc = self.lib.battn_attend_exact(self.h, _ptr(out), _ptr(q), _ptr(kvk), _ptr(kvv), _ptr(pos), _ptr(kslot),
                                         _ptr(act), _ptr(part), n_seq, rows, nsplit, int(is_swa), self._stream())
        self._check("battn_attend_exact", rc)

    def attn_partials(self, rec, q, kvk, kvv, pos, part, rows: int = 1, batch: int = 1, is_swa: bool = False,
                      kslot=None, act=None):
        """Split records (o, m, l) instead of the normalised output (bruce.cu:781-783)."""
        rc = self.lib.battn_partials(self.h, _ptr(rec), _ptr(q), _ptr(kvk), _ptr(kvv), _ptr(pos), _ptr(kslot),
                                     _ptr(act), _ptr(part), rows, batch, int(is_swa), self._stream())
        self._check("battn_partials", rc)

    def attn_combine(self, out, parts, n_parts: int, n_rows: int):
        """k_attn_combine over records gathered from several devices (bruce.cu:992-1007)."""
        rc = self.lib.battn_merge(self.h, _ptr(out), _ptr(parts), n_parts, n_rows, self._stream())
        self._check("battn_merge", rc)

    # ---- paged cache of a full-causal layer ------------------------------------------------------------
    def alloc_pages(self, n_pages: int, page_len: int, table: torch.Tensor, fill: int | None = None):
        """A pool of `n_pages` pages of `page_len` positions (K and V) and its `battn_pages` descriptor; `table` is
        the int32 device tensor [n_tables][max_pages] the kernels read the page numbers from (the host may edit it
        between launches).  Returns (descriptor, pool_k, pool_v); keep the tensors alive with the descriptor."""
        n = C.c_size_t()
        self._check("battn_pages_pool_bytes", self.lib.battn_pages_pool_bytes(self.h, n_pages, page_len, C.byref(n)))
        mk = (lambda: torch.empty(n.value, dtype=torch.uint8, device=self.device)) if fill is None else \
             (lambda: torch.full((n.value,), fill, dtype=torch.uint8, device=self.device))
        pk, pv = mk(), mk()
        assert table.dtype == torch.int32 and table.dim() == 2 and table.is_contiguous()
        desc = capi.CPages(pk.data_ptr(), pv.data_ptr(), table.data_ptr(), n_pages, table.shape[0], table.shape[1],
                           page_len)
        return desc, pk, pv

    def pages_copy(self, pages, from_page: int, to_page: int):
        """Copy on write: one physical page's K and V records into another page."""
        self._check("battn_pages_copy", self.lib.battn_pages_copy(self.h, C.byref(pages), from_page, to_page,
                                                                  self._stream()))

    def kv_append_paged(self, pages, k, v, pos, ktab=None, act=None, rows: int = 1):
        self._check("battn_kv_append_paged", self.lib.battn_kv_append_paged(
            self.h, C.byref(pages), _ptr(k), _ptr(v), _ptr(pos), _ptr(ktab), _ptr(act), pos.numel(), rows,
            self._stream()))

    def qkv_prep_paged(self, q_out, q, k, v, sqk, cs, sn, pages, pos, ktab=None, act=None, rows: int = 1,
                       theta_sel: int = 1):
        """The fused prologue (qkv_prep) storing its K/V rows into a paged cache."""
        self._check("battn_qkv_prep_paged", self.lib.battn_qkv_prep_paged(
            self.h, _ptr(q_out), _ptr(q), _ptr(k), _ptr(v), _ptr(sqk), _ptr(cs), _ptr(sn), int(theta_sel),
            C.byref(pages), _ptr(pos), _ptr(ktab), _ptr(act), pos.numel(), rows, self._stream()))

    def attn_paged(self, out, q, pages, pos, part, rows: int = 1, ktab=None, act=None, table_row: int = 0):
        """Attention over a paged cache: one row per sequence (decode), 2..8 rows (verify) or a prompt chunk of the
        sequence with table row `table_row`; the dispatch of launch_attn_m / launch_attn_ms."""
        st = self._stream()
        n_seq = pos.numel()
        if rows == 1:
            rc = self.lib.battn_decode_paged(self.h, _ptr(out), _ptr(q), C.byref(pages), _ptr(pos), _ptr(ktab),
                                             _ptr(act), _ptr(part), n_seq, st)
            self._check("battn_decode_paged", rc)
        elif rows * self.geom.group <= 32:
            rc = self.lib.battn_verify_paged(self.h, _ptr(out), _ptr(q), C.byref(pages), _ptr(pos), _ptr(ktab),
                                             _ptr(act), _ptr(part), rows, n_seq, st)
            self._check("battn_verify_paged", rc)
        else:
            rc = self.lib.battn_prefill_paged(self.h, _ptr(out), _ptr(q), C.byref(pages), table_row, _ptr(pos),
                                              _ptr(part), rows, st)
            self._check("battn_prefill_paged", rc)

    def attn_exact_paged(self, out, q, pages, pos, part, n_seq: int, rows: int, nsplit: int, ktab=None, act=None):
        rc = self.lib.battn_attend_exact_paged(self.h, _ptr(out), _ptr(q), C.byref(pages), _ptr(pos), _ptr(ktab),
                                               _ptr(act), _ptr(part), n_seq, rows, nsplit, self._stream())
        self._check("battn_attend_exact_paged", rc)

    # ---- sliding window with sinks ---------------------------------------------------------------------
    def _dev(self, name: str, t, dtype, n: int = 0):
        """The pointer of a device tensor the new calls read or write, after the checks a raw pointer cannot have."""
        if t.dtype is dtype and t.get_device() == self.device.index and t.is_contiguous() and t.numel() >= n:
            return t.data_ptr()
        raise ValueError(f"{name}: need a contiguous {dtype} tensor of at least {n} elements on {self.device}, "
                         f"got {t.dtype} {tuple(t.shape)} on {t.device}")

    def _seqs(self, pos, sel, act):
        """Pointers of the per-sequence arrays: positions, partitions (or table rows) and activity."""
        n = pos.numel()
        return (self._dev("pos", pos, torch.int32), None if sel is None else self._dev("kslot", sel, torch.int32, n),
                None if act is None else self._dev("act", act, torch.int32, n), n)

    def _cache_ptrs(self, kvk, kvv, is_swa: bool, layer: bool):
        """A layer's (or, for the single-sequence form, one slot's) K and V buffers."""
        g = self.geom
        n = (g.n_slots if layer else 1) * g.pstride(is_swa) * g.n_kv * g.rec
        return self._dev("kvk", kvk, torch.uint8, n), self._dev("kvv", kvv, torch.uint8, n)

    def _stream_here(self):
        # the handle of torch.cuda.current_stream(self.device) without building the Python object (2 us of a 10 us call)
        return torch._C._cuda_getCurrentRawStream(self.device.index)

    def alloc_sinks(self, n_sink: int):
        """Sink buffers of one window layer for all slots; returns (descriptor, k, v): keep the tensors alive with it."""
        cap, n = max(128, -(-n_sink // 128) * 128), C.c_size_t()
        self._check("battn_sinks_bytes", self.lib.battn_sinks_bytes(self.h, cap, C.byref(n)))
        k, v = (torch.zeros(n.value, dtype=torch.uint8, device=self.device) for _ in range(2))
        return self.sinks(n_sink, k, v), k, v

    def sinks(self, n_sink: int, k=None, v=None, cap: int | None = None):
        """The descriptor of `n_sink` sinks: over the buffers of a ring layer, without for a cache that keeps its first
        positions.  The buffers are those of all slots; for the single-sequence form (kslot None) one slot's, with `cap`."""
        if (k is None) != (v is None):
            raise ValueError("sinks: both buffers or neither")
        if k is None:
            return capi.CSinks(None, None, n_sink, 0)
        per = self.geom.n_kv * self.geom.rec
        n = self.geom.n_slots if cap is None else 1
        cap = k.numel() // (n * per) if cap is None else cap
        d = capi.CSinks(self._dev("k", k, torch.uint8, n * per * cap), self._dev("v", v, torch.uint8, n * per * cap), n_sink, cap)
        d.slots, d.bufs = min(k.numel(), v.numel()) // max(per * cap, 1), (k, v)
        return d

    def _sinks(self, sinks, kslot):
        """The descriptor for a call; partitions are named by kslot only over buffers that have one for every slot."""
        if kslot is not None and getattr(sinks, "slots", self.geom.n_slots) < self.geom.n_slots:
            raise ValueError(f"sinks: buffers of {sinks.slots} of {self.geom.n_slots} slots in a call that names slots")
        return C.byref(sinks)

    def _part(self, part, n: int, rows: int):
        """The scratch of an attention call, big enough for it."""
        need = self._ws_need.get((n, rows))
        if need is None:
            need = self._ws_need[n, rows] = self.workspace_bytes(n, rows)
        return self._dev("part", part, torch.uint8, need)

    def sinks_store(self, kvk, kvv, sinks, pos, kslot=None, act=None, rows: int = 1):
        """Behind the append of the same rows: the records of the first positions, ring -> sink buffers."""
        p, s, a, n = self._seqs(pos, kslot, act)
        k, v = self._cache_ptrs(kvk, kvv, True, kslot is not None)
        self._check("battn_sinks_store", self.lib.battn_sinks_store(self.h, k, v, self._sinks(sinks, kslot), p, s, a,
                                                                    n, rows, self._stream_here()))

    def attn_sinks(self, out, q, kvk, kvv, sinks, pos, part, rows: int = 1, kslot=None, act=None, is_swa: bool = True):
        """Sliding-window attention whose rows see the first n_sink positions too: `rows` rows of every sequence (decode,
        verify) or a prompt chunk of one."""
        p, s, a, n = self._seqs(pos, kslot, act)
        k, v = self._cache_ptrs(kvk, kvv, is_swa, kslot is not None)
        nq = n * rows * self.geom.n_head * self.geom.head_dim
        self._check("battn_attend_sinks", self.lib.battn_attend_sinks(
            self.h, self._dev("out", out, self.out_torch, nq), self._dev("q", q, self.q_torch, nq), k, v,
            self._sinks(sinks, kslot), p, s, a, self._part(part, n, rows), rows, n, int(is_swa), self._stream_here()))

    def attn_sinks_paged(self, out, q, pages, sinks, pos, part, rows: int = 1, ktab=None, act=None):
        p, s, a, n = self._seqs(pos, ktab, act)
        nq = n * rows * self.geom.n_head * self.geom.head_dim
        self._check("battn_attend_sinks_paged", self.lib.battn_attend_sinks_paged(
            self.h, self._dev("out", out, self.out_torch, nq), self._dev("q", q, self.q_torch, nq), C.byref(pages),
            C.byref(sinks), p, s, a, self._part(part, n, rows), rows, n, self._stream_here()))

    # ---- attention that accumulates its weights ------------------------------------------------------------
    def alloc_track_part(self, n_seq: int, rows: int, max_positions: int) -> torch.Tensor:
        n = C.c_size_t()
        self._check("battn_track_workspace_bytes",
                    self.lib.battn_track_workspace_bytes(self.h, n_seq, rows, max_positions, C.byref(n)))
        return torch.empty(n.value, dtype=torch.uint8, device=self.device)

    def _track_part(self, part):
        """Pointer and bytes of the scratch of a weight-accumulating call; the library checks that they suffice."""
        return self._dev("part", part, part.dtype), part.numel() * part.element_size()

    def _track_args(self, out, score_out, score_in, q, rows, n, scores):
        nq = n * rows * self.geom.n_head * self.geom.head_dim
        return (self._dev("out", out, self.out_torch, nq), self._dev("score_out", score_out, torch.float32, scores),
                None if score_in is None else self._dev("score_in", score_in, torch.float32, scores),
                self._dev("q", q, self.q_torch, nq))

    def attn_track(self, out, score_out, score_in, q, kvk, kvv, pos, part, rows: int = 1, kslot=None, act=None):
        """Full-causal attention (one row of every sequence, or 2..512 rows of one) that also adds the weight every cached
        position receives to score_in, into score_out (the same tensor, usually); score_in None: nothing so far."""
        g = self.geom
        p, s, a, n = self._seqs(pos, kslot, act)
        k, v = self._cache_ptrs(kvk, kvv, False, kslot is not None)
        args = self._track_args(out, score_out, score_in, q, rows, n, (1 if kslot is None else g.n_slots) * g.n_kv * g.slot_ctx)
        self._check("battn_attend_track", self.lib.battn_attend_track(
            self.h, *args, k, v, p, s, a, *self._track_part(part), rows, n, self._stream_here()))

    def attn_track_paged(self, out, score_out, score_in, q, pages, pos, part, rows: int = 1, ktab=None, act=None):
        p, s, a, n = self._seqs(pos, ktab, act)
        args = self._track_args(out, score_out, score_in, q, rows, n, (1 if ktab is None else pages.n_tables) *
                                self.geom.n_kv * pages.max_pages * pages.page_len)
        self._check("battn_attend_track_paged", self.lib.battn_attend_track_paged(
            self.h, *args, C.byref(pages), p, s, a, *self._track_part(part), rows, n, self._stream_here()))

    # ---- eviction by accumulated attention weight --------------------------------------------------------
    def alloc_evict_part(self, n_seq: int) -> torch.Tensor:
        n = C.c_size_t()
        self._check("battn_evict_workspace_bytes", self.lib.battn_evict_workspace_bytes(self.h, n_seq, C.byref(n)))
        return torch.empty(n.value, dtype=torch.uint8, device=self.device)

    def _evict_args(self, score, kept, pos_out, pos, part, budget, sel, sel_dst, act, scores: int):
        p, s, a, n = self._seqs(pos, sel, act)
        d = None if sel_dst is None else self._dev("kslot_dst", sel_dst, torch.int32, n)
        return n, (self._dev("score", score, torch.float32, scores),
                   self._dev("kept", kept, torch.int32, n * self.geom.n_kv * max(budget, 1)),
                   self._dev("pos_out", pos_out, torch.int32, n), p, s, d, a, self._dev("part", part, torch.uint8, 4 * n))

    def evict(self, kvk, kvv, score, kept, pos_out, pos, part, budget: int, n_sink: int = 0, n_recent: int = 0, kslot=None,
              kslot_dst=None, act=None):
        """Keeps `budget` of the pos[i] cached positions of every sequence: the first n_sink, the last n_recent and the best
        scored between them, moved to the front of the same partition or of kslot_dst[i]'s."""
        k, v = self._cache_ptrs(kvk, kvv, False, kslot is not None)
        g = self.geom
        n, args = self._evict_args(score, kept, pos_out, pos, part, budget, kslot, kslot_dst, act,
                                   (1 if kslot is None else g.n_slots) * g.n_kv * g.slot_ctx)
        self._check("battn_evict", self.lib.battn_evict(self.h, k, v, *args, budget, n_sink, n_recent, n, self._stream_here()))

    def evict_paged(self, pages, score, kept, pos_out, pos, part, budget: int, n_sink: int = 0, n_recent: int = 0, ktab=None,
                    ktab_dst=None, act=None):
        n, args = self._evict_args(score, kept, pos_out, pos, part, budget, ktab, ktab_dst, act,
                                   (1 if ktab is None else pages.n_tables) * self.geom.n_kv * pages.max_pages * pages.page_len)
        self._check("battn_evict_paged", self.lib.battn_evict_paged(self.h, C.byref(pages), *args, budget, n_sink, n_recent, n,
                                                                    self._stream_here()))

    # ---- the step after attention ------------------------------------------------------------------------
    def gate_norm(self, dst, aout, gate, sgate, xq, xd, xsum, rows: int):
        """k_gate_norm_vec4 (bruce.cu:1526): sigmoid gate, L2 norm, q8 activation copy; dst may be None."""
        rc = self.lib.battn_gate_norm(self.h, _ptr(dst), _ptr(aout), _ptr(gate), _ptr(sgate), _ptr(xq), _ptr(xd),
                                      _ptr(xsum), rows, self._stream())
        self._check("battn_gate_norm", rc)

    def prefill_gate_norm(self, dst, q, kvk, kvv, pos, part, gate, sgate, xq, xd, xsum, rows: int, is_swa: bool = False):
        """Prompt-chunk attention fused with the gate-norm step (k_combine_gate_norm_rows_opt, bruce.cu:1577)."""
        rc = self.lib.battn_prefill_gate_norm(self.h, _ptr(dst), _ptr(q), _ptr(kvk), _ptr(kvv), _ptr(pos), _ptr(part),
                                              _ptr(gate), _ptr(sgate), _ptr(xq), _ptr(xd), _ptr(xsum), rows, int(is_swa),
                                              self._stream())
        self._check("battn_prefill_gate_norm", rc)

    # ---- one sequence split by position range across devices ----------------------------------------
    def xchg_create(self, rank: int, world: int, max_rows: int = 8):
        """This device's receive area for the cross-device exchange of split records.  Returns (exchange, its
        IPC handle as bytes) -- the handle goes to the other processes."""
        x = C.c_void_p()
        buf = C.create_string_buffer(capi.IPC_HANDLE_BYTES)
        self._check("battn_xchg_create", self.lib.battn_xchg_create(self.h, rank, world, max_rows, C.byref(x), buf))
        return x, bytes(buf.raw)

    def xchg_connect(self, x, all_handles: bytes):
        self._check("battn_xchg_connect", self.lib.battn_xchg_connect(x, all_handles))

    def xchg_area(self, x):
        ptr, n = C.c_void_p(), C.c_size_t()
        self._check("battn_xchg_area", self.lib.battn_xchg_area(x, C.byref(ptr), C.byref(n)))
        return ptr.value, n.value

    def xchg_connect_ptrs(self, x, ptrs):
        arr = (C.c_void_p * len(ptrs))(*ptrs)
        self._check("battn_xchg_connect_ptrs", self.lib.battn_xchg_connect_ptrs(x, arr))

    def xchg_set_wait_polls(self, x, polls: int):
        self._check("battn_xchg_set_wait_polls", self.lib.battn_xchg_set_wait_polls(x, polls))

    def xchg_destroy(self, x):
        self.lib.battn_xchg_destroy(x)

    def attn_partials_push(self, x, out, q, kvk, kvv, pos, part, epoch, rows: int = 1, batch: int = 1,
                           is_swa: bool = False, kslot=None, act=None, epoch_advance: int = 1):
        """Decode on this device's shard, push the merged (o, m, l) records to every device of the group and --
        when `out` is given -- wait for the peers' records of the same step and merge them (one decode launch + one
        merge launch).  `epoch`: int32 device tensor holding this device's step counter (advanced on the device)."""
        rc = self.lib.battn_partials_push(self.h, x, _ptr(out), _ptr(q), _ptr(kvk), _ptr(kvv), _ptr(pos), _ptr(kslot),
                                          _ptr(act), _ptr(part), rows, batch, int(is_swa), _ptr(epoch),
                                          int(epoch_advance), self._stream())
        self._check("battn_partials_push", rc)

    def attn_merge_wait(self, x, out, n_rows: int, epoch):
        rc = self.lib.battn_merge_wait(self.h, x, _ptr(out), n_rows, _ptr(epoch), self._stream())
        self._check("battn_merge_wait", rc)

    # ---- diagnostics -------------------------------------------------------------------------------
    def device_status(self, clear: bool = True) -> int:
        bits = C.c_int()
        self._check("battn_device_status", self.lib.battn_device_status(self.h, C.byref(bits), int(clear)))
        return bits.value

    def profile_start(self, max_launches: int):
        """Bracket the main kernel of every following attention call with CUDA events."""
        self._check("battn_profile_start", self.lib.battn_profile_start(self.h, max_launches))
        self._prof_cap = max_launches

    def profile_stop(self):
        """Elapsed milliseconds of each bracketed launch since profile_start, in call order."""
        buf = (C.c_float * self._prof_cap)()
        n = C.c_int()
        self._check("battn_profile_stop", self.lib.battn_profile_stop(self.h, buf, self._prof_cap, C.byref(n)))
        return [buf[i] for i in range(min(n.value, self._prof_cap))]

    def launch_count(self) -> int:
        return int(self.lib.battn_launch_count(self.h))
