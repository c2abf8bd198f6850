"""Paged key-value cache on the GPU (kq_kv_*, include/pesti_decoder.h).

The keys and values of all sequences live in two pools of f16 pages
[pages][kv_heads][page_size][head_dim]; a block table names the pages of each
sequence.  ``PagedCache`` binds a pair of pools to a context and offers what a
decode step does with them: ``append`` rows, ``attention`` or
``rope_attention`` of one new token per sequence, and ``evict`` by accumulated
attention weight.  Tensors are CUDA tensors on the context's device; calls are
queued on the context's stream and return nothing: what they write is handed in.
"""
from __future__ import annotations

import ctypes

from . import kq


def _bind(lib: ctypes.CDLL) -> ctypes.CDLL:
    P, I, I32, I64, F, Z = (ctypes.c_void_p, ctypes.c_int, ctypes.c_int32, ctypes.c_int64, ctypes.c_float,
                            ctypes.c_size_t)
    sig = {
        "kq_kv_create": ([P, P, P, I64, I64, I, I, I, ctypes.POINTER(P)], I),
        "kq_kv_destroy": ([P], I),
        "kq_kv_set_table_cols": ([P, I64], I),
        "kq_kv_append": ([P, P, I64, I64, I, P, P, P, P, I64, I64, F, P, I64, P, I64], I),
        "kq_kv_append_tracked": ([P, P, I64, I64, I, P, P, P, P, I64, I64, F, P, I64, P, P, I64], I),
        "kq_kv_attention_scratch": ([P, I64, I, I64], Z),
        "kq_kv_attention": ([P, P, I64, P, I64, I64, I, P, I64, P, P, I64, P, Z], I),
        "kq_kv_rope_attention": ([P, P, I64, P, I64, I64, I, P, I64, P, P, F, P, P, I64, P, Z], I),
        "kq_kv_evict_scratch": ([P, I64, I64], Z),
        "kq_kv_evict": ([P, I64, P, I64, P, P, P, P, P, P, I64, P, I32, P, Z], I),
    }
    for name, (args, res) in sig.items():
        getattr(lib, name).argtypes = args
        getattr(lib, name).restype = res
    return lib


def _invalid(message: str) -> kq.KqError:
    return kq.KqError(kq.KQ_ERR_INVALID_ARG, message)


class PagedCache:
    """Two pools of pages (f16 CUDA tensors of one shape [pages][kv_heads]
    [page_size][head_dim], contiguous within a page) as one layer's cache."""

    def __init__(self, ctx: "kq.Context", k, v):
        import torch
        if k.dim() != 4 or 0 in k.shape or k.shape != v.shape or k.stride() != v.stride():
            raise _invalid(f"pools of shapes {tuple(k.shape)} and {tuple(v.shape)}: one shape and stride is wanted")
        if k.dtype != torch.float16 or v.dtype != torch.float16:
            raise _invalid(f"pools of {k.dtype} and {v.dtype}: float16 is wanted")
        self.pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        if not k[0].is_contiguous():
            raise _invalid(f"pool strides {k.stride()}: the pages must be contiguous")
        page_ld = k.stride(0) if self.pages > 1 else k[0].numel()
        self.device, self.index = torch.device("cuda", ctx.device), ctx.device
        if k.device != self.device or v.device != self.device:
            raise _invalid(f"pools on {k.device} and {v.device}, context on {self.device}")
        self.ctx, self.k, self.v = ctx, k, v
        self.lib = _bind(ctx.lib)
        self._types = torch.float32, torch.int32
        h = ctypes.c_void_p()
        ctx.check(self.lib.kq_kv_create(ctx.handle, k.data_ptr(), v.data_ptr(), self.pages, page_ld,
                                        self.page_size, self.kv_heads, self.head_dim, ctypes.byref(h)), "kq_kv_create")
        self.handle, self._cols = h, 0
        self._append, self._attention = self.lib.kq_kv_append_tracked, self.lib.kq_kv_attention
        self._rope_attention = self.lib.kq_kv_rope_attention

    # ---- argument checks (lean: they run before every call) ------------------------------
    def _rows(self, t, name: str, dtype, rows: int = -1):
        """The row stride of a matrix with unit inner stride."""
        try:
            n, cols = t.shape
            ld, inner = t.stride()
            if t.dtype is dtype and t.get_device() == self.index and (inner == 1 or cols <= 1) and (n == rows or rows < 0):
                return ld if n > 1 else cols
        except ValueError:  # not a matrix
            pass
        raise self._no_rows(t, name, dtype, rows)

    def _no_rows(self, t, name: str, dtype, rows: int) -> kq.KqError:
        return _invalid(f"{name}: {t.dtype} {tuple(t.shape)} strides {t.stride()} on {t.device}; "
                        f"{rows if rows >= 0 else 'any'} rows of {dtype} on {self.device} are wanted")

    def _table(self, t, batch: int = -1):
        """The row stride of a block table, which may be part of a wider one:
        its own width is what bounds the calls that follow."""
        try:
            n, cols = t.shape
            ld, inner = t.stride()
            if cols and t.dtype is self._types[1] and t.get_device() == self.index and (inner == 1 or cols == 1) and (
                    n == batch or batch < 0):
                if cols != self._cols:
                    self.ctx.check(self.lib.kq_kv_set_table_cols(self.handle, cols), "kq_kv_set_table_cols")
                    self._cols = cols
                return ld if n > 1 else cols
        except ValueError:  # not a matrix
            pass
        raise self._no_rows(t, "table", self._types[1], batch)

    def _vector(self, t, name: str, n: int):
        """The address of n contiguous int32."""
        if t is None or t.dtype is not self._types[1] or t.get_device() != self.index or t.shape != (n,) or (
                not t.is_contiguous()):
            raise _invalid(f"{name}: {n} contiguous int32 on {self.device} are wanted"
                           + ("" if t is None else f", not {t.dtype} {tuple(t.shape)} on {t.device}"))
        return t.data_ptr()

    def _track(self, t, name: str, dtype, batch: int, ld=None):
        """The address and track_ld of a contiguous [batch][kv_heads][track_ld] array."""
        shape = t.shape
        if t.dtype is not dtype or t.get_device() != self.index or len(shape) != 3 or not t.is_contiguous() or (
                shape[0] != batch or shape[1] != self.kv_heads):
            raise _invalid(f"{name}: {t.dtype} {tuple(shape)} on {t.device}; contiguous {dtype} [{batch}]"
                           f"[{self.kv_heads}][slots] is wanted")
        if ld and ld != shape[2]:
            raise _invalid(f"{name}: {shape[2]} slots where the others have {ld}")
        return t.data_ptr(), shape[2]

    def _scratch(self, t):
        if t.get_device() != self.index or not t.is_contiguous():
            raise _invalid(f"scratch on {t.device}: contiguous memory on {self.device} is wanted")
        return t.data_ptr(), t.nbytes

    # ---- calls -----------------------------------------------------------------------------
    def scratch(self, batch: int, heads: int, track_ld: int = 0):
        """Zeroed scratch of attention / rope_attention calls of up to these
        sizes (track_ld: that of the mass array, 0 without one); one call at a
        time may use it."""
        import torch
        n = self.lib.kq_kv_attention_scratch(self.handle, batch, heads, track_ld)
        if n == 0:
            raise _invalid(f"attention of {batch} sequences, {heads} query heads over {self.kv_heads}")
        return torch.zeros(n, dtype=torch.uint8, device=self.device)

    def evict_scratch(self, batch: int, track_ld: int):
        """Scratch of evict calls of these sizes; one call at a time may use it."""
        import torch
        n = self.lib.kq_kv_evict_scratch(self.handle, batch, track_ld)
        if n == 0:
            raise _invalid(f"eviction from {batch} sequences of {track_ld} tracked slots")
        return torch.empty(n, dtype=torch.uint8, device=self.device)

    def append(self, qkv, table, slots, *, theta: float, seqs=None, pos=None, q_out=None, mass=None,
               slot_pos=None) -> None:
        """Row r of qkv [rows][(heads + 2 kv_heads) head_dim] (q | k | v) into
        slot slots[r] (-1: none) of sequence seqs[r] (default r), turned to
        position pos[r] (default: the slot); the turned q into q_out.  The
        slots' mass starts at 0 (without it a slot used before keeps the weight
        of what lay there), and their positions go to slot_pos."""
        f32, i32 = self._types
        ld, table_ld = self._rows(qkv, "qkv", f32), self._table(table)
        rows, cols = qkv.shape
        batch, hd = table.shape[0], self.head_dim
        heads = cols // hd - 2 * self.kv_heads
        if (heads + 2 * self.kv_heads) * hd != cols:
            raise _invalid(f"qkv: rows of {cols} are not whole heads of {hd}")
        q_ptr, q_ld = None, 0
        if q_out is not None:
            q_ptr, q_ld = q_out.data_ptr(), self._rows(q_out, "q_out", f32, rows)
            if q_out.shape[1] < heads * hd:
                raise _invalid(f"q_out: rows of {q_out.shape[1]} for {heads} heads of {hd}")
        m, track = (None, 0) if mass is None else self._track(mass, "mass", f32, batch)
        sp = None
        if slot_pos is not None:
            sp, track = self._track(slot_pos, "slot_pos", i32, batch, track)
        rc = self._append(self.handle, qkv.data_ptr(), ld, rows, heads,
                          None if seqs is None else self._vector(seqs, "seqs", rows),
                          self._vector(slots, "slots", rows), None if pos is None else self._vector(pos, "pos", rows),
                          table.data_ptr(), table_ld, batch, theta, q_ptr, q_ld, m, sp, track)
        if rc:
            self.ctx.check(rc, "kq_kv_append")

    def attention(self, q, table, lens, out, scratch, mass=None) -> None:
        """out[b] = attention of q[b] [heads][head_dim] (turned already) over
        slots [0, lens[b]) of sequence b (0: zeros); mass accumulates each
        slot's weight, summed over the query heads of its kv head."""
        f32, i32 = self._types
        q_ld = self._rows(q, "q", f32)
        batch, cols = q.shape
        heads = cols // self.head_dim
        out_ld = self._rows(out, "out", f32, batch)
        if heads * self.head_dim != cols or out.shape[1] < cols:
            raise _invalid(f"q rows of {cols} and out rows of {out.shape[1]} for heads of {self.head_dim}")
        m, track = (None, 0) if mass is None else self._track(mass, "mass", f32, batch)
        rc = self._attention(self.handle, q.data_ptr(), q_ld, out.data_ptr(), out_ld, batch, heads, table.data_ptr(),
                             self._table(table, batch), self._vector(lens, "lens", batch), m, track,
                             *self._scratch(scratch))
        if rc:
            self.ctx.check(rc, "kq_kv_attention")

    def rope_attention(self, qkv, table, lens, out, scratch, *, theta: float, pos=None, mass=None,
                       slot_pos=None) -> None:
        """The same for the step's new tokens: q and k of qkv[b] (q | k | v)
        turned to pos[b] (default lens[b] - 1), k and v appended at slot
        lens[b] - 1, then the attention; the new slot's mass starts anew and its
        position goes to slot_pos."""
        f32, i32 = self._types
        ld = self._rows(qkv, "qkv", f32)
        batch, cols = qkv.shape
        hd = self.head_dim
        heads = cols // hd - 2 * self.kv_heads
        out_ld = self._rows(out, "out", f32, batch)
        if (heads + 2 * self.kv_heads) * hd != cols or out.shape[1] < heads * hd:
            raise _invalid(f"qkv rows of {cols} and out rows of {out.shape[1]} for heads of {hd}")
        m, track = (None, 0) if mass is None else self._track(mass, "mass", f32, batch)
        p = None
        if slot_pos is not None:
            p, track = self._track(slot_pos, "slot_pos", i32, batch, track)
        rc = self._rope_attention(self.handle, qkv.data_ptr(), ld, out.data_ptr(), out_ld, batch, heads,
                                  table.data_ptr(), self._table(table, batch),
                                  self._vector(lens, "lens", batch),
                                  None if pos is None else self._vector(pos, "pos", batch), theta, m, p, track,
                                  *self._scratch(scratch))
        if rc:
            self.ctx.check(rc, "kq_kv_rope_attention")

    def evict(self, table, lens, lens_out, mass, slot_pos, mass_out, pos_out, keep: int, scratch,
              recent_from=None) -> None:
        """Cut sequences of more than `keep` slots to `keep`: the slots at
        positions >= recent_from[b], then those of the greatest mass.  The
        outputs may be the inputs."""
        keep = min(keep, 2 ** 31 - 1)  # a greater budget would lose its upper bits on the way
        f32, i32 = self._types
        batch = table.shape[0]
        m, track = self._track(mass, "mass", f32, batch)
        p, _ = self._track(slot_pos, "slot_pos", i32, batch, track)
        mo, _ = self._track(mass_out, "mass_out", f32, batch, track)
        po, _ = self._track(pos_out, "pos_out", i32, batch, track)
        sp, sb = self._scratch(scratch)
        self.ctx.check(self.lib.kq_kv_evict(
            self.handle, batch, table.data_ptr(), self._table(table), self._vector(lens, "lens", batch),
            self._vector(lens_out, "lens_out", batch), m, p, mo, po, track,
            None if recent_from is None else self._vector(recent_from, "recent_from", batch), keep, sp, sb), "kq_kv_evict")

    def close(self) -> None:
        if getattr(self, "handle", None):
            self.lib.kq_kv_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
