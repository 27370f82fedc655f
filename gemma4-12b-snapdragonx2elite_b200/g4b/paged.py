"""Batches over a paged KV cache: one plan per step, its append and its attention.

``PagedPlan`` holds the sizes of a batch that a serving loop keeps (token rows, sequences, heads, page tables),
the plan in device memory and the attention's workspace.  A step calls ``update`` once, then ``append`` and
``attend`` in every layer of that kind (same heads and window):

    plan = PagedPlan(T, B, nH, nkv, hd, page_size, table_pages, prefix_pages, window)
    plan.update(q_start, kv_len, prefix_len)                        # int32 device tensors
    q = plan.append(qkv, qnw, knw, cos, sin, kc, vc, table, koff, voff)
    out = plan.attend(q, kc, vc, table, prefix_table)

The layout of the batch and of the cache is described at "batches over a paged KV cache" in include/g4b.h.
Every call is stream-ordered and can be captured; calls of one plan must be ordered among themselves, so
two graphs that may run at once need a plan each, and a plan lives at least as long as the graphs that use it.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib as L
from .ops import _DT, _is, _on, _ptr, _raw_stream


class PagedPlan:
    def __init__(self, tokens: int, seqs: int, nH: int, nkv: int, hd: int, page_size: int, table_pages: int,
                 prefix_pages: int = 0, window: int = 0, device="cuda"):
        self.T, self.B, self.nH, self.nkv, self.hd = tokens, seqs, nH, nkv, hd
        self.page_size, self.table_pages, self.prefix_pages, self.window = page_size, table_pages, prefix_pages, window
        dev = torch.device(device)
        if dev.type != "cuda":
            raise ValueError(f"a paged plan lives on a CUDA device, not on {dev}")
        self.index = torch.cuda.current_device() if dev.index is None else dev.index
        self.device = torch.device("cuda", self.index)
        self._lib = L.load()
        self._sizes = (tokens, seqs, nH, nkv, hd, page_size, table_pages, prefix_pages, window)
        with _on(self.index, None):
            plan, ws = self._lib.g4b_paged_plan_bytes(*self._sizes), self._lib.g4b_paged_workspace_bytes(*self._sizes)
            if not plan:
                raise L.G4BError("g4b_paged_plan_bytes", L.G4B_E_SHAPE, L.last_error())
            # a plan of zeros is nobody's: a call before the first update() writes nothing
            self._plan = torch.zeros(plan, dtype=torch.uint8, device=self.device)
            self._ws = torch.empty(ws, dtype=torch.uint8, device=self.device)
            if not torch.cuda.is_current_stream_capturing():
                torch.cuda.current_stream(self.index).synchronize()     # the zeros come before the calls of any stream
            self._streams = {_raw_stream(self.index)}
        self._plan_ptr, self._ws_ptr, self._ws_bytes = self._plan.data_ptr(), self._ws.data_ptr(), ws
        self._table_shape, self._head_shape = (seqs, table_pages), (hd,)

    def _bad(self, op: str, **tensors):
        """What a call was given, for the message of the error that it raises."""
        said = ", ".join(f"{n} {tuple(t.shape)} {str(t.dtype)[6:]} strides {t.stride()} on {t.device}" for n, t in
                         tensors.items() if t is not None)
        raise ValueError(f"{op}: for {self.T} tokens of {self.B} sequences, {self.nH} / {self.nkv} heads of {self.hd}, "
                         f"{self.table_pages} + {self.prefix_pages} pages of {self.page_size} on {self.device}, got {said}")

    def _rows(self, t: torch.Tensor, least: int) -> int:
        """Elements between the rows of a [T, >= least] view with unit element stride on the plan's device; 0: it
        is none.  (One row: its stride means nothing.)"""
        if t.dim() != 2 or t.get_device() != self.index:
            return 0
        (rows, width), (step, unit) = t.shape, t.stride()
        if rows != self.T or width < least or unit != 1:
            return 0
        return width if rows == 1 else step if step >= width else 0

    def _caches(self, kc: torch.Tensor, vc: torch.Tensor) -> int:
        """Pages of the caches; 0: they are none of this plan's."""
        shape = kc.shape
        if len(shape) != 4 or shape[1] != self.nkv or shape[2] != self.page_size or shape[3] != self.hd:
            return 0
        for t in (kc, vc):
            if not (_is(t, torch.float16, shape, self.index) or _is(t, torch.int16, shape, self.index)):
                return 0
        return shape[0]

    def _stream(self) -> int:
        """The current stream's handle; its work is done before the plan's memory serves anything else."""
        raw = _raw_stream(self.index)
        if raw not in self._streams:
            self._streams.add(raw)
            for t in (self._plan, self._ws):
                t.record_stream(torch.cuda.current_stream(self.index))
        return raw

    def _elsewhere(self, stream) -> bool:
        return stream is not None or torch.cuda.current_device() != self.index

    def update(self, q_start: torch.Tensor, kv_len: torch.Tensor, prefix_len: Optional[torch.Tensor] = None,
               stream: Optional[torch.cuda.Stream] = None) -> None:
        """Plan the batch: q_start [B + 1], kv_len [B] and, with prefix pages, prefix_len [1], int32."""
        if self._elsewhere(stream):
            with _on(self.index, stream):
                return self.update(q_start, kv_len, prefix_len)
        if (prefix_len is None) != (self.prefix_pages == 0):
            raise ValueError(f"paged_plan: prefix_len goes with prefix pages ({self.prefix_pages} here)")
        i32, index = torch.int32, self.index
        if not (_is(q_start, i32, (self.B + 1,), index) and _is(kv_len, i32, (self.B,), index)
                and (prefix_len is None or _is(prefix_len, i32, (1,), index))):
            self._bad("paged_plan", q_start=q_start, kv_len=kv_len, prefix_len=prefix_len)
        L.check("g4b_paged_plan", self._lib.g4b_paged_plan(
            q_start.data_ptr(), kv_len.data_ptr(), _ptr(prefix_len), *self._sizes, self._plan_ptr, self._plan.numel(),
            self._stream()))

    def append(self, qkv: torch.Tensor, qnw: torch.Tensor, knw: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
               kc: torch.Tensor, vc: torch.Tensor, table: torch.Tensor, koff: int, voff: int,
               q_out: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
        """The new tokens' normed, rotated keys and normed values into their pages of kc / vc
        [num_pages, nkv, page_size, hd]; returns their normed, rotated queries [T, nH * hd] f16.

        qkv [T, row] f32 or f16: q heads at 0, k heads at koff, v heads at voff (koff again for k = v);
        cos / sin [positions, hd] f32; table [B, table_pages] int32."""
        if self._elsewhere(stream):
            with _on(self.index, stream):
                return self.append(qkv, qnw, knw, cos, sin, kc, vc, table, koff, voff, q_out)
        nq, nk, index, f32 = self.nH * self.hd, self.nkv * self.hd, self.index, torch.float32
        if q_out is None:
            q_out = torch.empty((self.T, nq), dtype=torch.float16, device=self.device)
        dtype = _DT.get(qkv.dtype)
        step, q_step, pages, rot = self._rows(qkv, max(nq, koff + nk, voff + nk)), self._rows(q_out, nq), \
            self._caches(kc, vc), cos.shape
        if not (step and q_step and pages and dtype is not None and q_out.dtype is torch.float16 and len(rot) == 2
                and rot[1] == self.hd and _is(cos, f32, rot, index) and _is(sin, f32, rot, index)
                and _is(qnw, f32, self._head_shape, index) and _is(knw, f32, self._head_shape, index)
                and _is(table, torch.int32, self._table_shape, index)):
            self._bad("paged_append", qkv=qkv, qnw=qnw, knw=knw, cos=cos, sin=sin, kc=kc, vc=vc, table=table, q_out=q_out)
        L.check("g4b_paged_append", self._lib.g4b_paged_append(
            qkv.data_ptr(), dtype, step, qnw.data_ptr(), knw.data_ptr(), cos.data_ptr(), sin.data_ptr(), rot[0],
            kc.data_ptr(), vc.data_ptr(), pages, table.data_ptr(), q_out.data_ptr(), q_step, *self._sizes[:5], koff, voff,
            *self._sizes[5:], self._plan_ptr, self._stream()))
        return q_out

    def attend(self, q: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor, table: torch.Tensor,
               prefix_table: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
               out_dtype: torch.dtype = torch.float16, scale: float = 1.0,
               stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
        """Attention of the new tokens' queries q [T, nH * hd] f16 (append's result) over the cache; returns
        out [T, nH * hd] (or writes the given [T, row] view).  Padding rows of out are left as they are."""
        if self._elsewhere(stream):
            with _on(self.index, stream):
                return self.attend(q, kc, vc, table, prefix_table, out, out_dtype, scale)
        if (prefix_table is None) != (self.prefix_pages == 0):
            raise ValueError(f"paged_attn: prefix_table goes with prefix pages ({self.prefix_pages} here)")
        nq, index = self.nH * self.hd, self.index
        if out is None:
            out = torch.empty((self.T, nq), dtype=out_dtype, device=self.device)
        dtype = _DT.get(out.dtype)
        step, out_step, pages = self._rows(q, nq), self._rows(out, nq), self._caches(kc, vc)
        if not (step and out_step and pages and dtype is not None and q.dtype is torch.float16
                and _is(table, torch.int32, self._table_shape, index)
                and (prefix_table is None or _is(prefix_table, torch.int32, (self.prefix_pages,), index))):
            self._bad("paged_attn", q=q, kc=kc, vc=vc, table=table, prefix_table=prefix_table, out=out)
        L.check("g4b_paged_attn", self._lib.g4b_paged_attn(
            q.data_ptr(), step, kc.data_ptr(), vc.data_ptr(), pages, table.data_ptr(), _ptr(prefix_table), out.data_ptr(),
            dtype, out_step, scale, *self._sizes, self._plan_ptr, self._ws_ptr, self._ws_bytes, self._stream()))
        return out
