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
two graphs that may run at once need a plan each.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib as L
from .ops import _DT, _need, _on, _ptr, _stream_handle


class PagedPlan:
    def __init__(self, tokens: int, seqs: int, nH: int, nkv: int, hd: int, page_size: int, table_pages: int,
                 prefix_pages: int = 0, window: int = 0, device="cuda"):
        self.T, self.B, self.nH, self.nkv, self.hd = tokens, seqs, nH, nkv, hd
        self.page_size, self.table_pages, self.prefix_pages, self.window = page_size, table_pages, prefix_pages, window
        dev = torch.device(device)
        self.device = torch.device("cuda", torch.cuda.current_device() if dev.index is None else dev.index)
        self._lib = L.load()
        self._sizes = (tokens, seqs, nH, nkv, hd, page_size, table_pages, prefix_pages, window)
        with _on(self.device, None):
            plan, ws = self._lib.g4b_paged_plan_bytes(*self._sizes), self._lib.g4b_paged_workspace_bytes(*self._sizes)
            if not plan:
                raise L.G4BError("g4b_paged_plan_bytes", L.G4B_E_SHAPE, L.last_error())
            # a plan of zeros is nobody's: a call before the first update() writes nothing
            self._plan = torch.zeros(plan, dtype=torch.uint8, device=self.device)
            self._ws = torch.empty(ws, dtype=torch.uint8, device=self.device)

    def _check(self, op: str, t: torch.Tensor, name: str, dtype, shape) -> None:
        _need(t, name)
        if t.device != self.device:
            raise ValueError(f"{op}: {name} is on {t.device}, the plan on {self.device}")
        if t.dtype not in (dtype if isinstance(dtype, tuple) else (dtype,)):
            raise TypeError(f"{op}: {name} is {t.dtype}")
        if shape is not None and tuple(t.shape) != shape:
            raise ValueError(f"{op}: {name} is {tuple(t.shape)}, want {shape}")

    def _rows(self, op: str, t: torch.Tensor, name: str, dtypes, least: int) -> None:
        """A [T, row] view with unit element stride and rows of at least `least` elements."""
        if not t.is_cuda or t.device != self.device:
            raise ValueError(f"{op}: {name} must be a CUDA tensor on {self.device}")
        if t.dtype not in dtypes:
            raise TypeError(f"{op}: {name} is {t.dtype}")
        if t.dim() != 2 or t.shape[0] != self.T or t.shape[1] < least or t.stride(1) != 1 or \
                (self.T > 1 and t.stride(0) < t.shape[1]):
            raise ValueError(f"{op}: {name} must be [{self.T}, >= {least}] rows, got {tuple(t.shape)} "
                             f"with strides {t.stride()}")

    def _caches(self, op: str, kc: torch.Tensor, vc: torch.Tensor) -> int:
        pages = kc.shape[0]
        for t, n in ((kc, "kc"), (vc, "vc")):
            self._check(op, t, n, (torch.float16, torch.int16), (pages, self.nkv, self.page_size, self.hd))
        return pages

    def update(self, q_start: torch.Tensor, kv_len: torch.Tensor, prefix_len: Optional[torch.Tensor] = None,
               stream: Optional[torch.cuda.Stream] = None) -> None:
        """Plan the batch: q_start [B + 1], kv_len [B] and, with prefix pages, prefix_len [1], int32."""
        self._check("paged_plan", q_start, "q_start", torch.int32, (self.B + 1,))
        self._check("paged_plan", kv_len, "kv_len", torch.int32, (self.B,))
        if (prefix_len is None) != (self.prefix_pages == 0):
            raise ValueError(f"paged_plan: prefix_len goes with prefix pages ({self.prefix_pages} here)")
        if prefix_len is not None:
            self._check("paged_plan", prefix_len, "prefix_len", torch.int32, (1,))
        with _on(self.device, stream):
            L.check("g4b_paged_plan", self._lib.g4b_paged_plan(
                _ptr(q_start), _ptr(kv_len), _ptr(prefix_len), *self._sizes, _ptr(self._plan), self._plan.numel(),
                _stream_handle(stream, self.device)))

    def append(self, qkv: torch.Tensor, qnw: torch.Tensor, knw: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
               kc: torch.Tensor, vc: torch.Tensor, table: torch.Tensor, koff: int, voff: int,
               q_out: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
        """The new tokens' normed, rotated keys and normed values into their pages of kc / vc
        [num_pages, nkv, page_size, hd]; returns their normed, rotated queries [T, nH * hd] f16.

        qkv [T, row] f32 or f16: q heads at 0, k heads at koff, v heads at voff (koff again for k = v);
        cos / sin [positions, hd] f32; table [B, table_pages] int32."""
        op, nq, nk = "paged_append", self.nH * self.hd, self.nkv * self.hd
        self._rows(op, qkv, "qkv", _DT, max(nq, koff + nk, voff + nk))
        for t, n in ((qnw, "qnw"), (knw, "knw")):
            self._check(op, t, n, torch.float32, (self.hd,))
        for t, n in ((cos, "cos"), (sin, "sin")):
            self._check(op, t, n, torch.float32, (cos.shape[0], self.hd))
        pages = self._caches(op, kc, vc)
        self._check(op, table, "table", torch.int32, (self.B, self.table_pages))
        with _on(self.device, stream):
            if q_out is None:
                q_out = torch.empty((self.T, nq), dtype=torch.float16, device=self.device)
            self._rows(op, q_out, "q_out", (torch.float16,), nq)
            L.check("g4b_paged_append", self._lib.g4b_paged_append(
                _ptr(qkv), _DT[qkv.dtype], self._stride(qkv), _ptr(qnw), _ptr(knw), _ptr(cos), _ptr(sin), cos.shape[0],
                _ptr(kc), _ptr(vc), pages, _ptr(table), _ptr(q_out), self._stride(q_out), *self._sizes[:5], koff, voff,
                *self._sizes[5:], _ptr(self._plan), _stream_handle(stream, self.device)))
        return q_out

    def attend(self, q: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor, table: torch.Tensor,
               prefix_table: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
               out_dtype: torch.dtype = torch.float16, scale: float = 1.0,
               stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
        """Attention of the new tokens' queries q [T, nH * hd] f16 (append's result) over the cache; returns
        out [T, nH * hd] (or writes the given [T, row] view).  Padding rows of out are left as they are."""
        op, nq = "paged_attn", self.nH * self.hd
        self._rows(op, q, "q", (torch.float16,), nq)
        pages = self._caches(op, kc, vc)
        self._check(op, table, "table", torch.int32, (self.B, self.table_pages))
        if (prefix_table is None) != (self.prefix_pages == 0):
            raise ValueError(f"paged_attn: prefix_table goes with prefix pages ({self.prefix_pages} here)")
        if prefix_table is not None:
            self._check(op, prefix_table, "prefix_table", torch.int32, (self.prefix_pages,))
        with _on(self.device, stream):
            if out is None:
                out = torch.empty((self.T, nq), dtype=out_dtype, device=self.device)
            self._rows(op, out, "out", _DT, nq)
            L.check("g4b_paged_attn", self._lib.g4b_paged_attn(
                _ptr(q), self._stride(q), _ptr(kc), _ptr(vc), pages, _ptr(table), _ptr(prefix_table), _ptr(out),
                _DT[out.dtype], self._stride(out), float(scale), *self._sizes, _ptr(self._plan), _ptr(self._ws),
                self._ws.numel(), _stream_handle(stream, self.device)))
        return out

    @staticmethod
    def _stride(t: torch.Tensor) -> int:
        """Elements between rows (one row: its stride means nothing)."""
        return t.stride(0) if t.shape[0] > 1 else t.shape[1]
