"""The 8-bit paged KV cache (rvkv_q8_pool) from Python: the counterpart of
HipKvStorage with int8 codes and an f32 scale for every token and KV head.

Device buffers are torch tensors used as memory; every byte of work runs in
librvkv.so. Length, type and device checks that the C ABI cannot make are made
here, before the call.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _lib
from ._lib import RvkvError, check
from .kv_storage import (_DT, HipGatherPlan, _need, _on, _ptr,
                         rope_append_call)


class HipQ8Storage:
    """One 8-bit pool for all layers' K and V. memory: a contiguous uint8
    tensor of at least rvkv_q8_pool_bytes(...) bytes to use as the pool (as it
    is, so a cache can be handed on); by default zeroed memory of its own."""

    def __init__(self, n_layers: int, num_blocks: int, block_size: int,
                 n_kv_heads: int, head_dim: int, stream=None,
                 memory: Optional[torch.Tensor] = None):
        self._L = _lib.load()
        self._pool = None
        self.n_layers, self.num_blocks = n_layers, num_blocks
        self.block_size, self.n_kv_heads, self.head_dim = (
            block_size, n_kv_heads, head_dim)
        nbytes = self._L.rvkv_q8_pool_bytes(n_layers, num_blocks, block_size,
                                            n_kv_heads, head_dim)
        if not nbytes:
            # (the create call names the reason and its code)
            check(self._L.rvkv_q8_pool_create(
                n_layers, num_blocks, block_size, n_kv_heads, head_dim, None,
                0, None, ctypes.byref(ctypes.c_void_p())))
        if memory is None:
            memory = torch.zeros(
                nbytes, dtype=torch.uint8,
                device=torch.device("cuda", torch.cuda.current_device()))
        _need(memory.dtype == torch.uint8 and memory.is_contiguous() and
              memory.numel() >= nbytes,
              "q8_pool_create: memory must be contiguous uint8 of at least "
              "rvkv_q8_pool_bytes bytes")
        _need(memory.device.type != "cuda" or
              memory.device.index == torch.cuda.current_device(),
              "q8_pool_create: the current device is not the memory's")
        self.device, self.memory, self.nbytes = memory.device, memory, nbytes
        handle = ctypes.c_void_p()
        if stream is None and self.device.type == "cuda":
            stream = torch.cuda.current_stream(self.device)
        self.stream = stream
        self._views = {}  # (layer, which) -> codes, scales of this memory
        check(self._L.rvkv_q8_pool_create(
            n_layers, num_blocks, block_size, n_kv_heads, head_dim,
            _ptr(memory), memory.numel(),
            ctypes.c_void_p(stream.cuda_stream if stream else 0),
            ctypes.byref(handle)))
        self._pool = handle

    # -- lifetime -----------------------------------------------------------
    def close(self) -> None:
        if getattr(self, "_pool", None):
            self._L.rvkv_q8_pool_destroy(self._pool)
            self._pool = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def set_stream(self, stream) -> None:
        """Rebinds the pool to another stream (e.g. a graph-capture stream);
        later calls enqueue there."""
        check(self._L.rvkv_q8_pool_set_stream(
            self._pool, ctypes.c_void_p(stream.cuda_stream)))
        self.stream = stream

    # -- the cells, as views of the pool's memory -----------------------------
    def _record(self) -> int:
        n = self.n_kv_heads * self.block_size * (self.head_dim + 4)
        return -(-n // 256) * 256

    def _view(self, layer: int, which: int):
        got = self._views.get((layer, which))
        if got is None:
            _need(0 <= layer < self.n_layers and which in (0, 1),
                  "q8: layer or which out of range")
            rec, bs, hd = self._record(), self.block_size, self.head_dim
            nb, kv = self.num_blocks, self.n_kv_heads
            first = (2 * layer + which) * nb * rec
            # (as_strided counts from the storage's start, not the tensor's)
            bytes_, words = (self.memory[:self.nbytes].view(t) for t in
                             (torch.int8, torch.float32))
            codes = bytes_.as_strided(
                (nb, kv, bs, hd),
                (rec, bs * hd) + ((hd, 1) if which == 0 else (1, bs)),
                bytes_.storage_offset() + first)
            scales = words.as_strided(
                (nb, kv, bs), (rec // 4, bs, 1),
                words.storage_offset() + (first + kv * bs * hd) // 4)
            got = self._views[layer, which] = codes, scales
        return got

    def codes(self, layer: int, which: int) -> torch.Tensor:
        """int8 [num_blocks, n_kv, block_size, hd] of K (which 0) or V (1): a
        view, strided as the records lie (V's tokens are innermost)."""
        return self._view(layer, which)[0]

    def scales(self, layer: int, which: int) -> torch.Tensor:
        """f32 [num_blocks, n_kv, block_size]: a view."""
        return self._view(layer, which)[1]

    # -- append ---------------------------------------------------------------
    def rope_append(self, layer: int, q, k: torch.Tensor, v: torch.Tensor,
                    positions, inv_freq, slot_block: torch.Tensor,
                    slot_off: torch.Tensor, interleaved: bool = False,
                    attn_factor: float = 1.0, q_norm=None, k_norm=None,
                    eps: float = 1e-6, q_out=None):
        """rvkv_q8_rope_append: HipKvStorage.rope_append into the 8-bit
        cache."""
        return rope_append_call(self._L.rvkv_q8_rope_append, self, layer, q, k,
                                v, positions, inv_freq, slot_block, slot_off,
                                interleaved, attn_factor, q_norm, k_norm, eps,
                                q_out)

    def write_tokens(self, layer: int, block_ids: torch.Tensor,
                     offsets: torch.Tensor, k: torch.Tensor,
                     v: torch.Tensor) -> None:
        """HipKvStorage.write_tokens: k, v [n_tokens, n_kv, hd] as they are."""
        _need(k.numel() != 0, "kv_write: k/v len is 0")
        self.rope_append(layer, None, k, v, None, None, block_ids, offsets)

    # -- gather, copy-on-write ------------------------------------------------
    def gather(self, layer: int, plan: HipGatherPlan, out_k: torch.Tensor,
               out_v: torch.Tensor) -> None:
        """rvkv_q8_gather: [batch, n_kv, ctx_len, hd] into f32 or f16."""
        n = plan.batch * self.n_kv_heads * plan.ctx_len * self.head_dim
        _need(out_k.numel() == n and out_v.numel() == n and
              out_k.is_contiguous() and out_v.is_contiguous(),
              "kv_gather: output length must equal batch * n_kv_heads * "
              "ctx_len * head_dim")
        _need(out_k.dtype == out_v.dtype and out_k.dtype in _DT,
              "kv_gather: outputs must both be float32 or float16")
        _on(self, "kv_gather", (plan.block_idx, out_k, out_v))
        check(self._L.rvkv_q8_gather(
            self._pool, layer, _ptr(plan.block_idx), plan.batch,
            plan.max_blocks, plan.ctx_len, _ptr(out_k), _ptr(out_v),
            _DT[out_k.dtype]))

    def copy_blocks(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Copies src[i] -> dst[i] for all layers, K and V."""
        _need(src.numel() == dst.numel(),
              "copy_blocks: src and dst have different lengths")
        for t in (src, dst):
            _need(t.dtype == torch.int32 and t.is_contiguous(),
                  "copy_blocks: src and dst must be contiguous int32")
        _on(self, "copy_blocks", (src, dst))
        check(self._L.rvkv_q8_copy_blocks(self._pool, _ptr(src), _ptr(dst),
                                          src.numel()))

    # -- attention ------------------------------------------------------------
    def _check_attn(self, op, q, out, ints):
        shape, dtype = q.shape, q.dtype
        if (len(shape) != 3 or shape[2] != self.head_dim or dtype not in _DT or
                not q.is_contiguous()):
            raise RvkvError(f"{op}: q must be contiguous [rows, n_heads, "
                            "head_dim] float32 or float16")
        if out is None:
            out = torch.empty_like(q)
        elif (out.shape != shape or out.dtype != dtype or
              not out.is_contiguous()):
            raise RvkvError(f"{op}: out must match q")
        for t in ints:
            if t.dtype != torch.int32 or not t.is_contiguous():
                raise RvkvError(f"{op}: index tensors must be contiguous "
                                "int32")
        _on(self, op, (q, out, *ints))
        return out

    def _scratch(self, op, ws, need):
        if ws is None:
            if not need:
                return None
            ws = torch.empty(need, dtype=torch.uint8, device=self.device)
            # (the pool's stream may be another than torch's: the memory is
            # not handed out again before the work there is done)
            if torch.cuda.current_stream(self.device) != self.stream:
                ws.record_stream(self.stream)
            return ws
        if ws.device != self.device or not ws.is_contiguous():
            raise RvkvError(f"{op}: workspace must be contiguous and on the "
                            "storage's device")
        return ws

    def decode_workspace_bytes(self, batch: int, n_heads: int,
                               max_ctx_len: int, window: int = 0) -> int:
        return self._L.rvkv_q8_decode_workspace_bytes(
            self._pool, batch, n_heads, max_ctx_len, int(window or 0))

    def alloc_workspace(self, batch: int, n_heads: int, max_ctx_len: int,
                        window: int = 0) -> torch.Tensor:
        nbytes = self.decode_workspace_bytes(batch, n_heads, max_ctx_len,
                                             window)
        return torch.empty(max(nbytes, 256), dtype=torch.uint8,
                           device=self.device)

    def paged_decode(self, layer: int, q: torch.Tensor,
                     block_tables: torch.Tensor, ctx_lens: torch.Tensor,
                     max_ctx_len: int, out: Optional[torch.Tensor] = None,
                     ws: Optional[torch.Tensor] = None,
                     scale: Optional[float] = None,
                     window: int = 0) -> torch.Tensor:
        """rvkv_q8_paged_decode: HipKvStorage.paged_decode over the 8-bit
        cache, for f32 or f16 q (out has q's type)."""
        op = "paged_decode"
        out = self._check_attn(op, q, out, (block_tables, ctx_lens))
        batch, n_heads, hd = q.shape
        _need(block_tables.dim() == 2 and block_tables.shape[0] == batch,
              f"{op}: block_tables must be [batch, max_blocks]")
        _need(ctx_lens.numel() == batch,
              f"{op}: ctx_lens length must equal batch")
        window = int(window or 0)
        if ws is None:
            ws = self._scratch(op, None, self.decode_workspace_bytes(
                batch, n_heads, max_ctx_len, window))
        else:
            ws = self._scratch(op, ws, 0)
        check(self._L.rvkv_q8_paged_decode(
            self._pool, layer, q.data_ptr(), _DT[q.dtype],
            block_tables.data_ptr(), ctx_lens.data_ptr(), batch,
            block_tables.shape[1], n_heads, max_ctx_len,
            1.0 / math.sqrt(hd) if scale is None else scale, window,
            out.data_ptr(), None if ws is None else ws.data_ptr(),
            0 if ws is None else ws.numel() * ws.element_size()))
        return out

    def prefill_workspace_bytes(self, rows: int, batch: int, n_heads: int,
                                max_blocks: int, window: int = 0) -> int:
        return self._L.rvkv_q8_prefill_workspace_bytes(
            self._pool, rows, batch, n_heads, max_blocks, int(window or 0))

    def packed_prefill(self, layer: int, q: torch.Tensor,
                       row_start: torch.Tensor, block_tables: torch.Tensor,
                       pos_offset: torch.Tensor,
                       read_num_tokens: torch.Tensor,
                       out: Optional[torch.Tensor] = None,
                       ws: Optional[torch.Tensor] = None,
                       scale: Optional[float] = None,
                       window: int = 0) -> torch.Tensor:
        """rvkv_q8_packed_prefill: causal attention of several sequences' query
        rows, packed. q [rows, n_heads, hd] f32 or f16; row_start [batch + 1],
        block_tables [batch, max_blocks], pos_offset and read_num_tokens
        [batch] u32. Rows of no sequence are left as they were in out (an out
        made here holds anything there). ws: scratch of
        prefill_workspace_bytes(...), by default allocated here."""
        op = "packed_prefill"
        out = self._check_attn(op, q, out, (row_start, block_tables,
                                            pos_offset, read_num_tokens))
        batch = block_tables.shape[0] if block_tables.dim() == 2 else -1
        _need(batch >= 0, f"{op}: block_tables must be [batch, max_blocks]")
        _need(row_start.numel() == batch + 1,
              f"{op}: row_start must hold batch + 1 entries")
        _need(pos_offset.numel() == batch and read_num_tokens.numel() == batch,
              f"{op}: pos_offset/read_num_tokens length must equal batch")
        rows, n_heads, hd = q.shape
        wide, window = int(block_tables.shape[1]), int(window or 0)
        ws = self._scratch(op, ws, 0 if ws is not None else
                           self.prefill_workspace_bytes(rows, batch, n_heads,
                                                        wide, window))
        check(self._L.rvkv_q8_packed_prefill(
            self._pool, layer, q.data_ptr(), _DT[q.dtype],
            row_start.data_ptr(), rows, block_tables.data_ptr(),
            pos_offset.data_ptr(), read_num_tokens.data_ptr(), batch, wide,
            n_heads, 1.0 / math.sqrt(hd) if scale is None else scale, window,
            out.data_ptr(), None if ws is None else ws.data_ptr(),
            0 if ws is None else ws.numel() * ws.element_size()))
        return out
