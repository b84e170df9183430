"""The 8-bit key/value cache: torch owns device memory and the stream, the C ABI (fl_kv8_*) does the work.

    cache = KV8Cache(B, H, D, total_len, block_len=64, weights=True)
    op = KV8Attention(B, H, D, total_len, torch.float16, block_len=64, max_seq_len=1024)
    out = op.prefill(q, k, v, cache, freq_cis, attn_mask=mask)              # [B, H, S, D]
    out = op.decode(q, k, v, cache, freq_cis, start_pos=S)                  # [B, H*D]
    kept, rows = op.evict(cache, keep_blocks=8, recent_blocks=2, rows=S+1)  # in place
    k, v = op.read(cache, rows)                                             # values, [B, H, rows, D]
"""
from __future__ import annotations

import ctypes as C

import torch

from . import capi


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise capi.FlAttnError(capi.FL_ATTN_ERR_ARGUMENT, what)


# The handle of torch's current stream.  A decode step of a small batch takes less time on the GPU than its call on the host, and
# building a Stream object for its handle is a sixth of that call; the public way serves where torch lacks the short one.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


class KV8Cache:
    """The arrays of one layer: k, v int8 [B,H,L,D]; k_scale, v_scale float32 [B,H,L/block_len]; k_tail, v_tail float16
    [B,H,block_len,D]; weights float32 [B,H,L/block_len] or None."""

    def __init__(self, batch_size: int, head_num: int, size_per_head: int, total_len: int, block_len: int = 64,
                 weights: bool = False, device: str | torch.device = "cuda:0"):
        _need(block_len in (32, 64, 128) and total_len % block_len == 0, "block_len is 32, 64 or 128 and divides total_len")
        lead, n = (batch_size, head_num), total_len // block_len
        z = lambda dtype, *shape: torch.zeros(*lead, *shape, dtype=dtype, device=device)
        self._take(block_len, z(torch.int8, total_len, size_per_head), z(torch.int8, total_len, size_per_head),
                   z(torch.float32, n), z(torch.float32, n), z(torch.float16, block_len, size_per_head),
                   z(torch.float16, block_len, size_per_head), z(torch.float32, n) if weights else None)

    @classmethod
    def of(cls, block_len: int, k, v, k_scale, v_scale, k_tail, v_tail, weights=None) -> "KV8Cache":
        """A cache over tensors that the caller has."""
        self = cls.__new__(cls)
        self._take(block_len, k, v, k_scale, v_scale, k_tail, v_tail, weights)
        return self

    def _take(self, block_len, k, v, k_scale, v_scale, k_tail, v_tail, weights):
        _need(k.dim() == 4, "k is [B, H, L, D]")
        B, H, L, D = k.shape
        _need(block_len in (32, 64, 128) and L % block_len == 0, "block_len is 32, 64 or 128 and divides total_len")
        entries, tail = (B, H, L // block_len), (B, H, block_len, D)
        for name, t, dtype, shape in (("k", k, torch.int8, k.shape), ("v", v, torch.int8, k.shape),
                                      ("k_scale", k_scale, torch.float32, entries), ("v_scale", v_scale, torch.float32, entries),
                                      ("k_tail", k_tail, torch.float16, tail), ("v_tail", v_tail, torch.float16, tail),
                                      ("weights", weights, torch.float32, entries)):
            if name != "weights" or t is not None:
                _need(t.dtype == dtype and tuple(t.shape) == tuple(shape) and t.is_contiguous() and t.device == k.device,
                      f"{name} must be a contiguous {dtype} tensor {tuple(shape)} on {k.device}")
        self.block_len, self.shape, self.device = block_len, (B, H, L, D), k.device
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.k_tail, self.v_tail, self.weights = k_tail, v_tail, weights
        self.arrays = capi.Kv8CacheArrays(block_len=block_len, k=k.data_ptr(), v=v.data_ptr(), k_scale=k_scale.data_ptr(),
                                          v_scale=v_scale.data_ptr(), k_tail=k_tail.data_ptr(), v_tail=v_tail.data_ptr(),
                                          weights=None if weights is None else weights.data_ptr())
        self.ref = C.byref(self.arrays)


class KV8Attention:
    """Attention over caller-owned KV8Caches of one shape, with a workspace of its own: calls of one object come from one thread
    and go to one stream at a time.  dtype is the type of q, k_new, v_new (float32 or float16) and of what read() returns."""

    def __init__(self, batch_size: int, head_num: int, size_per_head: int, total_len: int, dtype: torch.dtype = torch.float16,
                 block_len: int = 64, max_seq_len: int = 1, nsplit: int = 0, softmax_scale: float = 0.0,
                 device: str | torch.device = "cuda:0"):
        self.lib = capi.load()
        if dtype not in (torch.float32, torch.float16):
            raise capi.FlAttnError(capi.FL_ATTN_ERR_DTYPE, "dtype must be float32 or float16")
        self.dtype, self.device = dtype, torch.device(device)
        if self.device.index is None:
            self.device = torch.device(self.device.type, torch.cuda.current_device())
        self._index = self.device.index
        self.block_len, self.max_seq_len = block_len, max_seq_len
        self.shape = (batch_size, head_num, total_len, size_per_head)
        self.desc = capi.AttnDesc(batch_size, head_num, size_per_head, total_len,
                                  capi.FL_ATTN_F16 if dtype == torch.float16 else capi.FL_ATTN_F32, nsplit, softmax_scale, 0)
        self._desc = C.byref(self.desc)
        n = C.c_size_t(0)
        with torch.cuda.device(self.device):
            capi.check(self.lib.fl_kv8_workspace_bytes(self._desc, block_len, max_seq_len, C.byref(n)))
            self.workspace = torch.empty(n.value, dtype=torch.uint8, device=self.device)
            stream = torch.cuda.current_stream(self.device)
            capi.check(self.lib.fl_kv8_workspace_init(self._desc, block_len, max_seq_len, self.workspace.data_ptr(), n.value,
                                                      stream.cuda_stream))
            stream.synchronize()  # the counters are zero for whatever stream the calls are made on
        self.io = capi.AttnIO(workspace=self.workspace.data_ptr(), workspace_bytes=n.value)
        self._io = C.byref(self.io)
        self.evict_args = capi.Kv8EvictArgs()
        self._evict_args = C.byref(self.evict_args)

    def _enqueue(self, call, *args) -> None:
        """call(*args, stream) on torch's current stream of this object's device."""
        stream = _raw_stream(self._index)
        if _current_device() == self._index:
            status = call(*args, stream)
        else:
            with torch.cuda.device(self.device):
                status = call(*args, stream)
        if status:
            capi.check(status)

    def _input(self, name: str, t: torch.Tensor, shape, dtype) -> int:
        if t.dtype is not dtype or t.shape != shape or not t.is_contiguous() or t.get_device() != self._index:
            _need(False, f"{name} must be a contiguous {dtype} tensor {shape} on {self.device}")
        return t.data_ptr()

    def _vector(self, name: str, t: torch.Tensor | None, dtype, numel: int) -> int | None:
        if t is None:
            return None
        if t.dtype is not dtype or t.numel() != numel or not t.is_contiguous() or t.get_device() != self._index:
            _need(False, f"{name} must hold {numel} contiguous {dtype} on {self.device}")
        return t.data_ptr()

    def _cache(self, cache: KV8Cache, shape=None) -> None:
        if cache.shape != (shape or self.shape) or cache.block_len != self.block_len or cache.device != self.device:
            B, H, L, D = shape or self.shape
            _need(False, f"the cache must be [B, H, L, D] = {(B, H, L, D)} in blocks of {self.block_len} on {self.device}")

    def _fill(self, q, k_new, v_new, seq_len, freq_cis, rope_rows, attn_mask, last, scales, out, out_shape, out_int8, out_scale):
        """Everything of io that both phases share; rope_rows: table rows the call uses (0: not known here), last: its last
        row of the cache."""
        B, H, _, D = self.shape
        io, shape = self.io, (B, seq_len, H, D)
        dtype = self.dtype if scales is None else torch.int32
        index = self._index
        if (q.dtype is not dtype or k_new.dtype is not dtype or v_new.dtype is not dtype or q.shape != shape or k_new.shape != shape
                or v_new.shape != shape or not q.is_contiguous() or not k_new.is_contiguous() or not v_new.is_contiguous()
                or q.get_device() != index or k_new.get_device() != index or v_new.get_device() != index):
            for name, t in (("q", q), ("k_new", k_new), ("v_new", v_new)):  # which one
                self._input(name, t, shape, dtype)
        io.q, io.k_new, io.v_new = q.data_ptr(), k_new.data_ptr(), v_new.data_ptr()
        rows = freq_cis.shape[0]
        if rows < rope_rows:
            _need(False, f"freq_cis has {rows} rows, the call uses {rope_rows}")
        io.freq_cis = self._input("freq_cis", freq_cis, (rows, D), torch.float32)
        if attn_mask is None:
            io.attn_mask = None
        else:
            if attn_mask.dtype is not torch.float32 or attn_mask.dim() != 2 or attn_mask.stride(1) != 1 or attn_mask.get_device() != self._index:
                _need(False, f"attn_mask must be float32 [rows, columns], columns contiguous, on {self.device}")
            n, m = attn_mask.shape
            if m <= last or (n != 1 and n <= last):
                _need(False, f"attn_mask is {n} x {m}, the call uses row and column {last}")
            io.attn_mask, io.mask_ld = attn_mask.data_ptr(), 0 if n == 1 else attn_mask.stride(0)
        if scales is None:
            io.qkv_inp_scale = io.q_weight_scale = io.k_weight_scale = io.v_weight_scale = None
        else:
            io.qkv_inp_scale = self._vector("qkv_inp_scale", scales[0], torch.float32, B * seq_len)
            io.q_weight_scale, io.k_weight_scale, io.v_weight_scale = (
                self._vector(n, t, torch.float32, H * D) for n, t in zip(("q_weight_scale", "k_weight_scale", "v_weight_scale"), scales[1:]))
        if out is None and out_int8 is None:
            out = torch.empty(*out_shape, dtype=torch.float32, device=self.device)  # (a tuple takes 0.3 us longer)
            io.out = out.data_ptr()
        else:
            io.out = None if out is None else self._input("out", out, out_shape, torch.float32)
        io.out_int8 = None if out_int8 is None else self._vector("out_int8", out_int8, torch.int8, B * seq_len * H * D)
        io.out_scale = None if out_scale is None else self._vector("out_scale", out_scale, torch.float32, B * seq_len)
        return out

    def decode(self, q, k_new, v_new, cache: KV8Cache, freq_cis, start_pos: int = 0, attn_mask=None, start_pos_per_seq=None,
               max_start_pos: int = -1, rope_row: int = capi.FL_ATTN_ROPE_AT_POSITION, rope_row_per_seq=None, scales=None,
               out=None, out_int8=None, out_scale=None):
        """One decode step: RoPE, append at row start_pos, attention over rows [0, start_pos].  q, k_new, v_new [B,1,H,D];
        returns out [B, H*D] float32.  start_pos_per_seq: int32 [B] on the device, up to max_start_pos.  rope_row or
        rope_row_per_seq: the table rows where they are not the positions (after an eviction).  scales: (qkv_inp_scale,
        q/k/v_weight_scale) for int32 accumulators."""
        B, H, L, D = self.shape
        self._cache(cache)
        last = start_pos if start_pos_per_seq is None else (L - 1 if max_start_pos < 0 else max_start_pos)
        # (rows named on the device are looked at there)
        rope_rows = 0 if rope_row_per_seq is not None else (last if rope_row < 0 else rope_row) + 1
        out = self._fill(q, k_new, v_new, 1, freq_cis, rope_rows, attn_mask, last, scales, out, (B, H * D), out_int8, out_scale)
        io = self.io
        io.start_pos_per_seq = None if start_pos_per_seq is None else self._vector("start_pos_per_seq", start_pos_per_seq, torch.int32, B)
        io.start_pos, io.max_start_pos, io.rope_row = start_pos, max_start_pos, rope_row
        io.flags = capi.FL_ATTN_IO_WORKSPACE_READY
        self._enqueue(self.lib.fl_kv8_decode_forward, self._desc, cache.ref, self._io,
                      None if rope_row_per_seq is None else self._vector("rope_row_per_seq", rope_row_per_seq, torch.int32, B), freq_cis.shape[0])
        return out

    def prefill(self, q, k_new, v_new, cache: KV8Cache, freq_cis, start_pos: int = 0, attn_mask=None, mask_tile_classes=None,
                rope_row: int = capi.FL_ATTN_ROPE_AT_POSITION, weight_queries: int = 0, scales=None, out=None, out_int8=None,
                out_scale=None, seq_len_per_seq=None):
        """The prompt phase: q, k_new, v_new [B,S,H,D] at positions start_pos .. start_pos+S-1 (causal by the mask); returns
        out [B,H,S,D] float32.  seq_len_per_seq: int32 [B] on the device, the tokens that each sequence brings of them: the
        padding behind is not stored, its output rows are zeros.  With cache.weights (up to size_per_head 128), the last weight_queries
        queries add theirs (0: all); beyond that size, zero cache.weights and pass KV8Cache.of() the other arrays alone.
        mask_tile_classes: PrefillAttention.classify_mask of the whole [L, L] mask."""
        B, H, L, D = self.shape
        S = q.shape[1] if q.dim() == 4 else 0
        _need(0 < S <= self.max_seq_len, f"q is [B, S, H, D] with 1 <= S <= max_seq_len = {self.max_seq_len}")
        self._cache(cache)
        out = self._fill(q, k_new, v_new, S, freq_cis, (start_pos if rope_row < 0 else rope_row) + S, attn_mask, start_pos + S - 1,
                         scales, out, (B, H, S, D), out_int8, out_scale)
        io = self.io
        io.start_pos_per_seq = None
        io.start_pos, io.max_start_pos, io.rope_row, io.flags = start_pos, -1, rope_row, 0
        if mask_tile_classes is None:
            io.mask_tile_classes = None
        else:
            n = -(-L // 32)
            io.mask_tile_classes = self._vector("mask_tile_classes", mask_tile_classes, torch.uint8, n * -(-n // 4) * 4)
        self._enqueue(self.lib.fl_kv8_prefill_forward, self._desc, cache.ref, self._io, S,
                      self._vector("seq_len_per_seq", seq_len_per_seq, torch.int32, B), weight_queries)
        return out

    def read(self, cache: KV8Cache, rows: int, rows_per_seq=None):
        """The values of rows [0, rows): k, v [B,H,rows,D] in dtype.  rows: of every sequence, or rows_per_seq int32 [B], how
        many each holds; zeros from there on."""
        B, H, _, D = self.shape
        self._cache(cache)
        k = torch.empty(B, H, max(rows, 0), D, dtype=self.dtype, device=self.device)
        v = torch.empty_like(k)
        self._enqueue(self.lib.fl_kv8_read, self._desc, cache.ref, rows, self._vector("rows_per_seq", rows_per_seq, torch.int32, B),
                      k.data_ptr(), v.data_ptr())
        return k, v

    def evict(self, cache: KV8Cache, keep_blocks: int, recent_blocks: int, rows: int, rows_per_seq=None, into: KV8Cache | None = None):
        """Keeps the last recent_blocks complete blocks and those of the largest weight, keep_blocks in all, in place or in
        `into` (its total_len may differ).  rows: rows in the cache, or rows_per_seq int32 [B].  Returns (kept [B,H,keep_blocks]
        int32, rows [B] int32 after the eviction)."""
        B, H, _, D = self.shape
        self._cache(cache)
        to = into if into is not None else cache
        self._cache(to, (B, H, to.shape[2], D))
        _need(cache.weights is not None and to.weights is not None, "the caches must have weights")
        kept = torch.empty(B, H, max(keep_blocks, 0), dtype=torch.int32, device=self.device)
        rows_out = torch.empty(B, dtype=torch.int32, device=self.device)
        args = self.evict_args
        args.rows, args.rows_per_seq = rows, self._vector("rows_per_seq", rows_per_seq, torch.int32, B)
        args.keep_blocks, args.recent_blocks, args.to_total_len = keep_blocks, recent_blocks, to.shape[2]
        args.kept, args.rows_out = kept.data_ptr(), rows_out.data_ptr()
        self._enqueue(self.lib.fl_kv8_evict, self._desc, cache.ref, to.ref, self._evict_args)
        return kept, rows_out
