"""Host-side API of the device-resident paged KV pool.

A CudaKvPool owns the HBM arenas that replace PagedKvPool's page storage
(worker/cpp/inferlab_runtime.cpp:649-1026). Block ids, block tables and
context lengths stay the caller's business, as in the reference where
the pool's host policy hands out page ids and the attention only follows the
table (docs/rfcs/0014-paged-kv-cache-prefix-ownership.md, "Logical block
tables"). Device arrays are torch tensors here only as HBM plumbing; every
kernel is a call into libinferlab_attention_cuda.so.
"""
from __future__ import annotations

import ctypes
import math
import weakref

import torch

from . import _lib
from .attention import AttentionError

KV_FP32, KV_F16, KV_BF16 = 0, 1, 2
TORCH_DTYPES = {KV_FP32: torch.float32, KV_F16: torch.float16, KV_BF16: torch.bfloat16}
_TYPESTR = {KV_FP32: "<f4", KV_F16: "<f2", KV_BF16: "<u2"}


def _check(status: int, error) -> None:
    if status != 0:
        raise AttentionError(error.value.decode())


def _vp(tensor):
    return None if tensor is None else ctypes.c_void_p(tensor.data_ptr())


def _stream_handle(device: int, stream) -> ctypes.c_void_p:
    if stream is None:
        stream = torch.cuda.current_stream(device)
    return ctypes.c_void_p(stream.cuda_stream)


def _torch_stream(device: int, stream) -> torch.cuda.Stream:
    """The stream a call runs on (default: the current one) as torch's own."""
    if stream is None:
        return torch.cuda.current_stream(device)
    if isinstance(stream, torch.cuda.Stream):
        return stream
    if stream.cuda_stream in (0, 1):  # both name the legacy stream
        return torch.cuda.default_stream(device)
    return torch.cuda.ExternalStream(stream.cuda_stream, device=device)


def _made(shape, dtype, device: int, stream) -> torch.Tensor:
    """Memory that a call fills on `stream`, allocated there: the current stream may still use what
    its own allocations reuse. It is then read on the current stream, as a rule, behind `stream`."""
    if stream is None or stream.cuda_stream == torch._C._cuda_getCurrentRawStream(device):
        return torch.empty(shape, dtype=dtype, device=device)
    here, there = torch.cuda.current_stream(device), _torch_stream(device, stream)
    near = torch.cuda.current_device() == device
    with _On(there, here) if near else torch.cuda.stream(there):
        made = torch.empty(shape, dtype=dtype, device=device)
    made.record_stream(here)
    return made


class _On:
    """torch.cuda.stream for two streams of the current device, of which `here` is current: what the
    general form costs is as much as a call."""

    def __init__(self, stream, here):
        self.stream, self.here = stream, here

    def __enter__(self):
        s = self.stream
        torch._C._cuda_setStream(stream_id=s.stream_id, device_index=s.device_index,
                                 device_type=s.device_type)

    def __exit__(self, *exc):
        s = self.here
        torch._C._cuda_setStream(stream_id=s.stream_id, device_index=s.device_index,
                                 device_type=s.device_type)


class _DeviceView:
    """Exposes a raw device range through __cuda_array_interface__. The tensor made from it keeps
    it, and so `owner`, whose memory it is, alive."""

    def __init__(self, ptr: int, shape, typestr: str, owner=None):
        self.owner = owner
        self.__cuda_array_interface__ = {
            "shape": tuple(shape), "typestr": typestr, "data": (ptr, False), "version": 3,
            "strides": None,
        }


def _require(tensor: torch.Tensor, name: str, dtype, device: int) -> torch.Tensor:
    if not isinstance(tensor, torch.Tensor):
        raise AttentionError(f"{name} must be a torch tensor on cuda:{device}")
    if tensor.device.type != "cuda" or tensor.device.index != device:
        raise AttentionError(f"{name} must live on cuda:{device}")
    if dtype is not None and tensor.dtype != dtype:
        raise AttentionError(f"{name} must have dtype {dtype}")
    if not tensor.is_contiguous():
        raise AttentionError(f"{name} must be contiguous")
    return tensor


_COUNTER_FRONT = 65536  # bytes at the front of a workspace that must start at zero


def _expect(tensor, name: str, dtype, device: int) -> int:
    """_require for the per-token calls, whose time is the host's: one pass over what a good
    tensor satisfies, the messages only for others. Returns the address."""
    if type(tensor) is not torch.Tensor or tensor.dtype is not dtype or \
            tensor.get_device() != device or not tensor.is_contiguous():
        _require(tensor, name, dtype, device)
    return tensor.data_ptr()


def _raw_stream(device: int, stream) -> int:
    return torch._C._cuda_getCurrentRawStream(device) if stream is None else stream.cuda_stream


class CudaKvPool:
    """HBM block pool: arenas [num_blocks][kv_heads][block_tokens][head_dim].

    kv_bits=4 holds the rows in 4 bits (inferlab_cuda_pool_create_kv4): dtype is
    then the 16-bit type that rows are rounded to before they are quantised and
    that queries, outputs and gathered rows have; block_tokens is a multiple of
    16 and head_dim 64 or 128. append, append_rotary, gather, gather_rows,
    decode, prefill, output_project and copy_blocks work on such a pool."""

    def __init__(self, device: int, dtype: int, num_blocks: int, block_tokens: int,
                 kv_heads: int, head_dim: int, kv_bits: int | None = None):
        self._lib = _lib.lib()
        if kv_bits not in (None, 4):
            raise AttentionError("paged KV kv_bits must be None or 4")
        create = (self._lib.inferlab_cuda_pool_create if kv_bits is None
                  else self._lib.inferlab_cuda_pool_create_kv4)
        handle = ctypes.c_void_p()
        error = _lib.error_buffer()
        _check(create(device, dtype, num_blocks, block_tokens, kv_heads, head_dim,
                      ctypes.byref(handle), error, len(error)), error)
        self._handle = handle
        self.kv_bits = kv_bits
        info = _lib.InferlabCudaPoolInfo()
        _check(self._lib.inferlab_cuda_pool_info(handle, ctypes.byref(info), error, len(error)),
               error)
        self.device = info.device
        self.dtype = info.dtype
        self.num_blocks = info.num_blocks
        self.block_tokens = info.block_tokens
        self.kv_heads = info.kv_heads
        self.head_dim = info.head_dim
        self.element_bytes = info.element_bytes
        self.block_bytes = info.block_bytes
        self.arena_bytes = info.arena_bytes
        # One token row of K and V over all kv-heads.
        self.row_bytes = info.block_bytes // info.block_tokens * (1 if kv_bits == 4 else 2)
        self._key_ptr = info.key_arena
        self._value_ptr = info.value_arena
        self._workspaces: dict = {}  # by stream
        self._fitting: dict = {}  # (stream, batch shape) -> a workspace that fits it
        self._arena_shape = (self.num_blocks, self.kv_heads, self.block_tokens, self.head_dim)
        self._views: dict = {}  # weak: a view keeps the pool, not the pool its views

    # -- lifetime -----------------------------------------------------------
    def close(self) -> None:
        if getattr(self, "_handle", None) is not None and self._handle.value:
            self._lib.inferlab_cuda_pool_destroy(self._handle)
            self._handle = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    # -- views ----------------------------------------------------------------
    @property
    def arena(self) -> torch.Tensor:
        """A 4-bit pool's packed arena as bytes [num_blocks][kv_heads][block_tokens / 16][tile]
        (no copy; it keeps the pool alive, until close(); the layout is in the C header)."""
        if self.kv_bits != 4:
            raise AttentionError("only a 4-bit pool has a packed arena")
        tiles = self.block_tokens // 16
        shape = (self.num_blocks, self.kv_heads, tiles,
                 self.block_bytes // (self.kv_heads * tiles))
        return torch.as_tensor(_DeviceView(self._key_ptr, shape, "|u1", self),
                               device=f"cuda:{self.device}")

    def _arena(self, ptr: int) -> torch.Tensor:
        if self.kv_bits == 4:
            raise AttentionError("a 4-bit pool has one packed arena (arena)")
        known = self._views.get(ptr)
        view = None if known is None else known()
        # A holder may have turned it into another view in place.
        if view is None or view.shape != self._arena_shape or not view.is_contiguous() or \
                view.data_ptr() != ptr or view.requires_grad:
            view = torch.as_tensor(_DeviceView(ptr, self._arena_shape, _TYPESTR[self.dtype], self),
                                   device=f"cuda:{self.device}")
            if self.dtype == KV_BF16:
                view = view.view(TORCH_DTYPES[self.dtype])
            self._views[ptr] = weakref.ref(view)
        return view

    @property
    def key_arena(self) -> torch.Tensor:
        """A torch view of the key arena (no copy; it keeps the pool alive, until close()). While one
        is held the same tensor is returned again, unless it was reshaped in place."""
        return self._arena(self._key_ptr)

    @property
    def value_arena(self) -> torch.Tensor:
        return self._arena(self._value_ptr)

    # -- kernels ----------------------------------------------------------------
    def synchronize(self, stream=None, timeout_ms: int = 0) -> None:
        """Bounded wait on the stream, then raise any error a kernel recorded."""
        error = _lib.error_buffer()
        _check(self._lib.inferlab_cuda_pool_synchronize(
            self._handle, _stream_handle(self.device, stream), timeout_ms, error, len(error)),
            error)

    def append(self, key_rows: torch.Tensor, value_rows: torch.Tensor,
               row_sequences: torch.Tensor, positions: torch.Tensor, block_tables: torch.Tensor,
               stream=None) -> None:
        """Write token rows [n][kv_heads][head_dim] at (sequence, position) via the tables."""
        dev = self.device
        row_dtype = KV_FP32 if key_rows.dtype == torch.float32 else self.dtype
        if key_rows.dtype not in (torch.float32, TORCH_DTYPES[self.dtype]):
            raise AttentionError("paged KV row dtype must be FP32 or the pool dtype")
        _require(key_rows, "key_rows", key_rows.dtype, dev)
        _require(value_rows, "value_rows", key_rows.dtype, dev)
        _require(row_sequences, "row_sequences", torch.int32, dev)
        _require(positions, "positions", torch.int32, dev)
        _require(block_tables, "block_tables", torch.int32, dev)
        rows = key_rows.shape[0]
        if key_rows.numel() != rows * self.kv_heads * self.head_dim or \
                value_rows.shape != key_rows.shape or row_sequences.numel() != rows or \
                positions.numel() != rows:
            raise AttentionError("paged KV append shapes do not match the pool")
        error = _lib.error_buffer()
        _check(self._lib.inferlab_cuda_kv_append(
            self._handle, _vp(key_rows), _vp(value_rows), row_dtype, _vp(row_sequences),
            _vp(positions), rows, _vp(block_tables), block_tables.shape[-1],
            _stream_handle(dev, stream), error, len(error)), error)

    def _rows(self, tensor: torch.Tensor, name: str, dtype, heads: int | None) -> int:
        """Checks token rows [n][heads][head_dim], heads and dims contiguous (a view of a wider
        projection output is fine); returns the elements between rows."""
        if not isinstance(tensor, torch.Tensor) or tensor.get_device() != self.device:
            raise AttentionError(f"{name} must live on cuda:{self.device}")
        if tensor.dtype is not dtype:
            raise AttentionError(f"{name} must have dtype {dtype}")
        shape = tensor.shape
        if len(shape) != 3 or shape[2] != self.head_dim or \
                (heads is not None and shape[1] != heads):
            raise AttentionError("paged KV append shapes do not match the pool")
        step, head, dim = tensor.stride()
        if (dim != 1 or (shape[1] > 1 and head != self.head_dim)) and tensor.numel():
            raise AttentionError(f"{name} must have contiguous heads")
        return step

    def append_rotary(self, queries: torch.Tensor | None, key_rows: torch.Tensor,
                      value_rows: torch.Tensor, cos_sin: torch.Tensor | None,
                      row_sequences: torch.Tensor, positions: torch.Tensor,
                      block_tables: torch.Tensor, interleaved: bool = False,
                      q_out: torch.Tensor | None = None, stream=None) -> torch.Tensor | None:
        """append with the position rotation on the way: Q and K rows are rotated by row
        positions[r] of cos_sin (fp32 [positions][rotary_dim]: cosines, then sines; None for no
        rotation), K and V go to the pool at (row_sequences[r], positions[r]), and the rotated Q is
        returned (queries None: nothing). Pairs are (i, i + rotary_dim / 2), or (2i, 2i + 1) when
        interleaved. Rows [n][heads][head_dim] are fp32 or the pool's type and may be views of one
        projection output; q_out (default: like the queries) may be either type. Rows of sequence
        -1 are padding: skipped, their q_out rows left as they were
        (inferlab_cuda_kv_append_rotary)."""
        dev = self.device
        dtype = key_rows.dtype
        pool_dtype = TORCH_DTYPES[self.dtype]
        if dtype is not torch.float32 and dtype is not pool_dtype:
            raise AttentionError("paged KV row dtype must be FP32 or the pool dtype")
        key_stride = self._rows(key_rows, "key_rows", dtype, self.kv_heads)
        value_stride = self._rows(value_rows, "value_rows", dtype, self.kv_heads)
        rows = key_rows.shape[0]
        sequences_at = _expect(row_sequences, "row_sequences", torch.int32, dev)
        positions_at = _expect(positions, "positions", torch.int32, dev)
        tables_at = _expect(block_tables, "block_tables", torch.int32, dev)
        if value_rows.shape[0] != rows or row_sequences.numel() != rows or \
                positions.numel() != rows or block_tables.dim() != 2:
            raise AttentionError("paged KV append shapes do not match the pool")
        angles_at, angle_rows, rotary_dim = None, 0, 0
        if cos_sin is not None:
            angles_at = _expect(cos_sin, "cos_sin", torch.float32, dev)
            if cos_sin.dim() != 2:
                raise AttentionError("cos_sin must be [positions][rotary_dim]")
            angle_rows, rotary_dim = cos_sin.shape
        queries_at, query_stride, q_heads, out_at, out_type = None, 0, 0, None, 0
        if queries is not None:
            query_stride = self._rows(queries, "queries", dtype, None)
            if queries.shape[0] != rows:
                raise AttentionError("paged KV append shapes do not match the pool")
            if q_out is None:
                q_out = _made(queries.shape, dtype, dev, stream)
            out_dtype = q_out.dtype
            out_at = _expect(q_out, "q_out", out_dtype, dev)
            if q_out.shape != queries.shape or \
                    (out_dtype is not torch.float32 and out_dtype is not pool_dtype):
                raise AttentionError("q_out must be shaped like the queries, FP32 or the pool dtype")
            queries_at, q_heads = queries.data_ptr(), queries.shape[1]
            out_type = KV_FP32 if out_dtype is torch.float32 else self.dtype
        elif q_out is not None:
            raise AttentionError("q_out needs queries")
        call = _lib.InferlabCudaRotaryAppend(
            queries_at, key_rows.data_ptr(), value_rows.data_ptr(),
            KV_FP32 if dtype is torch.float32 else self.dtype, q_heads, query_stride, key_stride,
            value_stride, angles_at, angle_rows, rotary_dim, 1 if interleaved else 0, sequences_at,
            positions_at, rows, tables_at, block_tables.shape[0], block_tables.shape[1], out_at,
            out_type, 0)
        error = _lib.call_error_buffer()
        if self._lib.inferlab_cuda_kv_append_rotary(self._handle, ctypes.byref(call),
                                                    _raw_stream(dev, stream), error, 512):
            raise AttentionError(error.value.decode())
        return q_out

    def project_append(self, hidden: torch.Tensor, weights: torch.Tensor, q_heads: int,
                       row_sequences: torch.Tensor, positions: torch.Tensor,
                       block_tables: torch.Tensor, q_out: torch.Tensor | None = None,
                       stream=None) -> torch.Tensor:
        """Q/K/V projection of hidden [tokens][model_dim] by the stacked
        weights [(q_heads + 2 kv_heads) head_dim][model_dim] (pool type, F16 or
        BF16 pools): returns Q [tokens][q_heads][head_dim] and writes every
        token's K/V rows into the pool at (row_sequences[t], positions[t])
        (inferlab_cuda_qkv_project_append)."""
        dev = self.device
        dtype = TORCH_DTYPES.get(self.dtype)
        _require(hidden, "hidden", dtype, dev)
        _require(weights, "weights", dtype, dev)
        _require(row_sequences, "row_sequences", torch.int32, dev)
        _require(positions, "positions", torch.int32, dev)
        _require(block_tables, "block_tables", torch.int32, dev)
        tokens, model_dim = hidden.shape
        if weights.shape != ((q_heads + 2 * self.kv_heads) * self.head_dim, model_dim) or \
                row_sequences.numel() != tokens or positions.numel() != tokens or \
                block_tables.dim() != 2:
            raise AttentionError("projection shapes do not match the pool")
        if q_out is None:
            q_out = _made((tokens, q_heads, self.head_dim), dtype, dev, stream)
        _require(q_out, "q_out", dtype, dev)
        error = _lib.error_buffer()
        _check(self._lib.inferlab_cuda_qkv_project_append(
            self._handle, _vp(hidden), _vp(weights), tokens, model_dim, q_heads,
            _vp(row_sequences), _vp(positions), _vp(block_tables), block_tables.shape[0],
            block_tables.shape[1], _vp(q_out), _stream_handle(dev, stream), error, len(error)),
            error)
        return q_out

    def output_project(self, attention: torch.Tensor, weights: torch.Tensor,
                       residual: torch.Tensor | None = None, out: torch.Tensor | None = None,
                       stream=None) -> torch.Tensor:
        """out = residual + attention @ weights.T on the tensor cores
        (inferlab_cuda_output_project): attention [tokens][in_dim] fp32 or
        the pool type, weights [out_dim][in_dim] in the pool type, residual /
        out [tokens][out_dim] fp32."""
        dev = self.device
        dtype = TORCH_DTYPES.get(self.dtype)
        if attention.dtype not in (torch.float32, dtype):
            raise AttentionError("projection input dtype must be FP32 or the pool dtype")
        _require(attention, "attention", attention.dtype, dev)
        _require(weights, "weights", dtype, dev)
        tokens, in_dim = attention.shape
        out_dim = weights.shape[0]
        if weights.shape[1] != in_dim:
            raise AttentionError("projection shapes do not match")
        if residual is not None:
            _require(residual, "residual", torch.float32, dev)
            if residual.shape != (tokens, out_dim):
                raise AttentionError("projection shapes do not match")
        if out is None:
            out = _made((tokens, out_dim), torch.float32, dev, stream)
        _require(out, "out", torch.float32, dev)
        a_dtype = KV_FP32 if attention.dtype == torch.float32 else self.dtype
        error = _lib.error_buffer()
        _check(self._lib.inferlab_cuda_output_project(
            self._handle, _vp(attention), a_dtype, _vp(weights),
            None if residual is None else _vp(residual), tokens, in_dim, out_dim, _vp(out),
            _stream_handle(dev, stream), error, len(error)), error)
        return out

    def gather(self, block_table: torch.Tensor, tokens: int, stream=None):
        """Contiguous copies [tokens][kv_heads][head_dim] of one sequence's K and V."""
        dev = self.device
        _require(block_table, "block_table", torch.int32, dev)
        if block_table.numel() != (tokens + self.block_tokens - 1) // self.block_tokens:
            raise AttentionError("paged KV block table length is inconsistent")
        shape = (tokens, self.kv_heads, self.head_dim)
        keys = _made(shape, TORCH_DTYPES[self.dtype], dev, stream)
        values = _made(shape, TORCH_DTYPES[self.dtype], dev, stream)
        error = _lib.error_buffer()
        _check(self._lib.inferlab_cuda_kv_gather(
            self._handle, _vp(block_table), tokens, _vp(keys), _vp(values),
            _stream_handle(dev, stream), error, len(error)), error)
        return keys, values

    def gather_rows(self, row_sequences: torch.Tensor, positions: torch.Tensor,
                    block_tables: torch.Tensor, stream=None):
        """The rows at (row_sequences[r], positions[r]): K and V [rows][kv_heads][head_dim] in the
        pool's type (a 4-bit pool's row type). Rows of sequence -1 are padding and left unset
        (inferlab_cuda_kv_gather_rows)."""
        dev = self.device
        sequences_at = _expect(row_sequences, "row_sequences", torch.int32, dev)
        positions_at = _expect(positions, "positions", torch.int32, dev)
        tables_at = _expect(block_tables, "block_tables", torch.int32, dev)
        rows = row_sequences.numel()
        if positions.numel() != rows or block_tables.dim() != 2:
            raise AttentionError("paged KV gather shapes do not match")
        keys, values = _made((2, rows, self.kv_heads, self.head_dim), TORCH_DTYPES[self.dtype], dev,
                             stream).unbind()
        error = _lib.call_error_buffer()
        if self._lib.inferlab_cuda_kv_gather_rows(
                self._handle, sequences_at, positions_at, rows, tables_at, block_tables.shape[0],
                block_tables.shape[1], keys.data_ptr(), values.data_ptr(),
                _raw_stream(dev, stream), error, 512):
            raise AttentionError(error.value.decode())
        return keys, values

    def workspace_size(self, num_seqs: int, q_heads: int, max_context_len: int,
                       max_query_count: int = 1) -> int:
        if self.kv_bits == 4:
            return int(self._lib.inferlab_cuda_kv4_workspace_size(
                self._handle, num_seqs, q_heads, max_query_count, max_context_len))
        return int(self._lib.inferlab_cuda_paged_decode_workspace_size(
            self._handle, num_seqs, q_heads, max_context_len))

    def make_workspace(self, num_seqs: int, q_heads: int, max_context_len: int,
                       stream=None, max_query_count: int = 1) -> torch.Tensor:
        """A zero-initialised decode workspace for this batch shape (max_query_count: the prefill
        of a 4-bit pool) and every smaller one."""
        size = max(16, self.workspace_size(num_seqs, q_heads, max_context_len, max_query_count))
        ws = _made(size, torch.uint8, self.device, stream)
        error = _lib.error_buffer()
        _check(self._lib.inferlab_cuda_paged_decode_workspace_init(
            _vp(ws), size, _stream_handle(self.device, stream), error, len(error)), error)
        return ws

    def set_decode_split(self, blocks_per_split: int) -> None:
        """Fixes later decodes' split length at blocks_per_split 16-token
        blocks (0: the planner chooses, the default). A tuning and test knob
        (inferlab_cuda_pool_set_decode_split)."""
        self._fitting.clear()
        error = _lib.error_buffer()
        _check(self._lib.inferlab_cuda_pool_set_decode_split(
            self._handle, int(blocks_per_split), error, len(error)), error)

    def _own_workspace(self, raw, stream, num_seqs, q_heads, max_query_count, max_context_len):
        """A workspace for a batch shape: the pool's own of the stream, as calls on one stream run
        in order and may share it, calls on two streams would race on its split counters and
        partials. A capture gets one of its own, zeroed by the graph, so that graphs replayed side
        by side share none and none outlives what it was captured with."""
        shape = (raw, num_seqs, q_heads, max_query_count, max_context_len)
        capturing = (torch.cuda.is_current_stream_capturing() if stream is None
                     else self._lib.inferlab_cuda_stream_is_capturing(raw) != 0)
        if not capturing:
            known = self._fitting.get(shape)
            if known is not None:
                return known
        need = self.workspace_size(num_seqs, q_heads, max_context_len, max_query_count)
        used = _torch_stream(self.device, stream)
        with torch.cuda.stream(used):  # the allocation belongs to that stream
            if capturing:
                return self._zeroed(need, used)
            ws = self._workspaces.get(raw)
            if ws is None or ws.numel() < need:
                ws = self._zeroed(need, used)
                self._workspaces[raw] = ws
                self._fitting.clear()  # nothing keeps the outgrown one
        if len(self._fitting) > 1024:
            self._fitting.clear()
        self._fitting[shape] = ws
        return ws

    def _zeroed(self, size: int, stream) -> torch.Tensor:
        """A workspace whose split counters, all in front, the (current) stream makes zero."""
        ws = torch.empty(max(16, size), dtype=torch.uint8, device=f"cuda:{self.device}")
        error = _lib.error_buffer()
        _check(self._lib.inferlab_cuda_paged_decode_workspace_init(
            _vp(ws), min(ws.numel(), _COUNTER_FRONT), ctypes.c_void_p(stream.cuda_stream), error,
            len(error)), error)
        return ws

    def decode(self, queries: torch.Tensor, block_tables: torch.Tensor,
               context_lens: torch.Tensor, max_context_len: int | None = None,
               out: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
               stream=None) -> torch.Tensor:
        """One decode step: queries [num_seqs][q_heads][head_dim] fp32 -> fp32 output. A 4-bit
        pool also takes queries of its row type and returns the queries' type; its context length
        0 is a slot without a sequence, whose output row is zero (inferlab_cuda_kv4_decode)."""
        dev = self.device
        if self.kv_bits == 4:
            return self._kv4_decode(queries, block_tables, context_lens, max_context_len, out,
                                    workspace, stream)
        _require(queries, "queries", torch.float32, dev)
        _require(block_tables, "block_tables", torch.int32, dev)
        _require(context_lens, "context_lens", torch.int32, dev)
        num_seqs, q_heads, hd = queries.shape
        if hd != self.head_dim or context_lens.numel() != num_seqs or \
                block_tables.shape[0] != num_seqs:
            raise AttentionError("paged decode shapes do not match the pool")
        if max_context_len is None:
            max_context_len = int(context_lens.max().item())
        if out is None:
            out = (torch.empty_like(queries) if stream is None
                   else _made(queries.shape, torch.float32, dev, stream))
        _require(out, "out", torch.float32, dev)
        if workspace is None:
            workspace = self._own_workspace(_raw_stream(dev, stream), stream, num_seqs, q_heads, 1,
                                            max_context_len)
        error = _lib.error_buffer()
        _check(self._lib.inferlab_cuda_paged_decode(
            self._handle, _vp(queries), _vp(block_tables), block_tables.shape[1],
            _vp(context_lens), num_seqs, q_heads, max_context_len, _vp(out), _vp(workspace),
            workspace.numel(), _stream_handle(dev, stream), error, len(error)), error)
        return out

    def decode_step_host(self, queries, block_tables, context_lens, new_keys=None,
                         new_values=None, out=None, stream=None, timeout_ms: int = 0,
                         block_copies=None):
        """One synchronous decode step from host (numpy) arrays: append the new
        token rows at context_lens - 1 (if given), decode every sequence, return
        the output as a host array. One C call (inferlab_cuda_decode_step_host).
        block_copies: per sequence the (from, to) copy-on-write pair that
        PageManager.prepare_append returned, or (-1, -1); the copies run in the
        same call before the rows are written (inferlab_cuda_decode_step_host_cow)."""
        import numpy as np

        q = np.ascontiguousarray(queries, dtype=np.float32)
        tables = np.ascontiguousarray(block_tables, dtype=np.int32)
        lens = np.ascontiguousarray(context_lens, dtype=np.int32)
        num_seqs, q_heads, _ = q.shape
        if out is None:
            out = np.empty_like(q)
        elif not (isinstance(out, np.ndarray) and out.dtype == np.float32 and
                  out.flags.c_contiguous and out.shape == q.shape):
            raise AttentionError("decode step output must be a contiguous float32 array shaped "
                                 "like the queries")
        keys = None if new_keys is None else np.ascontiguousarray(new_keys, dtype=np.float32)
        values = None if new_values is None else np.ascontiguousarray(new_values, dtype=np.float32)
        error = _lib.error_buffer()
        # Plain addresses: the per-step path avoids ctypes pointer objects.
        kp = None if keys is None else keys.ctypes.data
        vp = None if values is None else values.ctypes.data
        if block_copies is None:
            _check(self._lib.inferlab_cuda_decode_step_host(
                self._handle, q.ctypes.data, kp, vp, tables.ctypes.data, tables.shape[1],
                lens.ctypes.data, num_seqs, q_heads, out.ctypes.data,
                _stream_handle(self.device, stream), timeout_ms, error, len(error)), error)
            return out
        copies = np.ascontiguousarray(block_copies, dtype=np.int32)
        if copies.shape != (num_seqs, 2):
            raise AttentionError("decode step block copies must be [num_seqs][2]")
        _check(self._lib.inferlab_cuda_decode_step_host_cow(
            self._handle, q.ctypes.data, kp, vp, copies.ctypes.data, tables.ctypes.data,
            tables.shape[1], lens.ctypes.data, num_seqs, q_heads, out.ctypes.data,
            _stream_handle(self.device, stream), timeout_ms, error, len(error)), error)
        return out

    def decode_partials(self, queries: torch.Tensor, block_tables: torch.Tensor,
                        context_lens: torch.Tensor, max_context_len: int | None = None,
                        workspace: torch.Tensor | None = None, stream=None,
                        packed: torch.Tensor | None = None):
        """Split-KV partials (m, l, o) over this pool's part of each context.
        With `packed` (fp32, rows * (head_dim + 2) elements, rows = num_seqs *
        q_heads) they are written into it as [m | l | o], the layout
        lse_combine_packed merges after an all-gather."""
        dev = self.device
        _require(queries, "queries", torch.float32, dev)
        _require(block_tables, "block_tables", torch.int32, dev)
        _require(context_lens, "context_lens", torch.int32, dev)
        num_seqs, q_heads, hd = queries.shape
        if max_context_len is None:
            max_context_len = int(context_lens.max().item())
        if packed is not None:
            rows = num_seqs * q_heads
            _require(packed, "packed", torch.float32, dev)
            if packed.numel() != rows * (hd + 2):
                raise AttentionError("packed partials buffer has the wrong size")
            flat = packed.view(-1)
            m = flat[:rows].view(num_seqs, q_heads)
            l = flat[rows:2 * rows].view(num_seqs, q_heads)
            o = flat[2 * rows:].view(num_seqs, q_heads, hd)
        else:
            m = _made((num_seqs, q_heads), torch.float32, dev, stream)
            l = _made((num_seqs, q_heads), torch.float32, dev, stream)
            o = _made(queries.shape, torch.float32, dev, stream)
        if workspace is None:
            workspace = self._own_workspace(_raw_stream(dev, stream), stream, num_seqs, q_heads, 1,
                                            max_context_len)
        error = _lib.error_buffer()
        _check(self._lib.inferlab_cuda_paged_decode_partials(
            self._handle, _vp(queries), _vp(block_tables), block_tables.shape[1],
            _vp(context_lens), num_seqs, q_heads, max_context_len, _vp(m), _vp(l), _vp(o),
            _vp(workspace), workspace.numel(), _stream_handle(dev, stream), error, len(error)),
            error)
        return m, l, o

    def prefill(self, queries: torch.Tensor, block_tables: torch.Tensor,
                query_starts: torch.Tensor, query_counts: torch.Tensor,
                query_offsets: torch.Tensor, max_query_count: int,
                out: torch.Tensor | None = None, stream=None,
                max_context_len: int | None = None,
                workspace: torch.Tensor | None = None) -> torch.Tensor:
        """Causal (chunked) prefill of segments whose K/V are already in the pool. A 4-bit pool
        returns the queries' type; max_context_len (default: what the tables can hold) bounds its
        query_starts + query_counts and workspace is as for decode (inferlab_cuda_kv4_prefill)."""
        dev = self.device
        if self.kv_bits == 4:
            return self._kv4_prefill(queries, block_tables, query_starts, query_counts,
                                     query_offsets, max_query_count, out, stream, max_context_len,
                                     workspace)
        if queries.dtype == torch.float32:
            qtype = KV_FP32
        elif queries.dtype == TORCH_DTYPES[self.dtype]:
            qtype = self.dtype
        else:
            raise AttentionError("paged prefill query dtype must be FP32 or the pool dtype")
        _require(queries, "queries", None, dev)
        for name, t in (("block_tables", block_tables), ("query_starts", query_starts),
                        ("query_counts", query_counts), ("query_offsets", query_offsets)):
            _require(t, name, torch.int32, dev)
        total, q_heads, hd = queries.shape
        if hd != self.head_dim:
            raise AttentionError("paged prefill head_dim does not match the pool")
        if out is None:
            out = _made((total, q_heads, hd), torch.float32, dev, stream)
        _require(out, "out", torch.float32, dev)
        error = _lib.error_buffer()
        _check(self._lib.inferlab_cuda_paged_prefill(
            self._handle, _vp(queries), qtype, _vp(block_tables), block_tables.shape[1],
            _vp(query_starts), _vp(query_counts), _vp(query_offsets), query_starts.numel(),
            q_heads, max_query_count, total, _vp(out), _stream_handle(dev, stream), error,
            len(error)), error)
        return out

    def _kv4_operands(self, queries, out, stream):
        """The query / output type code, the addresses, and the output of a 4-bit attention call."""
        dtype = queries.dtype
        if dtype is not torch.float32 and dtype is not TORCH_DTYPES[self.dtype]:
            raise AttentionError("4-bit attention query dtype must be FP32 or the pool's row type")
        queries_at = _expect(queries, "queries", dtype, self.device)
        if queries.dim() != 3 or queries.shape[2] != self.head_dim:
            raise AttentionError("4-bit attention shapes do not match the pool")
        if out is None:
            out = (torch.empty_like(queries) if stream is None
                   else _made(queries.shape, dtype, self.device, stream))
            out_at = out.data_ptr()
        else:
            out_at = _expect(out, "out", dtype, self.device)
            if out.shape != queries.shape:
                raise AttentionError("4-bit attention output must be shaped like the queries")
        return KV_FP32 if dtype is torch.float32 else self.dtype, queries_at, out_at, out

    def _kv4_decode(self, queries, block_tables, context_lens, max_context_len, out, workspace,
                    stream):
        dev = self.device
        query_type, queries_at, out_at, out = self._kv4_operands(queries, out, stream)
        tables_at = _expect(block_tables, "block_tables", torch.int32, dev)
        lens_at = _expect(context_lens, "context_lens", torch.int32, dev)
        num_seqs, q_heads, _ = queries.shape
        table_shape = block_tables.shape
        if context_lens.numel() != num_seqs or len(table_shape) != 2 or table_shape[0] != num_seqs:
            raise AttentionError("4-bit attention shapes do not match the pool")
        if num_seqs == 0:
            return out
        if max_context_len is None:
            max_context_len = max(1, int(context_lens.max().item()))
        raw = _raw_stream(dev, stream)
        if workspace is None:
            workspace = self._own_workspace(raw, stream, num_seqs, q_heads, 1, max_context_len)
        workspace_at = _expect(workspace, "workspace", torch.uint8, dev)
        error = _lib.call_error_buffer()
        if self._lib.inferlab_cuda_kv4_decode(
                self._handle, queries_at, query_type, tables_at, table_shape[1], lens_at, num_seqs,
                q_heads, max_context_len, out_at, workspace_at, workspace.numel(), raw, error, 512):
            raise AttentionError(error.value.decode())
        return out

    def _kv4_prefill(self, queries, block_tables, query_starts, query_counts, query_offsets,
                     max_query_count, out, stream, max_context_len, workspace):
        dev = self.device
        query_type, queries_at, out_at, out = self._kv4_operands(queries, out, stream)
        segments = query_starts.numel()
        tables_at = _expect(block_tables, "block_tables", torch.int32, dev)
        starts_at = _expect(query_starts, "query_starts", torch.int32, dev)
        counts_at = _expect(query_counts, "query_counts", torch.int32, dev)
        offsets_at = _expect(query_offsets, "query_offsets", torch.int32, dev)
        table_shape = block_tables.shape
        if len(table_shape) != 2 or table_shape[0] != segments or \
                query_counts.numel() != segments or query_offsets.numel() != segments:
            raise AttentionError("4-bit attention shapes do not match the pool")
        total, q_heads, _ = queries.shape
        if segments == 0 or total == 0:
            return out
        if max_context_len is None:
            max_context_len = min(table_shape[1] * self.block_tokens, 0x7fffff00)
        raw = _raw_stream(dev, stream)
        if workspace is None:
            workspace = self._own_workspace(raw, stream, segments, q_heads, max_query_count,
                                            max_context_len)
        workspace_at = _expect(workspace, "workspace", torch.uint8, dev)
        error = _lib.call_error_buffer()
        if self._lib.inferlab_cuda_kv4_prefill(
                self._handle, queries_at, query_type, tables_at, table_shape[1], starts_at,
                counts_at, offsets_at, segments, q_heads, max_query_count, total, max_context_len,
                out_at, workspace_at, workspace.numel(), raw, error, 512):
            raise AttentionError(error.value.decode())
        return out


def lse_combine(part_m: torch.Tensor, part_l: torch.Tensor, part_o: torch.Tensor,
                out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Merge partials [parts][rows], [parts][rows][head_dim] in part order."""
    dev = part_o.device.index
    parts = part_o.shape[0]
    rows = math.prod(part_o.shape[1:-1])
    hd = part_o.shape[-1]
    for name, t in (("part_m", part_m), ("part_l", part_l), ("part_o", part_o)):
        _require(t, name, torch.float32, dev)
    if out is None:
        out = _made(part_o.shape[1:], torch.float32, dev, stream)
    error = _lib.error_buffer()
    _check(_lib.lib().inferlab_cuda_lse_combine(
        _vp(part_m), _vp(part_l), _vp(part_o), parts, rows, hd, _vp(out),
        _stream_handle(dev, stream), error, len(error)), error)
    return out


def lse_combine_packed(packed: torch.Tensor, parts: int, rows: int, head_dim: int,
                       out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Merge `parts` packed [m | l | o] partial blocks (part order) into
    [rows][head_dim]."""
    dev = packed.device.index
    _require(packed, "packed", torch.float32, dev)
    if packed.numel() != parts * rows * (head_dim + 2):
        raise AttentionError("packed partials buffer has the wrong size")
    if out is None:
        out = _made((rows, head_dim), torch.float32, dev, stream)
    error = _lib.error_buffer()
    _check(_lib.lib().inferlab_cuda_lse_combine_packed(
        _vp(packed), parts, rows, head_dim, _vp(out), _stream_handle(dev, stream), error,
        len(error)), error)
    return out
