"""Attention of a chunk of new tokens over vLLM's paged KV cache, on B200 (sm_100a): whole
prompts, parts of prompts whose earlier part is cached, drafted tokens and single tokens, as
one ragged batch.

`ChunkAttention` stands beside `DecodeAttention` (dory_decode_attention): it reads the same
cache views and block tables, takes the query as `dory_rotary_steps.rotary_append` returns it
(which also appends the chunk's keys and values, and must have run before), and gives the gated
output in BF16 for the output projection.  The reference has no counterpart: its prompts run
on vLLM's attention.

A call is enqueued on the current stream, allocates nothing and reads nothing on the host, so
it can be captured in a CUDA graph (lengths and tables may change between replays).  There is
no CPU or Triton path.
"""

from __future__ import annotations

import ctypes

import torch

import _native
from dory_decode_attention import _FP8_CACHE_DTYPES, _KV_DTYPES, _SQK_DTYPES

_pack = _native.packer(_native.DoryChunkParams)


class ChunkAttention:
    """Causal attention of the last n positions of each sequence of a batch, optionally
    windowed and gated, with one scratch buffer.  Calls on one instance must be ordered (one
    stream, or events between); graphs that may run at the same time need an instance each.

    kv_cache_dtype: "auto" / "bf16", or "fp8" / "fp8_e4m3" for caches of e4m3 bytes, as
    DecodeAttention takes them.  head_dim 64, 128 or 256 (FP8: 128 or 256), at most 64 query
    heads per KV head."""

    def __init__(self, num_heads: int, num_kv_heads: int, head_dim: int, device: torch.device,
                 kv_cache_dtype: str = "auto"):
        if num_heads < 1 or num_kv_heads < 1 or num_heads % num_kv_heads:
            raise ValueError("query heads must be a multiple of KV heads")
        if kv_cache_dtype not in _KV_DTYPES:
            raise ValueError(f"kv_cache_dtype must be one of {sorted(_KV_DTYPES)}")
        self.num_heads, self.num_kv_heads, self.head_dim = num_heads, num_kv_heads, head_dim
        self.kv_cache_dtype = kv_cache_dtype
        self._kv_code = _KV_DTYPES[kv_cache_dtype]
        self._cache_types = (_FP8_CACHE_DTYPES if self._kv_code == _native.DTYPE_FP8_E4M3
                             else (torch.bfloat16,))
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise RuntimeError("ChunkAttention runs on CUDA devices only (no CPU path)")
        self._lib = _native.load()
        with torch.cuda.device(self.device):
            nbytes = self._lib.dory_chunk_scratch_bytes(num_heads, num_kv_heads, head_dim)
            if nbytes <= 0:
                raise NotImplementedError("head_dim must be 64, 128 or 256, with at most 64 query "
                                          "heads per KV head")
            self.scratch = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
            _native.check(self._lib.dory_decode_scratch_init(
                self.scratch.data_ptr(), nbytes, torch.cuda.current_stream().cuda_stream))
        self._call = self._lib.dory_chunk_attention
        self._scratch = (self.scratch.data_ptr(), self.scratch.numel())
        self._dev_index = self.scratch.get_device()

    def __call__(self, q: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                 block_tables: torch.Tensor, query_start: torch.Tensor, seq_lens: torch.Tensor,
                 window: int, softmax_scale: float, out: torch.Tensor,
                 gate: torch.Tensor | None = None, *, k_scale: float = 1.0,
                 v_scale: float = 1.0) -> None:
        """q: BF16 [T, heads, head_dim] (or [T, heads * head_dim]), normalised and scaled as
        rotary_append leaves it; key_cache / value_cache: [blocks, block_size, kv_heads,
        head_dim] views that already hold the chunk's own rows; block_tables: int32 [S,
        max_blocks]; query_start: int32 [S + 1], sequence i owns rows query_start[i] ..
        query_start[i + 1] - 1 of q; seq_lens: int32 [S], positions including those rows (0:
        a padded request, zero rows); window: 0 for all earlier positions; gate: FP32, BF16 or
        FP16 [T, heads * head_dim] (e.g. post-sigmoid) or None; out: BF16 [T, heads *
        head_dim], whose span of memory lies apart from those of q and gate.  Rows that no
        sequence owns keep what out held.  A query_start that decreases or leaves [0, T] is
        reported (check_errors) and nothing is written."""
        heads, dim, dev = self.num_heads, self.head_dim, self._dev_index
        if q.dtype is not torch.bfloat16 or out.dtype is not torch.bfloat16:
            raise ValueError("q and out must be bfloat16")
        if not q.is_cuda:
            raise RuntimeError("ChunkAttention runs on CUDA tensors only (no CPU path)")
        _native.check_device_index(dev, q, key_cache, value_cache, block_tables, query_start,
                                   seq_lens, out, gate)
        shape, stride = q.shape, q.stride()
        tokens = shape[0]
        if len(shape) == 3 and shape[1] == heads and shape[2] == dim and stride[2] == 1:
            q_token, q_head = stride[0], stride[1]
        elif len(shape) == 2 and shape[1] == heads * dim and stride[1] == 1:
            q_token, q_head = stride[0], dim
        else:
            raise ValueError("q must be [tokens, heads, head_dim] with unit last stride")
        cache, strides = key_cache.shape, key_cache.stride()
        if strides != value_cache.stride() or strides[-1] != 1 or cache != value_cache.shape:
            raise ValueError("key and value caches need equal shapes and strides and unit last "
                             "stride")
        if len(cache) != 4 or cache[2] != self.num_kv_heads or cache[3] != dim:
            raise ValueError("cache view must be [blocks, block_size, kv_heads, head_dim]")
        if key_cache.dtype not in self._cache_types or value_cache.dtype is not key_cache.dtype:
            raise ValueError(f"caches must be of type {self._cache_types[0]}")
        table = block_tables.shape
        if (block_tables.dtype is not torch.int32 or query_start.dtype is not torch.int32
                or seq_lens.dtype is not torch.int32):
            raise ValueError("block_tables, query_start and seq_lens must be int32")
        seqs = seq_lens.numel()
        if (len(table) != 2 or table[0] < seqs or block_tables.stride(1) != 1
                or query_start.numel() < seqs + 1 or not seq_lens.is_contiguous()
                or not query_start.is_contiguous()):
            raise ValueError("block_tables must be [sequences, max_blocks] with unit last stride, "
                             "query_start [sequences + 1] and seq_lens [sequences] contiguous")
        if out.dim() != 2 or out.shape[0] != tokens or out.shape[1] != heads * dim \
                or out.stride(1) != 1 or (tokens > 1 and out.stride(0) < heads * dim):
            raise ValueError("out must be [tokens, heads * head_dim] with unit last stride")
        gate_ptr = gate_token = gate_code = 0
        if gate is not None:
            gate_code = _SQK_DTYPES.get(gate.dtype)
            if gate_code is None or gate.shape != out.shape or gate.stride(1) != 1:
                raise ValueError("gate must be [tokens, heads * head_dim], float32, bfloat16 or "
                                 "float16, with unit last stride")
            gate_ptr, gate_token = gate.data_ptr(), gate.stride(0)
        packed = _pack(
            q.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), block_tables.data_ptr(),
            query_start.data_ptr(), seq_lens.data_ptr(), gate_ptr, out.data_ptr(),
            *self._scratch, q_token, q_head, out.stride(0),
            gate_token, block_tables.stride(0), strides[0], strides[1], strides[2], cache[0],
            float(softmax_scale), float(k_scale), float(v_scale), tokens, seqs, table[1], heads,
            self.num_kv_heads, dim, cache[1], int(window), gate_code, self._kv_code)
        if torch._C._cuda_getDevice() != dev:
            with torch.cuda.device(dev):
                status = self._call(packed, torch._C._cuda_getCurrentRawStream(dev))
        else:
            status = self._call(packed, torch._C._cuda_getCurrentRawStream(dev))
        if status:
            _native.check(status)

    def fetch_errors(self, clear: bool = True) -> int:
        """Device error bits (DORY_DEVERR_*) recorded since the last clear.  Synchronises the
        current stream."""
        flags = ctypes.c_uint32(0)
        with torch.cuda.device(self.device):
            _native.check(self._lib.dory_decode_fetch_errors(
                self.scratch.data_ptr(), ctypes.byref(flags), int(clear),
                torch.cuda.current_stream().cuda_stream))
        return flags.value

    def check_errors(self) -> None:
        """Raises RuntimeError naming every device error bit recorded since the last check."""
        flags = self.fetch_errors(clear=True)
        if flags:
            names = [name for bit, name in _native.DEVERR_NAMES.items() if flags & bit]
            raise RuntimeError("chunk attention device errors: " + ", ".join(names))


__all__ = ["ChunkAttention"]
