"""Chunk attention on the host: struct layout and refusals before any launch, and the FP64
oracle against a dense softmax."""

from __future__ import annotations

import ctypes

import pytest
import torch

import _native
import build_native
import dory_prompt_oracle as P


@pytest.fixture(scope="module")
def lib():
    build_native.build()
    return _native.load()


def test_struct_layout(lib):
    assert lib.dory_chunk_params_bytes() == ctypes.sizeof(_native.DoryChunkParams)
    pack = _native.packer(_native.DoryChunkParams)
    values = [i + 1 for i in range(len(_native.DoryChunkParams._fields_))]
    raw = pack(*values).ljust(ctypes.sizeof(_native.DoryChunkParams), b"\0")
    p = _native.DoryChunkParams.from_buffer_copy(raw)
    assert [getattr(p, name) for name, _ in p._fields_] == values


def test_scratch_bytes(lib):
    assert lib.dory_chunk_scratch_bytes(32, 8, 128) >= 256
    for bad in ((30, 8, 128), (0, 8, 128), (32, 0, 128), (32, 8, 96), (130, 2, 128)):
        assert lib.dory_chunk_scratch_bytes(*bad) == 0


def params(**kw):
    p = _native.DoryChunkParams()
    for f in ("q", "key_cache", "value_cache", "block_tables", "query_start", "seq_lens", "gate",
              "out", "scratch"):
        setattr(p, f, 0x1000)  # never dereferenced: validation fails before any launch
    p.scratch_bytes = 1 << 40
    p.q_stride_token, p.q_stride_head, p.out_stride_token, p.gate_stride_token = 4096, 128, 4096, 4096
    p.table_stride, p.stride_block, p.stride_offset, p.stride_head = 8, 32768, 256, 4096
    p.num_cache_blocks, p.softmax_scale, p.k_scale, p.v_scale = 100, 0.1, 1.0, 1.0
    p.num_tokens, p.num_seqs, p.max_blocks, p.num_heads, p.num_kv_heads = 4, 1, 8, 32, 8
    p.head_dim, p.block_size = 128, 16
    for k, v in kw.items():
        setattr(p, k, v)
    return p


FP8 = _native.DTYPE_FP8_E4M3


@pytest.mark.parametrize("kw,status,message", [
    (dict(num_heads=30), _native.ERR_INVALID_ARGUMENT, "multiple of KV heads"),
    (dict(num_heads=520), _native.ERR_UNSUPPORTED, "max 64"),
    (dict(num_tokens=-1), _native.ERR_INVALID_ARGUMENT, "negative"),
    (dict(window=-1), _native.ERR_INVALID_ARGUMENT, "window"),
    (dict(head_dim=96), _native.ERR_UNSUPPORTED, "head_dim"),
    (dict(block_size=24), _native.ERR_UNSUPPORTED, "block_size"),
    (dict(kv_dtype=_native.DTYPE_F16), _native.ERR_INVALID_ARGUMENT, "kv_dtype"),
    (dict(kv_dtype=FP8, head_dim=64), _native.ERR_UNSUPPORTED, "FP8"),
    (dict(kv_dtype=FP8, v_scale=float("inf")), _native.ERR_INVALID_ARGUMENT, "scales"),
    (dict(kv_dtype=FP8, stride_offset=264), _native.ERR_ALIGNMENT, "16-byte"),
    (dict(softmax_scale=0.0), _native.ERR_INVALID_ARGUMENT, "softmax_scale"),
    (dict(softmax_scale=float("nan")), _native.ERR_INVALID_ARGUMENT, "softmax_scale"),
    (dict(gate_dtype=3), _native.ERR_INVALID_ARGUMENT, "gate"),
    (dict(num_cache_blocks=0), _native.ERR_INVALID_ARGUMENT, "empty"),
    (dict(max_blocks=0), _native.ERR_INVALID_ARGUMENT, "empty"),
    (dict(seq_lens=None), _native.ERR_INVALID_ARGUMENT, "null"),
    (dict(q=0x1008), _native.ERR_ALIGNMENT, "16-byte"),
    (dict(q_stride_token=4100), _native.ERR_ALIGNMENT, "16-byte"),
    (dict(out_stride_token=4100), _native.ERR_ALIGNMENT, "16-byte"),
    (dict(stride_block=4), _native.ERR_ALIGNMENT, "16-byte"),
    (dict(gate=0x1004), _native.ERR_ALIGNMENT, "16-byte"),
    (dict(scratch_bytes=16), _native.ERR_INVALID_ARGUMENT, "scratch too small"),
    (dict(out=0x1000 + 2 * 3 * 4096), _native.ERR_INVALID_ARGUMENT, "apart"),  # q's last row
    (dict(out=0x1000000, gate=0x1000000 + 2 * 3 * 4096 + 16), _native.ERR_INVALID_ARGUMENT, "apart"),
])
def test_host_validation(lib, kw, status, message):
    p = params(**kw)
    assert lib.dory_chunk_attention(ctypes.byref(p), None) == status
    assert message in lib.dory_decode_last_error().decode()


def test_nothing_to_do(lib):
    assert lib.dory_chunk_attention(ctypes.byref(params(num_tokens=0, q=None, out=None)), None) == 0
    assert lib.dory_chunk_attention(ctypes.byref(params(num_seqs=0)), None) == 0
    assert lib.dory_chunk_attention(None, None) == _native.ERR_INVALID_ARGUMENT


def test_constructor_refusals():
    from dory_chunk_attention import ChunkAttention
    with pytest.raises(RuntimeError, match="no CPU path"):
        ChunkAttention(8, 2, 128, torch.device("cpu"))
    with pytest.raises(ValueError, match="multiple of KV heads"):
        ChunkAttention(8, 3, 128, torch.device("cuda"))
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        ChunkAttention(8, 2, 128, torch.device("cuda"), kv_cache_dtype="int8")


def test_oracle_against_a_dense_softmax():
    g = torch.Generator().manual_seed(0)
    B, NKV, G, D, n, length, window = 4, 2, 3, 8, 5, 11, 6
    key, value = (torch.randn(6, B, NKV, D, generator=g, dtype=torch.float64) for _ in range(2))
    q = torch.randn(n + 2, NKV * G, D, generator=g, dtype=torch.float64)
    table = torch.tensor([[3, 0, 5, 1], [2, 2, 2, 2]], dtype=torch.int32)
    value[1] = float("nan")  # a block that neither sequence reaches
    for w in (0, window):
        out, size = P.chunk_attention(q, key, value, table, [0, n, n + 1], [length, 0], w, 0.3)
        flat_k, flat_v = (x[table[0, :3].long()].flatten(0, 1)[:length] for x in (key, value))
        for h in range(NKV * G):
            s = q[:n, h] @ flat_k[:, h // G].T * 0.3
            i, j = torch.arange(length - n, length)[:, None], torch.arange(length)[None]
            hide = (j > i) | ((j <= i - w) if w else torch.zeros_like(j > i))
            want = torch.softmax(s.masked_fill(hide, -torch.inf), -1) @ flat_v[:, h // G]
            torch.testing.assert_close(out[:n, h * D:(h + 1) * D], want)
        assert (out[n] == 0).all() and out[n + 1].isnan().all() and (size[:n] > 0).all()


def test_a_scratch_off_the_16_byte_grid_is_refused(lib):
    """The join reads it 16 bytes at a time."""
    for at in (0x1004, 0x1008):
        assert lib.dory_chunk_attention(ctypes.byref(params(scratch=at)), None) == _native.ERR_ALIGNMENT
        assert "scratch" in lib.dory_decode_last_error().decode()
