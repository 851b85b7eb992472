"""Rotary positions and the append of new tokens to the paged cache, on the B200 library:
the input side of chunk attention (dory_chunk_attention) for prompts, parts of prompts,
ragged batches and single tokens.

* `rotary_cos_sin(max_position, rotary_dim, ...)`: the table of angles, cos | sin, plain or
  scaled for a longer context ("linear", "llama3", "yarn").
* `rotary_embed(q, k, positions, cos_sin, q_out, k_out, ...)`: the rotation of q and k, half or
  interleaved pairs, the whole head or its first rotary_dim dims, in place or not;
  `inverse=True` rotates back, which is also the rotation's gradient.
* `rotary_append(q, k, v, positions, cos_sin, slot_mapping, key_cache, value_cache, q_out, ...)`:
  the rotation, the model's q/k normalisation (`sqk`) and the cache write (BF16 or e4m3) in
  one launch; q comes back in BF16, ready for ChunkAttention.

The reference has no counterpart: its prompts run on vLLM's rotary embedding and cache write.
Everything is enqueued on the current stream of the tensors' device, allocates nothing and
waits for nothing, so calls can be captured in CUDA graphs.
"""

from __future__ import annotations

import math

import torch

import _native
from dory_decode_attention import _SQK_DTYPES, EPS

_IO_DTYPES = _SQK_DTYPES  # float32, bfloat16, float16
_FP8_CACHE_DTYPES = (torch.float8_e4m3fn, torch.uint8)
_pack = _native.packer(_native.DoryRotaryParams)


def rotary_cos_sin(max_position: int, rotary_dim: int, base: float = 10000.0, *,
                   scaling: str | None = None, factor: float = 1.0,
                   original_max_position: int = 8192, low_freq_factor: float = 1.0,
                   high_freq_factor: float = 4.0, beta_fast: float = 32.0,
                   beta_slow: float = 1.0, attention_factor: float | None = None,
                   dtype: torch.dtype = torch.float32, device=None) -> torch.Tensor:
    """cos | sin of the angles position * w_i, w_i = base^(-2i / rotary_dim), as
    [max_position, rotary_dim] (cos of every pair, then sin).  The angles are formed in FP64:
    in FP32 those of far positions would be off by position * 2^-24 radians.

    scaling: None; "linear", w_i / factor; "llama3", w_i / factor where the wavelength
    exceeds original_max_position / low_freq_factor, w_i below original_max_position /
    high_freq_factor and a mix between; "yarn", w_i / factor for the pairs that turn less
    than beta_slow times within original_max_position, w_i above beta_fast turns, a ramp over
    the pairs between, and cos and sin times attention_factor (default 0.1 ln(factor) + 1)."""
    if rotary_dim < 2 or rotary_dim % 2 or max_position < 1:
        raise ValueError("rotary_dim must be even and positive, max_position positive")
    if not (factor > 0 and base > 1):
        raise ValueError("factor must be positive and base above 1")
    i = torch.arange(rotary_dim // 2, dtype=torch.float64, device=device)
    w = base ** (-2.0 * i / rotary_dim)
    size = 1.0
    if scaling == "linear":
        w = w / factor
    elif scaling == "llama3":
        if high_freq_factor <= low_freq_factor:
            raise ValueError("high_freq_factor must exceed low_freq_factor")
        turns = original_max_position * w / (2 * math.pi)
        mix = ((turns - low_freq_factor) / (high_freq_factor - low_freq_factor)).clamp(0, 1)
        w = w * mix + w / factor * (1 - mix)
    elif scaling == "yarn":
        def pair_of(turns):  # the (fractional) pair that turns that often in the original length
            return (rotary_dim * math.log(original_max_position / (turns * 2 * math.pi))
                    / (2 * math.log(base)))
        low = max(math.floor(pair_of(beta_fast)), 0)
        high = min(math.ceil(pair_of(beta_slow)), rotary_dim - 1)
        ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        w = w / factor * ramp + w * (1 - ramp)
        size = attention_factor if attention_factor is not None else \
            (0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0)
    elif scaling is not None:
        raise ValueError(f"unknown scaling {scaling!r}: None, 'linear', 'llama3' or 'yarn'")
    angle = torch.arange(max_position, dtype=torch.float64, device=device)[:, None] * w
    return (torch.cat([angle.cos(), angle.sin()], dim=1) * size).to(dtype)


def _heads(name: str, x: torch.Tensor, tokens: int, head_dim: int) -> tuple:
    """(data pointer, token stride, head stride, heads) of a [T, H, head_dim] tensor."""
    shape, stride = x.shape, x.stride()
    if len(shape) != 3 or shape[0] != tokens or shape[2] != head_dim:
        raise ValueError(f"{name} must be [tokens, heads, head_dim] like q and k")
    if stride[2] != 1 and head_dim > 1 and x.numel():
        raise ValueError(f"{name} needs unit last stride")
    return x.data_ptr(), stride[0], stride[1], shape[1]


def _end(rows: tuple, size: int, tokens: int, dim: int) -> int:
    """The address behind the last of `rows`, as _heads returns them."""
    ptr, token, head, heads = rows
    return ptr + ((tokens - 1) * token + (heads - 1) * head + dim) * size


def _check_output(name: str, out: tuple, out_size: int, x: tuple, x_size: int, tokens: int,
                  dim: int, in_place: bool) -> None:
    """ValueError if rows of an output lie on one another, or the output over its input `x`
    (unless it is that tensor itself and in_place allows it).  out, x: as _heads returns them;
    out_size, x_size: bytes of an element."""
    ptr, token, head, heads = out
    if not tokens or not heads:
        return
    if heads > 1 and tokens > 1:
        inner, outer, n = (head, token, heads) if head <= token else (token, head, tokens)
        bad = inner < dim or outer < (n - 1) * inner + dim
    else:
        bad = (heads > 1 and head < dim) or (tokens > 1 and token < dim)
    if bad:
        raise ValueError(f"{name}'s rows must not overlap")
    if ptr == x[0] and token == x[1] and head == x[2] and out_size == x_size:
        if in_place:
            return
        raise ValueError(f"{name} must not be its input")
    if ptr < _end(x, x_size, tokens, dim) and x[0] < _end(out, out_size, tokens, dim):
        raise ValueError(f"{name} must lie apart from its input" +
                         (" or be that tensor itself" if in_place else ""))


def _meet(a: tuple, a_size: int, b: tuple, b_size: int, tokens: int, dim: int) -> bool:
    """Whether rows of a and b, as _heads returns them, share memory; a_size, b_size: bytes of an
    element.  Slices of one fused projection lie between one another and do not."""
    a_ptr, a_token, a_head, a_heads = a
    b_ptr, b_token, b_head, b_heads = b
    if not tokens or not a_heads or not b_heads:
        return False
    if _end(a, a_size, tokens, dim) <= b_ptr or _end(b, b_size, tokens, dim) <= a_ptr:
        return False
    a_width = ((a_heads - 1) * a_head + dim) * a_size
    b_width = ((b_heads - 1) * b_head + dim) * b_size
    step = a_token * a_size
    if step and step == b_token * b_size and a_width <= (b_ptr - a_ptr) % step <= step - b_width:
        return False  # side by side in every token
    # heads between heads, or anything else: row by row
    starts, sizes = [], []
    for ptr, token, head, heads, size in ((a_ptr, a_token, a_head, a_heads, a_size),
                                          (b_ptr, b_token, b_head, b_heads, b_size)):
        rows = (torch.arange(tokens)[:, None] * token + torch.arange(heads) * head).flatten() * size
        starts.append(rows + ptr)
        sizes.append(torch.full_like(rows, dim * size))
    owner = torch.cat([torch.zeros_like(starts[0]), torch.ones_like(starts[1])])
    start, order = torch.cat(starts).sort()
    end, owner = start + torch.cat(sizes)[order], owner[order]
    # the furthest that rows of either have reached before each row of the other
    for mine in (0, 1):
        reached = torch.where(owner == mine, end, 0).cummax(0).values
        if ((owner[1:] != mine) & (reached[:-1] > start[1:])).any():
            return True
    return False


def _table(cos_sin, positions, tokens: int, head_dim: int) -> tuple:
    """(positions ptr, table ptr, rotary_dim, max_position, table dtype, positions dtype)."""
    if cos_sin is None:
        return 0, 0, 0, 0, 0, 0
    code = _IO_DTYPES.get(cos_sin.dtype)
    shape = cos_sin.shape
    if code is None or len(shape) != 2 or not cos_sin.is_contiguous():
        raise ValueError("cos_sin must be contiguous [max_position, rotary_dim], float32, "
                         "bfloat16 or float16")
    if shape[1] > head_dim or shape[1] % 2 or shape[1] == 0:
        raise ValueError("rotary_dim must be even, positive and at most head_dim")
    if positions is None or positions.numel() != tokens or not positions.is_contiguous():
        raise ValueError("positions must be contiguous with one entry per token")
    kind = positions.dtype
    if kind is not torch.int64 and kind is not torch.int32:
        raise ValueError("positions must be int64 or int32")
    return (positions.data_ptr(), cos_sin.data_ptr(), shape[1], shape[0], code,
            0 if kind is torch.int64 else 1)


def _error_ptr(error_word) -> int:
    if error_word is None:
        return 0
    if error_word.dtype != torch.int32 or not error_word.numel():
        raise ValueError("error_word must be an int32 tensor of at least one element")
    return error_word.data_ptr()


_functions: dict = {}


def _launch(name: str, device: int, packed: bytes) -> None:
    fn = _functions.get(name)
    if fn is None:
        fn = _functions[name] = getattr(_native.load(), name)
    if torch._C._cuda_getDevice() != device:
        with torch.cuda.device(device):
            status = fn(packed, torch._C._cuda_getCurrentRawStream(device))
    else:
        status = fn(packed, torch._C._cuda_getCurrentRawStream(device))
    if status:
        _native.check(status)


def rotary_embed(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor,
                 cos_sin: torch.Tensor, q_out: torch.Tensor, k_out: torch.Tensor | None = None,
                 *, interleaved: bool = False, inverse: bool = False,
                 error_word: torch.Tensor | None = None) -> None:
    """Rotates q [T, NH, D] and k [T, NKV, D] (or None) by the angles of positions [T] (int64
    or int32) into q_out and k_out, same shapes and type (BF16, FP16 or FP32); an output may be
    its own input itself, otherwise it must lie apart from it; the outputs lie apart from each
    other and from the other's input.  Any token and head strides, unit last stride.  cos_sin
    [max_position, rotary_dim]: the first rotary_dim dims turn, pairs (i, i + rotary_dim / 2) or,
    interleaved, (2i, 2i + 1); the others are copied.  inverse: the
    rotation back.  error_word (optional int32 device tensor) collects
    DORY_DEVERR_POSITION_OOB; such a token's outputs are zero."""
    code = _IO_DTYPES.get(q.dtype)
    if code is None or q_out.dtype is not q.dtype:
        raise ValueError("q and q_out must have one type: float32, bfloat16 or float16")
    if not q.is_cuda:
        raise RuntimeError("rotary_embed runs on CUDA tensors only (no CPU path)")
    if q.dim() != 3:
        raise ValueError("q must be [tokens, heads, head_dim]")
    if (k is None) != (k_out is None):
        raise ValueError("k and k_out go together")
    device = q.get_device()
    _native.check_device_index(device, q_out, k, k_out, positions, cos_sin, error_word)
    tokens, _, dim = q.shape
    size = q.element_size()
    q_ptr, q_t, q_h, heads = q_rows = _heads("q", q, tokens, dim)
    qo_ptr, qo_t, qo_h, out_heads = qo_rows = _heads("q_out", q_out, tokens, dim)
    if out_heads != heads:
        raise ValueError("q_out must have q's heads")
    _check_output("q_out", qo_rows, size, q_rows, size, tokens, dim, True)
    k_ptr = k_t = k_h = ko_ptr = ko_t = ko_h = kv_heads = 0
    if k is not None:
        if k.dtype is not q.dtype or k_out.dtype is not q.dtype:
            raise ValueError("k and k_out must have q's type")
        k_ptr, k_t, k_h, kv_heads = k_rows = _heads("k", k, tokens, dim)
        ko_ptr, ko_t, ko_h, out_heads = ko_rows = _heads("k_out", k_out, tokens, dim)
        if out_heads != kv_heads:
            raise ValueError("k_out must have k's heads")
        _check_output("k_out", ko_rows, size, k_rows, size, tokens, dim, True)
        qo_end, ko_end = _end(qo_rows, size, tokens, dim), _end(ko_rows, size, tokens, dim)
        if ((qo_ptr < ko_end and ko_ptr < qo_end and _meet(qo_rows, size, ko_rows, size, tokens, dim))
                or (ko_rows != k_rows and qo_ptr < _end(k_rows, size, tokens, dim) and k_ptr < qo_end
                    and _meet(qo_rows, size, k_rows, size, tokens, dim))
                or (qo_rows != q_rows and ko_ptr < _end(q_rows, size, tokens, dim) and q_ptr < ko_end
                    and _meet(ko_rows, size, q_rows, size, tokens, dim))):
            raise ValueError("the outputs must lie apart, from each other and from the other's input")
    pos_ptr, table, rotary, max_position, table_code, pos32 = _table(cos_sin, positions, tokens, dim)
    flags = ((_native.ROTARY_INTERLEAVED if interleaved else 0) |
             (_native.ROTARY_INVERSE if inverse else 0))
    _launch("dory_rotary_embed", device, _pack(
        q_ptr, k_ptr, 0, pos_ptr, table, 0, 0, qo_ptr, ko_ptr, 0, 0, _error_ptr(error_word),
        q_t, q_h, k_t, k_h, 0, 0, qo_t, qo_h, ko_t, ko_h, 0, 0, 0, 0, max_position,
        0.0, 0.0, 1.0, 1.0, tokens, heads, kv_heads, dim, rotary, 0, code, table_code, pos32, 0,
        0, flags))


def rotary_append(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor,
                  positions: torch.Tensor | None, cos_sin: torch.Tensor | None,
                  slot_mapping: torch.Tensor, key_cache: torch.Tensor,
                  value_cache: torch.Tensor, q_out: torch.Tensor | None, *,
                  sqk: torch.Tensor | None = None, sqk_factor: float = 1.0, eps: float = EPS,
                  interleaved: bool = False, k_scale: float = 1.0, v_scale: float = 1.0,
                  error_word: torch.Tensor | None = None) -> None:
    """Rotates q [T, NH, D] and k [T, NKV, D] (as rotary_embed; cos_sin None: not at all), with
    `sqk` ([NH * D]) normalises both (q = (sqk * sqk_factor)^2 * q / |q|, k = k / |k|, eps inside
    the root), and writes k and v [T, NKV, D] to the cache views [blocks, block_size, NKV, D]
    at slot_mapping[t] (int64, as vLLM's: block * block_size + row; negative: a padding token,
    nothing is written; no slot twice).  BF16 caches, or e4m3 (float8_e4m3fn or uint8) with the
    layer's k_scale / v_scale.  q_out: BF16 [T, NH, D] (or [T, NH * D]), apart from the
    inputs and the caches; q and q_out None: k and v alone.  q, k, v: one type, BF16, FP16 or FP32, e.g. slices of a fused projection.
    head_dim 64, 128 or 256.  error_word (optional int32 device tensor) collects
    DORY_DEVERR_SLOT_OOB (slot beyond the cache, skipped) and DORY_DEVERR_POSITION_OOB."""
    code = _IO_DTYPES.get(k.dtype)
    if code is None or v.dtype is not k.dtype or (q is not None and q.dtype is not k.dtype):
        raise ValueError("q, k and v must have one type: float32, bfloat16 or float16")
    if not k.is_cuda:
        raise RuntimeError("rotary_append runs on CUDA tensors only (no CPU path)")
    if k.dim() != 3:
        raise ValueError("k must be [tokens, kv_heads, head_dim]")
    if (q is None) != (q_out is None):
        raise ValueError("q and q_out go together")
    device = k.get_device()
    _native.check_device_index(device, q, v, positions, cos_sin, slot_mapping, key_cache,
                               value_cache, q_out, sqk, error_word)
    tokens, _, dim = k.shape
    k_ptr, k_t, k_h, kv_heads = k_rows = _heads("k", k, tokens, dim)
    v_ptr, v_t, v_h, v_heads = v_rows = _heads("v", v, tokens, dim)
    if v_heads != kv_heads:
        raise ValueError("v must have k's heads")
    q_ptr = q_t = q_h = qo_ptr = qo_t = qo_h = heads = 0
    if q is not None:
        if q_out.dtype is not torch.bfloat16:
            raise ValueError("q_out must be bfloat16")
        q_ptr, q_t, q_h, heads = q_rows = _heads("q", q, tokens, dim)
        if q_out.dim() == 2:
            if q_out.shape[1] != heads * dim or q_out.stride(1) != 1:
                raise ValueError("q_out must be [tokens, heads * head_dim]")
            q_out = q_out.unflatten(1, (heads, dim))
        qo_ptr, qo_t, qo_h, out_heads = qo_rows = _heads("q_out", q_out, tokens, dim)
        if out_heads != heads:
            raise ValueError("q_out must have q's heads")
        size = q.element_size()
        _check_output("q_out", qo_rows, 2, q_rows, size, tokens, dim, False)
        qo_end = _end(qo_rows, 2, tokens, dim)
        if ((qo_ptr < _end(k_rows, size, tokens, dim) and k_ptr < qo_end
             and _meet(qo_rows, 2, k_rows, size, tokens, dim))
                or (qo_ptr < _end(v_rows, size, tokens, dim) and v_ptr < qo_end
                    and _meet(qo_rows, 2, v_rows, size, tokens, dim))):
            raise ValueError("q_out must lie apart from k and v")
    pos_ptr, table, rotary, max_position, table_code, pos32 = _table(cos_sin, positions, tokens, dim)
    shape, stride = key_cache.shape, key_cache.stride()
    if stride != value_cache.stride() or stride[-1] != 1 or shape != value_cache.shape:
        raise ValueError("key and value caches need equal shapes and strides and unit last stride")
    if len(shape) != 4 or shape[2] != kv_heads or shape[3] != dim:
        raise ValueError("cache view must be [blocks, block_size, kv_heads, head_dim]")
    kind = key_cache.dtype
    if value_cache.dtype is not kind:
        raise ValueError("key and value caches must have one type")
    if kind is torch.bfloat16:
        kv_code = _native.DTYPE_BF16
    elif kind in _FP8_CACHE_DTYPES:
        kv_code = _native.DTYPE_FP8_E4M3
    else:
        raise ValueError("caches must be bfloat16, or float8_e4m3fn / uint8 for FP8")
    key, value = key_cache.data_ptr(), value_cache.data_ptr()
    if q is not None and tokens and shape[0] and shape[1]:
        reach = (shape[0] - 1) * stride[0] + (shape[1] - 1) * stride[1] \
            + (kv_heads - 1) * stride[2] + dim
        reach *= 2 if kv_code == _native.DTYPE_BF16 else 1
        if (qo_ptr < key + reach and key < qo_end) or (qo_ptr < value + reach and value < qo_end):
            raise ValueError("q_out must lie apart from the caches")
    if (slot_mapping.dtype is not torch.int64 or slot_mapping.numel() < tokens
            or not slot_mapping.is_contiguous()):
        raise ValueError("slot_mapping must be contiguous int64 with one entry per token")
    sqk_ptr = sqk_code = flags = 0
    if sqk is not None:
        sqk_code = _IO_DTYPES.get(sqk.dtype)
        if sqk_code is None or not sqk.is_contiguous() or (q is not None and sqk.numel() != heads * dim):
            raise ValueError("sqk must be contiguous with heads * head_dim entries")
        sqk_ptr, flags = sqk.data_ptr(), _native.ROTARY_NORM
    if interleaved:
        flags |= _native.ROTARY_INTERLEAVED
    _launch("dory_rotary_append", device, _pack(
        q_ptr, k_ptr, v_ptr, pos_ptr, table, sqk_ptr, slot_mapping.data_ptr(), qo_ptr, 0,
        key, value, _error_ptr(error_word),
        q_t, q_h, k_t, k_h, v_t, v_h, qo_t, qo_h, 0, 0, stride[0], stride[1], stride[2], shape[0],
        max_position, float(sqk_factor), float(eps), float(k_scale), float(v_scale), tokens,
        heads, kv_heads, dim, rotary, shape[1], code, table_code, pos32, sqk_code, kv_code, flags))


__all__ = ["rotary_cos_sin", "rotary_embed", "rotary_append"]
