"""Rotary positions on the host: the table of angles and the refusals, before any launch."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import _native
import build_native
from dory_rotary_steps import _check_output, _heads, _table, rotary_append, rotary_cos_sin, rotary_embed


@pytest.fixture(scope="module")
def lib():
    build_native.build()
    return _native.load()


def test_struct_layout(lib):
    assert lib.dory_rotary_params_bytes() == ctypes.sizeof(_native.DoryRotaryParams)
    pack = _native.packer(_native.DoryRotaryParams)
    values = [i + 1 for i in range(len(_native.DoryRotaryParams._fields_))]
    p = _native.DoryRotaryParams.from_buffer_copy(pack(*values))
    assert [getattr(p, name) for name, _ in p._fields_] == values


def test_plain_table():
    t = rotary_cos_sin(70000, 64, 10000.0, dtype=torch.float64)
    assert t.shape == (70000, 64)
    for p, i in ((0, 0), (1, 0), (69999, 0), (69999, 5), (12345, 31)):
        angle = p * 10000.0 ** (-2 * i / 64)
        assert t[p, i].item() == pytest.approx(math.cos(angle), abs=1e-10)
        assert t[p, 32 + i].item() == pytest.approx(math.sin(angle), abs=1e-10)
    assert rotary_cos_sin(10, 8).dtype == torch.float32


def angles(t):
    """Angle per position of every pair, from position 1 (unambiguous while below pi)."""
    half = t.shape[1] // 2
    return torch.atan2(t[1, half:], t[1, :half])


def test_scaled_tables():
    kw = dict(dtype=torch.float64)
    plain = angles(rotary_cos_sin(2, 128, 500000.0, **kw))
    linear = angles(rotary_cos_sin(2, 128, 500000.0, scaling="linear", factor=4.0, **kw))
    torch.testing.assert_close(linear, plain / 4)
    l3 = angles(rotary_cos_sin(2, 128, 500000.0, scaling="llama3", factor=8.0,
                               original_max_position=8192, **kw))
    wave = 2 * math.pi / plain
    short, long = wave < 8192 / 4, wave > 8192
    assert short.any() and long.any() and (~short & ~long).any()
    torch.testing.assert_close(l3[short], plain[short])
    torch.testing.assert_close(l3[long], plain[long] / 8)
    between = ~short & ~long
    mix = (8192 / wave[between] - 1) / (4 - 1)
    torch.testing.assert_close(l3[between], (1 - mix) * plain[between] / 8 + mix * plain[between])
    yarn = rotary_cos_sin(2, 128, 10000.0, scaling="yarn", factor=16.0, original_max_position=4096,
                          **kw)
    size = 0.1 * math.log(16) + 1
    assert yarn[0, 0].item() == pytest.approx(size)
    base = angles(rotary_cos_sin(2, 128, 10000.0, **kw))
    turns = 4096 * base / (2 * math.pi)
    fast, slow = turns > 32 * 1.4, turns < 1 / 1.4
    torch.testing.assert_close(angles(yarn)[fast], base[fast])
    torch.testing.assert_close(angles(yarn)[slow], base[slow] / 16)
    ratio = angles(yarn) / base
    assert (ratio[1:] <= ratio[:-1] + 1e-12).all()  # the ramp falls from 1 to 1/16


@pytest.mark.parametrize("kw", [dict(rotary_dim=7), dict(rotary_dim=0), dict(max_position=0),
                                dict(scaling="ntk"), dict(factor=0.0, scaling="linear"),
                                dict(scaling="llama3", low_freq_factor=4.0)])
def test_table_refusals(kw):
    args = dict(max_position=16, rotary_dim=8)
    args.update(kw)
    with pytest.raises(ValueError):
        rotary_cos_sin(**args)


def test_cpu_tensors_are_refused():
    q, out = torch.zeros(2, 4, 64), torch.zeros(2, 4, 64)
    table, pos = rotary_cos_sin(8, 64), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        rotary_embed(q, None, pos, table, out)
    cache = torch.zeros(2, 16, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        rotary_append(None, q, q, pos, table, pos, cache, cache, None)


def test_output_checks():
    def check(out, x, in_place):
        T, _, D = x.shape
        _check_output("o", _heads("o", out, T, D), out.element_size(), _heads("x", x, T, D),
                      x.element_size(), T, D, in_place)
    x = torch.zeros(4, 3, 8)
    check(x, x, True)                      # itself
    check(torch.zeros(4, 3, 8), x, False)  # apart
    check(torch.zeros(3, 4, 8).transpose(0, 1), x, False)
    check(torch.zeros(1, 3, 8).expand(4, 3, 8)[:1], x[:1], False)  # one token: any stride
    with pytest.raises(ValueError, match="must not be its input"):
        check(x, x, False)
    big = torch.zeros(5, 3, 8)
    with pytest.raises(ValueError, match="apart"):
        check(big[1:], big[:4], True)
    with pytest.raises(ValueError, match="apart"):  # another type over the same memory
        check(x.view(torch.float16)[..., :8], x, False)
    with pytest.raises(ValueError, match="rows must not overlap"):
        check(torch.zeros(1, 3, 8).expand(4, 3, 8), x, True)
    with pytest.raises(ValueError, match="rows must not overlap"):
        check(torch.zeros(100).as_strided((4, 3, 8), (12, 8, 1)), x, True)


def test_argument_checks():
    with pytest.raises(ValueError, match="unit last stride"):
        _heads("q", torch.zeros(2, 8, 4).transpose(1, 2), 2, 8)
    with pytest.raises(ValueError):
        _heads("q", torch.zeros(2, 8), 2, 8)
    pos = torch.zeros(2, dtype=torch.int64)
    for bad in (torch.zeros(4, 10), torch.zeros(4, 7), torch.zeros(4, 8, dtype=torch.float64),
                torch.zeros(4, 16)[:, :8], torch.zeros(4, 0)):
        with pytest.raises(ValueError):
            _table(bad, pos, 2, 8)
    for bad in (pos[:1], pos.float(), pos.to(torch.int16), torch.zeros(4, dtype=torch.int64)[::2],
                None):
        with pytest.raises(ValueError):
            _table(torch.zeros(4, 8), bad, 2, 8)


def params(**kw):
    p = _native.DoryRotaryParams()
    for f in ("q", "k", "v", "positions", "cos_sin", "sqk", "slot_mapping", "q_out", "k_out",
              "key_cache", "value_cache"):
        setattr(p, f, 0x1000)  # never dereferenced: validation fails before any launch
    p.num_tokens, p.num_heads, p.num_kv_heads, p.head_dim, p.rotary_dim = 1, 8, 2, 128, 128
    p.max_position, p.block_size, p.num_cache_blocks = 16, 16, 4
    p.k_scale = p.v_scale = 1.0
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("append,kw,status,message", [
    (False, dict(num_heads=0), _native.ERR_INVALID_ARGUMENT, "positive"),
    (False, dict(num_tokens=-1), _native.ERR_INVALID_ARGUMENT, "positive"),
    (False, dict(head_dim=2000), _native.ERR_UNSUPPORTED, "head_dim"),
    (False, dict(rotary_dim=3), _native.ERR_INVALID_ARGUMENT, "rotary_dim"),
    (False, dict(rotary_dim=130), _native.ERR_INVALID_ARGUMENT, "rotary_dim"),
    (False, dict(rotary_dim=0), _native.ERR_INVALID_ARGUMENT, "rotary_dim"),
    (False, dict(max_position=0), _native.ERR_INVALID_ARGUMENT, "max_position"),
    (False, dict(io_dtype=3), _native.ERR_INVALID_ARGUMENT, "dtype"),
    (False, dict(flags=_native.ROTARY_NORM), _native.ERR_INVALID_ARGUMENT, "append"),
    (False, dict(k_out=None), _native.ERR_INVALID_ARGUMENT, "null"),
    (True, dict(head_dim=80, rotary_dim=80), _native.ERR_UNSUPPORTED, "head_dim"),
    (True, dict(flags=_native.ROTARY_INVERSE), _native.ERR_INVALID_ARGUMENT, "forwards"),
    (True, dict(kv_dtype=_native.DTYPE_F16), _native.ERR_INVALID_ARGUMENT, "kv_dtype"),
    (True, dict(kv_dtype=_native.DTYPE_FP8_E4M3, k_scale=0.0), _native.ERR_INVALID_ARGUMENT,
     "scales"),
    (True, dict(num_cache_blocks=0), _native.ERR_INVALID_ARGUMENT, "block"),
    (True, dict(slot_mapping=None), _native.ERR_INVALID_ARGUMENT, "null"),
    (True, dict(flags=_native.ROTARY_NORM, sqk=None), _native.ERR_INVALID_ARGUMENT, "null"),
])
def test_host_validation(lib, append, kw, status, message):
    p = params(**kw)
    fn = lib.dory_rotary_append if append else lib.dory_rotary_embed
    assert fn(ctypes.byref(p), None) == status
    assert message in lib.dory_decode_last_error().decode()
    assert fn(None, None) == _native.ERR_INVALID_ARGUMENT


def _rows(x):
    return _heads("x", x, x.shape[0], x.shape[2])


def test_rows_that_share_memory_are_told_from_rows_side_by_side():
    from dory_rotary_steps import _meet
    T, D = 5, 8
    fused = torch.zeros(T, 7, D)
    q, k, v = fused.split([4, 2, 1], dim=1)

    def meet(a, b):
        got = _meet(_rows(a), a.element_size(), _rows(b), b.element_size(), T, D)
        assert got == _meet(_rows(b), b.element_size(), _rows(a), a.element_size(), T, D)
        return got
    for a, b in ((q, k), (k, v), (q, v), (q, torch.zeros(T, 2, D)), (q, fused[:, 4:])):
        assert not meet(a, b)
    for a, b in ((q, q), (q, fused[:, 3:5]), (fused, v)):
        assert meet(a, b)
    # heads between heads, as one projection a head leaves them
    each = torch.zeros(T, 4, 3, D)
    assert not meet(each[:, :, 0], each[:, :, 1]) and not meet(each[:, :, 2], each[:, 1:, 0])
    assert meet(each[:, :, 0], each[:, 2:, 0])
    # tokens between tokens, and another type over the same memory
    two = torch.zeros(2 * T, 3, D)
    assert not meet(two[::2], two[1::2]) and meet(two[::2], two[:T])
    wide = torch.zeros(T, 3, 2 * D)
    half = wide.view(torch.float16)
    assert meet(wide[..., :D], half[..., :D]) and not meet(wide[..., :D], half[..., 2 * D:3 * D])
    assert not meet(q, fused.view(torch.bfloat16)[:, 4:, :D])
    assert not _meet((64, 8, 8, 0), 4, _rows(k), 4, T, D)  # no heads
    # every pair of slices of a small buffer, against the bytes themselves
    memory = torch.zeros(64, dtype=torch.int16)
    g = torch.Generator().manual_seed(1)
    for _ in range(300):
        views = []
        for _ in range(2):
            token, head, start = (int(torch.randint(0, n, (), generator=g)) for n in (14, 7, 20))
            views.append(memory.as_strided((3, 2, 2), (token, head, 1), start))
        marks = []
        for x in views:
            memory.zero_()
            x.fill_(1)
            marks.append(memory.clone().bool())
        got = _meet(_rows(views[0]), 2, _rows(views[1]), 2, 3, 2)
        assert got == bool((marks[0] & marks[1]).any()), [x.stride() for x in views]
