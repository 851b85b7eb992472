"""rotary_embed and rotary_append on the GPU against the FP64 oracle.

Tolerances: u(T) = torch.finfo(T).eps / 2 is the rounding to the output type.  A rotated
element is a c - b s in FP32: two products and a sum, each off by at most 2^-24 of its size,
so 3 * 2^-24 (|a c| + |b s|).  The normalisation adds at most D + 2 FP32 roundings of the sum
of squares (halved by the root), rsqrtf's 2 ulp and four products: (D / 2 + 10) 2^-24 relative.
"""

from __future__ import annotations

import pytest
import torch

import _native
import dory_prompt_oracle as P
from dory_rotary_steps import rotary_append, rotary_cos_sin, rotary_embed

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32 = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def inputs(T, NH, NKV, D, R, dtype, seed=0, max_position=600, table=torch.float32):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(T, NH + 2 * NKV, D, generator=g).to(TYPES[dtype])
    pos = torch.randint(0, max_position, (T,), generator=g)
    return qkv, pos, rotary_cos_sin(max_position, R, dtype=table)


def check(got, want, size, dtype):
    u = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * u * 2  # half a step below the normal range
    tol = u * want.abs() + (1 + u) * 3 * F32 * size + tiny
    off = (got.double().cpu() - want).abs()
    assert (off <= tol).all(), (off - tol).max().item()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,NH,NKV,D,R", [
    (1, 32, 8, 128, 128), (7, 3, 1, 64, 64), (33, 4, 2, 256, 64), (5, 2, 2, 128, 34),
    (3, 5, 1, 80, 80), (2, 1, 1, 6, 2), (2, 2, 1, 129, 128), (300, 16, 4, 256, 256),
    (1500, 8, 2, 128, 64), (0, 4, 2, 64, 64)])
def test_embed(T, NH, NKV, D, R, interleaved, dtype):
    qkv, pos, table = inputs(T, NH, NKV, D, R, dtype)
    d = qkv.to(DEV)
    q, k = d[:, :NH], d[:, NH:NH + NKV]  # slices of a fused projection
    qo, ko = torch.empty(T, NH, D, dtype=d.dtype, device=DEV), torch.empty(T, NKV, D, dtype=d.dtype, device=DEV)
    rotary_embed(q, k, pos.to(DEV), table.to(DEV), qo, ko, interleaved=interleaved)
    want, size = P.rotary(qkv, pos, table, interleaved)
    check(qo, want[:, :NH], size[:, :NH], d.dtype)
    check(ko, want[:, NH:NH + NKV], size[:, NH:NH + NKV], d.dtype)
    # in place, the same numbers, v untouched
    rotary_embed(q, k, pos.to(DEV).int(), table.to(DEV), q, k, interleaved=interleaved)
    assert torch.equal(q, qo) and torch.equal(k, ko)
    assert torch.equal(d[:, NH + NKV:].cpu(), qkv[:, NH + NKV:])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,R", [(128, 128), (128, 32), (80, 10)])
def test_inverse_is_the_gradient(D, R, interleaved):
    T, NH = 9, 4
    qkv, pos, table = inputs(T, NH, 1, D, R, "f32", seed=3)
    grad = qkv[:, :NH].contiguous()
    x = torch.randn(T, NH, D, dtype=torch.float64, generator=torch.Generator().manual_seed(4),
                    requires_grad=True)
    c, s = table.double()[pos][:, None, :R // 2], table.double()[pos][:, None, R // 2:]
    at = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    a, b = x[..., at[0]], x[..., at[1]]
    loss = ((a * c - b * s) * grad[..., at[0]]).sum() + ((b * c + a * s) * grad[..., at[1]]).sum() \
        + (x[..., R:] * grad[..., R:]).sum()
    loss.backward()
    out = torch.empty(T, NH, D, device=DEV)
    rotary_embed(grad.to(DEV), None, pos.to(DEV), table.to(DEV), out, interleaved=interleaved,
                 inverse=True)
    _, size = P.rotary(grad, pos, table, interleaved, inverse=True)
    check(out, x.grad, size, torch.float32)
    # and a difference of the forward kernel along a direction agrees with it
    step = 2.0 ** -6
    up, down = torch.empty(T, NH, D, device=DEV), torch.empty(T, NH, D, device=DEV)
    x0, direction = x.detach().float(), grad.flip(0)
    for sign, o in ((1, up), (-1, down)):
        rotary_embed((x0 + sign * step * direction).to(DEV), None, pos.to(DEV), table.to(DEV), o,
                     interleaved=interleaved)
    along = ((up - down).double().cpu() / (2 * step) * grad.double()).sum()
    terms = (grad.double().abs().sum() * x0.abs().max() * 8 * F32 / step).item()
    assert abs(along - (out.double().cpu() * direction.double()).sum()) <= terms


@pytest.mark.parametrize("table", [torch.bfloat16, torch.float16])
def test_table_types_and_strides(table):
    T, NH, D = 21, 6, 128
    qkv, pos, cs = inputs(T, NH, 2, D, 96, "bf16", table=table)
    want, size = P.rotary(qkv[:, :NH], pos, cs)
    base = torch.zeros(NH, T, D + 8, dtype=torch.bfloat16, device=DEV)
    q = base[:, :, :D].transpose(0, 1)  # heads outermost, padded rows
    q.copy_(qkv[:, :NH])
    odd = torch.full((T, NH * D + 1), 7.0, dtype=torch.bfloat16, device=DEV)
    out = odd[:, 1:].unflatten(1, (NH, D))  # rows off the 16-byte grid
    rotary_embed(q, None, pos.to(DEV), cs.to(DEV), out)
    check(out, want, size, torch.bfloat16)
    assert (odd[:, 0] == 7).all() and (base[:, :, D:] == 0).all()


def test_bad_positions_are_reported():
    T, NH, D = 5, 2, 64
    qkv, pos, cs = inputs(T, NH, 1, D, 64, "f32", max_position=32)
    pos[1], pos[3] = 32, -1
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = torch.full((T, NH, D), 3.0, device=DEV)
    rotary_embed(qkv[:, :NH].to(DEV), None, pos.to(DEV), cs.to(DEV), out, error_word=word)
    assert word.item() == _native.DEVERR_POSITION_OOB
    want, size = P.rotary(qkv[:, :NH], pos, cs)
    check(out, want, size, torch.float32)
    assert (out[1] == 0).all() and (out[3] == 0).all()


# ---- append ----
def views(layout, blocks, B, NKV, D, dtype):
    shape = (blocks, NKV, B, 2 * D) if layout == "triton" else (blocks, 2, B, NKV, D)
    raw = torch.randint(0, 100, shape, generator=torch.Generator().manual_seed(9),
                        dtype=torch.uint8).to(dtype if dtype != torch.float8_e4m3fn else torch.uint8).to(DEV)
    raw = raw.view(dtype)
    return (raw, *(raw.transpose(1, 2).split(D, dim=-1) if layout == "triton" else raw.unbind(1)))


def run_append(T, NH, NKV, D, R, dtype, fp8, norm, interleaved, layout, B, seed=0):
    qkv, pos, table = inputs(T, NH, NKV, D, R or 2, dtype, seed=seed)
    table = table if R else None
    kind = torch.float8_e4m3fn if fp8 else torch.bfloat16
    blocks = -(-T // B) + 2
    raw, key, value = views(layout, blocks, B, NKV, D, kind)
    before = raw.view(torch.uint8).clone()
    g = torch.Generator().manual_seed(seed + 1)
    slots = torch.randperm(blocks * B, generator=g)[:T]
    if T > 2:
        slots[T // 2] = -1
    sqk = (torch.rand(NH * D, generator=g) + 0.5).to(torch.bfloat16) if norm else None
    ks, vs = (0.3, 0.07) if fp8 else (1.0, 1.0)
    d = qkv.to(DEV)
    q_out = torch.empty(T, NH * D, dtype=torch.bfloat16, device=DEV)
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    rotary_append(d[:, :NH], d[:, NH:NH + NKV], d[:, NH + NKV:], pos.to(DEV),
                  None if table is None else table.to(DEV), slots.to(DEV), key, value, q_out,
                  sqk=None if sqk is None else sqk.to(DEV), sqk_factor=0.7, eps=1e-6,
                  interleaved=interleaved, k_scale=ks, v_scale=vs, error_word=word)
    assert word.item() == 0
    turn = (lambda x: P.rotary(x, pos, table, interleaved)) if R else \
        (lambda x: (x.double(), torch.zeros_like(x, dtype=torch.float64)))
    q, q_size = turn(qkv[:, :NH])
    k, k_size = turn(qkv[:, NH:NH + NKV])
    more = 0.0
    if norm:
        q, f = P.normalised(q, 1e-6, sqk, 0.7)
        q_size, more = q_size * f, (D / 2 + 10) * F32
        k, f = P.normalised(k, 1e-6)
        k_size = k_size * f
    u = 2.0 ** -8

    def bf16_tol(want, size):
        exact = (u + more * (1 + u)) * want.abs() + (1 + u) * 3 * F32 * size
        return exact + 2.0 ** -133
    off = (q_out.view(T, NH, D).double().cpu() - q).abs()
    assert (off <= bf16_tol(q, q_size)).all()
    v = qkv[:, NH + NKV:].double()
    touched = torch.zeros(blocks * B, dtype=torch.bool)
    for name, cache, want, size, scale in (("k", key, k, k_size, ks),
                                           ("v", value, v, torch.zeros_like(v), vs)):
        got = cache.to(torch.float32).double().cpu().reshape(blocks * B, NKV, D) \
            if not fp8 else cache.float().double().cpu().reshape(blocks * B, NKV, D)
        for t in range(T):
            if slots[t] < 0:
                continue
            touched[slots[t]] = True
            tol = bf16_tol(want[t], size[t])
            if fp8:  # to e4m3 units; half a step there is 2^-4 of the value, 2^-10 below 2^-6
                w = (want[t] / scale).clamp(-448, 448)
                tol = tol / scale * (1 + 2.0 ** -4) + 2.0 ** -4 * w.abs() + 2.0 ** -10
            else:
                w = want[t]
            assert ((got[slots[t]] - w).abs() <= tol).all(), (name, t)
    # every other row is as it was
    after, old = raw.view(torch.uint8).cpu(), before.cpu()
    e = 1 if fp8 else 2
    if layout == "triton":
        same = (after == old).reshape(blocks, NKV, B, -1).all(-1).all(1).reshape(-1)
    else:
        same = (after == old).reshape(blocks, 2, B, NKV * D * e).all(-1).all(1).reshape(-1)
    assert same[~touched].all()
    return q_out, raw


@pytest.mark.parametrize("layout,B", [("triton", 16), ("unbind", 48)])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("T,NH,NKV,D,R,dtype,interleaved", [
    (1, 32, 8, 128, 128, "bf16", False), (37, 16, 4, 256, 64, "f32", True),
    (5, 3, 1, 64, 34, "f16", False), (5, 3, 1, 64, 34, "bf16", True),
    (700, 8, 4, 128, 128, "bf16", False), (700, 8, 4, 128, 96, "f32", True),
    (9, 4, 2, 128, 0, "bf16", False)])
def test_append(T, NH, NKV, D, R, dtype, interleaved, fp8, norm, layout, B):
    run_append(T, NH, NKV, D, R, dtype, fp8, norm, interleaved, layout, B)


def test_append_keys_alone_and_bad_slots():
    T, NKV, D = 6, 2, 128
    qkv, pos, table = inputs(T, 0, NKV, D, D, "bf16", max_position=64)
    raw, key, value = views("triton", 3, 16, NKV, D, torch.bfloat16)
    slots = torch.tensor([3, 48, 1 << 40, -5, 7, 47])
    pos[3] = 9999  # a padding token's position is nobody's business
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    before = raw.clone()
    rotary_append(None, qkv[:, :NKV].to(DEV), qkv[:, NKV:].to(DEV), pos.to(DEV), table.to(DEV),
                  slots.to(DEV), key, value, None, error_word=word)
    assert word.item() == _native.DEVERR_SLOT_OOB
    changed = (raw != before).reshape(3, NKV, 16, -1).any(-1).any(1).reshape(-1).nonzero().flatten()
    assert changed.tolist() == [3, 7, 47]
    want, _ = P.rotary(qkv[:, :NKV], pos, table)
    row = key.reshape(48, NKV, D)[7].double().cpu()
    assert ((row - want[4]).abs() <= 2.0 ** -8 * want[4].abs() + 1e-6).all()


def test_append_saturates_and_keeps_zero_rows():
    T, NKV, D = 3, 1, 64
    k = torch.zeros(T, NKV, D, device=DEV)
    k[0] = 1e6
    v = torch.full((T, NKV, D), -1e30, device=DEV)
    raw, key, value = views("unbind", 1, 16, NKV, D, torch.float8_e4m3fn)
    rotary_append(None, k, v, None, None, torch.arange(T, device=DEV), key, value, None)
    assert (key[0, 0].float() == 448).all() and (key[0, 1:3].float() == 0).all()
    assert (value[0, :3].float() == -448).all()
    # the normalisation of a zero row divides by sqrt(eps): zero
    rotary_append(None, k, v, None, None, torch.arange(T, device=DEV), key, value, None,
                  sqk=torch.ones(64, device=DEV))
    assert (key[0, 1:3].float() == 0).all()


def test_refusals():
    T, NH, NKV, D = 4, 4, 2, 128
    q, k = torch.zeros(T, NH, D, device=DEV), torch.zeros(T, NKV, D, device=DEV)
    table, pos = rotary_cos_sin(8, D, device=DEV), torch.zeros(T, dtype=torch.int64, device=DEV)
    cache = torch.zeros(2, 16, NKV, D, dtype=torch.bfloat16, device=DEV)
    qo = torch.empty(T, NH, D, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError):  # host table
        rotary_embed(q, None, pos, table.cpu(), q)
    with pytest.raises(ValueError):  # another type
        rotary_embed(q, None, pos, table, qo)
    with pytest.raises(ValueError):  # k without k_out
        rotary_embed(q, k, pos, table, q)
    for kw in (dict(v=k[:, :1]), dict(v=k.half()), dict(key=cache[:, :, :1]), dict(slots=pos.int()),
               dict(slots=pos[:2]), dict(value=cache.float()), dict(q_out=qo[:2]),
               dict(q_out=qo.float()), dict(sqk=torch.ones(5, device=DEV)),
               dict(key=torch.zeros(2, 16, NKV, 2 * D, dtype=torch.bfloat16, device=DEV)[..., :D])):
        a = dict(v=k, key=cache, value=cache, slots=pos, q_out=qo, sqk=None)
        a.update(kw)
        with pytest.raises(ValueError):
            rotary_append(q, k, a["v"], pos, table, a["slots"], a["key"], a["value"], a["q_out"],
                          sqk=a["sqk"])
    with pytest.raises(NotImplementedError):  # head_dim 80
        c80 = torch.zeros(2, 16, NKV, 80, dtype=torch.bfloat16, device=DEV)
        rotary_append(None, k[..., :80].contiguous(), k[..., :80].contiguous(), None, None, pos,
                      c80, c80, None)


def test_captured_and_on_another_stream():
    T, NH, NKV, D = 8, 4, 2, 128
    qkv, pos, table = inputs(T, NH, NKV, D, D, "bf16")
    d, p, cs = qkv.to(DEV), pos.to(DEV), table.to(DEV)
    raw, key, value = views("triton", 2, 16, NKV, D, torch.bfloat16)
    slots = torch.arange(T, device=DEV)
    out = torch.zeros(T, NH, D, dtype=torch.bfloat16, device=DEV)

    def call():
        rotary_append(d[:, :NH], d[:, NH:NH + NKV], d[:, NH + NKV:], p, cs, slots, key, value, out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    first, rows = out.clone(), raw.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    out.zero_()
    d.copy_(qkv.flip(0))
    p.copy_(pos.flip(0))
    slots.copy_(torch.arange(T, device=DEV).flip(0))
    graph.replay()
    assert torch.equal(out, first.flip(0)) and torch.equal(raw, rows)


@pytest.mark.parametrize("D,R", [(128, 128), (64, 24)])  # the wide kernel, and the general one
def test_an_unknown_position_appends_zeros_whatever_eps(D, R):
    q, k, v = (torch.randn(1, n, D, device=DEV) for n in (4, 2, 2))
    key = torch.full((2, 16, 2, D), 5.0, dtype=torch.bfloat16, device=DEV)
    value = key.clone()
    q_out = torch.full((1, 4, D), 5.0, dtype=torch.bfloat16, device=DEV)
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    rotary_append(q, k, v, torch.tensor([9], device=DEV), rotary_cos_sin(8, R, device=DEV),
                  torch.tensor([17], device=DEV), key, value, q_out,
                  sqk=torch.ones(4 * D, device=DEV), eps=0.0, error_word=word)
    assert word.item() == _native.DEVERR_POSITION_OOB
    assert (q_out == 0).all() and (key[1, 1] == 0).all()
    assert torch.equal(value[1, 1], v[0].to(torch.bfloat16))
    assert (key[0] == 5.0).all() and (key[1, 2:] == 5.0).all()


def test_a_block_walks_many_tokens():
    """More tokens than 32 a block, which the kernels read positions and slots of at a time, with
    positions and slots out of range everywhere."""
    T, D = 3552 * 70 + 5, 64
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(T, 4, D, generator=g, device=DEV).to(torch.bfloat16)
    q, k, v = x.split([2, 1, 1], dim=1)
    pos = torch.randint(-1, 4100, (T,), generator=g, device=DEV)
    blocks = T // 16 + 1
    slots = torch.randperm(T, generator=g, device=DEV)
    slots[pos % 7 == 1] = -1
    slots[pos % 7 == 2] += blocks * 16
    table = rotary_cos_sin(4096, D, device=DEV)
    key = torch.full((blocks, 16, 1, D), 5.0, dtype=torch.bfloat16, device=DEV)
    value = key.clone()
    q_out = torch.empty(T, 2, D, dtype=torch.bfloat16, device=DEV)
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    rotary_append(q, k, v, pos, table, slots, key, value, q_out, error_word=word)
    assert word.item() == _native.DEVERR_POSITION_OOB | _native.DEVERR_SLOT_OOB
    inside = (pos >= 0) & (pos < 4096)
    c, s = (t[:, None] for t in table[pos.clamp(0, 4095)].double().chunk(2, dim=1))
    a, b = x[:, :3].double().chunk(2, dim=2)
    want = torch.cat([a * c - b * s, b * c + a * s], dim=2) * inside[:, None, None]
    size = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()], dim=2)
    # each product and the sum rounded to FP32, then to bf16
    tol = 3 * 2.0 ** -24 * size + 2.0 ** -8 * want.abs() * (1 + 2.0 ** -20) + 1e-30
    assert ((q_out.double() - want[:, :2]).abs() <= tol[:, :2]).all()
    kept = (slots >= 0) & (slots < blocks * 16)
    at = slots[kept]
    flat_k, flat_v = key.view(-1, D), value.view(-1, D)
    assert ((flat_k[at].double() - want[kept, 2]).abs() <= tol[kept, 2]).all()
    assert torch.equal(flat_v[at], v[kept, 0])
    free = torch.ones(blocks * 16, dtype=torch.bool, device=DEV)
    free[at] = False
    assert (flat_k[free] == 5.0).all() and (flat_v[free] == 5.0).all()
    rotary_embed(q, k, pos, table, q_out, k_out := torch.empty_like(k))
    assert ((q_out.double() - want[:, :2]).abs() <= tol[:, :2]).all()
    assert ((k_out.double() - want[:, 2:]).abs() <= tol[:, 2:]).all()


@pytest.mark.parametrize("D,R", [(64, 64), (128, 64), (256, 256)])
def test_a_padding_token_of_unknown_position_is_not_reported(D, R):
    x = torch.randn(3, 4, D, device=DEV).to(torch.bfloat16)
    key = torch.full((2, 16, 1, D), 5.0, dtype=torch.bfloat16, device=DEV)
    value, word = key.clone(), torch.zeros(1, dtype=torch.int32, device=DEV)
    q_out = torch.empty(3, 2, D, dtype=torch.bfloat16, device=DEV)
    rotary_append(x[:, :2], x[:, 2:3], x[:, 3:], torch.tensor([0, 99, -4], device=DEV),
                  rotary_cos_sin(8, R, device=DEV), torch.tensor([3, -1, -1], device=DEV), key,
                  value, q_out, error_word=word)
    assert word.item() == 0 and (q_out[1:] == 0).all()
    assert torch.equal(value[0, 3], x[0, 3:]) and (value.view(-1, D)[4:] == 5.0).all()


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("dim_step", [1, 3])  # the wide kernel, and (odd strides) the general one
def test_append_offsets_pass_32_bits(D, dim_step):
    stride = 2 ** 25 + (dim_step - 1)
    buf = torch.empty(70 * stride, dtype=torch.bfloat16, device=DEV)
    key = buf.as_strided((70, 16, 2, D), (stride, 2 * D, D, 1))
    value = buf.as_strided((70, 16, 2, D), (stride, 2 * D, D, 1), 2 ** 24)
    for c in (key, value):
        c[[0, 5, 69]] = 5.0
    x = torch.randn(3, 6, D, device=DEV).to(torch.bfloat16)
    slots = torch.tensor([69 * 16 + 15, 3, 5 * 16], device=DEV)
    q_out = torch.empty(3, 2, D, dtype=torch.bfloat16, device=DEV)
    rotary_append(x[:, :2], x[:, 2:4], x[:, 4:], None, None, slots, key, value, q_out)
    assert torch.equal(q_out, x[:, :2])
    for c, rows in ((key, x[:, 2:4]), (value, x[:, 4:])):
        assert torch.equal(c[69, 15], rows[0]) and torch.equal(c[0, 3], rows[1])
        assert torch.equal(c[5, 0], rows[2])
        assert (c[69, :15] == 5.0).all() and (c[5, 1:] == 5.0).all() and (c[0, 4:] == 5.0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_rows_off_the_16_byte_grid_give_the_same_bits(dtype, interleaved):
    T, NH, NKV, D, R = 1500, 4, 2, 128, 96
    qkv, pos, table = inputs(T, NH, NKV, D, R, dtype, seed=24)
    d, p, cs = qkv.to(DEV), pos.to(DEV), table.to(DEV)
    odd = torch.zeros(T, (NH + 2 * NKV) * D + 1, dtype=d.dtype, device=DEV)[:, 1:].unflatten(1, (-1, D))
    odd.copy_(d)
    outs = []
    for x in (d, odd):
        q, k, v = x.split([NH, NKV, NKV], dim=1)
        qo, ko = torch.empty_like(q, memory_format=torch.contiguous_format), \
            torch.empty_like(k, memory_format=torch.contiguous_format)
        rotary_embed(q, k, p, cs, qo, ko, interleaved=interleaved)
        key = torch.zeros(T // 16 + 1, 16, NKV, D, dtype=torch.bfloat16, device=DEV)
        value, qb = key.clone(), torch.empty(T, NH, D, dtype=torch.bfloat16, device=DEV)
        rotary_append(q, k, v, p, cs, torch.arange(T, device=DEV), key, value, qb,
                      interleaved=interleaved)
        outs.append((qo, ko, key, value, qb))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


@pytest.mark.parametrize("D,R", [(64, 64), (128, 128), (128, 0), (256, 64), (128, 34)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_leaves_the_bits_of_the_other_normalising_calls(D, R, interleaved):
    """The rotated FP32 rows through qk_norm_cache give the query and the cache rows bit for bit."""
    from dory_sublayer_steps import qk_norm_cache
    T, NH, NKV = 1500, 4, 2
    qkv, pos, table = inputs(T, NH, NKV, D, R or 2, "f32", seed=21)
    d = qkv.to(DEV)
    # rows of many sizes, so that sums of squares come near every kind of rounding
    d[:, :NH + NKV] *= torch.exp2(torch.randint(-9, 9, (T, NH + NKV, 1), device=DEV).float())
    cs, p = table.to(DEV), pos.to(DEV)
    sqk = (torch.rand(NH * D, generator=torch.Generator().manual_seed(22)) + 0.5).to(DEV)
    slots = torch.randperm(T, generator=torch.Generator().manual_seed(23)).to(DEV)
    turned = d[:, :NH + NKV].contiguous()
    if R:
        rotary_embed(d[:, :NH], d[:, NH:NH + NKV], p, cs, turned[:, :NH], turned[:, NH:],
                     interleaved=interleaved)
    caches = [torch.zeros(T // 16 + 1, 16, NKV, D, dtype=torch.bfloat16, device=DEV) for _ in range(4)]
    q_out = [torch.empty(T, NH * D, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    qk_norm_cache(turned.view(T, -1), d[:, NH + NKV:].reshape(T, -1).contiguous(), sqk, 0.7, 1e-6, q_out[0], NH, D,
                  key_cache=caches[0], value_cache=caches[1], slot_mapping=slots)
    rotary_append(d[:, :NH], d[:, NH:NH + NKV], d[:, NH + NKV:], p, cs if R else None, slots,
                  caches[2], caches[3], q_out[1], sqk=sqk, sqk_factor=0.7, eps=1e-6,
                  interleaved=interleaved)
    assert torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])
    assert torch.equal(q_out[0], q_out[1])


@pytest.mark.parametrize("D,R", [(128, 128), (64, 24)])  # the wide kernel, and the general one
def test_a_norm_beyond_fp32_gives_zeros(D, R):
    """The sum of squares is an FP32 value: infinite from rows of 1e20 on."""
    x = torch.full((1, 3, D), 1e20, device=DEV)
    key = torch.full((1, 16, 1, D), 5.0, dtype=torch.bfloat16, device=DEV)
    value, q_out = key.clone(), torch.empty(1, 1, D, dtype=torch.bfloat16, device=DEV)
    rotary_append(x[:, :1], x[:, 1:2], x[:, 2:], torch.tensor([0], device=DEV),
                  rotary_cos_sin(8, R, device=DEV), torch.tensor([0], device=DEV), key, value, q_out,
                  sqk=torch.ones(D, device=DEV))
    assert (q_out == 0).all() and (key[0, 0] == 0).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_normalised_rows_off_the_16_byte_grid_give_the_same_bits(interleaved):
    T, NH, NKV, D, R = 1500, 4, 2, 128, 96
    qkv, pos, table = inputs(T, NH, NKV, D, R, "f32", seed=25)
    d, p, cs = qkv.to(DEV), pos.to(DEV), table.to(DEV)
    odd = torch.zeros(T, (NH + 2 * NKV) * D + 1, device=DEV)[:, 1:].unflatten(1, (-1, D))
    odd.copy_(d)
    outs = []
    for x in (d, odd):
        key = torch.zeros(T // 16 + 1, 16, NKV, D, dtype=torch.bfloat16, device=DEV)
        value, q_out = key.clone(), torch.empty(T, NH, D, dtype=torch.bfloat16, device=DEV)
        rotary_append(*x.split([NH, NKV, NKV], dim=1), p, cs, torch.arange(T, device=DEV), key, value,
                      q_out, sqk=torch.full((NH * D,), 1.3, device=DEV), sqk_factor=0.7,
                      interleaved=interleaved)
        outs.append((key, value, q_out))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_outputs_over_other_arguments_are_refused():
    T, NH, NKV, D = 6, 4, 2, 64
    fused = torch.randn(T, NH + 2 * NKV, D, device=DEV).to(torch.bfloat16)
    kept = fused.clone()
    q, k, v = fused.split([NH, NKV, NKV], dim=1)
    table, pos = rotary_cos_sin(8, D, device=DEV), torch.arange(T, device=DEV)
    other = torch.empty(T, NH, D, dtype=torch.bfloat16, device=DEV)
    cache = torch.zeros(3, 16, NKV, D, dtype=torch.bfloat16, device=DEV)
    value = torch.zeros_like(cache)
    for args in ((q, k, pos, table, fused[:, NH - 1:2 * NH - 1], torch.empty_like(k)),
                 (q, k, pos, table, other, fused[:, 1:1 + NKV]),
                 (q, k, pos, table, other, other[:, 1:1 + NKV])):
        with pytest.raises(ValueError, match="apart"):
            rotary_embed(*args)
    over = cache.view(-1)[:T * NH * D].view(T, NH, D)
    for out in (fused[:, NH:2 * NH], over, over.flatten(1)):
        with pytest.raises(ValueError, match="apart"):
            rotary_append(q, k, v, pos, table, pos, cache, value, out)
    with pytest.raises(ValueError, match="apart"):
        rotary_append(other, k, v, pos, table, pos, cache, value, fused[:, 2 * NKV:])
    pool = torch.zeros(8, 16, NKV, D, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="apart"):  # over the end of a cache
        rotary_append(q, k, v, pos, table, pos, pool[:3], value, pool[2:].view(-1)[16 * D:][:over.numel()]
                      .view_as(over))
    assert not pool.any()
    assert torch.equal(fused, kept) and not cache.any() and not value.any()
    rotary_append(q, k, v, pos, table, pos, pool[:3], value, pool[3:].view(-1)[:over.numel()]
                  .view_as(over))  # right behind it
    rotary_append(other, k, v, pos, table, pos, cache, value, q)  # beside k and v, token by token
    assert torch.equal(fused[:, NH:], kept[:, NH:])
    assert torch.equal(value.view(-1, NKV, D)[:T], v)
