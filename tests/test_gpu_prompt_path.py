"""The prompt path as a serving step runs it: VllmChunkBinding (rotated append, chunk attention)
over vLLM's metadata and cache layouts, in chunks, mixed with decodes, followed by the
framework's own decode call over the same cache.

Tolerances: the queries and cached rows are bf16, each within 2^-8 of the oracle's FP64 values (the
append's own tests), so a score is off by at most 2 * 2^-8 scale |q| |k| and a weight by twice
that; chunk attention adds its own (test_gpu_chunk): 2^-8 of the weighted mean of |v|, 2^-8 of it
for v's rounding and 2^-8 of the result.
"""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

import dory_prompt_oracle as P
from dory_chunk_attention import ChunkAttention
from dory_decode_attention import EPS, DecodeAttention
from dory_rotary_steps import rotary_cos_sin
from vllm_binding import VllmChunkBinding, kv_cache_views

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
NH, NKV, FACTOR = 8, 2, 0.7


class Layer:
    """One layer's weights-to-be, cache and sequences (projections are drawn per token)."""

    def __init__(self, lens, D=128, layout="unbind", fp8=False, norm=True, seed=0, interleaved=False,
                 rotary=None):
        g = torch.Generator().manual_seed(seed)
        self.D, self.fp8, self.interleaved = D, fp8, interleaved
        B = 16
        self.need = [-(-n // B) for n in lens]
        blocks = sum(self.need) + 2
        kind = torch.uint8 if fp8 else torch.bfloat16
        shape = (blocks, 2, B, NKV, D) if layout == "unbind" else (blocks, NKV, B, 2 * D)
        self.cache = torch.full(shape, 0x7f if fp8 else float("nan"), dtype=kind, device=DEV)
        perm = torch.randperm(blocks, generator=g).to(torch.int32)
        self.table = torch.zeros(len(lens), max(self.need) + 2, dtype=torch.int32)
        at = 0
        for i, n in enumerate(self.need):
            self.table[i, :n] = perm[at:at + n]
            at += n
        self.lens = lens
        self.qkv = [torch.randn(n, NH + 2 * NKV, D, generator=g).to(torch.bfloat16) for n in lens]
        self.gates = [torch.rand(n, NH * D, generator=g) for n in lens]
        self.sqk = (torch.rand(NH * D, generator=g) + 0.5).to(torch.bfloat16) if norm else None
        self.cos_sin = rotary_cos_sin(max(lens) + 8, rotary or D)
        self.scales = (0.02, 0.03) if fp8 else (1.0, 1.0)
        self.scale = 8.0 / D ** 0.5 if norm else D ** -0.5
        self.binding = VllmChunkBinding(ChunkAttention(NH, NKV, D, DEV,
                                                       kv_cache_dtype="fp8" if fp8 else "auto"))

    def step(self, spans, window=0, pad_tokens=0, pad_requests=0):
        """One serving step over spans[i] = (first, last) positions of sequence i (None: not in
        the batch); returns [(sequence, first, last, out rows)]."""
        rows = [(i, *s) for i, s in enumerate(spans) if s is not None]
        cat = lambda xs: torch.cat([xs[i][a:b] for i, a, b in rows])  # noqa: E731
        qkv, gate = cat(self.qkv), cat(self.gates)
        pos = torch.cat([torch.arange(a, b) for _, a, b in rows])
        slots = torch.cat([self.table[i, torch.arange(a, b) // 16].long() * 16 +
                           torch.arange(a, b) % 16 for i, a, b in rows])
        T = len(pos)
        if pad_tokens:  # as for a captured graph: stale rows, slot -1
            qkv = torch.cat([qkv, qkv[:1].expand(pad_tokens, -1, -1)])
            gate = torch.cat([gate, gate[:1].expand(pad_tokens, -1)])
            pos = torch.cat([pos, torch.full((pad_tokens,), 10 ** 6)])
            slots = torch.cat([slots, torch.full((pad_tokens,), -1)])
        starts = [0]
        for _, a, b in rows:
            starts.append(starts[-1] + b - a)
        starts += [starts[-1]] * pad_requests
        table = torch.cat([self.table[[i for i, _, _ in rows]],
                           torch.zeros(pad_requests, self.table.shape[1], dtype=torch.int32)])
        meta = SimpleNamespace(
            query_start_loc=torch.tensor(starts, dtype=torch.int32, device=DEV),
            seq_lens=torch.tensor([b for _, _, b in rows] + [0] * pad_requests, dtype=torch.int32,
                                  device=DEV),
            block_table=table.to(DEV), slot_mapping=slots.to(DEV))
        x = qkv.to(DEV)
        q, k, v = x.split([NH, NKV, NKV], dim=1)
        q_out = torch.empty(x.shape[0], NH, self.D, dtype=torch.bfloat16, device=DEV)
        out = torch.full((x.shape[0], NH * self.D), 3.0, dtype=torch.bfloat16, device=DEV)
        word = torch.zeros(1, dtype=torch.int32, device=DEV)
        self.binding.forward(
            meta, self.cache, q, k, v, pos.to(DEV), self.cos_sin.to(DEV), q_out, window, self.scale,
            out, gate.to(DEV), sqk=None if self.sqk is None else self.sqk.to(DEV), sqk_factor=FACTOR,
            interleaved=self.interleaved, k_scale=self.scales[0], v_scale=self.scales[1],
            error_word=word)
        self.binding.attention.check_errors()
        assert word.item() == 0
        assert (out[T:] == 3.0).all()
        return [(i, a, b, out[starts[j]:starts[j + 1]]) for j, (i, a, b) in enumerate(rows)]

    def oracle(self, i, window):
        """(out, mean of |v|, largest |q| |k|) of sequence i, FP64, straight from the formulas."""
        n, x = self.lens[i], self.qkv[i]
        q, _ = P.rotary(x[:, :NH], torch.arange(n), self.cos_sin, self.interleaved)
        k, _ = P.rotary(x[:, NH:NH + NKV], torch.arange(n), self.cos_sin, self.interleaved)
        v = x[:, NH + NKV:].double()
        if self.sqk is not None:
            q, _ = P.normalised(q, EPS, self.sqk, FACTOR)
            k, _ = P.normalised(k, EPS)
        if self.fp8:  # the cache's rows themselves
            key, value = kv_cache_views(self.cache.view(torch.float8_e4m3fn), NKV, self.D)
            place = torch.arange(n)
            ids = self.table[i, place // 16].long()
            got_k = key.float().cpu().double()[ids, place % 16] * self.scales[0]
            got_v = value.float().cpu().double()[ids, place % 16] * self.scales[1]
            # each within half a step of e4m3, and of bf16 before it
            for got, want, s in ((got_k, k, self.scales[0]), (got_v, v, self.scales[1])):
                want = (want / s).clamp(-448, 448) * s
                assert ((got - want).abs() <= 2.0 ** -4 * 1.07 * want.abs() + s * 2.0 ** -10
                        + 2.0 ** -8 * want.abs()).all()
            k, v = got_k, got_v
        dense = torch.arange(n, dtype=torch.int32)[None]  # one position a block
        out, size = P.chunk_attention(q, k[:, None], v[:, None], dense, [0, n], [n], window,
                                      self.scale, self.gates[i])
        size = size.maximum(P.chunk_attention(q, k[:, None], v[:, None].abs(), dense, [0, n], [n],
                                              window, self.scale, self.gates[i])[0].abs())
        qk = (q.norm(dim=-1).max() * k.norm(dim=-1).max()).item()
        return out, size, qk

    def check(self, rows, window=0):
        for i, a, b, out in rows:
            want, size, qk = self.oracle(i, window)
            rel = 2 * (2 * 2.0 ** -8 * self.scale * qk) + 2 * 2.0 ** -8 + 1e-4
            tol = rel * size[a:b] + 2.0 ** -8 * want[a:b].abs() * (1 + rel) + 1e-6
            off = (out.double().cpu() - want[a:b]).abs()
            assert (off <= tol).all(), (i, a, b, (off - tol).max().item())


@pytest.mark.parametrize("layout", ["unbind", "triton"])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("window", [0, 50])
def test_chunks_and_decodes(layout, fp8, window):
    """Three prompts in chunks of different sizes, steps that mix chunks with single tokens."""
    layer = Layer([150, 37, 260], layout=layout, fp8=fp8)
    steps = [[(0, 64), (0, 20), None], [(64, 65), (20, 37), (0, 200)], [(65, 150), None, (200, 201)],
             [None, None, (201, 260)]]
    rows = []
    for s in steps:
        rows += layer.step(s, window)
    layer.check(rows, window)


def test_whole_prompt_equals_its_chunks_and_padding_changes_nothing():
    whole = Layer([200, 90], seed=4)
    parts = Layer([200, 90], seed=4)
    full = whole.step([(0, 200), (0, 90)], pad_tokens=7, pad_requests=3)
    whole.check(full)
    first = parts.step([(0, 130), None])
    second = parts.step([(130, 200), (0, 90)])
    assert torch.equal(whole.cache.nan_to_num(7), parts.cache.nan_to_num(7))
    # the same values by another order of summation: both within the tolerance of the oracle
    parts.check(first)
    parts.check(second)


@pytest.mark.parametrize("D,norm,interleaved,rotary", [(256, True, False, None), (64, False, True, 32)])
def test_other_shapes(D, norm, interleaved, rotary):
    layer = Layer([70, 41], D=D, norm=norm, interleaved=interleaved, rotary=rotary, seed=5)
    layer.check(layer.step([(0, 70), (0, 40)]) + layer.step([None, (40, 41)]))


@pytest.mark.parametrize("fp8", [False, True])
def test_a_decode_step_reads_the_prompt(fp8):
    """DecodeAttention.from_raw for the next token over the cache the prompt path wrote gives the
    chunk call's own answer for that token."""
    n = 123
    layer = Layer([n], layout="triton", fp8=fp8, seed=6)
    layer.step([(0, n - 1)])
    before = layer.cache.clone()
    want = layer.step([(n - 1, n)])[0][3]
    after, layer.cache = layer.cache, before
    D, x = layer.D, layer.qkv[0][n - 1:]
    turned, _ = P.rotary(x[:, :NH + NKV], [n - 1], layer.cos_sin)
    key, value = kv_cache_views(layer.cache, NKV, D)
    attn = DecodeAttention(NH, NKV, D, DEV, kv_cache_dtype="fp8" if fp8 else "auto")
    out = torch.empty(8, NH * D // 8, device=DEV)
    slot = layer.table[0, (n - 1) // 16].long() * 16 + (n - 1) % 16
    attn.from_raw(turned.float().reshape(-1).to(DEV), x[:, NH + NKV:].float().reshape(-1).to(DEV),
                  layer.sqk.to(DEV), FACTOR, EPS, slot.reshape(1).to(DEV), key, value,
                  layer.table[0].to(DEV), torch.tensor([n], dtype=torch.int32, device=DEV), 0,
                  layer.scale, layer.gates[0][n - 1].to(DEV), out, k_scale=layer.scales[0],
                  v_scale=layer.scales[1])
    attn.check_errors()
    got = out.t().reshape(-1).double()
    torch.testing.assert_close(got, want[0].double(), atol=2e-2, rtol=1e-2)
    # and appends the row the prompt path would have, but for ties in its rounding
    a, b = layer.cache, after
    if fp8:
        a, b = a.view(torch.float8_e4m3fn), b.view(torch.float8_e4m3fn)
    changed = (a.float().nan_to_num(0) - b.float().nan_to_num(0)).abs()
    assert (changed <= 2.0 ** -3 * b.float().nan_to_num(0).abs() + 2.0 ** -8).all()


def test_captured_step():
    layer = Layer([64, 64], seed=7)
    eager = layer.step([(0, 64), (0, 64)])
    want, rows = torch.cat([r[3] for r in eager]).clone(), layer.cache.clone()
    # the same step captured, over a cleared cache
    meta = SimpleNamespace(
        query_start_loc=torch.tensor([0, 64, 128], dtype=torch.int32, device=DEV),
        seq_lens=torch.tensor([64, 64], dtype=torch.int32, device=DEV),
        block_table=layer.table.to(DEV),
        slot_mapping=torch.cat([layer.table[i, torch.arange(64) // 16].long() * 16 +
                                torch.arange(64) % 16 for i in range(2)]).to(DEV))
    q, k, v = torch.cat(layer.qkv).to(DEV).split([NH, NKV, NKV], dim=1)
    pos, cs = torch.arange(64, device=DEV).repeat(2), layer.cos_sin.to(DEV)
    gate, sqk = torch.cat(layer.gates).to(DEV), layer.sqk.to(DEV)
    q_out = torch.empty(128, NH, layer.D, dtype=torch.bfloat16, device=DEV)
    out = torch.zeros(128, NH * layer.D, dtype=torch.bfloat16, device=DEV)

    def call():
        layer.binding.forward(meta, layer.cache, q, k, v, pos, cs, q_out, 0, layer.scale, out, gate,
                              sqk=sqk, sqk_factor=FACTOR)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    layer.cache.fill_(float("nan"))
    out.zero_()
    graph.replay()
    assert torch.equal(out, want)
    assert torch.equal(layer.cache.nan_to_num(9), rows.nan_to_num(9))


def test_refusals():
    layer = Layer([20], seed=8)
    binding = layer.binding
    q = torch.zeros(4, NH, layer.D, dtype=torch.bfloat16, device=DEV)
    out = torch.zeros(4, NH * layer.D, dtype=torch.bfloat16, device=DEV)
    meta = SimpleNamespace(query_start_loc=torch.tensor([0], dtype=torch.int32, device=DEV),
                           seq_lens=torch.tensor([4], dtype=torch.int32, device=DEV),
                           block_table=layer.table.to(DEV), slot_mapping=None)
    with pytest.raises(ValueError, match="query_start_loc"):
        binding.attend(meta, layer.cache, q, 0, 1.0, out)
    meta.query_start_loc = torch.tensor([0, 4], dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="KV-cache shape"):
        binding.attend(meta, layer.cache[:, 0], q, 0, 1.0, out)


FIRST = """
import sys, torch
sys.path[:0] = [{package!r}]
from dory_chunk_attention import ChunkAttention
from dory_rotary_steps import rotary_append, rotary_cos_sin
dev, T = torch.device("cuda"), 40
q, k, v = torch.randn(T, 12, 128, device=dev).bfloat16().split([8, 2, 2], 1)
key = torch.zeros(8, 16, 2, 128, device=dev, dtype=torch.bfloat16)
value, at = key.clone(), torch.arange(T, device=dev)
table = rotary_cos_sin(64, 128, device=dev)
q_out = torch.empty(T, 8, 128, device=dev, dtype=torch.bfloat16)
blocks = torch.arange(8, device=dev, dtype=torch.int32)[None]
start = torch.tensor([0, T], device=dev, dtype=torch.int32)
out = torch.zeros(T, 1024, device=dev, dtype=torch.bfloat16)
attn = ChunkAttention(8, 2, 128, dev)
def step():
    rotary_append(q, k, v, at, table, at, key, value, q_out)
    attn(q_out, key, value, blocks, start, start[1:], 0, 0.09, out)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    step()
graph.replay()
attn.check_errors()
first = out.clone()
for x in (out, key, value):
    x.zero_()
step()
assert torch.equal(out, first) and out.any()
"""


def test_the_first_call_may_be_a_captured_one():
    package = str(Path(__file__).resolve().parents[1] / "dory-vllm-experiments_b200")
    subprocess.run([sys.executable, "-c", FIRST.format(package=package)], check=True, timeout=300)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("fp8", [False, True])
def test_the_decode_call_appends_the_prompt_paths_row(D, fp8):
    """DecodeAttention.from_raw on the FP32 rows that rotary_embed turned, and rotary_append on the
    rows themselves, leave the same bytes in the cache, everywhere."""
    from dory_rotary_steps import rotary_append, rotary_embed
    if fp8 and D == 64:
        pytest.skip("no FP8 caches of 64-dim heads")
    g = torch.Generator(device=DEV).manual_seed(12)
    n, steps = 16, 64
    cos_sin = rotary_cos_sin(n + 1, D, device=DEV)
    sqk = (torch.rand(NH * D, generator=g, device=DEV) + 0.5).to(torch.bfloat16)
    attn = DecodeAttention(NH, NKV, D, DEV, kv_cache_dtype="fp8" if fp8 else "auto")
    ks, vs = (0.02, 0.03) if fp8 else (1.0, 1.0)
    kind = torch.uint8 if fp8 else torch.bfloat16
    table = torch.tensor([1, 0], dtype=torch.int32, device=DEV)
    at, slot = torch.tensor([n], device=DEV), torch.tensor([0], device=DEV)
    for _ in range(steps):
        x = torch.randn(1, NH + 2 * NKV, D, generator=g, device=DEV) * 3
        q, k, v = x.split([NH, NKV, NKV], dim=1)
        caches = [torch.randint(0, 100, (2, 16, NKV, D), generator=g, device=DEV).to(kind)
                  for _ in range(2)]
        mine = [c.clone() for c in caches]
        rotary_append(q, k, v, at, cos_sin, slot, *mine, torch.empty(1, NH, D, dtype=torch.bfloat16,
                                                                     device=DEV),
                      sqk=sqk, sqk_factor=FACTOR, k_scale=ks, v_scale=vs)
        turned = x[:, :NH + NKV].contiguous()
        rotary_embed(q, k, at, cos_sin, turned[:, :NH], turned[:, NH:])
        attn.from_raw(turned.view(-1), v.reshape(-1), sqk, FACTOR, EPS, slot, *caches, table,
                      torch.tensor([n + 1], dtype=torch.int32, device=DEV), 0, 0.1,
                      torch.ones(NH * D, device=DEV), torch.empty(8, NH * D // 8, device=DEV),
                      k_scale=ks, v_scale=vs)
        attn.check_errors()
        assert all(torch.equal(a, b) for a, b in zip(mine, caches))
