"""ChunkAttention on the GPU against the FP64 oracle.

Tolerance of an element, with A = sum_c w_c |v_c| (the oracle's second result): the weights are
rounded to bf16 (2^-8 of each: 2^-8 A), a score is off by at most (D + 4) 2^-24 scale |q| |k| and
a weight by twice that share, the exponential by 3e-6 (its polynomial) and as much in the sum it
is divided by, the two sums by (8 + L) 2^-24 at most, and the result is rounded to bf16 (2^-8
|out|).  FP8 caches: the weights are f16 numbers of at most 2^15 whose row's largest is 2^7 or
more, so besides 2^-11 of each, a weight is off by up to half a step of f16's smallest, 2^-25,
which is 2^-32 of the largest: with L of them over a sum of at least the largest, 2^-32 L max|v|.
"""

from __future__ import annotations

import pytest
import torch

import _native
import dory_prompt_oracle as P
import workloads as W
from dory_chunk_attention import ChunkAttention

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
F32 = 2.0 ** -24


class Batch:
    """A ragged batch over a cache whose unused rows hold NaN (bf16 and e4m3 alike)."""

    def __init__(self, lens, NH=8, NKV=2, D=128, B=16, layout="triton", fp8=False, seed=0,
                 rows_after=0, spare=3, spread=1.0, poison=True):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.NH, self.NKV, self.D, self.B, self.fp8 = NH, NKV, D, B, fp8
        self.lens = lens
        need = [max(1, -(-n // B)) for _, n in lens]
        self.blocks = sum(need) + spare
        kind = torch.float8_e4m3fn if fp8 else torch.bfloat16
        _, key, value = W.cache_views(self.blocks, B, NKV, D, layout, DEV, torch.float32)
        raw, self.key, self.value = W.cache_views(self.blocks, B, NKV, D, layout, DEV, kind)
        for c in (key, value):
            c.copy_(torch.randn(c.shape, generator=g, device=DEV) * spread)
        perm = torch.randperm(self.blocks, generator=g, device=DEV).to(torch.int32)
        width = max(need) + 1
        self.tables = torch.full((len(lens), width), -7, dtype=torch.int32, device=DEV)
        used = torch.zeros(self.blocks, B, dtype=torch.bool, device=DEV)
        at = 0
        for i, (_, n) in enumerate(lens):
            ids = perm[at:at + need[i]]
            at += need[i]
            self.tables[i, :need[i]] = ids
            pos = torch.arange(n, device=DEV)
            used[ids[pos // B].long(), pos % B] = True
        if poison:
            key[~used], value[~used] = float("nan"), float("nan")
        self.key.copy_(key.to(kind))
        self.value.copy_(value.to(kind))
        starts = [0]
        for n, _ in lens:
            starts.append(starts[-1] + n)
        self.T = starts[-1] + rows_after
        self.query_start = torch.tensor(starts, dtype=torch.int32, device=DEV)
        self.seq_lens = torch.tensor([n for _, n in lens], dtype=torch.int32, device=DEV)
        self.q = torch.randn(self.T, NH, D, generator=g, device=DEV).to(torch.bfloat16)
        self.gate = torch.rand(self.T, NH * D, generator=g, device=DEV)
        self.out = torch.full((self.T, NH * D), 5.0, dtype=torch.bfloat16, device=DEV)
        self.scales = (0.7, 1.3) if fp8 else (1.0, 1.0)
        self.scale = D ** -0.5

    def attention(self):
        return ChunkAttention(self.NH, self.NKV, self.D, DEV,
                              kv_cache_dtype="fp8" if self.fp8 else "auto")

    def run(self, window=0, gate=None, attn=None, errors=0, q=None, out=None):
        attn = attn or self.attention()
        attn(self.q if q is None else q, self.key, self.value, self.tables, self.query_start,
             self.seq_lens, window, self.scale, self.out if out is None else out, gate=gate,
             k_scale=self.scales[0], v_scale=self.scales[1])
        assert attn.fetch_errors() == errors
        return self.out if out is None else out

    def oracle(self, window=0, gate=None):
        return P.chunk_attention(self.q, self.key.float() * self.scales[0],
                                 self.value.float() * self.scales[1], self.tables,
                                 self.query_start.tolist(), self.seq_lens.tolist(), window,
                                 self.scale, gate)

    def check(self, out, window=0, gate=None):
        want, size = self.oracle(window, gate)
        owned = ~want.isnan().all(1)
        owned[self.query_start[-1].item():] = False
        longest = max([n for _, n in self.lens] + [1])
        k = self.key.float().nan_to_num(0, 0, 0).norm(dim=-1).max().item() * self.scales[0]
        score = (self.D + 4) * F32 * self.scale * self.q.float().norm(dim=-1).max().item() * k
        rel = 2.0 ** -8 + 2 * score + 6e-6 + (8 + longest) * F32
        tol = rel * size + 2.0 ** -8 * want.abs() * (1 + rel) + 2.0 ** -130
        if self.fp8:
            v = self.value.float().nan_to_num(0, 0, 0).abs().max().item() * self.scales[1]
            tol = tol + 2.0 ** -32 * longest * v * (1 if gate is None else gate.double())
        off = (out.double() - want).abs()
        bad = ~(off <= tol) & owned[:, None]
        assert not bad.any(), (bad.sum().item(), bad.nonzero()[0].tolist(),
                               out[bad][:4].tolist(), want[bad][:4].tolist())
        if (~owned).any():
            assert (out[~owned] == 5.0).all()


RAGGED = [(1, 1), (0, 50), (7, 7), (1, 130), (300, 300), (2, 1000), (64, 65), (1, 16), (33, 257)]


@pytest.mark.parametrize("lens", [[(1, 1)], [(1, 17)], [(1, 2000)], [(4, 640)], [(5, 5)], [(128, 128)],
                                  [(129, 300)], [(64, 64)], [(16, 4099)], [(700, 1500)], RAGGED])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_lengths(lens, D):
    b = Batch(lens, D=D)
    b.check(b.run())
    b.check(b.run(gate=b.gate), gate=b.gate)


@pytest.mark.parametrize("window", [1, 2, 16, 100, 128, 129, 1024])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_windows(window, D):
    b = Batch([(300, 700), (1, 1), (1, 1500), (40, 40), (130, 2000)], D=D, seed=1)
    b.check(b.run(window=window, gate=b.gate), window, b.gate)


@pytest.mark.parametrize("NH,NKV", [(1, 1), (2, 2), (4, 2), (3, 1), (5, 1), (12, 2), (7, 1), (8, 1),
                                    (16, 1), (33, 1), (64, 1), (32, 8)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_head_groups(NH, NKV, D):
    b = Batch([(150, 170), (1, 33), (9, 400)], NH=NH, NKV=NKV, D=D, seed=2)
    b.check(b.run())


@pytest.mark.parametrize("layout", W.LAYOUTS)
@pytest.mark.parametrize("B", [16, 32, 48, 64, 80, 128, 256, 272])
def test_cache_layouts(layout, B):
    b = Batch([(90, 600), (3, 3), (200, 200)], B=B, layout=layout, seed=3)
    b.check(b.run(window=150), 150)


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("layout,B", [("triton", 16), ("unbind", 48), ("bench", 128)])
@pytest.mark.parametrize("window", [0, 77])
def test_fp8(D, layout, B, window):
    b = Batch(RAGGED + [(260, 900)], D=D, B=B, layout=layout, fp8=True, seed=4)
    b.check(b.run(window=window, gate=b.gate), window, b.gate)


@pytest.mark.parametrize("D", [128, 256])
def test_fp8_groups_and_query_sizes(D):
    b = Batch([(150, 170), (1, 33), (9, 400)], NH=10, NKV=2, D=D, fp8=True, seed=5)
    # rows of very different sizes, some beyond the range of half precision
    b.q *= torch.exp2(torch.randint(-24, 20, (b.T, b.NH, 1), device=DEV).float()).to(torch.bfloat16)
    b.scale = 1e-5
    b.check(b.run())


@pytest.mark.parametrize("gate_type", [torch.float32, torch.bfloat16, torch.float16])
def test_gate_types_and_strides(gate_type):
    b = Batch(RAGGED, seed=6, rows_after=5)
    wide = torch.zeros(b.T, b.NH * b.D + 64, dtype=gate_type, device=DEV)
    gate = wide[:, 64:]
    gate.copy_(b.gate)
    fused = torch.zeros(b.T, b.NH + 4, b.D, dtype=torch.bfloat16, device=DEV)
    fused[:, 2:2 + b.NH] = b.q
    out = torch.full((b.T, b.NH * b.D + 8), 5.0, dtype=torch.bfloat16, device=DEV)
    b.run(gate=gate, q=fused[:, 2:2 + b.NH], out=out[:, :b.NH * b.D])
    b.check(out[:, :b.NH * b.D], gate=gate.float())
    assert (out[:, b.NH * b.D:] == 5.0).all()
    heads_first = b.q.transpose(0, 1).contiguous().transpose(0, 1)
    other = b.run(q=heads_first)
    b.check(other)


@pytest.mark.parametrize("fp8", [False, True])
def test_empty_and_padded_requests(fp8):
    b = Batch([(5, 20), (3, 3), (2, 40), (4, 10)], fp8=fp8, rows_after=4)
    b.seq_lens[1] = 0   # padded: zero rows
    b.seq_lens[3] = 2   # fewer positions than rows: the first two rows have none
    out = b.run()
    b.check(out)
    assert (out[5:8] == 0).all() and (out[10:12] == 0).all() and (out[12:14] != 0).any()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("fp8", [False, True])
def test_bad_blocks_are_left_out(D, fp8):
    if fp8 and D == 64:
        pytest.skip("no FP8 caches of 64-dim heads")
    b = Batch([(40, 300), (1, 200), (200, 200)], D=D, fp8=fp8, seed=7)
    b.tables[0, 3], b.tables[1, 0], b.tables[2, 5] = b.blocks, -1, 1 << 30
    b.check(b.run(errors=_native.DEVERR_BLOCK_OOB))
    # a length beyond the table: the positions it cannot name are left out
    b = Batch([(4, 100)], D=D, fp8=fp8, seed=8)
    b.tables = b.tables[:, :5].contiguous()
    b.seq_lens[0] = 84
    b.check(b.run(errors=_native.DEVERR_BLOCK_OOB))
    b.seq_lens[0] = 2_000_000_000  # every visible position is beyond the table
    b.tables = b.tables[:, :2].contiguous()
    out = b.run(window=16, errors=_native.DEVERR_BLOCK_OOB)
    assert (out == 0).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 40])
def test_hidden_rows_may_hold_anything(bad, D, window):
    """A later token's K or V, or one before a row's window, must not reach that row."""
    b = Batch([(150, 400), (1, 50), (60, 60)], D=D, seed=9)
    table = b.tables[0]
    for pos, which in ((399, b.value), (320, b.value), (380, b.key)):
        which[table[pos // 16].long(), pos % 16, 0, ::3] = bad
    first = 400 - 150
    if window:  # positions that only the first rows see
        b.value[table[(first - 30) // 16].long(), (first - 30) % 16, 1, 5] = bad
    out = b.run(window=window).double()
    want, size = b.oracle(window)
    clean = want.isfinite() & size.isfinite()
    assert (~clean).any() and clean.any()
    assert out[clean].isfinite().all()
    off, tol = (out - want)[clean].abs(), (2.0 ** -6 * size + 1e-6)[clean]
    assert (off <= tol).all()
    assert (out[want.isnan()].isnan()).all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens", [[(20, 200)], [(1, 3000)]])  # whole items, and parts joined
def test_a_visible_nan_key_reaches_its_rows(D, lens):
    """Wherever in a tile the position lies."""
    b = Batch(lens, D=D, seed=31)
    clean = b.run().clone().view(b.T, b.NH, D)
    groups = b.NH // b.NKV
    for pos in list(range(100, 117)) + [0, 33, 63, 64, 127, 128]:
        row = b.key[b.tables[0, pos // 16].long(), pos % 16, 1]
        kept = row.clone()
        row[5] = float("nan")
        out = b.run().view(b.T, b.NH, D)
        assert out[:, groups:].isnan().all(), pos
        assert torch.equal(out[:, :groups], clean[:, :groups])
        row.copy_(kept)


def test_a_single_token_of_any_stride():
    b = Batch([(1, 90)], NH=4, NKV=1, seed=32)
    want = b.run(gate=b.gate).clone()
    q = b.q.as_strided((1, 4, 128), (4 * 128 + 1, 128, 1))
    gate, out = (x.as_strided(x.shape, (x.shape[1] + 3, 1)) for x in (b.gate, b.out))
    b.out.fill_(5.0)
    b.key, b.value = (c.as_strided(c.shape, (c.stride(0), c.stride(1), 1, 1))
                      for c in (b.key, b.value))
    assert torch.equal(b.run(gate=gate, q=q, out=out), want)


@pytest.mark.parametrize("starts", [[0, 30, 20, 40], [-1, 10, 20, 40], [0, 10, 20, 41],
                                    [0, 40, 0, 40]])
def test_a_broken_query_start_is_reported_and_nothing_written(starts):
    b = Batch([(10, 50), (10, 20), (20, 20)], seed=33)
    b.query_start.copy_(torch.tensor(starts, dtype=torch.int32))
    out = b.run(errors=_native.DEVERR_QUERY_START)
    assert (out == 5.0).all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("spread", [0.0, 8.0, 60.0])
def test_flat_and_steep_scores(D, spread):
    b = Batch([(260, 1500), (3, 700)], D=D, seed=10, spread=1.0)
    if spread == 0.0:
        b.q.zero_()
    else:  # scores that grow with the position, so the running maximum moves all the time
        b.q[:, :, 0] = spread
        for i, (_, n) in enumerate(b.lens):
            pos = torch.arange(n, device=DEV)
            b.key[b.tables[i][pos // 16].long(), pos % 16, :, 0] = \
                (pos[:, None] / 16).to(torch.bfloat16).expand(-1, b.NKV)
    b.check(b.run())


@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_long_prompt_many_times(D):
    """Many tiles an item and many items an SM, so every role gets ahead of the others."""
    b = Batch([(4096, 4096)], D=D, seed=15)
    attn = b.attention()
    first = b.run(attn=attn).clone()
    b.check(first)
    for _ in range(20):
        assert torch.equal(b.run(attn=attn), first)


@pytest.mark.parametrize("D,fp8", [(64, False), (128, False), (256, False), (128, True), (256, True)])
@pytest.mark.parametrize("most", [3, 40, 200])
def test_many_short_sequences(D, fp8, most):
    """Several items an SM, of one tile or a few: loads and conversions run items ahead of the
    softmax, whose warps are at the output of the item before."""
    g = torch.Generator().manual_seed(most)
    n = torch.randint(1, most + 1, (400,), generator=g)
    extra = torch.randint(0, 3 * most, (400,), generator=g) * (torch.rand(400, generator=g) < 0.7)
    b = Batch([(int(x), int(x + y)) for x, y in zip(n, extra)], NH=8, NKV=4, D=D, fp8=fp8, seed=16)
    # rows of different sizes: a scale that belongs to another item shows
    b.q *= torch.exp2(torch.randint(-6, 3, (b.T, 1, 1), device=DEV).float()).to(torch.bfloat16)
    attn = b.attention()
    first = b.run(attn=attn, gate=b.gate).clone()
    b.check(first, gate=b.gate)
    for _ in range(10):
        assert torch.equal(b.run(attn=attn, gate=b.gate), first)


def test_long_cache_offsets_pass_32_bits():
    """Block strides that take element and byte offsets past 2^32."""
    NKV, D, B, blocks = 8, 128, 16, 140_000  # 32,768 elements a block: 4.6e9 elements
    raw, key, value = W.cache_views(blocks, B, NKV, D, "triton", DEV)
    g = torch.Generator(device=DEV).manual_seed(11)
    b = Batch([(37, 500)], NH=16, NKV=NKV, D=D, seed=11)
    ids = blocks - 1 - torch.randperm(2000, generator=g, device=DEV)[:b.tables.shape[1]]
    for i in range(b.tables.shape[1] - 1):
        key[ids[i]] = b.key[b.tables[0, i].long()]
        value[ids[i]] = b.value[b.tables[0, i].long()]
    want = b.run().clone()
    b.key, b.value, b.tables = key, value, ids.to(torch.int32)[None].contiguous()
    assert torch.equal(b.run(), want)


def test_same_results_every_time_and_per_split():
    b = Batch([(20, 5000), (600, 900), (1, 3001)], NH=32, NKV=8, seed=12)
    first = b.run().clone()
    for _ in range(5):
        b.out.fill_(1.0)
        assert torch.equal(b.run(), first)


@pytest.mark.parametrize("D,fp8", [(64, False), (128, False), (256, False), (128, True), (256, True)])
@pytest.mark.parametrize("NH,NKV", [(6, 2), (33, 1), (7, 1)])
def test_same_results_whatever_ran_before(D, fp8, NH, NKV):
    """Groups that do not fill a tile's 128 rows: the others hold what shared memory held."""
    g = torch.Generator().manual_seed(D + NH)
    lens = [(n, int(n + torch.randint(0, 900, (), generator=g)))
            for n in torch.randint(1, 90, (40,), generator=g).tolist()]
    b = Batch(lens, NH=NH, NKV=NKV, D=D, fp8=fp8, seed=40)
    b.scale *= 4  # maxima that grow past the rescaling's slack here and there
    attn = b.attention()
    first = b.run(window=300, gate=b.gate, attn=attn).clone()
    b.check(first, 300, b.gate)
    other = Batch([(600, 900)], NH=8, NKV=8, D=D, seed=41, spread=30.0, fp8=fp8)
    for size in (1.0, 1e3, float("nan"), 1e-3):
        other.run(q=other.q * size)
        assert torch.equal(b.run(window=300, gate=b.gate, attn=attn), first), size


def test_captured_with_changing_lengths_and_two_instances():
    b = Batch([(40, 500), (8, 700)], NH=16, NKV=4, seed=13)
    attn = b.attention()
    b.run(attn=attn)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attn(b.q, b.key, b.value, b.tables, b.query_start, b.seq_lens, 0, b.scale, b.out)
    b.out.fill_(5.0)
    b.query_start.copy_(torch.tensor([0, 3, 48], dtype=torch.int32))
    b.seq_lens.copy_(torch.tensor([499, 650], dtype=torch.int32))
    graph.replay()
    b.check(b.out)
    # another instance on another stream, at the same time
    c = Batch([(300, 2000)], NH=16, NKV=4, seed=14)
    other, side = c.attention(), torch.cuda.Stream()
    c.run(attn=other)
    want_b, want_c = b.out.clone(), c.out.clone()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        b.out.zero_()
        c.out.zero_()
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            other(c.q, c.key, c.value, c.tables, c.query_start, c.seq_lens, 0, c.scale, c.out)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(b.out, want_b) and torch.equal(c.out, want_c)


def test_refusals():
    b = Batch([(4, 20)])
    attn = b.attention()

    def call(**kw):
        a = dict(q=b.q, key=b.key, value=b.value, tables=b.tables, start=b.query_start,
                 lens=b.seq_lens, out=b.out, gate=None)
        a.update(kw)
        attn(a["q"], a["key"], a["value"], a["tables"], a["start"], a["lens"], 0, b.scale, a["out"],
             gate=a["gate"])
    for kw in (dict(q=b.q.float()), dict(q=b.q[:, :4]), dict(q=b.q.transpose(1, 2)),
               dict(key=b.key.float()), dict(key=b.key[:, :, :1], value=b.value[:, :, :1]),
               dict(value=b.value.contiguous()), dict(tables=b.tables.long()),
               dict(tables=b.tables[0]), dict(start=b.query_start[:1]), dict(lens=b.seq_lens.long()),
               dict(out=b.out.float()), dict(out=b.out[:2]), dict(gate=b.gate[:, :5]),
               dict(gate=b.gate.double()), dict(lens=b.seq_lens.cpu()), dict(gate=b.gate.cpu())):
        with pytest.raises(ValueError):
            call(**kw)
    flat = b.q.view(b.T, -1)
    for kw in (dict(out=flat), dict(q=b.q[:3], out=flat[1:], gate=b.gate[:3]),
               dict(gate=b.out)):  # rows may be read again after others have been written
        with pytest.raises(ValueError, match="apart"):
            call(**kw)
    with pytest.raises(ValueError):  # an FP8 instance over a bf16 cache
        ChunkAttention(b.NH, b.NKV, b.D, DEV, kv_cache_dtype="fp8")(
            b.q, b.key, b.value, b.tables, b.query_start, b.seq_lens, 0, b.scale, b.out)
    with pytest.raises(NotImplementedError):
        ChunkAttention(8, 2, 96, DEV)
    assert (b.out == 5.0).all()
    call(q=b.q[:0], out=b.out[:0])  # nothing to do


@pytest.mark.parametrize("D,fp8", [(64, False), (128, False), (256, False), (128, True), (256, True)])
@pytest.mark.parametrize("column", [7, 0.75])
@pytest.mark.parametrize("hidden", [False, True])
def test_one_bad_value_in_a_cut_item_spoils_its_column_alone(D, fp8, column, hidden):
    """An item cut between SMs into parts of several tiles, whose maxima keep growing by less than
    makes O be rescaled, and one NaN in V, in either half of the columns: the rows that see it
    have that column NaN, and everything else is right, wherever it was computed again."""
    column = column if isinstance(column, int) else int(column * D)
    n, length = 20, 40000
    b = Batch([(n, length)], D=D, fp8=fp8, seed=51)
    b.q[:, :, 0] = 4.0
    pos = torch.arange(length, device=DEV)
    ids = b.tables[0, pos // 16].long()
    # 1.2 more in log2 units from a tile to the next, six tiles long
    step = 1.2 / 1.4427 / (4.0 * b.scale * b.scales[0])
    b.key[ids, pos % 16, :, 0] = (pos // 128 % 6 * step)[:, None].expand(-1, b.NKV).to(b.key.dtype)
    at = length - 3 if hidden else length // 2
    row = b.value[ids[at], at % 16]
    row[1, column] = float("nan")
    out = b.run().double()
    k = b.key.float().nan_to_num(0, 0, 0).norm(dim=-1).max().item() * b.scales[0]
    score = (D + 4) * F32 * b.scale * b.q.float().norm(dim=-1).max().item() * k
    rel = 2.0 ** -8 + 2 * score + 6e-6 + (8 + length) * F32
    want, size = b.oracle()
    tol = rel * size + 2.0 ** -8 * want.abs() * (1 + rel) + 2.0 ** -130
    if fp8:
        v = b.value.float().nan_to_num(0, 0, 0).abs().max().item() * b.scales[1]
        tol = tol + 2.0 ** -32 * length * v
    spoilt = torch.zeros(b.T, b.NH, D, dtype=torch.bool, device=DEV)
    spoilt[n - 3 if hidden else 0:, b.NH // b.NKV:, column] = True
    spoilt = spoilt.view(b.T, -1)
    assert torch.equal(want.isnan(), spoilt) and torch.equal(out.isnan(), spoilt)
    off = (out - want).abs()
    assert (off <= tol)[~spoilt].all(), (off / tol)[~spoilt].max().item()


@pytest.mark.parametrize("D,fp8", [(64, False), (128, False), (256, False), (128, True), (256, True)])
@pytest.mark.parametrize("why", ["short", "blocks"])
def test_rows_that_see_nothing_are_zero_beside_rows_that_see_a_bad_value(D, fp8, why):
    b = Batch([(40, 40), (3, 9)], D=D, fp8=fp8, seed=52, poison=False)
    if why == "short":
        b.seq_lens[0] = 30  # ten rows before the first position
        seen = torch.arange(40, device=DEV) - 10
        errors = 0
    else:
        b.tables[0, 0] = b.blocks
        seen = torch.arange(40, device=DEV) - 16
        errors = _native.DEVERR_BLOCK_OOB
    b.value[b.tables[0, 1].long(), 4] = float("nan")  # position 20
    out = b.run(errors=errors)[:40]
    assert (out[seen < 0] == 0).all()
    sees_it = torch.arange(40, device=DEV) - (10 if why == "short" else 0) >= 20
    assert out[sees_it].isnan().all() and out[~sees_it].isfinite().all()
    assert (out[(seen >= 0) & ~sees_it] != 0).any()


@pytest.mark.parametrize("D,fp8", [(64, False), (128, False), (256, False), (128, True), (256, True)])
def test_one_bad_value_does_not_slow_a_prompt_down(D, fp8):
    """Rows that see a NaN are NaN by the formula itself; only rows that share a tile with it and
    do not see it have to be computed again."""
    b = Batch([(2048, 2048)], NH=16, NKV=2, D=D, fp8=fp8, seed=53)
    attn = b.attention()

    def milliseconds():
        times = []
        for _ in range(4):
            e = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
            e[0].record()
            b.run(attn=attn)
            e[1].record()
            torch.cuda.synchronize()
            times.append(e[0].elapsed_time(e[1]))
        return min(times[1:])
    clean, want = milliseconds(), b.out.clone().view(b.T, b.NH, D)
    b.value[b.tables[0, 20].long(), 5, 1, 9] = float("nan")  # position 325
    bad, out = milliseconds(), b.out.view(b.T, b.NH, D)
    assert out[325:, 8:, 9].isnan().all() and out[:325].isfinite().all() and out[:, :8].isfinite().all()
    out[325:, 8:, 9] = want[325:, 8:, 9]
    # rows computed again differ by the rounding of their weights and of the result
    assert ((out - want).float().abs() <= 2.0 ** -6 * (want.float().abs() + 1)).all()
    assert bad < 8 * clean, (bad, clean)


@pytest.mark.parametrize("D,fp8", [(64, False), (128, False), (256, False), (128, True), (256, True)])
@pytest.mark.parametrize("window", [0, 70])
@pytest.mark.parametrize("seed", [0, 1, 2])
def test_scattered_bad_values(D, fp8, window, seed):
    """NaN and Inf all over V, whole items and cut ones, bad blocks and rows before the sequence:
    every element is what the formula gives from the positions that its row sees."""
    g = torch.Generator().manual_seed(60 + seed)
    b = Batch([(70, 90), (3, 3), (33, 2500), (20, 12), (1, 40), (90, 300)], NH=6, NKV=2, D=D, fp8=fp8,
              seed=60 + seed)
    b.tables[2, 7] = b.blocks  # positions 112 to 127: with the window, none of the last rows sees them
    for _ in range(25):
        i = int(torch.randint(0, 6, (), generator=g))
        n = max(int(b.seq_lens[i]) - int(torch.randint(0, 100, (), generator=g)), 1)
        at = int(torch.randint(max(0, n - 60), n, (), generator=g))
        block = int(b.tables[i, at // 16])
        if 0 <= block < b.blocks:
            bad = [float("nan"), float("inf"), -float("inf")][int(torch.randint(0, 3, (), generator=g))]
            columns = torch.randint(0, D, (int(torch.randint(1, 4, (), generator=g)),), generator=g)
            b.value[block, at % 16, int(torch.randint(0, 2, (), generator=g)), columns.to(DEV)] = \
                torch.tensor(bad, device=DEV).to(b.value.dtype)
    out = b.run(window=window, gate=b.gate, errors=0 if window else _native.DEVERR_BLOCK_OOB)
    want, size = b.oracle(window, b.gate)
    assert torch.equal(out.isnan(), want.isnan())
    infinite = want.isinf()
    assert torch.equal(out.double()[infinite], want[infinite])
    clean = want.isfinite()
    k = b.key.float().nan_to_num(0, 0, 0).norm(dim=-1).max().item() * b.scales[0]
    score = (D + 4) * F32 * b.scale * b.q.float().norm(dim=-1).max().item() * k
    rel = 2.0 ** -8 + 2 * score + 6e-6 + (8 + 2500) * F32
    tol = rel * size + 2.0 ** -8 * want.abs() * (1 + rel) + 2.0 ** -130
    if fp8:
        v = b.value.float().nan_to_num(0, 0, 0).abs().max().item() * b.scales[1]
        tol = tol + 2.0 ** -32 * 2500 * v
    assert ((out.double() - want).abs() <= tol)[clean].all()


@pytest.mark.parametrize("D,fp8", [(64, False), (128, False), (256, False), (128, True), (256, True)])
def test_bad_values_among_many_sequences_and_in_a_replay(D, fp8):
    """More sequences than a warp looks at once, several whole items an SM, and values that turn bad
    between the capture of a graph and its replay."""
    g = torch.Generator().manual_seed(70)
    lens = [(int(n), int(n + x)) for n, x in zip(torch.randint(1, 40, (150,), generator=g),
                                                 torch.randint(0, 200, (150,), generator=g))]
    b = Batch(lens, NH=4, NKV=2, D=D, fp8=fp8, seed=71)
    attn = b.attention()
    first = b.run(attn=attn, gate=b.gate).clone()
    b.check(first, gate=b.gate)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attn(b.q, b.key, b.value, b.tables, b.query_start, b.seq_lens, 0, b.scale, b.out, gate=b.gate,
             k_scale=b.scales[0], v_scale=b.scales[1])
    spoilt = torch.zeros(b.T, b.NH, D, dtype=torch.bool)
    for i in range(0, 150, 3):  # every third sequence: a position of its chunk, one column
        n, length = lens[i]
        at = length - 1 - int(torch.randint(0, n, (), generator=g))
        column, head = int(torch.randint(0, D, (), generator=g)), i // 3 % 2
        b.value[b.tables[i, at // 16].long(), at % 16, head, column] = float("nan")
        start = int(b.query_start[i])
        spoilt[start + at - (length - n):start + n, 2 * head:2 * head + 2, column] = True
    spoilt = spoilt.view(b.T, -1).to(DEV)
    b.out.fill_(5.0)
    graph.replay()
    replayed = b.out.clone()
    assert torch.equal(replayed.isnan(), spoilt)
    # the others as before, but for the rounding of rows that were computed again
    off = (replayed.float() - first.float()).abs()[~spoilt]
    assert (off <= 2.0 ** -6 * (first.float().abs() + 1)[~spoilt]).all()
    again = b.run(attn=attn, gate=b.gate)
    assert torch.equal(again.isnan(), spoilt) and torch.equal(again[~spoilt], replayed[~spoilt])
    whole = torch.tensor([i % 3 != 0 for i in range(150)]).repeat_interleave(
        torch.tensor([n for n, _ in lens])).to(DEV)
    assert torch.equal(replayed[whole], first[whole])
