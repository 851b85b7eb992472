"""The prompt side of the attention path: rotary positions, the append of a chunk's keys and
values to the paged cache, and the attention of the chunk over that cache.

Each operator is here in its plain form (elementary torch operations in FP32), in the call a
user makes of the framework's kernels, and from its definition in FP64.  Notation: T new
tokens of S sequences, NH query heads, NKV key/value heads, D dims a head, G = NH / NKV.

* rotary: y = x rotated by its token's angles.  The first R dims of a head are pairs, dims
  (i, i + R/2) or, interleaved, (2i, 2i + 1); pair (a, b) becomes (a c - b s, b c + a s) with
  c, s = cos_sin[position, i], cos_sin[position, R/2 + i].  Other dims stay.
* append: q, k rotated, then (where sqk is given) brought to unit length, x / sqrt(sum x^2 +
  eps), q also times (sqk * sqk_factor)^2; k and v go to their cache slots (as bf16, or as
  e4m3(bf16(x) / scale)), a negative slot writes nothing; q comes back in bf16.
* chunk: token i of a sequence's n new ones is at position p = seq_len - n + i and attends
  the cached positions j <= p (and j > p - window), out = sum_j softmax_j(scale q.k_j) v_j
  times the gate; the cache's pages are found through the sequence's block table.
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False

EPS = 1e-6
ROOT = Path(__file__).resolve().parent.parent


# ---------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------
def rotary_case(tokens, heads, kv_heads, head_dim, rotary_dim, interleaved=False, dtype="bf16",
                max_position=8192, batch=False):
    return dict(op="rotary", tokens=tokens, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                rotary_dim=rotary_dim, interleaved=interleaved, dtype=dtype,
                max_position=max_position, batch=batch)


def append_case(tokens, heads, kv_heads, head_dim, rotary_dim, interleaved=False, dtype="bf16",
                max_position=8192, batch=False, norm=True, fp8=False, block=16, padding=0,
                layout="triton"):
    return dict(op="append", tokens=tokens, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                rotary_dim=rotary_dim, interleaved=interleaved, dtype=dtype,
                max_position=max_position, batch=batch, norm=norm, fp8=fp8, block=block,
                padding=padding, layout=layout)


def chunk_case(seqs, chunk, context, heads, kv_heads, head_dim, window=0, fp8=False, block=16,
               gate=True, layout="triton", spread=0):
    """`seqs` sequences of up to `chunk` new tokens after up to `context` cached ones: the
    first has exactly these, the others' are drawn below them by random.Random(spread)."""
    return dict(op="chunk", seqs=seqs, chunk=chunk, context=context, heads=heads,
                kv_heads=kv_heads, head_dim=head_dim, window=window, fp8=fp8, block=block,
                gate=gate, layout=layout, spread=spread)


def listed():
    return [
        # one sequence's next token, as an eager decode step rotates it: latency
        dict(rotary_case(1, 32, 8, 128, 128), name="rotary_one_token"),
        # a whole prompt of the longest context the benchmark uses
        dict(rotary_case(8192, 32, 8, 128, 128), name="rotary_prompt"),
        # 256-dim heads rotated in part, pairs interleaved, FP32 as the sublayers hand it on,
        # positions far into a lengthened context
        dict(rotary_case(1777, 16, 4, 256, 64, interleaved=True, dtype="f32",
                         max_position=131072), name="rotary_partial_far"),
        # the decode step of 512 sequences, one new token each
        dict(append_case(512, 32, 8, 128, 128, batch=True), name="append_decode_batch"),
        # a whole prompt into the cache
        dict(append_case(8192, 32, 8, 128, 128, norm=True), name="append_prompt"),
        # a ragged batch padded as for a captured graph, into an FP8 cache, FP32 inputs
        dict(append_case(2051, 16, 4, 256, 128, interleaved=True, dtype="f32", fp8=True,
                         padding=37, layout="unbind"), name="append_fp8_padded"),
        # four drafted tokens checked against a short cache: latency
        dict(chunk_case(1, 4, 636, 32, 8, 128), name="chunk_draft"),
        # a chunk of a long prompt whose earlier part is cached
        dict(chunk_case(1, 509, 7683, 32, 8, 128, gate=False), name="chunk_late_part"),
        # the largest: a whole prompt at once
        dict(chunk_case(1, 8192, 0, 32, 8, 128), name="chunk_prompt"),
        # the sliding-window layers of the 256-dim model
        dict(chunk_case(1, 2048, 4096, 16, 4, 256, window=1024), name="chunk_window_256"),
        # a serving step's ragged batch: chunks of 1 to 400 tokens, caches of all lengths
        dict(chunk_case(24, 400, 4000, 32, 8, 128, spread=3), name="chunk_ragged"),
        # the same kind of step over an FP8 cache
        dict(chunk_case(8, 601, 7100, 32, 8, 128, fp8=True, spread=5, layout="unbind"),
             name="chunk_fp8"),
    ]


def spread_int(rng, low, high):
    """A whole number in [low, high], even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low),
                                                             math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "append", "chunk", "chunk", "chunk"])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8])
    fp8 = op != "rotary" and rng.random() < 0.3
    head_dim = rng.choice([128, 256] if fp8 else [64, 128, 256])
    while kv_heads * group * head_dim > 4096:
        group = max(1, group // 2)
    heads = kv_heads * group
    if op != "chunk":
        rotary_dim = rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4])
        common = dict(interleaved=rng.random() < 0.4, dtype=rng.choice(["bf16", "bf16", "f32", "f16"]),
                      max_position=rng.choice([8192, 32768, 131072]), batch=rng.random() < 0.3)
        tokens = spread_int(rng, 1, 8192 if common["dtype"] != "f32" else 4096)
        if op == "rotary":
            return rotary_case(tokens, heads, kv_heads, head_dim, rotary_dim, **common)
        return append_case(tokens, heads, kv_heads, head_dim, rotary_dim,
                           norm=rng.random() < 0.6, fp8=fp8, block=rng.choice([16, 16, 32, 48]),
                           padding=rng.choice([0, 0, min(tokens - 1, 5)]),
                           layout=rng.choice(["triton", "unbind"]), **common)
    chunk, context = spread_int(rng, 1, 8192), spread_int(rng, 1, 8192) - 1
    seqs = spread_int(rng, 1, 32)
    # at most the largest listed case's score matrix and tokens
    while seqs > 1 and seqs * heads * chunk * (chunk + context) > 32 * 8192 * 8192 // 4:
        seqs //= 2
    while seqs * heads * chunk * (chunk + context) * head_dim > 32 * 8192 * 8192 * 128 // 2:
        chunk, context = (chunk + 1) // 2, context // 2
    return chunk_case(seqs, chunk, context, heads, kv_heads, head_dim,
                      window=rng.choice([0, 0, 1024, spread_int(rng, 1, 4096)]), fp8=fp8,
                      block=rng.choice([16, 16, 32, 48]), gate=rng.random() < 0.5,
                      layout=rng.choice(["triton", "unbind"]), spread=rng.randrange(1 << 30))


def lengths(case):
    """[(new tokens, seq_len)] of a chunk case's sequences."""
    rng = random.Random(case["spread"])
    both = [(case["chunk"], case["context"])]
    both += [(spread_int(rng, 1, case["chunk"]), spread_int(rng, 1, case["context"] + 1) - 1)
             for _ in range(case["seqs"] - 1)]
    return [(n, n + c) for n, c in both]


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def table(max_position, rotary_dim, device):
    """cos | sin of every position's angles, FP32 [max_position, rotary_dim]; past 8192
    positions the angles are stretched by the same factor (linear scaling)."""
    i = torch.arange(rotary_dim // 2, dtype=torch.float64, device=device)
    inv = 10000.0 ** (-2.0 * i / rotary_dim) / max(1.0, max_position / 8192)
    angle = torch.arange(max_position, dtype=torch.float64, device=device)[:, None] * inv
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


def caches(case, blocks, g, fill):
    """Key and value views [blocks, block, kv_heads, head_dim] of one pool."""
    nkv, d, b = case["kv_heads"], case["head_dim"], case["block"]
    shape = (blocks, nkv, b, 2 * d) if case["layout"] == "triton" else (blocks, 2, b, nkv, d)
    raw = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) if fill else \
        torch.zeros(shape, device="cuda")
    raw = raw.to(torch.float8_e4m3fn if case["fp8"] else torch.bfloat16)
    if case["layout"] == "triton":
        return raw.transpose(1, 2).split(d, dim=-1)
    return raw.unbind(1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = torch.device("cuda")
    nh, nkv, d = case["heads"], case["kv_heads"], case["head_dim"]
    s = dict(case=case)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev)

    if case["op"] != "chunk":
        t, dt = case["tokens"], DTYPES[case["dtype"]]
        # one projection's output: q heads, k heads, v heads of a token side by side
        qkv = normal(t, nh + 2 * nkv, d).to(dt)
        s["q"], s["k"], s["v"] = qkv.split([nh, nkv, nkv], dim=1)
        last = case["max_position"]
        if case["batch"]:  # one token each of many sequences
            s["positions"] = torch.randint(0, last, (t,), generator=g, device=dev)
        else:              # consecutive tokens, the last at the end of the context
            s["positions"] = torch.arange(last - t, last, device=dev)
        s["cos_sin"] = table(last, case["rotary_dim"], dev)
        s["q_out"] = torch.empty(t, nh, d, dtype=dt if case["op"] == "rotary" else torch.bfloat16,
                                 device=dev)
        s["k_out"] = torch.empty(t, nkv, d, dtype=dt, device=dev)
        if case["op"] == "append":
            b = case["block"]
            blocks = -(-t // b) + 3
            s["key"], s["value"] = caches(case, blocks, g, False)
            if case["batch"]:
                slots = torch.randperm(blocks * b, generator=g, device=dev)[:t]
            else:
                page = torch.randperm(blocks, generator=g, device=dev)
                at = torch.arange(t, device=dev)
                slots = page[at // b] * b + at % b
            if case["padding"]:
                slots[t - case["padding"]:] = -1
            s["slots"] = slots
            s["sqk"] = (torch.rand(nh * d, generator=g, device=dev) + 0.5).to(torch.bfloat16) \
                if case["norm"] else None
            s["sqk_factor"], s["k_scale"], s["v_scale"] = 0.7, 0.5, 0.25
            if not case["fp8"]:
                s["k_scale"] = s["v_scale"] = 1.0
        return s

    lens = lengths(case)
    b = case["block"]
    need = [-(-n // b) for _, n in lens]
    blocks = sum(need) + 5
    s["key"], s["value"] = caches(case, blocks, g, True)
    s["k_scale"], s["v_scale"] = (0.8, 1.1) if case["fp8"] else (1.0, 1.0)
    perm = torch.randperm(blocks, generator=g, device=dev).to(torch.int32)
    first = [sum(need[:i]) for i in range(len(need))]
    at = torch.arange(max(need))
    rows = torch.tensor(first)[:, None] + torch.minimum(at[None], torch.tensor(need)[:, None] - 1)
    s["tables"] = perm[rows.to(dev)].contiguous()
    starts = [0]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    t = starts[-1]
    s["query_start"] = torch.tensor(starts, dtype=torch.int32, device=dev)
    s["seq_lens"] = torch.tensor([n for _, n in lens], dtype=torch.int32, device=dev)
    s["q"] = normal(t, nh, d).to(torch.bfloat16)
    s["gate"] = torch.sigmoid(normal(t, nh * d)) if case["gate"] else None
    s["out"] = torch.empty(t, nh * d, dtype=torch.bfloat16, device=dev)
    s["scale"] = d ** -0.5
    if own:  # the handle a program keeps: the scratch of one attention instance
        s["attention"] = framework()[1].ChunkAttention(
            nh, nkv, d, dev, kv_cache_dtype="fp8" if case["fp8"] else "auto")
    return s


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------
def framework():
    """The framework's modules of these operators."""
    package = str(ROOT / "dory-vllm-experiments_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import dory_chunk_attention
    import dory_rotary_steps
    return dory_rotary_steps, dory_chunk_attention


def run(state):
    op = state["case"]["op"]
    if own:
        return {"rotary": own_rotary, "append": own_append, "chunk": own_chunk}[op](state)
    return {"rotary": plain_rotary, "append": plain_append, "chunk": plain_chunk}[op](state)


def own_rotary(s):
    framework()[0].rotary_embed(s["q"], s["k"], s["positions"], s["cos_sin"], s["q_out"],
                                s["k_out"], interleaved=s["case"]["interleaved"])
    return {"q": s["q_out"], "k": s["k_out"]}


def own_append(s):
    framework()[0].rotary_append(s["q"], s["k"], s["v"], s["positions"], s["cos_sin"], s["slots"],
                                 s["key"], s["value"], s["q_out"], sqk=s["sqk"],
                                 sqk_factor=s["sqk_factor"], eps=EPS,
                                 interleaved=s["case"]["interleaved"], k_scale=s["k_scale"],
                                 v_scale=s["v_scale"])
    return {"q": s["q_out"], "key": s["key"], "value": s["value"]}


def own_chunk(s):
    s["attention"](s["q"], s["key"], s["value"], s["tables"], s["query_start"], s["seq_lens"],
                   s["case"]["window"], s["scale"], s["out"], gate=s["gate"],
                   k_scale=s["k_scale"], v_scale=s["v_scale"])
    return s["out"]


def rotated(x, s):
    """x [T, H, D] (FP32 or FP64) rotated by the angles of s["positions"]."""
    r = s["case"]["rotary_dim"]
    cs = s["cos_sin"].to(x.dtype)[s["positions"]][:, None]
    c, sn = cs[..., :r // 2], cs[..., r // 2:]
    if s["case"]["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack([a * c - b * sn, b * c + a * sn], dim=-1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat([a * c - b * sn, b * c + a * sn], dim=-1)
    return torch.cat([turned, x[..., r:]], dim=-1)


def plain_rotary(s):
    return {n: rotated(s[n].float(), s).to(s[n].dtype) for n in ("q", "k")}


def plain_append(s):
    case = s["case"]
    q, k, v = rotated(s["q"].float(), s), rotated(s["k"].float(), s), s["v"].float()
    if case["norm"]:
        q = q / torch.sqrt((q * q).sum(-1, keepdim=True) + EPS)
        k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + EPS)
        w = s["sqk"].float() * s["sqk_factor"]
        q = q * (w * w).view(1, case["heads"], case["head_dim"])
    live = case["tokens"] - case["padding"]
    slots = s["slots"][:live]
    page, row = slots // case["block"], slots % case["block"]
    for cache, x, scale in ((s["key"], k, s["k_scale"]), (s["value"], v, s["v_scale"])):
        x = x[:live].to(torch.bfloat16)
        if case["fp8"]:  # bf16 first: the values that a bf16 cache would hold
            x = (x.float() / scale).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
            cache.view(torch.uint8)[page, row] = x.view(torch.uint8)
        else:
            cache[page, row] = x
    return {"q": q.to(torch.bfloat16), "key": s["key"], "value": s["value"]}


def padded(s):
    """(token of each (sequence, chunk row), whether it is one, its position): the ragged
    chunks as one [S, longest] batch."""
    starts, lens = s["query_start"].long(), s["seq_lens"].long()
    n = starts[1:] - starts[:-1]
    i = torch.arange(s["case"]["chunk"], device=n.device)
    real = i[None] < n[:, None]
    token = torch.where(real, starts[:-1, None] + i, 0)
    return token, real, lens[:, None] - n[:, None] + i


def plain_chunk(s):
    case = s["case"]
    nh, nkv, d = case["heads"], case["kv_heads"], case["head_dim"]
    token, real, position = padded(s)
    seqs, rows = token.shape
    tables = s["tables"].long()
    span = tables.shape[1] * case["block"]
    k = s["key"][tables].float().reshape(seqs, span, nkv, d).permute(0, 2, 3, 1) * s["k_scale"]
    v = s["value"][tables].float().reshape(seqs, span, nkv, d).permute(0, 2, 1, 3) * s["v_scale"]
    q = s["q"][token].float().reshape(seqs, rows, nkv, nh // nkv, d).permute(0, 2, 3, 1, 4)
    score = torch.matmul(q.reshape(seqs, nkv, -1, d) * s["scale"], k)
    score = score.view(seqs, nkv, nh // nkv, rows, span)
    j = torch.arange(span, device=k.device)
    seen = (j <= position[..., None]) & (j < s["seq_lens"].long()[:, None, None])
    if case["window"]:
        seen &= j > position[..., None] - case["window"]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    score -= score.amax(-1, keepdim=True)
    p = score.exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(seqs, nkv, -1, span), v).view(seqs, nkv, -1, rows, d) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(seqs, rows, nh * d)
    out = o[real]  # sequence by sequence, as the tokens lie
    if case["gate"]:
        out = out * s["gate"]
    return out.to(torch.bfloat16)


# ---------------------------------------------------------------------------------------
# the work of a pass, and its exact answer
# ---------------------------------------------------------------------------------------
def work(case):
    nh, nkv, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] != "chunk":
        t, e = case["tokens"], 4 if case["dtype"] == "f32" else 2
        angles = t * (4 * case["rotary_dim"] + 8)
        if case["op"] == "rotary":
            return {"bytes": 2 * t * (nh + nkv) * d * e + angles,
                    "flops": 3 * t * (nh + nkv) * case["rotary_dim"]}
        live, held = t - case["padding"], 1 if case["fp8"] else 2
        moved = (t * nh + 2 * live * nkv) * d * e + t * nh * d * 2 + 2 * live * nkv * d * held
        return {"bytes": moved + angles + 8 * t + (nh * d * 2 if case["norm"] else 0),
                "flops": 3 * t * (nh + nkv) * case["rotary_dim"]
                + (6 * t * (nh + nkv) * d if case["norm"] else 0)}
    pairs = rows = tokens = 0
    w = case["window"] or 1 << 40
    for n, length in lengths(case):
        first = length - n
        # token at position p sees min(p + 1, w) positions
        short = max(0, min(length, w) - first)  # tokens that see p + 1
        pairs += short * (2 * first + short + 1) // 2 + (n - short) * (0 if n == short else w)
        rows += length - max(0, first + 1 - w)
        tokens += n
    held = 1 if case["fp8"] else 2
    moved = 2 * rows * nkv * d * held + 4 * tokens * nh * d
    if case["gate"]:
        moved += 4 * tokens * nh * d
    pages = sum(-(-n // case["block"]) for _, n in lengths(case))
    return {"bytes": moved + 4 * pages + 8 * case["seqs"], "flops": 4 * pairs * nh * d}


def exact(case, seed):
    s = prepare(case, seed)
    nh, nkv, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] != "chunk":
        r = case["rotary_dim"]
        angles = s["cos_sin"].double()[s["positions"]]
        spin = torch.complex(angles[:, :r // 2], angles[:, r // 2:])[:, None]

        def turn(x):  # the pairs as complex numbers
            y = x.double().clone()
            at = (slice(0, r, 2), slice(1, r, 2)) if case["interleaved"] else \
                (slice(0, r // 2), slice(r // 2, r))
            z = torch.complex(y[..., at[0]].contiguous(), y[..., at[1]].contiguous()) * spin
            y[..., at[0]], y[..., at[1]] = z.real, z.imag
            return y

        q, k = turn(s["q"]), turn(s["k"])
        if case["op"] == "rotary":
            return {"q": q, "k": k}
        if case["norm"]:
            k = k * (k.square().sum(-1, keepdim=True) + EPS).rsqrt()
            w = (s["sqk"].double() * s["sqk_factor"]).square().view(nh, d)
            q = q * (q.square().sum(-1, keepdim=True) + EPS).rsqrt() * w
        key, value = s["key"].double(), s["value"].double()
        for t0 in range(0, case["tokens"] - case["padding"], 4096):
            part = slice(t0, min(t0 + 4096, case["tokens"] - case["padding"]))
            at = s["slots"][part]
            index = (torch.div(at, case["block"], rounding_mode="floor"), at % case["block"])
            key[index] = (k[part] / s["k_scale"]).clamp(-448, 448) if case["fp8"] else k[part]
            new = s["v"][part].double()
            value[index] = (new / s["v_scale"]).clamp(-448, 448) if case["fp8"] else new
        return {"q": q, "key": key, "value": value}

    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    t0 = 0
    for i, (n, length) in enumerate(lengths(case)):
        pages = s["tables"][i, :-(-length // case["block"])].long()
        low = max(0, length - n + 1 - case["window"]) if case["window"] else 0
        place = torch.arange(low, length, device="cuda")
        row = torch.arange(length - n, length, device="cuda")
        hidden = place[None, :] > row[:, None]
        if case["window"]:
            hidden |= place[None, :] <= row[:, None] - case["window"]
        for h in range(nkv):
            k = s["key"][pages, :, h].double().flatten(0, 1)[low:length] * s["k_scale"]
            v = s["value"][pages, :, h].double().flatten(0, 1)[low:length] * s["v_scale"]
            for head in range(h * (nh // nkv), (h + 1) * (nh // nkv)):
                logit = s["q"][t0:t0 + n, head].double() @ k.T * s["scale"]
                weight = torch.softmax(logit.masked_fill(hidden, -math.inf), dim=-1)
                out[t0:t0 + n, head * d:(head + 1) * d] = weight @ v
        t0 += n
    if case["gate"]:
        out *= s["gate"].double()
    return out
