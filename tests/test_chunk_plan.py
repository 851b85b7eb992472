"""The scheduling warp of chunk attention (plan_role, csrc/dory_chunk.cu) on the host: its source
compiled by g++ with a one-lane stand-in for the warp, so that what it does when a wait gives up
can be seen without a GPU that waits."""

from __future__ import annotations

import subprocess
from pathlib import Path

import pytest

SOURCE = Path(__file__).resolve().parents[1] / "dory-vllm-experiments_b200" / "csrc" / "dory_chunk.cu"

HARNESS = r"""
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <cmath>
#include <algorithm>
#include <vector>
using std::max;
using std::min;
#define __device__
#define __forceinline__ inline
struct __nv_bfloat16 { uint16_t x; };
struct float2 { float x, y; };
struct Dim { int x; };
static Dim blockIdx, gridDim;
enum { DORY_DEVERR_QUERY_START = 32, DORY_DEVERR_BLOCK_OOB = 1 };
static uint32_t smem_u32(const void*) { return 0; }
static void mbar_arrive(uint32_t) {}
static void __syncwarp() {}
static int __ffs(uint32_t x) { return __builtin_ffs(int(x)); }
static uint32_t __ballot_sync(uint32_t, bool p) { return p; }
static bool __any_sync(uint32_t, bool p) { return p; }
template <class T> static T __shfl_sync(uint32_t, T x, int) { return x; }
template <class T> static T __shfl_up_sync(uint32_t, T x, int) { return x; }
static int __reduce_add_sync(uint32_t, int x) { return x; }
template <class T> static void atomicOr(T* p, uint32_t x) { *p |= x; }
template <int HD, bool KV8> struct Shape { static constexpr int kTiles = HD == 256 ? 1 : 2; };
static int waits_left;
static std::vector<int32_t> pushed;
static bool wait_warp(uint64_t, uint32_t, int*, uint32_t*) { return waits_left-- > 0; }
@CONSTANTS@
@ROWS@
@ITEM@
template <int HD, bool KV8> struct Control {
  uint64_t item_full[kQueue], item_empty[kQueue];
  Item items[kQueue];
  int abort;
};
@PLAN@

// argv: HD CTAs waits NKV TB window S, then (query_start[i + 1], seq_len[i]) of each sequence
template <int HD> void run(int argc, char** argv) {
  const int ctas = atoi(argv[2]), allowed = atoi(argv[3]);
  ChunkArgs a;
  memset(&a, 0, sizeof(a));
  a.NKV = atoi(argv[4]);
  a.TB = atoi(argv[5]);
  a.window = atoi(argv[6]);
  a.S = atoi(argv[7]);
  a.table_span = 1 << 20;
  std::vector<int32_t> starts{0}, lens, joins(8 * ctas);
  for (int i = 0; i < a.S; ++i) {
    starts.push_back(atoi(argv[8 + 2 * i]));
    lens.push_back(atoi(argv[9 + 2 * i]));
  }
  a.T = starts.back();
  a.query_start = starts.data();
  a.seq_lens = lens.data();
  uint32_t err = 0;
  a.err = &err;
  for (int c = 0; c < ctas; ++c)  // what a call with more rows left behind
    for (int i = 0; i < 8; ++i) joins[8 * c + i] = 1000000;
  a.joins = joins.data();
  gridDim.x = ctas;
  struct At { int seq, kvh, m, off; };
  std::vector<At> units;
  const int tokens = Shape<HD, false>::kTiles * a.TB;
  for (int i = 0; i < a.S; ++i)
    for (int h = 0; h < a.NKV; ++h) {
      const Seq s = sequence(a, i);
      for (int m = 0; m * tokens < s.n; ++m) {
        int first, tiles;
        const int n = item_units(a, s, m, tokens, first, tiles);
        for (int u = 0; u < n; ++u) units.push_back({i, h, m, u});
      }
    }
  const int total = int(units.size()), per = max((total + ctas - 1) / ctas, 1);
  for (int cta = 0; cta < ctas; ++cta) {
    blockIdx.x = cta;
    Piece p{min(cta * per, total), 0, per, 0, 0, 0, 0};
    p.u1 = min(p.u0 + per, total);
    if (p.u0 < p.u1) {
      const At& at = units[p.u0];
      p.seq = at.seq;
      p.kvh = at.kvh;
      p.m = at.m;
      p.off = at.off;
    }
    Control<HD, false> c;
    memset(&c, 0, sizeof(c));
    waits_left = allowed;
    plan_role<HD, false>(a, c, p, 0);
  }
  printf("T %d\n", a.T);
  for (int c = 0; c < ctas; ++c)
    printf("join %d %d %d %d\n", joins[8 * c], joins[8 * c + 1], joins[8 * c + 2], joins[8 * c + 3]);
}
int main(int argc, char** argv) {
  if (atoi(argv[1]) == 256) run<256>(argc, argv);
  else run<128>(argc, argv);
}
"""


def between(text: str, first: str, last: str) -> str:
    return text[text.index(first):text.index(last)]


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    text = SOURCE.read_text()
    parts = {
        "@CONSTANTS@": between(text, "constexpr float kLog2e", "struct Maps {"),
        "@ROWS@": between(text, "// Rows [t0, t1) of sequence i", "// The block of a sequence"),
        "@ITEM@": between(text, "enum : int { kItemEnd", "template <int HD, bool KV8>\nstruct Control"),
        "@PLAN@": between(text, "// The cache tiles that rows at positions", "// ---- loader ----"),
    }
    code = HARNESS
    for mark, part in parts.items():
        code = code.replace(mark, part)
    folder = tmp_path_factory.mktemp("plan")
    (folder / "plan.cpp").write_text(code)
    subprocess.run(["g++", "-std=c++17", "-w", "-o", str(folder / "plan"), str(folder / "plan.cpp")],
                   check=True)

    def run(head_dim, ctas, waits, kv_heads, tile_tokens, window, seqs):
        args = [head_dim, ctas, waits, kv_heads, tile_tokens, window, len(seqs)]
        end = 0
        for n, length in seqs:
            end += n
            args += [end, length]
        out = subprocess.run([str(folder / "plan"), *map(str, args)], check=True,
                             capture_output=True, text=True).stdout.split("\n")
        return int(out[0].split()[1]), [tuple(map(int, x.split()[1:])) for x in out if x[:4] == "join"]
    return run


SEQS = [(20, 900), (3, 3), (0, 50), (200, 200), (1, 5000), (65, 70)]


@pytest.mark.parametrize("head_dim", [128, 256])
@pytest.mark.parametrize("ctas", [1, 7, 148])
@pytest.mark.parametrize("window", [0, 100])
def test_the_record_of_a_cut_item_is_this_calls_own(plan, head_dim, ctas, window):
    """However early a wait gives up: no CTA leaves an earlier call's record to the join."""
    for waits in range(0, 40):
        T, joins = plan(head_dim, ctas, waits, 2, 32, window, SEQS)
        assert len(joins) == ctas
        for parts, first, tokens, kv_head in joins:
            assert parts == 0 or (2 <= parts <= ctas and tokens >= 1 and 0 <= first <= T - tokens
                                  and kv_head in (0, 1))
    # the call that gives up nowhere: one CTA cuts nothing, several cut the 40 tiles of 5000 (a cut
    # that falls on an item's output, as may be with the window, needs no join)
    if ctas == 1 or not window:
        assert any(parts for parts, *_ in joins) == (ctas > 1)


def test_an_empty_batch_leaves_no_record(plan):
    for seqs in ([(0, 0)], [(0, 100), (0, 5)]):
        T, joins = plan(128, 9, 100, 2, 32, 0, seqs)
        assert T == 0 and all(parts == 0 for parts, *_ in joins)


def test_no_role_waits_without_a_limit():
    """A role that gives up leaves its loop, so nothing inside the roles may wait for another warp
    except through an mbarrier with a limit: the only block barriers are the kernel's own, before
    the roles and after them."""
    text = SOURCE.read_text()
    header = (SOURCE.parent / "dory_sm100.cuh").read_text()
    for name in ("bar.sync", "barrier.sync", "barrier.cta", "named_barrier", "cooperative_groups"):
        assert name not in text and name not in header, name
    kernel = between(text, "    chunk_kernel(const __grid_constant__", "template <int N>")
    assert text.count("__syncthreads()") == kernel.count("__syncthreads()") == 2
    # a failed wait is never ignored: every call of these is tested
    for line in text.split("\n"):
        code = line.split("//")[0].strip()
        if code.startswith(("meet()", "wait_warp(", "wait_bar(", "wait_sum(", "wait_stage(")):
            assert False, line
    # and every spin on a barrier has the clock in its condition or body
    for at in [i for i in range(len(text)) if text.startswith("while (!mbar_try", i)]:
        assert "clock64()" in text[at:at + 260], text[at:at + 80]
