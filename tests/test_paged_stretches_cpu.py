"""The stretches that attention over a cache is cut into, on the host: every item ends in a stretch that is launched, whatever
the requests' offsets add up to.  A second launch reads the workspace at the stretches from an item's first to its last,
so one behind the grid would be a read behind the workspace.

csrc/kf_stretch.h is plain arithmetic; it is compiled for the host, and walked as the kernels walk it.
"""

from __future__ import annotations

import ctypes
import subprocess

import pytest

from kernelforge import build

WALK = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#define __device__
#define __forceinline__ inline
#include "kf_stretch.h"

struct Request { int items, cost; };

// The largest stretch that an item of the requests ends in, and the units that the stretches walk.
static int walk(const std::vector<Request>& requests, int stretches, int begin_cost, long long* units) {
  int total = 0;
  for (const Request& r : requests) total = kf::add_work(total, r.items * r.cost);
  if (total == kf::kNoWork) total = 0;
  const int per = total / stretches + (total % stretches ? 1 : 0);
  int worst = -1;
  *units = 0;
  for (int me = 0; me < stretches; ++me) {
    const kf::Stretch s = kf::stretch_of(total, per, me);
    if (s.begin < 0 || s.end < s.begin || s.end > total) exit(2);
    *units += s.end - s.begin;
    int owners = 0, before = 0;
    size_t seq = 0, owner = 0;
    int owner_at = 0;
    for (; seq < requests.size(); ++seq) {  // a run of one request each
      const int mine = requests[seq].items * requests[seq].cost;
      if (s.begins_in(before, mine)) owners++, owner = seq, owner_at = before;
      before = kf::add_work(before, mine);
    }
    if (owners != (s.begin < s.end)) exit(3);
    int seq_at = owner_at;
    seq = owner;
    for (int at = s.begin; at < s.end;) {
      int n;
      while ((n = requests[seq].items * requests[seq].cost) <= at - seq_at) {
        seq_at += n;
        if (++seq >= requests.size()) exit(4);
      }
      const int cost = requests[seq].cost, item_at = seq_at + (at - seq_at) / cost * cost;
      if (item_at + cost > total) exit(5);
      // The kernels' pieces begin where the item's first units, which stand for beginning it, are done.
      if (at <= item_at + begin_cost && s.end > item_at + begin_cost) {
        const int last = kf::last_stretch(item_at, cost, per);
        if (last < me) exit(6);
        worst = last > worst ? last : worst;
      }
      at = item_at + cost;
    }
  }
  return worst;
}

int main(int argc, char** argv) {
  const int requests = atoi(argv[1]), items = atoi(argv[2]), cost = atoi(argv[3]), stretches = atoi(argv[4]);
  const bool ascending = atoi(argv[5]);
  std::vector<Request> r;
  for (int i = 0; i < requests; ++i) r.push_back({ascending || i % 2 == 0 ? items : 0, cost + (ascending ? i % 7 : 0)});
  long long units;
  const int worst = walk(r, stretches, 2, &units);
  printf("%d %lld\n", worst, units);
}
"""


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    d = tmp_path_factory.mktemp("stretches")
    (d / "walk.cpp").write_text(WALK)
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I", str(build.SRC_DIR),
                    str(d / "walk.cpp"), "-o", str(d / "walk")], check=True, timeout=120)

    def run(*args):
        out = subprocess.run([str(d / "walk"), *map(str, args)], capture_output=True, text=True, timeout=60)
        assert out.returncode == 0, (out.returncode, out.stderr[-300:])
        return tuple(map(int, out.stdout.split()))
    return run


def wrapped(sums: int) -> int:
    return (sums + 2 ** 31) % 2 ** 32 - 2 ** 31


@pytest.mark.parametrize("requests,tokens", [(512, 8192), (4096, 4096)])
def test_offsets_that_do_not_ascend(walk, requests, tokens):
    """Offsets 0, T, 0, T, ..: half the requests have all T tokens (32 heads on 4, row tiles of 16, keys in units of 128 of
    131072).  In 32 bits the work wraps to a small sum, against which the item that crosses it ends in stretch 256 of 256."""
    items, cost, grid = tokens * 8 // 16 * 4, 131072 // 128 + 2, 256
    assert items * cost < 2 ** 31
    total = wrapped(requests // 2 * items * cost)
    assert total > 0
    item_at = (total - 1) // cost * cost
    assert (item_at + cost - 1) // -(-total // grid) == grid  # what sums in 32 bits led to
    last, units = walk(requests, items, cost, grid, 0)
    assert last < grid and units == 0


@pytest.mark.parametrize("requests,items,cost,grid", [
    (1, 4, 3, 12), (1, 1, 5000, 256), (64, 2, 66, 256), (300, 7, 12, 512), (9, 131072, 1700, 256), (1, 131071, 16384, 512)])
def test_offsets_that_ascend(walk, requests, items, cost, grid):
    last, units = walk(requests, items, cost, grid, 1)
    assert 0 <= last < grid and units == sum(items * (cost + i % 7) for i in range(requests))


class AttnArgs(ctypes.Structure):
    """kf::AttnArgs of csrc/kf_launch.h."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("q", "k", "v", "out", "cu", "seq_lens", "table")] + \
        [(n, ctypes.c_int64) for n in ("table_stride", "q_token", "q_head", "out_token", "out_head", "k_page", "k_head",
                                       "k_token", "v_page", "v_head", "v_token")] + \
        [(n, ctypes.c_int) for n in ("tokens", "seqs", "heads", "kv_heads", "head_dim", "table_width", "log2_block",
                                     "num_pages", "zero_rest")] + \
        [("scale", ctypes.c_float), ("scale_log2", ctypes.c_float), ("rep", ctypes.c_int), ("min_rows", ctypes.c_int),
         ("ws", ctypes.c_void_p), ("pieces", ctypes.c_void_p)]


class FewPlan(ctypes.Structure):
    """kf::FewPlan of csrc/kf_launch.h."""
    _fields_ = [("row_tiles", ctypes.c_int), ("waves", ctypes.c_int), ("cut", ctypes.c_bool), ("grid", ctypes.c_int),
                ("most_units", ctypes.c_int64)]


def few_rows_plan(tokens, seqs, heads, kv_heads, d, keys, rows, max_rows, beside):
    plan = ctypes.CDLL(str(build.LIB_PATH))._ZN2kf13few_rows_planERKNS_8AttnArgsEliib
    plan.restype = FewPlan
    plan.argtypes = [ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_int, ctypes.c_bool]
    args = AttnArgs(tokens=tokens, seqs=seqs, heads=heads, kv_heads=kv_heads, head_dim=d, table_width=keys // 16, log2_block=4)
    return plan(ctypes.byref(args), rows, max_rows, 256, beside)


ALL = 2 ** 31 - 1


@pytest.mark.parametrize("beside", [False, True])
@pytest.mark.parametrize("tokens,seqs,heads,kv_heads,d,keys", [
    (32768, 2, 128, 8, 128, 1 << 20), (4096, 2, 1024, 8, 8, 1 << 20), (40000, 3, 64, 8, 64, 1 << 20)])
def test_work_beside_long_requests(tokens, seqs, heads, kv_heads, d, keys, beside):
    """Requests of more rows than the kernel of few rows takes are none of its work: a long chunk beside a single token
    over long tables is not more than a launch takes."""
    p = few_rows_plan(tokens, seqs, heads, kv_heads, d, keys, 64, 64, beside)
    unit = 32 * p.waves
    items = seqs * -(-64 // (16 * p.row_tiles)) * kv_heads
    assert p.most_units == items * (keys // unit + 2) < 2 ** 31 - 1


def test_work_of_one_kernel_for_all():
    """Without the other kernel every row counts: both sides of what a launch takes."""
    for tokens, fits in ((32000, True), (33000, False)):
        p = few_rows_plan(tokens, 2, 128, 8, 128, 1 << 20, 64, ALL, True)
        items = (tokens * 16 // 32 + 2) * 8
        assert p.most_units == items * ((1 << 20) // 64 + 2) and (p.most_units < 2 ** 31 - 1) == fits
