"""The rule that splits the keys of drafted trees, replayed on the host with the
kernels' own functions: whatever the batch, its items, its partials and its
merges fit what the host laid out for them, and every split holds keys."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]

# Batches of random shapes, for item sizes and residents of all tile kernels; the
# reciprocal, exact on the host, is also tried a unit in the last place off.
PROGRAM = r"""
#include "tree_items.h"
#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>

static int cus = 256;
namespace mvllm {
int device_cu_count() { return cus; }
}
using namespace mvllm;

int main() {
  std::mt19937_64 rng(11);
  auto log_int = [&](double lo, double hi) {
    return static_cast<int64_t>(std::exp(std::uniform_real_distribution<double>(std::log(lo), std::log(hi + 1))(rng)));
  };
  const int32_t heads[] = {1, 2, 3, 4, 5, 8, 9, 16, 32, 64, 128}, rows[] = {16, 32, 64, 128};
  int64_t batches = 0, split_batches = 0, tightest = 1 << 30;
  for (int shape = 0; shape < 60000; ++shape) {
    cus = rng() % 4 ? 256 : 64;
    TreeArgs a = {};
    a.num_requests = log_int(1, shape % 8 ? 300 : 3000);
    a.num_kv_heads = heads[rng() % 11];
    a.group = 1 + static_cast<int32_t>(rng() % 16);
    a.head_dim = 128;
    a.block_size = 16;
    a.width = log_int(1, rng() % 4 ? 2500 : 60000);
    const int64_t reach = a.width * a.block_size;
    const int64_t most_nodes = log_int(1, 200), least = rng() % 2 ? 1 : log_int(1, reach);
    const bool apart = rng() % 3 == 0;  // a few long requests among short ones
    std::vector<TreeReq> batch;
    const int32_t size = rows[rng() % 4];
    a.num_tokens = rng() % 4 ? 0 : static_cast<int64_t>(rng() % 50);  // tokens outside
    for (int64_t r = 0; r < a.num_requests; ++r) {
      TreeReq q = {0, 0, 0, 0, 0, 0};
      q.nodes = rng() % 16 ? static_cast<int32_t>(1 + rng() % most_nodes) : 0;
      if (q.nodes) {
        const bool small = apart && rng() % 10;
        const int64_t top = small ? std::min<int64_t>(reach, 100) : reach, low = std::min(least, top);
        q.keys = rng() % 50 ? static_cast<int32_t>(low + static_cast<int64_t>(rng() % (top - low + 1))) : 0;
        q.blocks = static_cast<int32_t>((static_cast<int64_t>(q.nodes) * a.group + size - 1) / size);
      }
      a.num_tokens += q.nodes;
      batch.push_back(q);
    }
    const int32_t shortest = size == 16 ? 128 : 384;
    const int64_t residents = size == 16 ? 1 : 1 + static_cast<int64_t>(rng() % 3);
    tree_layout(a, size, shortest, residents, nullptr);
    // plan_split's choice.
    float total = 0.f, blocks = 0.f;
    for (const TreeReq& q : batch) total += static_cast<float>(tree_load(q)), blocks += static_cast<float>(q.blocks);
    int32_t split = a.shortest;
    if (!all_shortest(a, total, blocks)) {
      const float off[] = {1.0f, 1.0f - 0x1p-23f, 1.0f + 0x1p-23f};
      const float share = split_share(a, total) * off[rng() % 3];
      split = 0;
      if (blocks < static_cast<float>(a.target))
        for (int c = 0; c < kAttempts && !split; ++c) {
          const int32_t length = split_length(a, share, c);
          int64_t count = 0;
          for (const TreeReq& q : batch) count += split_count(q.blocks, q.keys, length);
          if (count <= a.target) split = length;
        }
      if (!split) split = split_length(a, share, kAttempts);
    }
    int64_t items = 0, partials = 0, merges = 0;
    bool sound = split >= a.shortest && split % 64 == 0;
    for (const TreeReq& q : batch) {
      if (!q.blocks) continue;
      const int32_t ns = tree_splits(a, q, split), share = tree_share(q, ns);
      items += static_cast<int64_t>(ns) * q.blocks;
      if (ns > 1) partials += static_cast<int64_t>(ns) * q.blocks, merges += q.blocks;
      // The splits before the last are whole tiles, the last one holds keys, none is longer than the rule's length.
      if (ns > 1) sound = sound && share % 64 == 0 && share <= split && static_cast<int64_t>(ns - 1) * share < q.keys &&
                          static_cast<int64_t>(ns) * share >= q.keys;
      split_batches += ns > 1;
    }
    sound = sound && items <= a.capacity && partials <= a.slots && merges <= a.merge_capacity;
    if (a.merge_capacity) tightest = std::min(tightest, a.capacity - items);
    if (!sound) {
      std::printf("requests %lld heads %d group %d rows %d reach %lld split %d: items %lld of %d, partials %lld of %d, merges %lld of %d\n",
                  (long long)a.num_requests, a.num_kv_heads, a.group, size, (long long)reach, split, (long long)items, a.capacity,
                  (long long)partials, a.slots, (long long)merges, a.merge_capacity);
      return 1;
    }
    ++batches;
  }
  std::printf("%lld batches, %lld split requests, %lld places left at least\n", (long long)batches, (long long)split_batches, (long long)tightest);
  return split_batches > 100000 ? 0 : 2;
}
"""


def test_every_split_of_a_tree_batch_fits(tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not Path(hipcc).exists():
        pytest.skip("hipcc not found")
    source, program = tmp_path / "rule.hip", tmp_path / "rule"
    source.write_text(PROGRAM)
    subprocess.run(
        [hipcc, "--offload-host-only", "-O2", "-std=c++17", "-Wno-unused-function", f"-I{ROOT / 'include'}",
         f"-I{ROOT / 'micro-vllm_amd' / 'csrc'}", str(source), "-o", str(program)],
        check=True, capture_output=True, text=True, timeout=300,
    )
    done = subprocess.run([str(program)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout
