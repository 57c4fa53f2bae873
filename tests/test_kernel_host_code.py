"""Host code of csrc/ that only shows its faults in rare orders of events, compiled by itself and driven through them on the CPU."""

import ctypes
import os
import subprocess

import pytest

from omniserver_b200.ops import library


def compiled(tmp_path, name, source, *flags):
    """The source, which may include csrc's headers, as a shared library."""
    src, out = tmp_path / f"{name}.cu", tmp_path / f"{name}.so"
    src.write_text(source)
    cmd = [library._find_nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O1", "-shared", "-Xcompiler", "-fPIC", "-I",
           library._CSRC, str(src), "-o", str(out), *flags]
    p = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert p.returncode == 0, p.stdout
    return ctypes.CDLL(str(out))


RING = r"""
#include <random>
#include <vector>
#include "attn_tree.cuh"

// The ring of the tree attention's tensor-core kernel: two producers put the tiles K0, K1, V0, K2, V1, .. of each stretch into it, the
// product S = Q K^T of a tile waits for its keys and for the product P V of the tile before the last, P V for S and its values; a tile
// leaves its place when its product is complete. Events happen in a random order. Counts the tiles, at every moment, that are under way and
// that the producers, if they stopped now, would not wait for: out[0]; if each waited for the last two that it put: out[1]. And the places
// whose wait would not end when everything has landed, since the barrier is in a later phase of the same parity: out[2].
template <int STAGES> void run(unsigned seed, int stretches, int most, long long* out) {
  std::mt19937 rng(seed);
  std::vector<int> keys, values;          // the ring's tile of each key tile, counted on across stretches
  for (int k = 0, i0 = 0; k < stretches; ++k) {
    const int n = 1 + (int)(rng() % most);
    for (int t = 0; t < n; ++t) {
      keys.push_back(i0 + (t == 0 ? 0 : 2 * t - 1));
      values.push_back(i0 + (t + 1 < n ? 2 * t + 2 : 2 * t + 1));
    }
    i0 += 2 * n;
  }
  const int U = (int)keys.size();
  enum { NOT_YET, UNDER_WAY, LANDED, USED };
  std::vector<int> state(2 * U, NOT_YET);
  attn_tree::LastPut<STAGES> now[2][STAGES];
  int put[2] = {0, 0}, s = 0, s_done = 0, pv = 0, pv_done = 0;
  std::vector<int> last[2];
  int phases[STAGES] = {};                // of each place's barrier that have begun
  while (pv_done < U) {
    const int what = (int)(rng() % 8);
    if (what < 2) {                                            // a producer
      if (put[what] == U) continue;
      const int i = (what == 0 ? keys : values)[put[what]];
      if (i >= STAGES && state[i - STAGES] != USED) continue;  // waits for `empty`
      ++put[what];
      state[i] = UNDER_WAY;
      ++phases[i % STAGES];
      for (int k = 0; k < STAGES; ++k) now[what][k].put(k, i);
      last[what].push_back(i);
    } else if (what < 4) {                                     // a tile lands
      std::vector<int> flying;
      for (int i = 0; i < 2 * U; ++i)
        if (state[i] == UNDER_WAY) flying.push_back(i);
      if (!flying.empty() && rng() % 4 == 0) state[flying[rng() % flying.size()]] = LANDED;
    } else if (what == 4) {
      if (s < U && state[keys[s]] == LANDED && (s < 2 || pv_done > s - 2)) ++s;
    } else if (what == 5) {
      if (s_done < s) state[keys[s_done++]] = USED;
    } else if (what == 6) {
      if (pv < s_done && state[values[pv]] == LANDED) ++pv;
    } else if (pv_done < pv) {
      state[values[pv_done++]] = USED;
    }
    int noted[STAGES];
    for (int k = 0; k < STAGES; ++k) {
      noted[k] = now[0][k].tile > now[1][k].tile ? now[0][k].tile : now[1][k].tile;
      out[2] += noted[k] >= 0 && ((noted[k] / STAGES) & 1) == (phases[k] & 1);
    }
    for (int i = 0; i < 2 * U; ++i) {
      if (state[i] != UNDER_WAY) continue;
      out[0] += noted[i % STAGES] != i;
      bool among = false;
      for (const auto& l : last)
        for (size_t k = l.size() < 2 ? 0 : l.size() - 2; k < l.size(); ++k) among = among || l[k] == i;
      out[1] += !among;
    }
  }
}
extern "C" __attribute__((visibility("default"))) void ring(int stages, unsigned seed, int stretches, int most, long long* out) {
  if (stages == 4) run<4>(seed, stretches, most, out);
  else run<8>(seed, stretches, most, out);
}
"""


def test_a_tree_attention_that_gives_up_waits_for_every_copy_under_way(tmp_path):
    lib = compiled(tmp_path, "ring", RING)
    for stages in (4, 8):
        out = (ctypes.c_longlong * 3)()
        for seed in range(200):
            lib.ring(stages, ctypes.c_uint(seed), 1 + seed % 4, 1 + seed % 13, out)
        assert out[0] == 0, f"{stages} places: a copy under way that nothing waits for"
        assert out[2] == 0, f"{stages} places: a wait that does not end"
        assert out[1] > 0, "the events no longer reach more than two tiles under way"


ALLOW = r"""
#include <cuda_runtime.h>
#include <stdlib.h>
#include <atomic>
#include <chrono>
#include <thread>

// The runtime's calls, as far as this test goes: one device, one kernel. Of two calls that set what the kernel may have, the smaller one
// waits for the larger one to come past it, for half a second at most.
static std::atomic<int> may_have{0}, larger_set{0}, smaller_in{0};
template <typename K> static cudaError_t fake_set(K, cudaFuncAttribute, int bytes) {
  if (bytes == 60000) {
    smaller_in = 1;
    for (int i = 0; i < 500 && !larger_set; ++i) std::this_thread::sleep_for(std::chrono::milliseconds(1));
  }
  may_have = bytes;
  if (bytes == 100000) larger_set = 1;
  return cudaSuccess;
}
static cudaError_t fake_device(int* dev) {
  *dev = 0;
  return cudaSuccess;
}
#define cudaFuncSetAttribute fake_set
#define cudaGetDevice fake_device
#include "common.cuh"

__global__ void some_kernel() {}

// what the kernel may have when both calls have returned, -1 if one of them failed
extern "C" __attribute__((visibility("default"))) int allow() {
  int rc[2] = {0, 0};
  std::thread small([&] { rc[0] = osb_allow_smem<some_kernel>(60000); });
  while (!smaller_in) std::this_thread::yield();
  std::thread large([&] { rc[1] = osb_allow_smem<some_kernel>(100000); });
  small.join();
  large.join();
  return rc[0] || rc[1] ? -1 : (int)may_have;
}
"""


def test_two_calls_at_once_leave_a_kernel_the_larger_shared_memory(tmp_path):
    assert compiled(tmp_path, "allow", ALLOW).allow() == 100000
