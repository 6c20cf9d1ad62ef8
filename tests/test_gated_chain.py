"""How a segment of the gated linear recurrence gets the value that enters it, the kernel's own header compiled for the host: a wave
is a few threads that meet where the wave's lanes do, and waves run one after the other in any order, so that waits run out."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "linrec_amd", "csrc")

# What the header takes from the others.  A lane that is `late` sees of every word what was there before its last store in this
# launch, as a lane of a wave may while another wave overwrites the words of a place.
SHIM = r"""
#pragma once
#include <atomic>
#include <barrier>
#include <cmath>
#include <cstdint>
#include <map>
#include <mutex>
#include <vector>
#define __device__
#define __forceinline__ inline
#define __HIP_MEMORY_SCOPE_AGENT 0
constexpr int LANES = 6;
inline thread_local int lane_of_thread = 0;
inline std::barrier<> meet(LANES);
inline bool votes[LANES];
inline uint64_t __ballot(bool v) {
  votes[lane_of_thread] = v;
  meet.arrive_and_wait();
  uint64_t all = 0;
  for (int i = 0; i < LANES; ++i) all |= uint64_t(votes[i]) << i;
  meet.arrive_and_wait();
  return all;
}
inline int __builtin_amdgcn_readfirstlane(int v) { return v; }
inline void __builtin_amdgcn_s_sleep(int) {}
template <typename T>
T __hip_atomic_fetch_add(T* p, T v, int, int) { return __atomic_fetch_add(p, v, __ATOMIC_RELAXED); }
namespace linrec {
constexpr uint32_t STATUS_AGGREGATE = 1u, STATUS_INCLUSIVE = 2u;
struct CarryHeader { uint32_t seq, gave_up; };
struct TileArgs { CarryHeader* ws; int spin_limit; };
inline uint64_t pack_desc(uint32_t flag, float v) { return (uint64_t(flag) << 32) | __builtin_bit_cast(uint32_t, v); }
inline std::mutex guard;
inline std::map<const uint64_t*, std::vector<uint64_t>> stores;
inline bool late[LANES];
inline uint64_t ld_desc(const uint64_t* p) {
  std::lock_guard<std::mutex> lock(guard);
  const auto it = stores.find(p);
  if (it == stores.end()) return 0;
  const std::vector<uint64_t>& all = it->second;
  return all[late[lane_of_thread] && all.size() > 1 ? all.size() - 2 : all.size() - 1];
}
inline void st_desc(uint64_t* p, uint64_t v) {
  std::lock_guard<std::mutex> lock(guard);
  stores[p].push_back(v);
}
}
"""

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <thread>
#include "gated_chain.hpp"
using namespace linrec;
// argv: segments, spin limit, late lanes (a mask), segments that hold a start (comma separated, - for none), the order of the segments
int main(int argc, char** argv) {
  const int segments = std::atoi(argv[1]);
  const unsigned mask = std::atoi(argv[3]);
  std::vector<char> cut(segments, 0);
  if (argv[4][0] != '-')
    for (char* at = argv[4]; *at;) { cut[std::strtol(at, &at, 10)] = 1; if (*at == ',') ++at; }
  for (int i = 0; i < LANES; ++i) late[i] = mask >> i & 1;
  // maps whose products stay in range; what enters, in double
  std::vector<std::vector<float>> a(segments, std::vector<float>(LANES)), b = a;
  std::vector<std::vector<double>> enters(segments + 1, std::vector<double>(LANES));
  for (int i = 0; i < LANES; ++i) {
    enters[0][i] = 3.0 + i;
    for (int k = 0; k < segments; ++k) {
      a[k][i] = 0.5f + 0.4f * ((k * 7 + i * 3) % 11) / 11.0f;
      b[k][i] = 1.0f + (k * 5 + i) % 13;
      enters[k + 1][i] = cut[k] ? b[k][i] : a[k][i] * enters[k][i] + b[k][i];
    }
  }
  std::vector<uint64_t> words(2 * LANES * chain_places(segments));
  CarryHeader header{7, 0};
  const TileArgs args{&header, std::atoi(argv[2])};
  int wrong = 0, ran = 0;
  for (char* at = argv[5]; *at; ++ran) {
    const int k = std::strtol(at, &at, 10);
    if (*at == ',') ++at;
    std::vector<float> got(LANES);
    std::vector<std::thread> wave;
    for (int i = 0; i < LANES; ++i)
      wave.emplace_back([&, i] {
        lane_of_thread = i;
        const Chain chain{words.data(), uint32_t(i) * 8, 2 * LANES, k, segments, header.seq};
        got[i] = enter_segment<LANES>(args, chain, i, float(enters[0][i]), a[k][i], b[k][i], cut[k], [&] { return float(enters[k][i]); });
      });
    for (std::thread& t : wave) t.join();
    for (int i = 0; i < LANES; ++i)
      if (!(std::fabs(got[i] - enters[k][i]) <= 1e-5 * enters[k][i])) {  // (a few dozen roundings of positive terms)
        std::printf("segment %d lane %d: %g enters, not %g\n", k, i, got[i], enters[k][i]);
        ++wrong;
      }
  }
  std::printf("%u\n", header.gave_up);
  return ran != segments ? 3 : wrong != 0;
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    where = tmp_path_factory.mktemp("chain")
    (where / "collook_kernel.hpp").write_text(SHIM)
    (where / "chain.cpp").write_text(PROGRAM)
    shutil.copy(os.path.join(CSRC, "gated_chain.hpp"), where)
    subprocess.run(["g++", "-std=c++20", "-O1", "-pthread", "-ffp-contract=off", str(where / "chain.cpp"), "-o", str(where / "chain")], check=True)
    return str(where / "chain")


def run(program, order, spin=2, late=0b101010, cuts=()):
    """Number of waits that ran out."""
    got = subprocess.run([program, str(len(order)), str(spin), str(late), ",".join(map(str, cuts)) or "-", ",".join(map(str, order))],
                         stdout=subprocess.PIPE, text=True, timeout=100)
    assert got.returncode == 0, (got.returncode, got.stdout)
    return int(got.stdout.split()[-1])


@pytest.mark.parametrize("cuts", [(), (0,), (3, 4, 7), (24, 25, 49), (12, 60)])
@pytest.mark.parametrize("segments", [1, 2, 5, 6, 26, 77, 130])
def test_in_order_nobody_gives_up(program, segments, cuts):
    assert run(program, list(range(segments)), late=0, cuts=[c for c in cuts if c < segments]) == 0


def test_a_group_whose_wait_runs_out_after_its_map_was_published(program):
    # segment 9 closes the second group with all of that group's maps there, and does not find the first group's: segment 4
    # comes later.  Lanes of the segments from 10 on see the words of the second group before and after whatever 9 stored then.
    order = [0, 1, 2, 3, 5, 6, 7, 8, 9, 4] + list(range(10, 60))
    assert run(program, order) > 0
    assert run(program, order, late=0) > 0


@pytest.mark.parametrize("late", [0, 0b000111, 0b101010])
@pytest.mark.parametrize("seed", range(6))
def test_any_order(program, seed, late):
    import random
    rng = random.Random(seed)
    segments = rng.choice([11, 30, 64, 130])
    order = list(range(segments))
    if seed % 2:
        rng.shuffle(order)
    else:  # a few stay behind
        for k in rng.sample(order, segments // 6):
            order.remove(k)
            order.insert(rng.randrange(len(order) + 1), k)
    cuts = rng.sample(range(segments), rng.choice([0, 1, segments // 8]))
    assert run(program, order, late=late, cuts=cuts) > 0 or seed % 2 == 0
