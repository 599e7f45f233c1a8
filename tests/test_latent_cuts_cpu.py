"""How the line of tiles of the absorbed form is cut into shares (csrc/latent_absorbed_kernel.h: latent_cut, latent_cut_step, latent_shares),
checked on the host against the same in 128 bits, for lines up to the 2^41 steps that a call may have."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdint>
#include <cstdio>
#include <hip/hip_runtime.h>
#include "latent_absorbed_kernel.h"

typedef __int128 wide;
static long checked = 0;

template <typename T>
int check(int64_t total, int groups, int64_t start, int steps, int cost_steps) {
  auto cut = [&](int g) { return (int64_t)((wide)total * g / groups); };
  int wrong = 0, g = 0;
  const int64_t cost = cost_steps + T::kStart;
  if (start + cost > total) return 0;
  while (cut(g + 1) <= start) ++g;
  if (cut(g + 1) >= start + cost) return 0;  // not cut
  // steps of the tile that share k has
  auto upto = [&](int k) {
    const wide in = (wide)cut(k) - start - T::kStart;
    return in < 0 ? 0 : in > steps ? steps : (int)in;
  };
  int first = -1, last = -1;
  for (int k = g; k < groups; ++k) {
    wrong += fa::latent_cut(total, groups, k) != cut(k);
    wrong += fa::latent_cut_step<T>(cut(k) - start, steps) != upto(k);
    if (upto(k) < upto(k + 1)) {
      if (first < 0) first = k;
      last = k;
    }
  }
  const fa::LatentShares s = fa::latent_shares<T>(total, groups, g, start, steps);
  wrong += s.first != first || s.last != last;
  if (wrong)
    printf("line of %lld in %d shares, tile at %lld of %d steps: shares %d .. %d, not %d .. %d\n", (long long)total, groups, (long long)start, steps,
           s.first, s.last, first, last);
  ++checked;
  return wrong;
}

template <typename T>
int check_all() {
  int wrong = 0;
  for (long long total : {1LL << 12, (1LL << 31) - 1, 1LL << 31, 2148302860LL, (1LL << 32) + 5, 3LL << 33, (1LL << 40) + 12345, 1LL << 41})
    for (int groups : {2, 8, 64, 248, 256})
      for (int g = 1; g < groups; g += groups > 16 ? 31 : 1) {
        const int64_t at = (int64_t)((wide)total * g / groups);
        for (int cost_steps : {1, 5, 700, 32780, 1 << 25})
          for (int less : {0, 1, cost_steps / 2})  // a tile whose last rows see fewer keys than those of the tile beside it
            for (int before : {1, T::kStart + 0, T::kStart + 1, T::kStart + cost_steps / 3, T::kStart + cost_steps - 1})
              if (cost_steps - less > 0 && at >= before) wrong += check<T>(total, groups, at - before, cost_steps - less, cost_steps);
      }
  return wrong;
}
int main() {
  const int wrong = check_all<fa::LatentSteps<false, 32>>() + check_all<fa::LatentSteps<false, 64>>() + check_all<fa::LatentSteps<false, 128>>() +
                    check_all<fa::LatentSteps<true, 32>>() + check_all<fa::LatentSteps<true, 128>>();
  printf("%ld checked\n", checked);
  return wrong == 0 && checked > 10000 ? 0 : 1;
}
"""


def test_cuts_and_joined_shares(tmp_path):
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    source = tmp_path / "cuts.hip"
    source.write_text(PROGRAM)
    subprocess.run([hipcc, "--offload-host-only", "-O1", "-std=c++17", "-I", os.path.join(ROOT, "flash_attention_factory_amd", "csrc"),
                    str(source), "-o", str(tmp_path / "cuts")], check=True, capture_output=True)
    said = subprocess.run([str(tmp_path / "cuts")], capture_output=True, text=True, timeout=100)
    assert said.returncode == 0, said.stdout[-4000:]
