"""What the wavefronts of the absorbed form do at the start of a tile (csrc/latent_absorbed_kernel.h: LatentAbsorbed), checked on the host for
every instance and number of rows: each step of the ring is loaded once, each strip's queries are asked for, and no wavefront
comes to the barrier in front of the first scores while rows of the first step that it has asked for may be on their way."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include <hip/hip_runtime.h>
#include "latent_absorbed_kernel.h"

template <int L, bool KV8, int M>
int check() {
  using T = fa::LatentAbsorbed<L, fa::BF16, KV8, M>;
  int wrong = 0;
  for (int rows = 1; rows <= 2 * M; ++rows) {
    int loaded = 0, asked[M / 16] = {}, scored[M / 16] = {};
    for (int wave = 0; wave < 8; ++wave) {
      const int strip = T::strip_of(wave), part = T::key_part_of(wave);
      const bool scores = T::has_scores(strip, rows);
      if (scores && strip >= M / 16) { ++wrong; continue; }
      if (scores) ++scored[strip];
      if (scores && T::asks_for_queries(scores, part)) asked[strip] += T::kParts == 1 ? 16 : 8;
      if (!T::loads(wave)) continue;
      loaded += T::kOwn;
      // rows that are decoded are waited for by decode(), in front of the same barrier
      const bool waits = T::kDecodes || T::asks_for_queries(scores, part) || T::waits_for_first_step(scores, part);
      if (!waits) {
        printf("L %d, FP8 %d, tiles of %d rows, %d in use: wavefront %d does not wait for its rows of the first step\n", L, KV8, M, rows, wave);
        ++wrong;
      }
    }
    wrong += loaded != T::kKeys;
    for (int strip = 0; strip < M / 16; ++strip) {
      const bool used = strip * 16 < (rows < M ? rows : M);
      if (used || scored[strip]) wrong += scored[strip] != T::kParts || asked[strip] != 16;
    }
  }
  return wrong;
}
template <int L>
int check_all() {
  return check<L, false, 32>() + check<L, false, 64>() + check<L, false, 128>() + check<L, true, 32>() + check<L, true, 64>() + check<L, true, 128>();
}
int main() { return check_all<256>() + check_all<512>() == 0 ? 0 : 1; }
"""


def test_no_wavefront_leaves_the_first_step_on_its_way(tmp_path):
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    source = tmp_path / "waits.hip"
    source.write_text(PROGRAM)
    subprocess.run([hipcc, "--offload-host-only", "-O1", "-std=c++17", "-I", os.path.join(ROOT, "flash_attention_factory_amd", "csrc"),
                    str(source), "-o", str(tmp_path / "waits")], check=True, capture_output=True)
    said = subprocess.run([str(tmp_path / "waits")], capture_output=True, text=True)
    assert said.returncode == 0, said.stdout
