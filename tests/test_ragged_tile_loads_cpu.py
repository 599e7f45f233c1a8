"""Which rows of the pool the threads of the tile form load (csrc/ragged_tile_kernel.h: RaggedTile::load_key), checked on the host for
every instance and block size: no row past the end of a block, every 16 bytes of a step once."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include <vector>
#include <hip/hip_runtime.h>
#include "ragged_tile_kernel.h"

template <int D, int KVF, int MAPS, int NW>
int check() {
  using T = fa::RaggedTile<D, KVF, MAPS, NW>;
  int wrong = 0;
  for (int shift = 4; shift <= 12; ++shift) {
    const int in_block = (1 << shift) - 1;
    for (int step = 0; step < 130; ++step) {
      std::vector<int> times(fa::kTileKeys * T::kPerRow);
      for (int pass = 0; pass < T::kPasses; ++pass)
        for (int tid = 0; tid < T::kThreads; ++tid) {
          const int load_row = tid / T::kPerRow, key = T::load_key(pass, load_row);
          const bool loads = T::kRowsPerPass <= fa::kTileKeys || load_row < fa::kTileKeys;
          // the kernel's address: a row of the thread's own, and where the step lies in a block of more than 64
          const int row = (key & in_block) + (step * fa::kTileKeys & in_block);
          const int col = (step * fa::kTileKeys >> shift) + (key >> shift), at = step * fa::kTileKeys + key;
          wrong += key < 0 || key >= fa::kTileKeys || row > in_block || col != at >> shift || row != (at & in_block);
          if (loads) ++times[key * T::kPerRow + tid % T::kPerRow];
        }
      for (int n : times) wrong += n != 1;
    }
  }
  if (wrong) printf("D %d, cache format %d, maps %d, %d wavefronts: %d wrong\n", D, KVF, MAPS, NW, wrong);
  return wrong;
}
template <int D, int KVF>
int check_all() {
  return check<D, KVF, 1, 4>() + check<D, KVF, 1, 8>() + check<D, KVF, 2, 4>() + check<D, KVF, 2, 8>();
}
int main() {
  return check_all<64, fa::kKv16>() + check_all<128, fa::kKv16>() + check_all<64, fa::kKvI8>() + check_all<128, fa::kKvI8>() +
                 check_all<64, fa::kKvE4M3>() + check_all<128, fa::kKvE5M2>() == 0 ? 0 : 1;
}
"""


def test_loads_stay_within_their_blocks(tmp_path):
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    source = tmp_path / "loads.hip"
    source.write_text(PROGRAM)
    subprocess.run([hipcc, "--offload-host-only", "-O1", "-std=c++17", "-I", os.path.join(ROOT, "flash_attention_factory_amd", "csrc"),
                    str(source), "-o", str(tmp_path / "loads")], check=True, capture_output=True)
    said = subprocess.run([str(tmp_path / "loads")], capture_output=True, text=True)
    assert said.returncode == 0, said.stdout
