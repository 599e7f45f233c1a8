"""Scales of the rows of FP8 latent pools (csrc/latent_cache_kernel.h: row_scale_exponent), checked on the host: the least power of two, 2^-100 or
more, that brings the largest magnitude to 448 or less, for every finite 32-bit one."""
import math
import os
import subprocess
from fractions import Fraction

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include <hip/hip_runtime.h>
#include "latent_cache_kernel.h"
int main() {
  uint32_t bits;
  while (scanf("%u", &bits) == 1) printf("%d\n", fa::row_scale_exponent(__builtin_bit_cast(float, bits)));
  return 0;
}
"""


def test_row_scale_exponents(tmp_path):
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    source = tmp_path / "scales.hip"
    source.write_text(PROGRAM)
    subprocess.run([hipcc, "--offload-host-only", "-O1", "-std=c++17", "-I", os.path.join(ROOT, "flash_attention_factory_amd", "csrc"),
                    str(source), "-o", str(tmp_path / "scales")], check=True, capture_output=True)
    # every exponent, with mantissas at and beside 1.75 (448 = 1.75 * 2^8) and at the ends
    most = [(e << 23) | m for e in range(255) for m in (0, 1, 0x5fffff, 0x600000, 0x600001, 0x7fffff)]
    said = subprocess.run([str(tmp_path / "scales")], input="\n".join(map(str, most)), capture_output=True, text=True, check=True).stdout.split()
    values = torch.tensor(most, dtype=torch.int32).view(torch.float32).double().tolist()
    for value, e in zip(values, map(int, said)):
        least = -100
        if value > 0:
            least = max(-100, math.frexp(value)[1] - 10)  # below the answer, or the answer
            while Fraction(value) > 448 * Fraction(2) ** least:
                least += 1
        assert e == least, (value, e, least)
