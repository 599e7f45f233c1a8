"""Which way ragged attention takes -- shares of a line of tiles or a work-group each, four or eight wavefronts, units in
shares or whole contexts -- against the 64-bit forms, and what a window hides."""
import math

import pytest
import torch

from flash_attention_factory_amd import torch_ops  # noqa: F401

import _ragged as R
from test_gpu_ragged_attention import _close, _differential, _pools, _query, _ragged, _strided

pytestmark = pytest.mark.gpu

# Sequences and heads with two tiles and more for each of 256 compute units: a work-group for each tile.
GRIDS = {
    "four_wavefronts_many_sequences": (R.Batch([20] * 130 + [0, 3], [(k * 29) % 150 for k in range(132)], B=16), 16, 8),
    "four_wavefronts": (R.Batch([30 - k % 3 for k in range(64)], [(k * 29) % 150 for k in range(64)], B=16), 64, 16),
    "eight_wavefronts": (R.Batch([33, 0, 40] + [37] * 40, [1600] + [(k * 29) % 150 for k in range(42)], B=16), 64, 8),
    "eight_wavefronts_many_sequences": (R.Batch([65] * 66, [(k * 29) % 150 for k in range(65)] + [1700], B=16), 32, 8),
}


@pytest.mark.parametrize("name", sorted(GRIDS))
@pytest.mark.parametrize("kv", ["16", "i8"])
def test_a_work_group_for_each_tile(name, kv):
    batch, H, Hk = GRIDS[name]
    _ragged(batch, H, Hk, 64, kv, torch.bfloat16, window=100 if kv == "i8" else -1)
    _differential(batch, H, Hk, 64, kv, torch.float16, window=-1 if kv == "i8" else 100)


@pytest.mark.parametrize("kv", ["16", "i8"])
@pytest.mark.parametrize("H,Hk", [(2, 2), (6, 3), (12, 12), (8, 1)])
def test_short_contexts_with_and_without_shares(kv, H, Hk):
    batch = R.Batch([1, 2, 1, 0, 1], [509, 0, 128, 7, 255], B=16)
    for longest in (510, 513):
        _ragged(batch, H, Hk, 128, kv, torch.float16, longest=longest)
        _differential(batch, H, Hk, 128, kv, torch.bfloat16, longest=longest)


@pytest.mark.parametrize("lens", [[4000], [5000, 20, 3000], [8300, 8100, 8200], [5000] * 9])
@pytest.mark.parametrize("kv", ["16", "i8"])
def test_numbers_of_shares(kv, lens):
    """From fewer units than compute units to many for each."""
    batch = R.Batch([1] * len(lens), lens, B=64)
    _ragged(batch, 8, 8, 64, kv, torch.float16)
    _differential(batch, 10, 5, 64, kv, torch.float16)


@pytest.mark.parametrize("new,old", [([1, 1, 1, 1], [300, 70, 129, 700]), ([70, 1, 40], [300, 600, 4]), ([300], [900])])
@pytest.mark.parametrize("window", [0, 20, 130])
@pytest.mark.parametrize("kv", ["16", "i8"])
def test_what_the_window_hides_may_be_anything(new, old, window, kv):
    """Keys and values before every new token's window are NaN (bytes: with NaN for the scales of whole blocks)."""
    batch = R.Batch(new, old, B=16)
    for s, (n, o) in enumerate(zip(new, old)):
        hidden = max(0, o - window)
        for block in range((hidden + 15) // 16):
            batch.used[int(batch.tables[s, block]), :hidden - block * 16] = False
    _ragged(batch, 4, 2, 64, kv, torch.float16, window=window)
    _differential(batch, 4, 2, 64, kv, torch.float16, window=window)
