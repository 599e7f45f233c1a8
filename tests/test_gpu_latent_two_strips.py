"""Absorbed attention over FP8 pools in tiles of 32 rows of which 17 to 32 are in use: every wavefront has scores, and half of them load as well.
Contexts of one step and of many, whole and cut; pool rows behind a context, and their scales, are NaN."""
import pytest

from test_gpu_latent import BF16, F16, _absorbed

pytestmark = pytest.mark.gpu

SHORT, LONG = [1, 2, 33, 50, 63, 64, 65, 128, 129, 200], [257, 300, 320, 321, 1000, 2000, 2049]


@pytest.mark.parametrize("L", [256, 512])
@pytest.mark.parametrize("dtype,H,n", [(F16, 17, 1), (BF16, 20, 1), (F16, 24, 1), (BF16, 32, 1), (BF16, 16, 2), (F16, 8, 3), (BF16, 8, 4)])
@pytest.mark.parametrize("B", [16, 64])
def test_whole_contexts(L, dtype, H, n, B):
    keys = [max(n, k) for k in SHORT]
    _absorbed(dtype, "e4m3", L, H, B, [n] * len(keys), [k - n for k in keys])


@pytest.mark.parametrize("L", [256, 512])
@pytest.mark.parametrize("dtype,H,n", [(F16, 17, 1), (BF16, 20, 1), (F16, 24, 1), (BF16, 32, 1), (BF16, 16, 2), (F16, 8, 4)])
def test_contexts_that_are_cut(L, dtype, H, n):
    keys = LONG + SHORT
    _absorbed(dtype, "e4m3", L, H, 16, [n] * len(keys), [max(n, k) - n for k in keys])
    for k in (257, 300, 2000):  # alone: shares of few steps
        _absorbed(dtype, "e4m3", L, H, 16, [n], [k - n], seed=k)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_rows_in_use_differ_from_sequence_to_sequence(dtype):
    _absorbed(dtype, "e4m3", 512, 8, 16, [4, 1, 2, 3, 0, 4, 2], [60, 63, 700, 31, 5, 1, 0])
    _absorbed(dtype, "e4m3", 256, 32, 32, [1] * 70, [7 * k for k in range(70)])


def test_references_move():
    _absorbed(BF16, "e4m3", 512, 32, 16, [1, 1], [900, 333], size=4.0, layout="tokens")
