"""Scored attention of wide windows: up to 64 tokens, several tiles of rows, the last rows that the
split kernels take (128 a kv head) and the first that they leave to the general ones."""
import pytest

from test_gpu_scored import TYPES, check, pytestmark  # noqa: F401


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("window,rows,hq,hkv", [(17, 17, 2, 2), (24, 24, 4, 1), (33, 5, 4, 2), (64, 64, 2, 1),
                                                (64, 1, 2, 1), (43, 43, 3, 1), (64, 64, 3, 1), (64, 7, 2, 2)])
def test_wide_windows(cuda_device, dtype, cache, window, rows, hq, hkv):
    check(cuda_device, dtype, cache, (1, window, 16, 65, 0, 301), hq, hkv, 128, 16, window=window, rows=rows, seed=window)


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("bs", [8, 32])
def test_wide_windows_over_several_splits(cuda_device, dtype, cache, bs):
    check(cuda_device, dtype, cache, (1500, 40), 8, 4, 128, bs, window=20, rows=20, seed=bs, bound=2048)
