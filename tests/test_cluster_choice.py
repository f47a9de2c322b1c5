"""Attention of few rows gives a cluster of CTAs to each segment only where the device can place it; else it takes the line of pages,
whose partial results need a workspace."""
import pytest
import torch

from onebitsparsemul_b200 import _lib, build

# (table width, tokens, sequences, heads, kv_heads, head_dim, max_new) that clusters are taken for: of 16, 8, 4, 2 and 1 CTAs
SHAPES = [(64, 1, 1, 4, 4, 128, 1), (40, 1, 1, 32, 32, 128, 1), (20, 8, 8, 32, 8, 64, 1), (12, 16, 16, 32, 8, 128, 1), (16, 64, 64, 32, 8, 64, 1), (12, 48, 16, 30, 10, 128, 3)]


@pytest.fixture(scope="module")
def workspace():
    build.build_library()
    return _lib.load().onebit_cache_attend_workspace


def test_without_a_place_for_clusters_the_line_is_taken(workspace):
    if torch.cuda.is_available():
        pytest.skip("this device has a place for them")
    for shape in SHAPES:
        assert workspace(*shape) > 0


@pytest.mark.gpu
def test_clusters_are_taken_where_they_fit(workspace):
    for shape in SHAPES:
        assert workspace(*shape) == 0
