"""What KVCache8 takes as a cache (no GPU)."""
import pytest
import torch

import onebitsparsemul_b200 as ob
from onebitsparsemul_b200 import build


@pytest.fixture(scope="module", autouse=True)
def extension():
    build.build_torch_extension()


def test_a_cache_s_tensors_are_apart():
    """With heads of 64 values keys and values have one shape: one tensor for both, or for both scales, was taken."""
    c = ob.KVCache8.empty(3, 2, 64, device="cpu")
    ob.KVCache8(c.k_pages, c.v_pages, c.k_scale, c.v_scale)
    both = torch.zeros(4, 2, 64, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    scales = torch.zeros(4, 2)
    inside = c.k_pages.view(torch.uint8).view(-1)[64:64 + 24].view(torch.float32).view(3, 2)
    for tensors in ((c.k_pages, c.k_pages, c.k_scale, c.v_scale), (c.k_pages, c.v_pages, c.k_scale, c.k_scale), (both[:3], both[1:], c.k_scale, c.v_scale),
                    (c.k_pages, c.v_pages, scales[:3], scales[1:]), (c.k_pages, c.v_pages, inside, c.v_scale), (c.k_pages, c.v_pages, c.k_scale, inside)):
        with pytest.raises(ValueError):
            ob.KVCache8(*tensors)
    whole = torch.zeros(6, 2, 64, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    ob.KVCache8(whole[:3], whole[3:], scales[:3], torch.zeros(3, 2))                 # parts of one allocation, apart
