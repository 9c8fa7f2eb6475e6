"""Bounds of pages whose channels lie many powers of two apart: every code is the
definition's and no key lies outside its bounds, however small beside the page's scale."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import attention_oracle as A
from test_gpu_blocks import bounds_on_gpu, check_bounds

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _gpu(gpu_available):
    torch.cuda.set_device(0)


@pytest.mark.parametrize("dtype", (BF, FP))
@pytest.mark.parametrize("dim", (64, 96, 128, 256))
def test_bounds_of_channels_far_below_the_scale(dtype, dim):
    """A key that a division by the scale takes below the least float still lies between its bounds."""
    page, pages = 4, 8
    info = torch.finfo(dtype)
    least = info.smallest_normal * info.eps  # the smallest value of the type
    k, _ = A.make_cache(np.random.default_rng(dim), pages, page, 2, dim, dtype)
    for p, (large, small) in enumerate(((info.max, least), (info.max, info.smallest_normal), (2.0 ** 127, 2.0 ** -30), (1e20, 7e-28), (1e20, 9e-28), (1.0, least),
                                        (-info.max, least), (0.0, least))):
        k[p] = 0
        k[p, 1, :, 0] = min(large, info.max)
        k[p, :, :, 1], k[p, :, :, 2] = small, -small
        k[p, 2, :, 5], k[p, 3, :, 6], k[p, :3, :, dim - 1] = small, -small, -small
    check_bounds(k, list(range(pages * page)))
    codes, scales = (t.cpu().double() for t in bounds_on_gpu(k, list(range(pages * page))))
    bounds = codes * scales[:, :, None, None]
    keys = k.double()
    assert bool((keys <= bounds[:, None, :, 0]).all()) and bool((keys >= bounds[:, None, :, 1]).all())
