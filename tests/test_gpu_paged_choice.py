"""The choice of blocks on the GPU, list for list, against a plain implementation in 64 bits
(paged8_choices.py): scales out of range."""
import numpy as np
import pytest

from paged8_choices import Choice

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from gpu_util import vxfa
    c = vxfa.Context(0)
    yield c
    c.close()


def current():
    import torch
    return torch.cuda.current_stream().cuda_stream


def nan(payload):
    return np.array([payload], np.uint32).view(np.float32)[0]


@pytest.mark.parametrize("rows", [9600, 100 * 16])
def test_scales_that_are_no_numbers(ctx, rows):
    """NaN of any payload count as 2^-64, what lies outside the range as its end, also where a
    workgroup searches together (more than 512 blocks, 128 workgroups and more); the lists keep to their places."""
    c = Choice([(rows, 1)] * 16, 8, 8, 64, 64, 16, 8, seed=rows)
    rng = np.random.default_rng(1)
    odd = np.array([0x7FFFFFFC, 0x7FFFFFFE], np.uint32).view(np.float32)
    c.bs = odd[rng.integers(0, 2, c.bs.shape)]
    c.check(ctx, current())
    some = np.array([0x7FFFFFFC, 0x7FFFFFFD, 0x7FFFFFFE, 0x7FFFFFFF, 0xFFFFFFFF, 0xFFC00000, 0x7F800001, 0x7F800000, 0xFF800000, 0, 1,
                     0x80000000, 0xBF800000, 0x7F7FFFFF, 0x3F800000, 0x40000000], np.uint32).view(np.float32)
    c.bs = some[rng.integers(0, len(some), c.bs.shape)]
    c.n_sink, c.n_recent = 1, 2
    c.check(ctx, current())
