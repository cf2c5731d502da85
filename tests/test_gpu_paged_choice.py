"""The choice of blocks on the GPU, list for list, against a plain implementation in 64 bits
(paged8_choices.py): scales out of range, scores of all sizes."""
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


@pytest.mark.parametrize("rows", [9600, 1600])
def test_scores_of_infinite_queries_and_keys(ctx, rows):
    """Infinities count as 127 2^64: scores of up to 2^150, past the range of F32, are told apart, and so are those of
    the least queries and scales, down to 2^-94."""
    c = Choice([(rows, 1)] * 16, 8, 8, 64, 64, 16, 8, seed=rows)
    c.bs[:] = 2.0 ** 64
    c.q[:8, :, 5] = np.inf
    c.q[:8, 4:, 6] = -np.inf
    c.check(ctx, current())
    c.bs[:] = 2.0 ** -64
    c.q[8:] = np.random.default_rng(2).choice([-1, 0, 1], c.q[8:].shape) * 2.0 ** -24
    c.check(ctx, current())
    c.bs[:] = 2.0 ** np.random.default_rng(3).choice([-64, -63, 0, 63, 64], c.bs.shape)
    c.check(ctx, current())
