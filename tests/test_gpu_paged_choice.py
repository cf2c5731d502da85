"""The choice of blocks on the GPU, list for list, against a plain implementation in 64 bits
(paged8_choices.py): scales out of range, scores of all sizes, the
search of long streams by 16 wavefronts and the join of their segments."""
import numpy as np
import pytest

from paged8_choices import LONG, Choice, long_choice

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


@pytest.mark.parametrize("name", LONG)
def test_long_streams(ctx, name):
    """(test_paged8_routes.py looks at which kernels these are.)"""
    c = long_choice(name, seed=len(name))
    c.max_nkv = max(n for n, _ in c.sizes)
    c.check(ctx, current())
    # among first and last blocks, scores alike, other pages
    c = long_choice(name, seed=len(name) + 1, few=2, n_sink=c.top // 3, n_recent=c.top // 4)
    c.max_nkv = max(n for n, _ in c.sizes)
    c.check(ctx, current())


def test_segments_in_a_graph(ctx):
    """Segments and their join captured once and replayed with other queries and sizes, another choice of the same
    context between, whose segments lie in the same workspace."""
    import torch
    from gpu_util import vxfa
    own = vxfa.Context(0)
    try:
        c, other = long_choice("5120_pairs", seed=1), long_choice("three_segments_1800_pairs", seed=2)
        c.max_nkv, other.max_nkv = 20000 * 16, 9000 * 16
        args, more = c.place(), other.place()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=side):
            own.paged_select(*args, stream=side.cuda_stream)
        rng = np.random.default_rng(3)
        for turn in range(4):
            c.q = c.host["q"] = rng.standard_normal(c.q.shape).astype(np.float16)
            c.sizes = [(int(n), 1) for n in rng.integers(1, 20000 * 16, 2)]
            c.n_kv = c.host["n_kv"] = np.array([n for n, _ in c.sizes], np.int32)
            for k in ("q", "n_kv"):
                c.dev[k].copy_(torch.from_numpy(c.host[k].reshape(-1).view(np.uint8)))
            c.dev["list"].fill_(0xA5)
            torch.cuda.synchronize()
            graph.replay()
            own.paged_select(*more, stream=current())
            c.same()
            other.same()
    finally:
        own.close()
