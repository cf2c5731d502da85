"""Single tokens where the host's bound of a stream's rows lies far above them, as in a graph captured for
the longest stream: pages of F16 and 8 bits against a plain implementation in 64 bits (paged8_util.py)."""
import math

import numpy as np
import pytest

import paged8_util as p8
from paged8_util import Batch8, Device8
from paged_util import Batch, check_out

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from gpu_util import vxfa
    c = vxfa.Context(0)
    yield c
    c.close()


def attend(ctx, c, bound, **opt):
    import torch
    c.table = np.concatenate([c.table, np.full((c.B, bound // c.page - c.max_pages), -1, np.int32)], 1)
    c.max_pages = bound // c.page
    d = Device8(c)
    scale, args = 1 / math.sqrt(c.hd), (opt.get("bias", 0.0), opt.get("cap", 0.0))
    st = torch.cuda.current_stream().cuda_stream
    if isinstance(c, Batch8):
        ctx.flash_attn_ext_paged_q8(d.q, d.k, d.ks, d.v, d.vs, d.batch, d.dst, scale, *args, stream=st)
    else:
        ctx.flash_attn_ext_paged(d.q, d.k, d.v, d.batch, d.dst, scale, *args, stream=st)
    torch.cuda.synchronize()
    want, err = p8.reference(c, scale, **opt)
    check_out(d.out(), want, err, True)
    d.check_guards()


@pytest.mark.parametrize("kind", [Batch, Batch8])
@pytest.mark.parametrize("hq,hkv,hd", [(8, 8, 128), (32, 8, 128), (8, 8, 64), (4, 2, 64)])
@pytest.mark.parametrize("rows", [1, 40, 3000, 20000])
def test_one_stream(ctx, kind, hq, hkv, hd, rows):
    """The join reads only the records that there are, of up to 513 that the bound allows."""
    attend(ctx, kind([(rows, 1)], hq, hkv, hd, 64, seed=rows), 131072)


@pytest.mark.parametrize("kind", [Batch, Batch8])
@pytest.mark.parametrize("hd", [128, 64])
def test_few_streams(ctx, kind, hd):
    attend(ctx, kind([(700, 1), (5000, 1)], 8, 8, hd, 64, seed=hd), 65536, cap=30.0)
    attend(ctx, kind([(3000, 1), (1, 1), (0, 0), (90, 2)], 16, 8, hd, 64, seed=hd), 65536, bias=4.0)
    attend(ctx, kind([(2500, 3)], 8, 8, hd, 64, seed=hd), 131072)
