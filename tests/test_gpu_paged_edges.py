"""Edges of the operators of a paged KV cache (lux/gpu/paged_ext.h): what lies beside a sequence's last key, faults that meet in one wait, rows of
many heads, block numbers out of range."""
import math

import pytest
import torch

from test_gpu_paged import Batch, buf  # noqa: F401  (a fixture)
from webgpu_b200 import backend as B

pytestmark = pytest.mark.gpu


# ---- attention: values behind the last key ----------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D,page", [(128, 1), (128, 2), (128, 4), (128, 5), (128, 8), (128, 12), (128, 16), (128, 24), (128, 64), (64, 1), (64, 8), (64, 24)])
def test_attention_bits_do_not_depend_on_what_was_there_before(ctx, buf, dtype, D, page):
    """Sequences that end anywhere in a key tile, behind others whose values are no numbers: what an earlier tile (or call) left in shared memory
    behind the last key takes no part, so that the outputs are those of a call without it, bit for bit."""
    ends = [1, 8, 24, 40, 56, 1000, 9, 33, 64, 90, 108, 130, 186, 300]
    lens = [n for e in ends for n in (700, e)] * 4             # every other one is to be spoiled; several items to a CTA
    b = Batch(dtype, 8, 8, D, page, [1] * len(lens), lens)
    b.run(ctx, buf)
    b.check()
    want = b.out[1::2].clone(), b.lse[1::2].clone()
    for s in range(0, len(lens), 2):
        for at in b.table[s].tolist():
            if at >= 0:
                b.vc[at] = math.nan
    for _ in range(2):                                         # (the second time every CTA's ring has seen them)
        b.run(ctx, buf)
        torch.cuda.synchronize()
        assert b.out[::2].isnan().all()
        assert torch.equal(b.out[1::2], want[0]) and torch.equal(b.lse[1::2], want[1])
