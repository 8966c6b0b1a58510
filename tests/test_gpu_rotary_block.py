"""The example block that runs the general operators together with the engine's attention, against itself in 64 bits.

The int8 rounding of a row is at most half a step of top / 127 per value, uniform: 1 / sqrt(12) of a step. Rows of
normal values have their top near 3 to 4 deviations, so a product's relative error is about 4 / 127 / sqrt(12) = 0.9 %;
five of them follow one another, each passed on at most once through the softmax and the residual sums: 5 x 0.9 % is
the bound on the norm, and the same again for rows whose top is larger."""
import os
import sys

import numpy as np
import pytest
import torch

from arctic_embed_s_int8 import Engine

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.mark.parametrize("lengths", [[1], [7, 1, 33], [128] * 4, [300, 5, 512]])
def test_block(lengths):
    import rotary_block as rb

    engine, block = Engine(0), rb.random_block(len(lengths))
    cu = torch.from_numpy(np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)).cuda()
    x = torch.randn(sum(lengths), rb.HIDDEN, generator=torch.Generator().manual_seed(2)).cuda()
    got, want = rb.run_block(engine, block, x, cu, max(lengths)), rb.plain_block(block, x, cu)
    engine.sync()
    for name, value in got.items():
        assert float((value.double() - want[name]).norm() / want[name].norm()) < 0.09, name
    # packed sequences do not see one another: each alone gives the same rows
    for a, b in zip(cu[:-1].tolist(), cu[1:].tolist()):
        one = rb.run_block(engine, block, x[a:b].contiguous(), torch.tensor([0, b - a], dtype=torch.int32).cuda(), b - a)
        assert torch.equal(one["qkv"], got["qkv"][a:b])
    engine.sync()
    engine.close()
