"""The quantization of more rows than are resident at once, so that a block takes several: 32, 128 or 512 threads to a row
with each count of 16-byte pieces to a thread. Against the formula restated in float32, through a product whose integer
sums are exact."""
import numpy as np
import pytest
import torch

from arctic_embed_s_int8 import Engine
from conftest import rng
from test_gpu_linear_i8 import TYPES, check, dev, make, pitched, quantize

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    e = Engine(0)
    yield e
    e.close()


# 1,024 threads on each of 148 SMs hold 4,736 rows of 32 threads, 1,184 of 128, 296 of 512
@pytest.mark.parametrize("x_type", TYPES)
@pytest.mark.parametrize("pieces,rows", [(17, 4737), (32, 9999), (47, 9473), (64, 4740), (100, 5001), (128, 14209), (200, 1185),
                                         (256, 3001), (300, 2369), (512, 1500), (700, 297), (1024, 893), (1500, 593),
                                         (2048, 301), (2049, 297)])
def test_more_rows_than_are_resident(eng, x_type, pieces, rows):
    size = 4 if x_type == torch.float32 else 2
    N = 33
    for K, pitch, smooth in ((pieces * (16 // size), 0, False), (pieces * (16 // size) - 1, pieces * (16 // size), True),
                             (pieces * (16 // size) - 1, 0, False)):
        r = rng(pieces + K)
        _, w, _, w_s, b = make(1, N, K, pieces)
        x = torch.from_numpy((r.normal(0, 1, (rows, K)) * np.exp(r.normal(0, 1, (rows, 1)))).astype(np.float32))
        x[[0, rows // 2, rows - 1]] = 0
        x[rows - 2, 0] = float("nan")
        x = x.to(x_type)
        s = np.exp(r.normal(0, 0.5, K)).astype(np.float32) if smooth else None
        out = torch.full((rows, N), float("inf"), device="cuda")
        eng.linear_i8(pitched(x, pitch) if pitch else x.cuda(), dev(w), dev(w_s), out, bias=dev(b),
                      inv_smooth=None if s is None else dev(s))
        eng.sync()
        assert out[rows - 2].isnan().all()
        keep = np.arange(rows) != rows - 2
        a, a_s = quantize(x.float().numpy()[keep], s)
        check(out[torch.from_numpy(keep).cuda()], a, a_s, w, w_s, b)
