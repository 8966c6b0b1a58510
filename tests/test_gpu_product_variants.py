"""Every tile that the product's estimate chooses on 148 SMs: one CTA or a pair, 16 to 256 tokens, depths split over 2, 3, 4 or 8
CTAs; with one tile to a CTA and with several; stored as boxes, as boxes with the last channels from the lanes, and
from the lanes alone; and the walk of eight token tiles. Against the exact integer sums, with test_gpu_linear_i8's tolerance
(|error| <= 2.01 u |sum a_scale w_scale| + (u + v) |out|, + 2^-25 for float16), computed in float64 on the GPU, and bit
for bit against the same rows in a product of a few tokens."""
import pytest
import torch

from arctic_embed_s_int8 import Engine
from conftest import rng
from test_gpu_linear_i8 import ROUNDOFF, TYPES, check, dev, make, pitched, quantize

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    e = Engine(0)
    yield e
    e.close()


def operands(M, N, K, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def ints(r):
        rows = torch.empty(r, -(-K // 16) * 16, dtype=torch.int8, device="cuda")[:, :K]  # whole 16 bytes: read in place
        return rows.copy_(torch.randint(-128, 128, (r, K), generator=g, dtype=torch.int8, device="cuda"))

    def uniform(n, lo, hi):
        return torch.rand(n, generator=g, device="cuda") * (hi - lo) + lo

    return ints(M), uniform(M, 1e-3, 1e-2), ints(N), uniform(N, 1e-4, 1e-3), uniform(N, -0.6, 0.6)


def run(eng, M, N, K, dtype, pitch, ops, term):
    a, a_s, w, w_s, b = ops
    buf = torch.full((M + 2, pitch), 7.0, dtype=dtype, device="cuda")
    out = buf[1:M + 1, :N]
    out.fill_(float("nan"))
    eng.matmul_i8(a, a_s, w, w_s, out, bias=b)
    eng.sync()
    assert (buf[0] == 7).all() and (buf[M + 1] == 7).all() and (buf[1:M + 1, N:] == 7).all()
    u, v = 2.0 ** -24, ROUNDOFF[dtype]
    want = term + b.double()
    tol = 2.01 * u * term.abs() + (u + v) * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0)
    bad = ~((out.double() - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3].tolist())
    for first in {0, M // 2, max(0, M - 3)}:
        few = torch.empty(min(3, M - first), N, dtype=dtype, device="cuda")
        eng.matmul_i8(a[first:first + 3], a_s[first:first + 3], w, w_s, few, bias=b)
        eng.sync()
        assert torch.equal(few, out[first:first + 3])


def run_all(eng, M, N, K, types=TYPES):
    ops = operands(M, N, K, M + N + K)
    a, a_s, w, w_s, _ = ops
    term = torch.mm(a.double(), w.double().t()) * (a_s.double()[:, None] * w_s.double())
    whole = -(-N // 16) * 16
    for dtype in types:
        for pitch in sorted({N, whole, whole + 1}):
            run(eng, M, N, K, dtype, pitch, ops, term)


# one tile to a CTA or cluster
@pytest.mark.parametrize("M,N,K", [
    (1, 32, 64), (1, 38, 67),                                             # 16 tokens
    (2408, 40, 69), (2613, 42, 74), (268, 3840, 148),                     # 32
    (4791, 32, 75), (5914, 33, 72),                                       # 64
    (9580, 40, 85), (16066, 39, 70),                                      # 128
    (31982, 32, 69), (30443, 55, 73),                                     # 256
    (3766, 392, 136), (5114, 135, 316),                                   # 128 to a pair
    (14672, 176, 66), (16105, 157, 64),                                   # 256 to a pair
    (1141, 35, 2192), (280, 144, 1444), (282, 37, 1285), (2, 32, 935),    # 16, split 2, 3, 4, 8
    (795, 148, 3249), (1226, 33, 2409), (904, 33, 1967), (17, 1152, 1186),  # 32
    (2920, 40, 5008), (1203, 136, 3526), (1642, 34, 3335), (37, 1432, 3073)])  # 64
def test_tiles(eng, M, N, K):
    run_all(eng, M, N, K)


# several, the accumulators taken in turn
@pytest.mark.parametrize("M,N,K", [
    (293, 1914, 66), (65, 7128, 65),       # 16 tokens
    (909, 1162, 181), (9580, 40, 85),      # 32
    (22475, 40, 64), (24681, 38, 77),      # 64
    (36672, 48, 132), (37394, 38, 142),    # 128
    (20050, 296, 69), (19326, 303, 85),    # 256
    (526, 6624, 73), (608, 6253, 90),      # 128 to a pair
    (29366, 168, 68), (28761, 129, 78),    # 256 to a pair
    # deeper than the ring of stages
    (9001, 1500, 1700), (20000, 96, 2300), (5000, 2507, 2100), (1300, 4099, 1800)])
def test_tiles_in_turn(eng, M, N, K):
    run_all(eng, M, N, K)


@pytest.mark.parametrize("M", [2501, 2048, 700, 129])
@pytest.mark.parametrize("N,K", [(8200, 8300), (20011, 3500)])
def test_walk_of_eight_tiles(eng, M, N, K):
    """Weights over 64 MB, with a last group of fewer token tiles and without."""
    run_all(eng, M, N, K, [TYPES[0], TYPES[2]])


# quantized inside the product, with the depth of a few tokens whole or split over each count of CTAs
@pytest.mark.parametrize("x_type", TYPES)
@pytest.mark.parametrize("M,N,K", [(1, 30522, 384), (1, 9000, 2000), (1, 6037, 1467), (1, 5200, 3001), (1, 4000, 4000),
                                   (2, 6037, 1400), (3, 5000, 1300), (4, 4100, 1000), (7, 2100, 580), (16, 1000, 250)])
def test_fused_quantization(eng, x_type, M, N, K):
    r = rng(M + N + K)
    _, w, _, w_s, b = make(M, N, K, M + K)
    x = torch.from_numpy((r.normal(0, 1, (M, K))).astype("float32")).to(x_type)
    dw = pitched(torch.from_numpy(w), -(-K // 16) * 16)
    for dtype in TYPES:
        out = torch.full((M, N), float("nan"), dtype=dtype, device="cuda")
        eng.linear_i8(x.cuda(), dw, dev(w_s), out, bias=dev(b))
        eng.sync()
        a, a_s = quantize(x.float().numpy(), None)
        check(out, a, a_s, w, w_s, b)
