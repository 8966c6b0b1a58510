"""The general int8 product (ae_matmul_i8) and the product from float activations (ae_linear_i8) against
their formulas in 64 bits.

Tolerance, with u the unit roundoff of float32 (2^-24) and v that of the output's type (2^-24, 2^-11, 2^-8):
the integer sum is exact, float(sum) and a_scale * w_scale are each off by u, and the fused multiply-add by u
of its result, so |error| <= 2.01 u |sum a_scale w_scale| + (u + v) |out| (+ half the smallest float16
subnormal, 2^-25). The quantization of the float activations is restated in float32, whose elementwise steps
are the same everywhere, and checked against 64 bits by a product with the identity."""
import numpy as np
import pytest
import torch

from arctic_embed_s_int8 import AeError, Engine
from conftest import rng

pytestmark = pytest.mark.gpu

ROUNDOFF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TYPES = list(ROUNDOFF)


@pytest.fixture(scope="module")
def eng():
    e = Engine(0)  # the operators need no model
    yield e
    e.close()


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def pitched(a, pitch, lead=0):
    """The device matrix a in rows of `pitch` elements that start `lead` elements into a 256-byte aligned buffer."""
    r, c = a.shape
    buf = torch.zeros(lead + max(r, 1) * pitch, dtype=a.dtype, device="cuda")
    view = buf[lead:].view(max(r, 1), pitch)[:r, :c]
    view.copy_(a)
    return view


def guarded(M, N, dtype, pitch=None):
    """An output filled with NaN inside a buffer filled with 7."""
    pitch = pitch or N
    buf = torch.full((M + 2, pitch), 7.0, dtype=dtype, device="cuda")
    out = buf[1:M + 1, :N]
    out.fill_(float("nan"))
    return buf, out


def guards_hold(buf, M, N):
    b = buf.float().cpu().numpy()
    return (b[0] == 7).all() and (b[M + 1] == 7).all() and (b[1:M + 1, N:] == 7).all()


def make(M, N, K, seed, bias=True):
    r = rng(seed)
    a = r.integers(-128, 128, (M, K), dtype=np.int8)
    w = r.integers(-128, 128, (N, K), dtype=np.int8)
    a_s = r.uniform(1e-3, 1e-2, M).astype(np.float32)
    w_s = r.uniform(1e-4, 1e-3, N).astype(np.float32)
    b = r.normal(0, 0.3, N).astype(np.float32) if bias else None
    return a, w, a_s, w_s, b


def int_product(a, w):
    """Exact: the sums of 8-bit products stay far inside a double's 53 bits."""
    return a.astype(np.float64) @ w.astype(np.float64).T


def check(out, a, a_s, w, w_s, b):
    acc = int_product(a, w)
    term = acc * (a_s.astype(np.float64)[:, None] * w_s.astype(np.float64))
    want = term + (0 if b is None else b.astype(np.float64))
    u, v = 2.0 ** -24, ROUNDOFF[out.dtype]
    tol = 2.01 * u * np.abs(term) + (u + v) * np.abs(want) + (2.0 ** -25 if out.dtype == torch.float16 else 0)
    got = out.double().cpu().numpy()
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3], got[bad][:3], want[bad][:3])


def run_matmul(eng, M, N, K, dtype, seed, bias=True, pitch=None, **kw):
    a, w, a_s, w_s, b = make(M, N, K, seed, bias)
    buf, out = guarded(M, N, dtype, pitch)
    da, dw = kw.get("a", dev)(a), kw.get("w", dev)(w)
    eng.matmul_i8(da, dev(a_s), dw, dev(w_s), out, bias=None if b is None else dev(b))
    eng.sync()
    assert guards_hold(buf, M, N)
    check(out, a, a_s, w, w_s, b)


# every side of the row, channel and depth tiles
@pytest.mark.parametrize("M", [1, 2, 16, 17, 33, 64, 65, 129])
@pytest.mark.parametrize("N,K", [(1, 1), (3, 16), (128, 128), (129, 127), (257, 384), (64, 129), (1001, 1003)])
def test_sizes(eng, M, N, K):
    for i, dt in enumerate(TYPES):
        run_matmul(eng, M, N, K, dt, M * 1000 + N + K + i, bias=(M + i) % 2 == 0)


@pytest.mark.parametrize("M,N,K", [(300, 1152, 384), (1000, 384, 1536), (2049, 515, 272), (1, 30522, 384),
                                   (5, 4096, 4096), (16, 129, 8192), (700, 33, 5000), (4099, 1031, 640)])
def test_larger_sizes(eng, M, N, K):
    run_matmul(eng, M, N, K, TYPES[(M + N) % 3], M + N + K)


@pytest.mark.parametrize("M", [1, 40, 300])
@pytest.mark.parametrize("a_pitch,a_lead,w_pitch,w_lead", [(208, 0, 240, 16), (201, 0, 200, 0), (208, 3, 224, 0),
                                                           (224, 16, 224, 1), (200, 0, 333, 7)])
def test_pitches_and_offsets(eng, M, a_pitch, a_lead, w_pitch, w_lead):
    """Rows that start anywhere: read in place where they lie on 16 bytes, laid out first elsewhere."""
    for dt, pitch in ((torch.float32, 133), (torch.bfloat16, 140), (torch.float16, 131)):
        run_matmul(eng, M, 131, 200, dt, M + a_pitch + w_lead, pitch=pitch,
                   a=lambda x: pitched(torch.from_numpy(x), a_pitch, a_lead),
                   w=lambda x: pitched(torch.from_numpy(x), w_pitch, w_lead))


@pytest.mark.parametrize("M,N,K,pitch", [(1500, 1031, 640, 1032), (4099, 1025, 200, 1040), (300, 8190, 384, 8200),
                                         (6000, 397, 130, 400)])
def test_rows_that_end_inside_16_bytes(eng, M, N, K, pitch):
    """Outputs whose rows start on 16 bytes and end elsewhere: what follows a row's end is not written."""
    for i, dt in enumerate(TYPES):
        run_matmul(eng, M, N, K, dt, M + N + i, pitch=pitch)


def far(x, pitch):
    """x in rows `pitch` elements apart, in a buffer that is not cleared."""
    r, c = x.shape
    view = torch.empty((r - 1) * pitch + c, dtype=x.dtype, device="cuda").as_strided((r, c), (pitch, 1))
    view.copy_(x)
    return view


@pytest.mark.parametrize("pitch", [2 ** 30, 2 ** 30 + 1])
def test_offsets_beyond_32_bits(eng, pitch):
    """Rows 2^30 elements apart, read in place or laid out first, and results stored as far apart."""
    M, N, K = 5, 200, 130
    a, w, a_s, w_s, b = make(M, N, K, 7)
    out = torch.empty(2 * pitch + N, dtype=torch.float16, device="cuda").as_strided((3, N), (pitch, 1))
    eng.matmul_i8(dev(a[:3]), dev(a_s[:3]), dev(w), dev(w_s), out, bias=dev(b))
    eng.sync()
    check(out, a[:3], a_s[:3], w, w_s, b)
    del out
    near = torch.empty(M, 5, dtype=torch.float32, device="cuda")
    eng.matmul_i8(far(torch.from_numpy(a), pitch), dev(a_s), far(torch.from_numpy(w[:5]), pitch), dev(w_s[:5]), near)
    eng.sync()
    check(near, a, a_s, w[:5], w_s[:5], None)
    x = torch.randn(3, K, dtype=torch.float16, device="cuda")
    here, there = (torch.empty(3, N, dtype=torch.float32, device="cuda") for _ in range(2))
    eng.linear_i8(x, dev(w), dev(w_s), here)
    eng.linear_i8(far(x, pitch), dev(w), dev(w_s), there)
    eng.sync()
    assert torch.equal(here, there)


@pytest.mark.parametrize("N", [58000, 58001])
def test_outputs_beyond_32_bits(eng, N):
    """2.3 billion results, as boxes and from the lanes: rows from all over them."""
    M, K = 40000, 40
    a, w, a_s, w_s, b = make(M, N, K, 8)
    out = torch.full((M, N), float("nan"), dtype=torch.bfloat16, device="cuda")
    eng.matmul_i8(dev(a), dev(a_s), dev(w), dev(w_s), out, bias=dev(b))
    eng.sync()
    assert not out[::97].isnan().any()
    rows = [0, 255, 256, 18511, 18512, 37025, 37026, 37027, 39998, 39999]
    check(out[rows], a[rows], a_s[rows], w, w_s, b)


@pytest.mark.parametrize("M", [1, 130])
def test_largest_sums(eng, M):
    """-128 * -128 over the deepest product is just inside int32."""
    K, N = 131071, 130
    a = np.full((M, K), -128, np.int8)
    w = np.full((N, K), -128, np.int8)
    a_s, w_s = np.full(M, 1e-4, np.float32), np.full(N, 1e-4, np.float32)
    buf, out = guarded(M, N, torch.float32)
    eng.matmul_i8(dev(a), dev(a_s), dev(w), dev(w_s), out)
    eng.sync()
    check(out, a, a_s, w, w_s, None)


def test_no_rows(eng):
    a, w, a_s, w_s, b = make(0, 32, 64, 1)
    out = torch.empty(0, 32, device="cuda")
    eng.matmul_i8(dev(a), dev(a_s), dev(w), dev(w_s), out)
    eng.linear_i8(torch.empty(0, 64, device="cuda"), dev(w), dev(w_s), out)
    eng.sync()


def test_scales_keep_infinities_and_nan_in_their_rows_and_columns(eng):
    M, N, K = 40, 150, 100
    a, w, a_s, w_s, b = make(M, N, K, 3)
    a_s[7], w_s[140] = np.nan, np.inf
    buf, out = guarded(M, N, torch.float32)
    eng.matmul_i8(dev(a), dev(a_s), dev(w), dev(w_s), out, bias=dev(b))
    eng.sync()
    got = out.cpu().numpy()
    assert np.isnan(got[7]).all() and not np.isfinite(got[:, 140]).any()
    keep = np.ones((M, N), bool)
    keep[7], keep[:, 140] = False, False
    assert np.isfinite(got[keep]).all()


def test_same_bits_every_time(eng):
    for M, N, K in ((3, 1000, 4096), (100, 384, 1536), (5000, 1152, 384)):
        a, w, a_s, w_s, b = (dev(x) for x in make(M, N, K, M))
        outs = [torch.empty(M, N, dtype=torch.bfloat16, device="cuda") for _ in range(3)]
        for o in outs:
            eng.matmul_i8(a, a_s, w, w_s, o, bias=b)
        eng.sync()
        assert all(torch.equal(outs[0], o) for o in outs[1:])


# ------------------------------------------------------------------------------- float activations
def quantize(x, inv_smooth):
    """ae_linear_i8's quantization, each step rounded to float32."""
    y = x.astype(np.float32)
    if inv_smooth is not None:
        y = y * inv_smooth
    top = np.abs(y).max(axis=1) if y.size else np.zeros(len(y), np.float32)
    any_ = top >= np.float32(2.0 ** -119)
    inv = np.where(any_, np.float32(127) / np.where(any_, top, 1), 0).astype(np.float32)
    return np.rint(y * inv[:, None]).astype(np.int8), np.where(any_, top / np.float32(127), 0).astype(np.float32)


def run_linear(eng, M, N, K, x_type, dtype, seed, smooth=True, bias=True, x_pitch=None, lead=0):
    _, w, _, w_s, b = make(M, N, K, seed, bias)
    r = rng(seed + 1)
    x = torch.from_numpy((r.normal(0, 1, (M, K)) * np.exp(r.normal(0, 1, K))).astype(np.float32)).to(x_type)
    s = np.exp(r.normal(0, 0.5, K)).astype(np.float32) if smooth else None
    buf, out = guarded(M, N, dtype)
    dx = pitched(x, x_pitch, lead) if x_pitch else x.cuda()
    eng.linear_i8(dx, dev(w), dev(w_s), out, bias=None if b is None else dev(b),
                  inv_smooth=None if s is None else dev(s))
    eng.sync()
    assert guards_hold(buf, M, N)
    a, a_s = quantize(x.float().numpy(), s)
    check(out, a, a_s, w, w_s, b)


@pytest.mark.parametrize("x_type", TYPES)
@pytest.mark.parametrize("M,N,K", [(1, 384, 384), (1, 1, 64), (2, 3, 130), (5, 1, 1003), (1, 129, 4096), (2, 64, 1), (7, 100, 1003), (16, 1536, 384),
                                   (17, 40, 1536), (64, 384, 1536), (130, 257, 2050), (509, 1001, 1003), (1, 16, 20001),
                                   (3, 128, 16392), (600, 384, 4104)])
def test_linear(eng, x_type, M, N, K):
    run_linear(eng, M, N, K, x_type, TYPES[(M + K) % 3], M + N + K, smooth=K % 2 == 0, bias=M % 2 == 0)


@pytest.mark.parametrize("x_type", TYPES)
@pytest.mark.parametrize("M", [1, 9, 200])
def test_linear_pitches_and_offsets(eng, x_type, M):
    for pitch, lead in ((208, 0), (201, 0), (208, 8), (208, 1)):
        run_linear(eng, M, 70, 200, x_type, torch.float32, M + pitch, x_pitch=pitch, lead=lead)


@pytest.mark.parametrize("M", [1, 12, 200])
@pytest.mark.parametrize("K", [64, 384, 1000])
def test_quantization_in_64_bits(eng, M, K):
    """A product with the identity gives the quantized rows back: each is the nearest step of top / 127,
    up to the three roundings on the way to it (3 u of at most 127 steps)."""
    r = rng(M + K)
    x = (r.normal(0, 1, (M, K)) * np.exp(r.normal(0, 2, (M, 1)))).astype(np.float32)
    out = torch.empty(M, K, device="cuda")
    eng.linear_i8(dev(x), dev(np.eye(K, dtype=np.int8)), dev(np.ones(K, np.float32)), out)
    eng.sync()
    step = np.abs(x.astype(np.float64)).max(1, keepdims=True) / 127
    steps = out.double().cpu().numpy() / step
    q = np.rint(steps)
    assert np.abs(steps - q).max() <= 127 * 3 * 2.0 ** -24
    assert np.abs(q).max(1).min() == 127 and np.abs(q).max() == 127
    assert np.abs(q - x / step).max() <= 0.5 + 127 * 3 * 2.0 ** -24


@pytest.mark.parametrize("x_type", TYPES)
@pytest.mark.parametrize("M,K", [(6, 384), (6, 20001), (40, 1000)])
def test_rows_without_a_scale(eng, x_type, M, K):
    """Zeros and values under the smallest scale give the bias; an infinity or a NaN gives a row of NaN; the
    rows beside them are as ever."""
    N = 70
    _, w, _, w_s, b = make(M, N, K, 5)
    x = torch.from_numpy(rng(6).normal(0, 1, (M, K)).astype(np.float32)).to(x_type)
    x[0] = 0
    x[1, K // 2] = float("inf")
    x[2, K - 1] = float("nan")
    x[3] = 2.0 ** -130 if x_type != torch.float16 else 0
    x[4, 0] = -float("inf")
    out = torch.empty(M, N, device="cuda")
    eng.linear_i8(x.cuda(), dev(w), dev(w_s), out, bias=dev(b))
    eng.sync()
    got = out.cpu().numpy()
    np.testing.assert_array_equal(got[[0, 3]], np.stack([b, b]))
    assert np.isnan(got[[1, 2, 4]]).all()
    a, a_s = quantize(x[5:].float().numpy(), None)
    check(out[5:], a, a_s, w, w_s, b)


def test_streams(eng):
    """Calls on two streams at once each have scratch of their own; the rows are laid out there."""
    M, N, K = 700, 515, 1003
    cases = [make(M, N, K, s) for s in (11, 12)]
    x = [torch.from_numpy(rng(s).normal(0, 1, (M, K)).astype(np.float32)).cuda() for s in (1, 2)]
    dw = [dev(c[1]) for c in cases]
    ws = [dev(c[3]) for c in cases]
    want = [torch.empty(M, N, device="cuda") for _ in x]
    for i in range(2):
        eng.linear_i8(x[i], dw[i], ws[i], want[i])
    eng.sync()
    streams = [torch.cuda.Stream() for _ in x]
    outs = [[torch.empty(M, N, device="cuda") for _ in range(20)] for _ in x]
    torch.cuda.synchronize()
    try:
        for j in range(20):
            for i in range(2):
                eng.set_stream(streams[i])
                eng.linear_i8(x[i], dw[i], ws[i], outs[i][j])
        torch.cuda.synchronize()
    finally:
        eng.set_stream(None)
    for i in range(2):
        assert all(torch.equal(want[i], o) for o in outs[i])


@pytest.mark.parametrize("M", [1, 64, 700])
def test_operands_written_just_before(eng, M):
    """Weights, activations and scales that the kernel ahead on the stream has just written, call after call with
    nothing in between: each result is that of the operands as they stood."""
    N, K, rounds = 512, 2048, 24
    r = rng(M)
    ws = torch.from_numpy(r.integers(-127, 128, (rounds, N, K), dtype=np.int8)).cuda()
    xs = torch.from_numpy(r.normal(0, 1, (rounds, M, K)).astype(np.float32)).cuda()
    w_s = torch.from_numpy(r.uniform(1e-4, 1e-3, (rounds, N)).astype(np.float32)).cuda()
    want = torch.empty(rounds, M, N, device="cuda")
    for i in range(rounds):
        eng.linear_i8(xs[i], ws[i], w_s[i], want[i])
        eng.sync()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = torch.empty_like(want)
    try:
        eng.set_stream(s)
        with torch.cuda.stream(s):
            w, x, sc = torch.zeros_like(ws[0]), torch.zeros_like(xs[0]), torch.zeros_like(w_s[0])
            for i in range(rounds):
                x.copy_(xs[i])
                sc.copy_(w_s[i])
                w.copy_(ws[i])
                eng.linear_i8(x, w, sc, got[i])
        s.synchronize()
    finally:
        eng.set_stream(None)
    eng.sync()
    assert torch.equal(got, want)


def test_calls_in_a_chain(eng):
    """One call's result is the next one's input."""
    M, D = 300, 1024
    r = rng(8)
    w = [torch.from_numpy(r.integers(-127, 128, (D, D), dtype=np.int8)).cuda() for _ in range(6)]
    ws = torch.full((D,), 1.0 / (127 * 18), device="cuda")
    x = torch.from_numpy(r.normal(0, 1, (M, D)).astype(np.float32)).cuda()
    steps = [x]
    for v in w:
        steps.append(torch.empty(M, D, device="cuda"))
        eng.linear_i8(steps[-2], v, ws, steps[-1])
        eng.sync()
    again = [torch.empty(M, D, device="cuda") for _ in w]
    for i, v in enumerate(w):
        eng.linear_i8(x if i == 0 else again[i - 1], v, ws, again[i])
    eng.sync()
    assert all(torch.equal(a, b) for a, b in zip(again, steps[1:]))


def test_graph_capture(eng):
    """A captured call replays on new inputs."""
    M, N, K = 4, 1152, 384
    a, w, a_s, w_s, b = make(M, N, K, 21)
    x = torch.from_numpy(rng(3).normal(0, 1, (M, K)).astype(np.float32)).cuda()
    dw, dws, out = dev(w), dev(w_s), torch.empty(M, N, device="cuda")
    s = torch.cuda.Stream()
    try:
        with torch.cuda.stream(s):
            eng.set_stream(s)
            eng.linear_i8(x, dw, dws, out)
            s.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                eng.linear_i8(x, dw, dws, out)
            x.mul_(-3)
            g.replay()
            s.synchronize()
    finally:
        eng.set_stream(None)
    q, q_s = quantize(x.cpu().numpy(), None)
    check(out, q, q_s, w, w_s, None)


def test_refusals(eng):
    M, N, K = 4, 32, 48
    a, w, a_s, w_s, b = (dev(x) for x in make(M, N, K, 1))
    out = torch.empty(M, N, device="cuda")
    x = torch.zeros(M, K, device="cuda")
    with pytest.raises(ValueError):
        eng.matmul_i8(a, a_s, w[:, :47], w_s, out)          # depths differ
    with pytest.raises(ValueError):
        eng.matmul_i8(a.float(), a_s, w, w_s, out)          # not int8
    with pytest.raises(ValueError):
        eng.matmul_i8(a, a_s, w, w_s.half(), out)           # scales are float32
    with pytest.raises(ValueError):
        eng.matmul_i8(a, a_s, w, w_s, out.double())         # no such output type
    with pytest.raises(ValueError):
        eng.matmul_i8(a, a_s, w, w_s, out.cpu())            # not on the GPU
    with pytest.raises(ValueError):
        eng.matmul_i8(a, a_s, w, w_s, torch.empty(N, M, device="cuda").t())  # columns not contiguous
    with pytest.raises(AeError) as e:
        eng.matmul_i8(a[:1].expand(M, K), a_s, w, w_s, out)  # rows that lie over one another
    assert e.value.code == -1
    with pytest.raises(ValueError):
        eng.linear_i8(x.int(), w, w_s, out)
    with pytest.raises(ValueError):
        eng.linear_i8(x, w, w_s, out, inv_smooth=torch.ones(K + 1, device="cuda"))
    with pytest.raises(AeError) as e:
        eng.matmul_i8(torch.empty(1, 0, dtype=torch.int8, device="cuda"), a_s[:1],
                      torch.empty(N, 0, dtype=torch.int8, device="cuda"), w_s, out[:1])
    assert e.value.code == -1
    eng.sync()


def test_refusals_of_the_c_abi(eng):
    """Status -1 and a message, whatever the argument; nothing is launched."""
    from arctic_embed_s_int8 import _lib

    lib, h = _lib.lib(), eng.handle
    M, N, K = 4, 32, 48
    a, w, a_s, w_s, b = (dev(x) for x in make(M, N, K, 1))
    x, out = torch.zeros(M, K, device="cuda"), torch.full((M, N), 3.0, device="cuda")
    p = {"a": a.data_ptr(), "as": a_s.data_ptr(), "w": w.data_ptr(), "ws": w_s.data_ptr(), "b": b.data_ptr(),
         "o": out.data_ptr(), "x": x.data_ptr()}

    def matmul(M=M, N=N, K=K, a=p["a"], lda=K, a_s=p["as"], w=p["w"], ldw=K, w_s=p["ws"], b=p["b"], t=0, o=p["o"], ldo=N):
        return lib.ae_matmul_i8(h, M, N, K, a, lda, a_s, w, ldw, w_s, b, t, o, ldo)

    def linear(xt=0, x=p["x"], ldx=K, s=None, **kw):
        v = dict(M=M, N=N, K=K, w=p["w"], ldw=K, w_s=p["ws"], b=p["b"], t=0, o=p["o"], ldo=N) | kw
        return lib.ae_linear_i8(h, v["M"], v["N"], v["K"], xt, x, ldx, s, v["w"], v["ldw"], v["w_s"], v["b"], v["t"],
                                v["o"], v["ldo"])

    shared = [dict(N=0), dict(K=0), dict(K=131072, ldw=131072), dict(M=2 ** 30 + 1), dict(N=2 ** 30 + 1), dict(w=None),
              dict(w_s=None), dict(o=None), dict(t=3), dict(t=-1), dict(ldw=K - 1), dict(ldo=N - 1),
              dict(ldo=2 ** 39), dict(ldw=2 ** 39), dict(w_s=p["ws"] + 2), dict(b=p["b"] + 1), dict(o=p["o"] + 2)]
    launches = eng.kernel_launches()
    for kw in shared + [dict(a=None), dict(a_s=None), dict(lda=K - 1), dict(lda=2 ** 39), dict(a_s=p["as"] + 1)]:
        assert matmul(**({"lda": kw["K"]} if "K" in kw else {}) | kw) == -1, kw
        assert b"ae_matmul_i8" in lib.ae_last_error(h)
    for kw in shared + [dict(x=None), dict(xt=4), dict(ldx=K - 1), dict(ldx=2 ** 39), dict(x=p["x"] + 2),
                        dict(s=p["b"] + 2)]:
        assert linear(**({"ldx": kw["K"]} if "K" in kw else {}) | kw) == -1, kw
        assert b"ae_linear_i8" in lib.ae_last_error(h)
    assert matmul(M=0, a=None, a_s=None, o=None) == 0 and linear(M=0, x=None, o=None) == 0
    assert eng.kernel_launches() == launches
    eng.sync()
    assert (out == 3).all()
    assert matmul() == 0 and linear() == 0
    eng.sync()
