"""The norm and rotation of queries and keys (ae_qk_norm_rope) against its formula in 64 bits.

Tolerance, with u = 2^-24 and v the unit roundoff of the heads' type: a sum of at most 512 squares in which no
value passes more than 32 additions is off by at most 32 u of itself, its root by half that, and the root, the
quotient and the two products of y by u each: y is off by at most 24 u |y|. A rotated value adds two rounded
products: |error| <= 26 u (|y_i| + |y_j|) + v |out| (+ half the smallest float16 subnormal)."""
import numpy as np
import pytest
import torch

from arctic_embed_s_int8 import AeError, Engine, rope_table
from conftest import rng

pytestmark = pytest.mark.gpu

ROUNDOFF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TYPES = list(ROUNDOFF)
EPS = 1e-6


@pytest.fixture(scope="module")
def eng():
    e = Engine(0)
    yield e
    e.close()


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def wanted(x, weight, table, pos, neighbours, norm, eps=EPS):
    """(formula, sum of the magnitudes it adds), in float64. x [T, H, D]."""
    y = x.astype(np.float64)
    if norm:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * (1 if weight is None else weight.astype(np.float64))
    out, mag = y.copy(), np.abs(y)
    r = 0 if table is None else table.shape[1]
    if r:
        i = np.arange(r // 2)
        a, b = (2 * i, 2 * i + 1) if neighbours else (i, i + r // 2)
        c, s = (t.astype(np.float64)[pos][:, None] for t in (table[:, :r // 2], table[:, r // 2:]))
        out[..., a] = y[..., a] * c - y[..., b] * s
        out[..., b] = y[..., b] * c + y[..., a] * s
        mag[..., a] = mag[..., b] = np.abs(y[..., a]) + np.abs(y[..., b])
    return out, mag


def check(got, x, *how, **kw):
    want, mag = wanted(x.float().cpu().numpy(), *how, **kw)
    v = ROUNDOFF[got.dtype]
    tol = 26 * 2.0 ** -24 * mag + v * np.abs(want) + (2.0 ** -25 if got.dtype == torch.float16 else 0)
    g = got.double().cpu().numpy()
    bad = ~(np.abs(g - want) <= tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3], g[bad][:3], want[bad][:3])


def heads(T, H, D, dtype, seed):
    r = rng(seed)
    x = r.normal(0, 1, (T, H, D)) * np.exp(r.normal(0, 1, (T, H, 1)))
    return torch.from_numpy(x.astype(np.float32)).to(dtype).cuda()


def run(eng, T, Hq, Hk, D, R, dtype, seed, neighbours=False, norm=True, weights=True, cu=None, rows=300):
    q, k = heads(T, Hq, D, dtype, seed), heads(T, Hk, D, dtype, seed + 1)
    r = rng(seed + 2)
    qw, kw = ((1 + r.normal(0, 0.3, D)).astype(np.float32) for _ in range(2)) if weights else (None, None)
    table = rope_table(rows, R) if R else None
    d_cu = pos = d_pos = None
    if cu is not None:
        pos = np.concatenate([np.arange(b - a) for a, b in zip(cu[:-1], cu[1:])])
        d_cu = dev(np.asarray(cu, np.int32))
    else:
        pos = r.integers(0, rows, T).astype(np.int32)
        d_pos = dev(pos)
    qo, ko = (torch.full_like(x, float("nan")) for x in (q, k))
    eng.qk_norm_rope(q, k, qo, ko, None if table is None else dev(table), positions=d_pos, cu=d_cu,
                     q_weight=None if qw is None else dev(qw), k_weight=None if kw is None else dev(kw), eps=EPS,
                     neighbours=neighbours, norm=norm)
    eng.sync()
    check(qo, q, qw, table, pos, neighbours, norm)
    check(ko, k, kw, table, pos, neighbours, norm)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("D,R", [(32, 32), (64, 64), (128, 128), (256, 256), (512, 512), (128, 64), (80, 64), (96, 96),
                                 (80, 20), (64, 16), (112, 28), (33, 6), (1, 0), (2, 2), (100, 50), (128, 0), (511, 510),
                                 (6, 6), (40, 24)])
def test_dims(eng, dtype, neighbours, D, R):
    run(eng, 37, 5, 3, D, R, dtype, D + R, neighbours=neighbours)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,Hq,Hk", [(1, 32, 8), (1, 1, 1), (3, 12, 12), (1000, 1, 0), (257, 0, 2), (129, 40, 1),
                                     (2, 15, 5)])
def test_heads(eng, dtype, T, Hq, Hk):
    run(eng, T, Hq, Hk, 64, 64, dtype, T + Hq)
    run(eng, T, Hq, Hk, 128, 128, dtype, T + Hk)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("neighbours", [False, True])
def test_without_norm_or_weights(eng, dtype, neighbours):
    run(eng, 50, 4, 2, 64, 32, dtype, 1, neighbours=neighbours, norm=False)
    run(eng, 50, 4, 2, 64, 32, dtype, 2, neighbours=neighbours, weights=False)
    run(eng, 50, 4, 2, 36, 36, dtype, 3, neighbours=neighbours, norm=False, weights=False)


@pytest.mark.parametrize("cu", [[0, 1], [0, 0, 5, 5, 5, 130, 130], [0, 300], [0] + list(range(1, 200)),
                                [0, 0, 0, 64, 364, 365]])
def test_ragged_positions(eng, cu):
    run(eng, cu[-1], 12, 12, 32, 32, torch.float32, len(cu), cu=cu)
    run(eng, cu[-1], 2, 1, 96, 48, torch.bfloat16, len(cu), cu=cu)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,R", [(64, 64), (40, 20)])
@pytest.mark.parametrize("lead", [0, 1])
def test_packed_in_place(eng, dtype, D, R, lead):
    """Queries and keys rotated where a packed projection has them, at aligned and unaligned addresses; the
    values and everything around stay as they were."""
    T, Hq, Hk = 45, 6, 2
    width = (Hq + 2 * Hk) * D + 8
    x = heads(1, T, width, dtype, 9).view(-1)
    buf = torch.cat([x.new_zeros(lead), x])[lead:].view(T, width)
    before = buf.clone()
    q, k = buf[:, :Hq * D].view(T, Hq, D), buf[:, Hq * D:(Hq + Hk) * D].view(T, Hk, D)
    q0, k0 = q.clone(), k.clone()
    table, pos = rope_table(60, R), rng(2).integers(0, 60, T).astype(np.int32)
    eng.qk_norm_rope(q, k, q, k, dev(table), positions=dev(pos))
    eng.sync()
    check(q, q0, None, table, pos, False, True, eps=1e-6)
    check(k, k0, None, table, pos, False, True, eps=1e-6)
    assert torch.equal(buf[:, (Hq + Hk) * D:], before[:, (Hq + Hk) * D:])


@pytest.mark.parametrize("D", [64, 50])
def test_head_major_strides(eng, D):
    """[heads, tokens, dim] in and [tokens, heads, dim] out."""
    T, H = 33, 4
    base, table = heads(H, T, D, torch.bfloat16, 4), rope_table(40, D)
    q, pos = base.transpose(0, 1), np.arange(T, dtype=np.int32)
    out, k = torch.empty(T, H, D, dtype=torch.bfloat16, device="cuda"), base.new_empty(T, 0, D)
    eng.qk_norm_rope(q, k, out, k, dev(table), positions=dev(pos))
    eng.sync()
    check(out, q, None, table, pos, False, True, eps=1e-6)


def test_special_values(eng):
    """A head of zeros stays zero; an infinity makes its own value NaN and the others of its head zero, as the
    formula has it; a NaN stays in its head."""
    T, H, D = 4, 2, 64
    x = heads(T, H, D, torch.float32, 7)
    x[0, 0], x[1, 1, 5], x[2, 0, 9] = 0, float("inf"), float("nan")
    table = rope_table(8, 32)
    out, k = torch.empty_like(x), x.new_empty(T, 0, D)
    pos = np.zeros(T, np.int32)  # angle 0: the rotation keeps every value
    eng.qk_norm_rope(x, k, out, k, dev(table), positions=dev(pos))
    eng.sync()
    got = out.cpu().numpy()
    assert (got[0, 0] == 0).all()
    assert np.isnan(got[1, 1, 5]) and (np.delete(got[1, 1], [5, 21]) == 0).all()
    assert np.isnan(got[2, 0]).all()
    rest = [(0, 1), (1, 0), (2, 1), (3, 0), (3, 1)]
    for t, h in rest:
        check(out[t:t + 1, h:h + 1], x[t:t + 1, h:h + 1], None, table, pos[:1], False, True)


@pytest.mark.parametrize("D,R", [(64, 64), (36, 36)])
@pytest.mark.parametrize("by_cu", [False, True])
def test_position_outside_the_table(eng, D, R, by_cu):
    """Reported by the next synchronisation; those tokens are left alone, the others done."""
    T, rows = 30, 10
    x = heads(T, 3, D, torch.float32, 1)
    out, k = torch.full_like(x, 5.0), x.new_empty(T, 0, D)
    pos = np.arange(T) % 10
    how = {}
    if by_cu:
        how["cu"] = dev(np.array([0, 10, 22, 28], np.int32))  # rows 20 and 21 at 10 and 11; 28 and 29 in none
        pos = np.array([*range(10), *range(12), *range(6), 0, 0])
        bad = [20, 21, 28, 29]
    else:
        pos[[3, 17]] = -1, rows
        how["positions"] = dev(pos.astype(np.int32))
        bad = [3, 17]
    eng.qk_norm_rope(x, k, out, k, dev(rope_table(rows, R)), **how)
    with pytest.raises(AeError) as e:
        eng.sync()
    assert e.value.code == -6 and "position" in str(e.value)
    eng.sync()  # reported once; the engine stays usable
    good = np.setdiff1d(np.arange(T), bad)
    assert (out[bad] == 5).all()
    check(out[good], x[good], None, rope_table(rows, R), pos[good], False, True)


def test_long_strides(eng):
    """Element offsets beyond 32 bits."""
    D, T = 64, 3
    buf = torch.zeros(2 ** 31 + 4096, dtype=torch.float16, device="cuda")
    x = buf.as_strided((T, 1, D), (2 ** 30, D, 1))
    x.copy_(heads(T, 1, D, torch.float16, 3))
    out, k = torch.empty(T, 1, D, dtype=torch.float16, device="cuda"), buf.new_empty(T, 0, D)
    table, pos = rope_table(4, D), np.arange(T, dtype=np.int32)
    eng.qk_norm_rope(x, k, out, k, dev(table), positions=dev(pos))
    eng.sync()
    check(out, x, None, table, pos, False, True)


def test_refusals(eng):
    T, D = 4, 32
    q, k = heads(T, 2, D, torch.float32, 1), heads(T, 1, D, torch.float32, 2)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    table, pos = dev(rope_table(8, D)), torch.zeros(T, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        eng.qk_norm_rope(q, k, qo, ko, table)                                # no positions
    with pytest.raises(ValueError):
        eng.qk_norm_rope(q, k, qo, ko, table, positions=pos.long())
    with pytest.raises(ValueError):
        eng.qk_norm_rope(q, k.half(), qo, ko, table, positions=pos)          # types differ
    with pytest.raises(ValueError):
        eng.qk_norm_rope(q, k, qo[:3], ko, table, positions=pos)
    with pytest.raises(ValueError):
        eng.qk_norm_rope(q, k, qo, ko, table, positions=pos, q_weight=torch.ones(D + 1, device="cuda"))
    with pytest.raises(ValueError):
        eng.qk_norm_rope(q, k, qo, ko, table[:, ::2], positions=pos)
    with pytest.raises(AeError) as e:
        eng.qk_norm_rope(q, k, qo, ko, dev(rope_table(8, D + 2)), positions=pos)  # rotates more than the head
    assert e.value.code == -1
    with pytest.raises(AeError) as e:
        eng.qk_norm_rope(q, k, qo, ko, table, positions=pos, eps=-1.0)
    assert e.value.code == -1
    wide = heads(T, 2, 514, torch.float32, 1)
    with pytest.raises(AeError) as e:
        eng.qk_norm_rope(wide, wide, torch.empty_like(wide), torch.empty_like(wide))
    assert e.value.code == -1
    eng.sync()


def test_no_tokens(eng):
    for T, Hq, Hk in ((0, 2, 1), (3, 0, 0)):
        q, k = torch.empty(T, Hq, 32, device="cuda"), torch.empty(T, Hk, 32, device="cuda")
        eng.qk_norm_rope(q, k, q, k, dev(rope_table(8, 32)), positions=torch.zeros(T, dtype=torch.int32, device="cuda"))
    eng.sync()


def test_refusals_of_the_c_abi(eng):
    """Status -1 and a message, whatever the argument; nothing is launched."""
    from arctic_embed_s_int8 import _lib

    lib, h, T, D = _lib.lib(), eng.handle, 4, 32
    x, table = torch.full((T, 2, D), 3.0, device="cuda"), dev(rope_table(8, D))
    pos = torch.zeros(T, dtype=torch.int32, device="cuda")
    P, S = x.data_ptr(), (2 * D, D)

    def call(type=0, T=T, Hq=1, Hk=1, D=D, R=D, flags=0, q=(P, *S), k=(P + 4 * D, *S), qo=(P, *S), ko=(P + 4 * D, *S),
             qw=None, kw=None, eps=1e-6, table=table.data_ptr(), rows=8, pos=pos.data_ptr(), cu=None, n=0):
        return lib.ae_qk_norm_rope(h, type, T, Hq, Hk, D, R, flags, *q, *k, *qo, *ko, qw, kw, eps, table, rows, pos, cu, n)

    launches = eng.kernel_launches()
    null = (None, *S)
    for kw in (dict(type=3), dict(type=-1), dict(flags=4), dict(D=0, R=0), dict(D=513, R=0), dict(R=34), dict(R=31),
               dict(Hq=65536), dict(T=2 ** 30 + 1), dict(eps=-1.0), dict(eps=float("nan")), dict(q=null), dict(k=null),
               dict(qo=null), dict(ko=null), dict(table=None), dict(rows=0), dict(pos=None), dict(rows=2 ** 31),
               dict(pos=None, cu=pos.data_ptr(), n=0), dict(q=(P + 2, *S)), dict(qw=P + 1), dict(pos=pos.data_ptr() + 2),
               dict(k=(P, 2 ** 32, D))):
        assert call(**kw) == -1, kw
        assert b"ae_qk_norm_rope" in lib.ae_last_error(h)
    assert call(T=0, q=null, k=null, qo=null, ko=null, pos=None) == 0
    assert call(Hq=0, Hk=0) == 0
    assert eng.kernel_launches() == launches
    eng.sync()
    assert (x == 3).all()
    assert call() == 0
    eng.sync()
