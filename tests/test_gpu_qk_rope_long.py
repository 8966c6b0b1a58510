"""The norm and rotation of batches long enough for four heads to a thread (from 256 threads an SM on), which
test_gpu_qk_rope.py's sizes stay below: against the same formula in 64 bits with the same tolerance."""
import numpy as np
import pytest
import torch

from arctic_embed_s_int8 import AeError, Engine, rope_table
from conftest import rng
from test_gpu_qk_rope import TYPES, check, dev, heads, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    e = Engine(0)
    yield e
    e.close()


def tokens(Hq, Hk, D, piece, more=3):
    """Tokens for 256 threads on each of 148 SMs with pieces of `piece` elements, and some more."""
    return -(-256 * 148 // ((-(-Hq // 4) - (-Hk // 4)) * (D // (2 * piece)))) + more


def piece(dtype, D, R):
    """The largest piece that divides both halves of a head and of its rotated dims."""
    most = 4 if dtype == torch.float32 else 8
    return next(p for p in (most, most // 2, most // 4) if D % (2 * p) == 0 and R % (2 * p) == 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("D,R", [(32, 32), (64, 64), (128, 128), (256, 64), (128, 0), (80, 64), (96, 48), (40, 24), (36, 20),
                                 (20, 4), (112, 28)])
def test_dims(eng, dtype, neighbours, D, R):
    T = tokens(5, 3, D, piece(dtype, D, R))
    run(eng, T, 5, 3, D, R, dtype, D + R, neighbours=neighbours, rows=T)


@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("D,R", [(6, 6), (2, 2), (10, 6), (62, 30)])
def test_single_values(eng, neighbours, D, R):
    """Halves of an odd count of floats: pieces of one value."""
    run(eng, tokens(5, 3, D, 1), 5, 3, D, R, torch.float32, D + R, neighbours=neighbours)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (2, 1), (3, 0), (0, 6), (4, 4), (7, 2), (9, 8), (15, 5), (32, 8), (41, 1)])
def test_heads(eng, dtype, Hq, Hk):
    """Last groups of one to four heads."""
    run(eng, tokens(Hq, Hk, 64, 4 if dtype == torch.float32 else 8), Hq, Hk, 64, 64, dtype, Hq * 50 + Hk)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("neighbours", [False, True])
def test_without_norm_or_weights(eng, dtype, neighbours):
    T = tokens(6, 3, 64, 4 if dtype == torch.float32 else 8)
    run(eng, T, 6, 3, 64, 32, dtype, 1, neighbours=neighbours, norm=False)
    run(eng, T, 6, 3, 64, 64, dtype, 2, neighbours=neighbours, weights=False)


@pytest.mark.parametrize("kind", ["one", "short", "mixed", "empty"])
@pytest.mark.parametrize("dtype,Hq,Hk,D", [(torch.float32, 12, 12, 32), (torch.bfloat16, 7, 2, 96), (torch.float16, 3, 1, 256)])
def test_ragged_positions(eng, kind, dtype, Hq, Hk, D):
    """Places counted from cu: blocks that hold many sequences' tokens, few, or parts of one."""
    T, r = tokens(Hq, Hk, D, 4 if dtype == torch.float32 else 8), rng(4)
    if kind == "one":
        cu = [0, T]
    elif kind == "short":
        cu = [*range(0, T, 2), T]
    elif kind == "mixed":
        cu = sorted([0, T, *r.integers(0, T, 60).tolist()])
    else:
        cu = sorted([0, 0, T, T, T, *([T // 2] * 90), *r.integers(0, T, 1100).tolist()])
    run(eng, T, Hq, Hk, D, D // 2, dtype, D, cu=cu, rows=T)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,R,lead", [(64, 64, 0), (64, 64, 1), (40, 24, 0), (40, 24, 2)])
def test_packed_in_place(eng, dtype, D, R, lead):
    """Where a packed projection has them, at addresses that lie on whole pieces, on smaller ones, or on none."""
    Hq, Hk = 6, 2
    T, width = tokens(Hq, Hk, D, 1), (Hq + 2 * Hk) * D + 8
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


def test_head_major_strides(eng):
    """[heads, tokens, dim] in and [tokens, heads, dim] out."""
    D, H = 64, 6
    T = tokens(H, 0, D, 8)
    base, table = heads(H, T, D, torch.bfloat16, 4), rope_table(T, D)
    q, pos = base.transpose(0, 1), np.arange(T, dtype=np.int32)
    out, k = torch.empty(T, H, D, dtype=torch.bfloat16, device="cuda"), base.new_empty(T, 0, D)
    eng.qk_norm_rope(q, k, out, k, dev(table), positions=dev(pos))
    eng.sync()
    check(out, q, None, table, pos, False, True, eps=1e-6)


def test_special_values(eng):
    """An infinity or a NaN stays in its head, beside others of the same thread and token."""
    D, H = 64, 7
    T = tokens(H, 0, D, 4)
    x = heads(T, H, D, torch.float32, 7)
    x[5, 0], x[5, 1, 5], x[5, 2, 9], x[T - 1, 6, 40] = 0, float("inf"), float("nan"), -float("inf")
    table, pos = rope_table(8, 32), np.zeros(T, np.int32)
    out, k = torch.empty_like(x), x.new_empty(T, 0, D)
    eng.qk_norm_rope(x, k, out, k, dev(table), positions=dev(pos))
    eng.sync()
    got = out.cpu().numpy()
    assert (got[5, 0] == 0).all() and np.isnan(got[5, 2]).all()
    assert np.isnan(got[5, 1, 5]) and (np.delete(got[5, 1], [5, 21]) == 0).all()
    assert np.isnan(got[T - 1, 6, 40]) and (np.delete(got[T - 1, 6], 40) == 0).all()
    rest = np.ones((T, H), bool)
    rest[5, :3] = rest[T - 1, 6] = False
    assert np.isfinite(got[rest]).all()
    check(out[5:6, 3:], x[5:6, 3:], None, table, pos[:1], False, True)


@pytest.mark.parametrize("by_cu", [False, True])
def test_position_outside_the_table(eng, by_cu):
    """Reported by the next synchronisation; those tokens are left alone, the others done."""
    D, Hq, Hk, rows = 64, 5, 3, 50
    T = tokens(Hq, Hk, D, 4)
    q, k = heads(T, Hq, D, torch.float32, 1), heads(T, Hk, D, torch.float32, 2)
    qo, ko = torch.full_like(q, 5.0), torch.full_like(k, 5.0)
    bad = np.zeros(T, bool)
    if by_cu:
        cu = np.array([2, *range(40, T - 60, 40), T - 1], np.int32)  # tokens 0, 1 and T - 1 in none, the last over the table
        pos = np.arange(T) - cu[np.maximum(np.searchsorted(cu, np.arange(T), side="right") - 1, 0)]
        bad[[0, 1, T - 1]] = True
        bad |= pos >= rows
        how = {"cu": dev(cu)}
    else:
        pos = rng(3).integers(0, rows, T).astype(np.int32)
        pos[[0, 77, T - 1]] = -1, rows, 2 ** 31 - 1
        bad = (pos < 0) | (pos >= rows)
        how = {"positions": dev(pos)}
    eng.qk_norm_rope(q, k, qo, ko, dev(rope_table(rows, D)), **how)
    with pytest.raises(AeError) as e:
        eng.sync()
    assert e.value.code == -6 and "position" in str(e.value)
    eng.sync()
    for x, out in ((q, qo), (k, ko)):
        assert (out[bad] == 5).all()
        check(out[~bad], x[~bad], None, rope_table(rows, D), pos[~bad], False, True)
