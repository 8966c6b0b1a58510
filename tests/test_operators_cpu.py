"""The general operators without a GPU: null contexts, the rotation table, and the tensor checks that come before
any call."""
import numpy as np
import pytest
import torch

from arctic_embed_s_int8 import _lib, rope_table


def test_null_context_is_refused():
    lib = _lib.lib()
    assert lib.ae_matmul_i8(None, 1, 1, 1, None, 1, None, None, 1, None, None, 0, None, 1) == -1
    assert lib.ae_linear_i8(None, 1, 1, 1, 0, None, 1, None, None, 1, None, None, 0, None, 1) == -1
    assert lib.ae_qk_norm_rope(None, 0, 1, 1, 1, 32, 32, 0, *[None, 0, 0] * 4, None, None, 1e-6, None, 0, None, None,
                               0) == -1


@pytest.mark.parametrize("rows,dim,base", [(1, 2, 1e4), (512, 32, 1e4), (300, 128, 5e5)])
def test_rope_table(rows, dim, base):
    t = rope_table(rows, dim, base)
    assert t.shape == (rows, dim) and t.dtype == np.float32
    p, i = rows - 1, dim // 2 - 1
    angle = p / base ** (2 * i / dim)
    # float64 angles up to `rows` are off by at most rows * 2^-52, the entries by half a float32 unit more
    assert abs(t[p, i] - np.cos(angle)) <= 2.0 ** -24 + rows * 2.0 ** -50
    assert abs(t[p, dim // 2 + i] - np.sin(angle)) <= 2.0 ** -24 + rows * 2.0 ** -50
    np.testing.assert_array_equal(t[0], [1.0] * (dim // 2) + [0.0] * (dim // 2))


def test_tensors_are_checked_before_any_call():
    m = _lib.tensors()
    a, w, s = torch.zeros(2, 8, dtype=torch.int8), torch.zeros(4, 8, dtype=torch.int8), torch.zeros(2)
    good = [0, 0, a, s, w, torch.zeros(4), torch.zeros(2, 4), None]

    def refused(call, args, word):
        with pytest.raises(ValueError, match=word):
            call(*args)

    refused(m.matmul_i8, good, "device memory")                      # host tensors
    refused(m.matmul_i8, [*good[:2], None, *good[3:]], "torch tensor")
    refused(m.matmul_i8, [*good[:2], a[0], *good[3:]], "tokens, in_features")
    refused(m.matmul_i8, [*good[:4], w[0], *good[5:]], "out_features, in_features")
    refused(m.linear_i8, [0, 0, torch.zeros(2, 8), None, *good[4:]], "device memory")
    with pytest.raises(TypeError):
        m.matmul_i8(*good[:-1])
    q = torch.zeros(3, 2, 8)
    refused(m.qk_norm_rope, [0, 0, q.double(), q, q, q, None, None, None, None, None, 1e-6, 0], "float32")
    refused(m.qk_norm_rope, [0, 0, q, q[0], q, q, None, None, None, None, None, 1e-6, 0], "tokens, heads, dim")
