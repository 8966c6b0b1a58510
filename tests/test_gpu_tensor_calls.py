"""The general operators' calls next to autograd, which they take no part in."""
import pytest
import torch

from arctic_embed_s_int8 import Engine, rope_table

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    e = Engine(0)
    yield e
    e.close()


def test_results_written_over_saved_tensors_are_noticed(eng):
    """A backward pass that saved what a call has since written over raises, as after any operation in place."""
    M, N, K, D = 3, 32, 48, 32
    a, w = (torch.ones(n, K, dtype=torch.int8, device="cuda") for n in (M, N))
    s, ws, x = torch.ones(M, device="cuda"), torch.ones(N, device="cuda"), torch.ones(M, K, device="cuda")
    table, pos = torch.from_numpy(rope_table(8, D)).cuda(), torch.zeros(M, dtype=torch.int32, device="cuda")
    heads = torch.ones(M, 2, D, device="cuda")
    calls = {"matmul": lambda out: eng.matmul_i8(a, s, w, ws, out), "linear": lambda out: eng.linear_i8(x, w, ws, out),
             "q": lambda out: eng.qk_norm_rope(heads, heads, out, torch.empty_like(heads), table, positions=pos),
             "k": lambda out: eng.qk_norm_rope(heads, heads, torch.empty_like(heads), out, table, positions=pos)}
    for name, call in calls.items():
        out = torch.ones(M, 2, D, device="cuda") if name in "qk" else torch.ones(M, N, device="cuda")
        p = torch.ones_like(out, requires_grad=True)
        (p * out).sum().backward()
        loss = (p * out).sum()
        call(out)
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()
    eng.sync()


def test_parameters_under_no_grad_and_inference_mode(eng):
    M, N, K = 3, 32, 48
    w = torch.ones(N, K, dtype=torch.int8, device="cuda")
    ws = torch.nn.Parameter(torch.ones(N, device="cuda"))
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            x, out = torch.ones(M, K, device="cuda"), torch.zeros(M, N, device="cuda")
            eng.linear_i8(x, w, ws, out)
            eng.sync()
            # 127 steps of 1 / 127, K times: the quotient and the product of the scales are rounded once each
            assert (out - K).abs().max() <= 2 * K * 2.0 ** -24
