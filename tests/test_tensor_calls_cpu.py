"""The general operators' calls on torch tensors that hold no memory of a GPU, or not what their address says."""
import os
import subprocess
import sys

import pytest

from conftest import PKG, ROOT

# Tensors of cuda:0 without a GPU: `plain` ones have the address 0, which the C ABI would refuse (as it does the null context),
# and those in a batch, as torch.func.vmap passes them, have none and throw when asked for it.
HOLLOW = """
import torch
from torch._C._functorch import _add_batch_dim
from arctic_embed_s_int8 import _lib

class Hollow(torch.Tensor):
    @staticmethod
    def __new__(cls, *size, dtype=torch.float32):
        return torch.Tensor._make_wrapper_subclass(cls, size, dtype=dtype, device="cuda:0")

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise NotImplementedError(str(func))

def batched(*size, dtype=torch.float32):
    return _add_batch_dim(Hollow(3, *size, dtype=dtype), 0, 1)

m = _lib.tensors()
"""


def run(lines: str) -> str:
    """What a process of its own prints."""
    r = subprocess.run([sys.executable, "-c", HOLLOW + lines], capture_output=True, text=True, cwd=ROOT,
                       env={**os.environ, "PYTHONPATH": PKG})
    assert r.returncode == 0, (r.returncode, r.stdout, r.stderr[-500:])
    return r.stdout


@pytest.mark.parametrize("call,args", [
    ("matmul_i8", ["Hollow(2, 8, dtype=i8)", "Hollow(2)", "Hollow(4, 8, dtype=i8)", "Hollow(4)", "Hollow(2, 4)", "None"]),
    ("linear_i8", ["Hollow(2, 8)", "Hollow(8)", "Hollow(4, 8, dtype=i8)", "Hollow(4)", "Hollow(2, 4)", "Hollow(4)"]),
    ("qk_norm_rope", ["Hollow(2, 3, 8)", "Hollow(2, 1, 8)", "Hollow(2, 3, 8)", "Hollow(2, 1, 8)", "Hollow(5, 4)",
                      "Hollow(2, dtype=torch.int32)", "None", "Hollow(8)", "Hollow(8)", "1e-6", "0"])])
def test_tensors_without_an_address_raise(call, args):
    """Whichever operand it is, and with the interpreter's lock held (the process ends otherwise)."""
    lines = f"i8 = torch.int8\nassert m.{call}(0, 0, {', '.join(args)}) == -1\n"
    for i, a in enumerate(args):
        if "Hollow" not in a:
            continue
        one = [*args[:i], a.replace("Hollow", "batched"), *args[i + 1:]]
        lines += f"try:\n    m.{call}(0, 0, {', '.join(one)})\nexcept RuntimeError as e:\n    print('storage' in str(e))\n"
    assert run(lines).split() == ["True"] * sum("Hollow" in a for a in args)


def test_gradients_are_not_dropped():
    """The calls compute none: a float operand or result that requires one is refused while gradients are recorded, whichever
    it is, and taken under no_grad."""
    operands = {
        "matmul_i8": ["Hollow(2, 8, dtype=i8)", "grad(2)", "Hollow(4, 8, dtype=i8)", "grad(4)", "grad(2, 4)", "grad(4)"],
        "linear_i8": ["grad(2, 8)", "grad(8)", "Hollow(4, 8, dtype=i8)", "grad(4)", "grad(2, 4)", "grad(4)"],
        "qk_norm_rope": ["grad(2, 3, 8)", "grad(2, 1, 8)", "grad(2, 3, 8)", "grad(2, 1, 8)", "grad(5, 4)",
                         "Hollow(2, dtype=torch.int32)", "None", "grad(8)", "grad(8)", "1e-6", "0"]}
    lines = "i8 = torch.int8\ndef grad(*size): return Hollow(*size).requires_grad_()\n"
    count = 0
    for call, args in operands.items():
        for i, a in enumerate(args):
            if "grad" in a:
                one = [x.replace("grad", "Hollow") if j != i else x for j, x in enumerate(args)]
                count += 1
                lines += (f"args = [0, 0, {', '.join(one)}]\ntry:\n    m.{call}(*args)\nexcept ValueError as e:\n"
                          f"    print('requires grad' in str(e))\nwith torch.no_grad():\n    assert m.{call}(*args) == -1\n")
    assert run(lines).split() == ["True"] * count


def test_tensors_that_stand_for_their_negatives_are_refused():
    """A lazily negated view (the imaginary part of a conjugate) holds the negatives of its values."""
    import torch

    from arctic_embed_s_int8 import _lib

    z = torch.ones(4, 1, dtype=torch.complex64)
    x = z.conj().imag
    assert x.is_neg()
    m, w = _lib.tensors(), torch.zeros(3, 1, dtype=torch.int8)
    with pytest.raises(ValueError, match="resolve_neg"):
        m.linear_i8(0, 0, x, None, w, torch.zeros(3), torch.zeros(4, 3), None)
    with pytest.raises(ValueError, match="device memory"):  # as it is refused for being on the host otherwise
        m.linear_i8(0, 0, x.resolve_neg(), None, w, torch.zeros(3), torch.zeros(4, 3), None)


def test_a_closed_engine_is_refused_as_everywhere():
    """AeError, as the engine's other calls raise it."""
    lines = """
from arctic_embed_s_int8 import AeError, Engine
e = Engine.__new__(Engine)
e._h, e.device, i8 = None, 0, torch.int8
h, w = Hollow(2, 1, 8), Hollow(4, 8, dtype=i8)
for call in (lambda: e.sync(), lambda: e.matmul_i8(Hollow(2, 8, dtype=i8), Hollow(2), w, Hollow(4), Hollow(2, 4)),
             lambda: e.linear_i8(Hollow(2, 8), w, Hollow(4), Hollow(2, 4)), lambda: e.qk_norm_rope(h, h, h, h)):
    try:
        call()
    except AeError as x:
        print(x.code)
"""
    assert run(lines).split() == ["-1"] * 4
