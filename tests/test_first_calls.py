"""The first call of a process, which is the first to need torch: each in a
process of its own, refused before any device work."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CALLS = ["grouped_linear(t, t)", "grouped_linear_grad(t)", "expert_layer(t, t, t, t, t)", "distill_loss(t, t, t, t)",
         "distill_loss_grad(t, t, t, t, t)", "grouped_matmul(t, t)", "block8_pack(t)"]

LEAF = """
import torch
import proxima_amd as px


class Leaf:  # of a float64 leaf on a GPU, what is looked at before anything runs
    is_cuda, requires_grad, dtype, shape = True, True, torch.float64, torch.Size((4, 8))

    def get_device(self):
        return 0

    def stride(self, d=None):
        return (8, 1) if d is None else (8, 1)[d]

    def dim(self):
        return 2


t = Leaf()
with torch.set_grad_enabled(GRAD):
    try:
        px.CALL
    except ValueError as e:
        print(e)
"""


def _fresh(source):
    run = subprocess.run([sys.executable, "-c", source], capture_output=True, text=True, cwd=ROOT)
    assert run.returncode == 0, run.stderr
    return run.stdout


@pytest.mark.parametrize("call", CALLS)
def test_the_first_call_may_have_an_operand_that_requires_grad(call):
    source = LEAF.replace("CALL", call)
    # in grad mode it is refused for that (products and packing look at the type first), without it for its type
    assert ("requires grad" if CALLS.index(call) < 5 else "must be") in _fresh(source.replace("GRAD", "True"))
    assert "must be" in _fresh(source.replace("GRAD", "False"))


@pytest.mark.parametrize("call", ["block8_unpack(p)", "block8_matmul(p, p)", "block8_linear(p, p)"])
def test_packed_rows_from_another_process_may_come_first(call):
    # unpickled ones are made without Block8's constructor
    assert "must be on one device" in _fresh("""
import torch
from proxima_amd import experts


class Elsewhere:
    def get_device(self):
        return 5

    def data_ptr(self):
        return 4096


p = experts.Block8.__new__(experts.Block8)
p._codes, p._scales, p._cols = torch.zeros(4, 128, dtype=torch.uint8), Elsewhere(), 100
try:
    experts.CALL
except ValueError as e:
    print(e)
""".replace("CALL", call))


def test_two_first_calls_at_once():
    # what tells another thread that all is filled is filled last
    assert _fresh("""
import sys, torch
from proxima_amd import experts

seen = []


class Watched:
    def __getattr__(self, name):
        seen.append(experts._torch)
        return getattr(torch, name)


sys.modules["torch"] = Watched()
experts._setup()
print(len(seen) > 0 and not any(seen), experts._torch is sys.modules["torch"])
""") == "True True\n"
