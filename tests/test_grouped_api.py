"""What the Python operators of the grouped products hand to the C functions, without a GPU."""
import ctypes

import numpy as np
import pytest
import torch

from ops_sparse_b200 import _lib as L
from ops_sparse_b200 import api


class Recorded(api._Grouped):
    """A product whose C functions note the scalars that they are given."""

    name = "product"

    def __init__(self, monkeypatch):
        self.seen = []

        class Lib:
            def __getattr__(lib, name):
                return self.take

        monkeypatch.setattr(L, "lib", Lib)
        self.buffer = torch.empty(64, dtype=torch.uint8)

    def _args(self, pa, pb):
        return pa, pb

    def take(self, pa, pb, last):
        self.seen.append(tuple(ctypes.cast(p, ctypes.POINTER(ctypes.c_float))[0] for p in (pa, pb)))
        return L.SUCCESS


@pytest.mark.parametrize("make", [lambda v: torch.tensor(v), lambda v: torch.tensor([v]), lambda v: np.full((), v)])
def test_a_scalar_that_changes_its_value_is_read_at_every_call(monkeypatch, make):
    op = Recorded(monkeypatch)
    beta = make(0.5)
    op(1.0, beta)
    beta[...] = 2.0
    op(1.0, beta)
    op(2, np.float32(0.25))
    op(True, 1)
    assert op.seen[-4:] == [(1.0, 0.5), (1.0, 2.0), (2.0, 0.25), (1.0, 1.0)]
