"""Microscaled 4-bit operators where they can go wrong: alignment, ranges, padding, derivatives other than the
plain gradient, saved state.  Values against the definition in float64 (tests/mx4_oracle.py)."""
import numpy as np
import pytest
import torch

import mx4_oracle as mo
from perm_b200 import _native as nat
from perm_b200 import mx4
from test_mx4_gpu import DTYPES, FMTS, HALF, chain, check_operand, check_product, f64, make_x, operand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 3, 8, 16])
def test_few_tokens_at_every_alignment_of_x(fmt, dtype, T):
    """x starts anywhere its type may, and its rows end inside a group of 256 columns: the asynchronous copies
    take 16-byte sources only."""
    dt = DTYPES[dtype]
    for n in (200, 248, 520):
        w, wv = operand(130, n, fmt, n)
        base = make_x(T + 1, n + 9, n, dt, 0.5).reshape(-1)
        for at in range(1, 9):
            x = base[at:at + T * n].view(T, n)
            check_product(mx4.linear(x, w), f64(x), wv, dt)
            x = base[at:at + T * (n + 3)].view(T, n + 3)[:, :n]
            check_product(mx4.linear(x, w), f64(x), wv, dt)
    mx4.status()
