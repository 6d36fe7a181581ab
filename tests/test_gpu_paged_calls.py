"""How the paged cache is called from Python: what is refused, whose workspace a call uses, what a table's
shape lets the kernels read.  The numbers are held to oracle/paged_ref.py as in test_gpu_paged.py."""
import math
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_gpu_paged import BF16, F16, F32, Case, paged  # noqa: E402,F401

from oracle import paged_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu


def test_tables_on_another_device_are_refused(paged, kq):  # noqa: F811
    """A batch's or a rotary table's pointers go to a kernel on the cache's device."""
    c = Case(paged, [2], [20], 4, 2, 64, F32, F32, 16, seed=30)
    rope = paged.Rope.make(32, 64)
    c.cache.append(1, c.batch, c.q, c.nk, c.nv, rope=rope)
    rope.device = torch.device("cuda", 1)   # as one made there has it
    with pytest.raises(ValueError, match="rotary"):
        c.cache.append(1, c.batch, c.q, c.nk, c.nv, rope=rope)
    c.batch.device = torch.device("cuda", 1)
    with pytest.raises(ValueError, match="batch"):
        c.cache.append(1, c.batch, c.q, c.nk, c.nv)
    with pytest.raises(ValueError, match="batch"):
        c.cache.attend(1, c.batch, c.q)
