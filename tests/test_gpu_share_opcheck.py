"""torch.library.opcheck of the operators on shared pages: their schemas name what
they change, and their fake implementations give what they return."""
import importlib

import numpy as np
import pytest
import torch

from _gpu import up

pytestmark = pytest.mark.gpu

ops = importlib.import_module("cuda-operators_amd.torch_ops") and torch.ops.kvq
TESTS = ("test_schema", "test_faketensor")


def state():
    st = {"lengths": [20, 5, 0], "block_table": [[3, 4], [6, 0], [0, 0]], "shares": [0] * 8, "free_pages": [7, 5, 2, 1, 0] + [0] * 3,
          "free_count": [5]}
    return [up(np.asarray(x, np.int32)) for x in st.values()]


def i32(*x):
    return up(np.asarray(x, np.int32))


@pytest.mark.parametrize("keep", [None, (20, 18, 1 << 30)])
def test_page_fork(keep):
    torch.library.opcheck(ops.page_fork, (i32(0, 0, 1), None if keep is None else i32(*keep), *state(), 16), test_utils=TESTS)


@pytest.mark.parametrize("layers", [None, 2])
@pytest.mark.parametrize("bounds", [False, True])
def test_page_copy(layers, bounds):
    lead = (8,) if layers is None else (layers, 8)
    code = lambda *s: torch.randint(-127, 128, lead + s, dtype=torch.int8, device="cuda")  # noqa: E731
    pool = [code(1, 16, 32), code(1, 16, 32), torch.rand((*lead, 1, 16), device="cuda"), torch.rand((*lead, 1, 16), device="cuda")]
    more = [code(1, 2, 32), torch.rand((*lead, 1), device="cuda")] if bounds else [None, None]
    torch.library.opcheck(ops.page_copy, (i32(3, -1), i32(5, -1), *pool, *more), test_utils=TESTS)


@pytest.mark.parametrize("shares", [True, False])
def test_page_compact(shares):
    lengths, table, s, free, count = state()
    torch.library.opcheck(ops.page_compact, (lengths, table, s if shares else None, free, count, 16, 4), test_utils=TESTS)
