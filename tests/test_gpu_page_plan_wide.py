"""kv_page_plan from 32768 tokens on, where a thread takes four neighbours: against the plan made token by token."""
import numpy as np
import pytest
import torch

from test_gpu_serving_ops import check_plan

pytestmark = pytest.mark.gpu
WIDE = 32768


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from wfamd import _lib
    assert _lib.kernel_available(), "gfx950 kernels must load (no fallback)"
    torch.cuda.set_device(0)


@pytest.mark.parametrize("page", [1, 32, 33, 64])
@pytest.mark.parametrize("batch,kind", [(3, "long"), (200, "ragged"), (1999, "mixed"), (2048, "mixed"), (2049, "mixed"), (4001, "ragged")])
def test_four_tokens_a_thread(batch, kind, page):
    rng = np.random.default_rng(batch + page)
    if kind == "long":
        new = np.array([20001, 0, 15011])
    elif kind == "ragged":
        new = rng.integers(0, 2 * 45000 // batch, batch)
    else:  # four neighbours of several sequences: mostly 0 to 3 new tokens, a few long ones among them
        new = rng.integers(0, 4, batch)
        new[rng.integers(0, batch, 12)] = 3001
    n = int(new.sum())
    assert n >= WIDE + 4
    cached = rng.integers(0, 100, batch)
    cols = -(-int((cached + new).max()) // page)
    need = -(-(cached + new) // page) - -(-cached // page)
    free, table = rng.permutation(int(need.sum()) + 5), rng.integers(0, 10 ** 6, (batch, cols))
    for tokens in (n, n - 1, n - 2, n - 3, n + 5):  # all that four leave over; fewer tokens than there are, and more
        check_plan(cached, new, free, table, tokens, page)
    # refused in the middle: rows too short for the long ones, and a free list that ends on the way
    short = max(1, cols // 2)
    check_plan(cached, new, free, table[:, :short], n, page)
    check_plan(cached, new, free[: len(free) // 2], table, n + 2, page)
