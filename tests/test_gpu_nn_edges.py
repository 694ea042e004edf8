"""``cp.nn`` at the limits of its plans and arguments, against plain NumPy in
64 bits."""
import numpy as np
import pytest

import macmetalpy_amd as cp
from macmetalpy_amd import nn

pytestmark = pytest.mark.gpu


def _sums(tok, grad, rows):
    """Sums of whole numbers by token, exact in any order."""
    want = np.zeros((rows, grad.shape[1]), np.float32)
    keep = (tok >= 0) & (tok < rows)
    np.add.at(want, tok[keep], grad[keep].astype(np.float32))
    return want


# ------------------------------------------------------------- embedding
@pytest.mark.parametrize("rows", [1 << 24, (1 << 24) + 1, (1 << 24) + 5, (1 << 25) + 3])
def test_embedding_grad_rows_beyond_24_bits(rows):
    """Rows that differ only in their bits from 24 on, the first and the last."""
    g = np.random.default_rng(rows)
    tok = g.integers(0, rows, 700)
    tok[:8] = [0, rows - 1, rows, -1, 5, min(rows - 1, (1 << 24) + 5 - 4), 1, rows - 1]
    tok[8:300] = g.integers(0, 3, 292) + (rows - 3)
    tok[300:400] = g.integers(0, 5, 100)
    grad = g.integers(-8, 9, (700, 1)).astype(np.float16)
    got = nn.embedding_grad(cp.array(grad), cp.array(tok), rows).get()
    assert np.array_equal(got.astype(np.float32), _sums(tok, grad, rows))
