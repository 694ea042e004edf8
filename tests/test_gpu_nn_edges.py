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


# ------------------------------------------------------------------ norm
def test_clip_refuses_outputs_that_overlap():
    """An output on another array's memory, or on a part of its own, would be
    scaled once or twice; arrays that only touch are others."""
    h = np.arange(1, 41, dtype=np.float32)
    a, b = cp.array(h), cp.array(h + 1)
    bad = [([a, a], [a, a]),                     # tied weights' gradients
           ([a, b], [b, a]),                     # two arrays that change places
           ([a[:15], b[:15]], [a[20:35], a[25:40]]),
           ([a[:20]], [a[1:21]]),                # a part of its own
           ([a[:20], b[:20]], [a[:20], a[10:30]]),
           ([a, b], [a, a]), ([a, a], [a, b])]
    for arrays, out in bad:
        with pytest.raises(ValueError, match="overlaps another array"):
            nn.clip_by_global_norm(arrays, 1.0, out=out)
    assert np.array_equal(a.get(), h) and np.array_equal(b.get(), h + 1)
    norm = np.sqrt(2 * (h.astype(np.float64) ** 2).sum())
    (c, d), n = nn.clip_by_global_norm([a, a], 1.0)  # read twice, written elsewhere
    assert np.isclose(n.get(), norm, rtol=1e-6)
    assert np.allclose(c.get(), h / norm, rtol=1e-6) and np.array_equal(c.get(), d.get())
    parts = [a[:10], a[10:10], a[10:11], a[11:]]     # side by side, one of them empty
    nn.clip_by_global_norm(parts, 1.0, out=parts)
    assert np.allclose(a.get(), h / np.linalg.norm(h), rtol=1e-6)
