"""The serving operators where settings and sizes are at their ends: equal logits at temperatures that are no power of two."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_drafts import DT, gen, i32  # noqa: E402
from test_gpu_serving import check_draw  # noqa: E402


def halves():
    """(largest logit, temperature) whose product of 32 largest / temperature lies next to a half in f32, rounded up to it
    or, below 0, down: to the nearest number it is then more than a half away.  The logits have 8 bits."""
    tops = np.unique(np.outer(np.arange(1, 256), 2.0 ** -np.arange(10)))
    tops = np.concatenate([tops, -tops])
    out = []
    for temp in (0.3, 0.35, 0.6, 0.7, 0.9, 1.2):
        per = np.float64(np.float32(32) / np.float32(temp))
        product = (tops * per).astype(np.float32).astype(np.float64)
        at = np.nonzero(np.rint(product) - tops * per > 0.5)[0]
        out += [(float(tops[i]), temp) for i in at[:: max(1, len(at) // 5)]]
    return out


@pytest.mark.parametrize("ty", list(DT))
def test_draw_equal_logits_at_temperatures(pk, ty):
    """The largest logit is in the first bin of the order also where its product with the bins a unit is a rounded half."""
    pairs = halves()
    assert len(pairs) >= 20
    rows = len(pairs)
    temp = torch.tensor([t for _, t in pairs], dtype=torch.float32, device="cuda")
    u = torch.rand(rows, generator=gen(3), device="cuda")
    for n in (900, 20000):
        x = torch.tensor([v for v, _ in pairs], device="cuda")[:, None].expand(rows, n).to(DT[ty]).contiguous()
        for spread in (False, True):
            if spread:
                x[:, ::3] -= 5.0
                x[:, 7] = -math.inf
            for k in (17, 250, n // 2, n - 3):
                for p in (1.0, 0.6):
                    check_draw(pk, x, u, temp=temp, top_k=i32([k] * rows), top_p=torch.full((rows,), p, device="cuda"))
