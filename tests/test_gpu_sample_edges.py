"""sample() where an empty place of a row could decide a token: rows masked with the lowest f32.  Tokens are compared with the
64-bit restatement of test_gpu_sample."""
import numpy as np
import pytest

from test_gpu_sample import checked, kv  # noqa: F401 (kv is a fixture)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

LOWEST = float(np.finfo(np.float32).min)
f32 = np.float32


def all_of(rows, **kw):
    types = dict(k=np.int32)
    return {key: np.full(rows, v, types.get(key, np.float32)) for key, v in kw.items()}


@pytest.mark.parametrize("n,copies", [(1, 1), (3, 1), (5001, 1), (50257, 1), (128001, 1), (262143, 1), (300001, 1),
                                      (3, 90), (5001, 30), (5001, 80), (50257, 20)])  # many rows: smaller blocks, off the chip
@pytest.mark.parametrize("kw", [{}, dict(p=0.9), dict(k=7), dict(k=900, p=0.8), dict(m=0.5), dict(p=0.7, m=0.5)], ids=str)
def test_rows_masked_with_the_lowest_value(kv, n, copies, kw):
    # every finite logit is the maximum: an element of -inf, a NaN and what fills a row up to whole quads weigh nothing beside it
    g = np.random.Generator(np.random.Philox(key=n))
    x = np.full((6, n), LOWEST, f32)
    x[1, g.random(n) < 0.3] = -np.inf
    x[2, g.random(n) < 0.3] = np.nan
    x[3, :] = -np.inf
    x[3, n // 2:] = LOWEST
    x[4, : n // 2] = LOWEST
    x[4, n // 2 + 1:] = -np.inf
    x[4, n // 3] = LOWEST  # (a row of one keeps a number)
    x[5, g.random(n) < 0.9] = -np.inf
    rows = 6 * copies
    checked(kv, torch.from_numpy(x).cuda().repeat(copies, 1), g.random(rows), **all_of(rows, **kw))


@pytest.mark.parametrize("temperature", [1e30, 1e-3, 0.7])
@pytest.mark.parametrize("mode", [{}, dict(p=0.9), dict(k=3000, p=0.95)], ids=str)
def test_the_two_lowest_values(kv, temperature, mode):
    n = 4099
    above = float(np.nextafter(f32(LOWEST), f32(0)))
    x = np.full((3, n), LOWEST, f32)
    x[0, 5::7] = above
    x[1, 17] = above
    x[2, ::2] = above
    x[2, 1::4] = -np.inf
    checked(kv, torch.from_numpy(x).cuda(), [0.3, 0.6, 0.97], **all_of(3, t=temperature, **mode))
