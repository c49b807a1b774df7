"""sample() where a rounding or an empty place of a row could decide a token: rows masked with the lowest f32, logits at the borders of
the histogram's bins, lists that every CTA of a row fills.  Tokens are compared with the 64-bit restatement of test_gpu_sample."""
import numpy as np
import pytest

from test_gpu_sample import checked, kv, model_logits  # noqa: F401 (kv is a fixture)

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


def bins_of(difference, zscale):
    """Bins of the depth difference * zscale, rounded to the nearest whole number after the product was rounded (as the kernel's rule
    has it), and from the unrounded product."""
    rounded = (difference * zscale).astype(f32).astype(np.float64) + 2.0 ** 23
    exact = difference.astype(np.longdouble) * zscale.astype(np.longdouble) + 2 ** 23
    return rounded.astype(f32).view(np.uint32) & 1023, exact.astype(f32).view(np.uint32) & 1023


def zscale_of(t):
    """Bins per unit of the logits: 1023 bins over 28 octaves."""
    return f32(f32(1.4426950408889634) / f32(t)) * f32(f32(1023) / f32(28))


@pytest.mark.parametrize("n,copies", [(1000, 1), (9000, 1), (1000, 12)])
def test_logits_at_the_border_of_a_bin(kv, n, copies):
    # Two logits, the second at a depth whose product with the bins per unit lies next to k + 1/2: where it is counted, it has
    # to be found.  p and n ask for the deepest bins (log2(n / (1 - p)) > 28).
    lo, hi = (np.array([v], f32).view(np.uint32)[0] for v in (4.0, 10.0))
    depth = np.random.default_rng(1).integers(lo, hi, 4_000_000).astype(np.uint32).view(f32)
    depth = np.concatenate([np.array([0x4102120A], np.uint32).view(f32), depth])
    a, b = bins_of(depth, zscale_of(1.0))
    depth = depth[a != b][:40]
    assert len(depth) == 40 and depth[0] == f32(8.129404)
    rows = len(depth)
    g = np.random.default_rng(2)
    for neighbour in (False, True):  # alone; beside one that lies in the middle of the bin which the other rule names
        x = np.full((rows, n), -np.inf, f32)
        x[:, 0] = 0
        x[np.arange(rows), g.integers(1, n // 2, rows)] = -depth
        if neighbour:
            x[np.arange(rows), g.integers(n // 2, n, rows)] = -(b[a != b][:rows].astype(np.float64) / float(zscale_of(1.0))).astype(f32)
        u = 1 - np.exp(-depth) * g.uniform(0.2, 0.8, rows)
        checked(kv, torch.from_numpy(x).cuda().repeat(copies, 1), np.tile(u, copies), **all_of(rows * copies, p=0.999999))


@pytest.mark.parametrize("copies", [1, 20])
def test_equal_logits_at_the_border_of_a_bin(kv, copies):
    # fifty equal bf16 logits at such a depth: all of them or none
    values = (np.arange(0x4080, 0x4120, dtype=np.uint32) << 16).view(f32)
    g = np.random.default_rng(2)
    found = []
    while len(found) < 24:
        t = f32(g.uniform(0.7, 2))
        a, b = bins_of(values, zscale_of(t))
        found += [(t, v) for v in values[(a != b) & (values / t < 9)]]
    rows, n = len(found), 1000
    t, v = (np.array(c, f32) for c in zip(*found))
    x = np.full((rows, n), -np.inf, f32)
    x[:, 500] = 0
    for r in range(rows):
        x[r, g.permutation(np.r_[0:500, 501:n])[:50]] = -v[r]
    u = 1 - 50 * np.exp(-v / t) / (1 + 50 * np.exp(-v / t)) * g.uniform(0.1, 0.9, rows)
    logits = torch.from_numpy(x).cuda().to(torch.bfloat16).repeat(copies, 1)
    checked(kv, logits, np.tile(u, copies), np.tile(t, copies), **all_of(rows * copies, p=0.999999))


@pytest.mark.parametrize("rows,n", [(15, 8192), (30, 4096), (60, 2048), (9, 8200), (100, 60000)])
def test_lists_that_every_cta_of_a_row_fills(kv, rows, n):
    # short slices, where the CTAs of a row run apart the most, and up to 100 candidates in each: the same token every time, the
    # right one at first
    x, g = model_logits(rows + n, rows, n)
    u, t = g.random(rows), 0.5 + g.random(rows)
    dev = lambda a, dt=torch.float32: torch.as_tensor(a, dtype=dt, device="cuda")
    for k, p in ((2, 1.0), (199, 0.9), (700, 1.0)):
        want = torch.from_numpy(checked(kv, x, u, t, **all_of(rows, k=k, p=p))).cuda()
        args = dict(temperature=dev(t), top_k=dev(np.full(rows, k), torch.int32), top_p=dev(np.full(rows, p)))
        outs = [torch.empty(rows, dtype=torch.int32, device="cuda") for _ in range(300)]
        for out in outs:  # one after the other without a pause
            kv.sample(x, dev(u), out=out, **args)
        assert bool((torch.stack(outs) == want).all())
