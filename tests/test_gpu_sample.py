"""sample(): tokens against a plain implementation in 64 bits.  The result is a whole number, so it has to be equal -- except
where a border of the distribution and the draw lie closer together than 44 fractional bits can tell apart; the inputs are
seeded, and `borders_apart` shows for each case that no such border is near."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def kv():
    import tract_b200

    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    tract_b200.lib()
    return tract_b200


def plain_row(x, t, k, p, m, u):
    """(token, distance of the draw from the nearest border) of one row of float64 logits, one step of the definition at a time."""
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return 0, 1.0
    if not t > 0:
        return int(np.argmax(x)), 1.0
    if top == np.inf:
        w = (x == np.inf).astype(np.float64)
    else:
        with np.errstate(over="ignore"):
            w = np.exp((x - top) / t)
    order = np.lexsort((np.arange(len(x)), -x))
    ws = w[order]
    n = len(x)
    if 0 < k < n:
        n = k
    if p <= 0:
        n = 1
    elif p < 1:
        cum = np.cumsum(ws[:n])
        reached = np.nonzero(cum >= p * cum[-1])[0]
        n = int(reached[0]) + 1
    if m > 0:
        n = min(n, int((ws >= min(m, 1.0)).sum()))
    kept = np.zeros(len(x))
    kept[order[:n]] = ws[:n]
    cdf = np.cumsum(kept)
    goal = min(max(u, 0.0), 1.0) * cdf[-1]
    token = min(int(np.searchsorted(cdf, goal, side="right")), int(np.nonzero(kept)[0][-1]))
    # kept weights of 1 only: sums are whole numbers and u times a sum is exact (24 + 17 bits), here as in fixed point, so a draw on
    # a border is decided the same way
    if (kept[kept > 0] == 1.0).all():
        return token, 1.0
    borders = np.unique(cdf)
    return token, float(np.abs(borders - goal).min() / cdf[-1]) if u > 0 else 1.0


def checked(kv, logits, u, t=None, k=None, p=None, m=None, near=2.0 ** -36):
    """All rows against plain_row.  Fixed-point weights are off by at most 2^-45, n of them by n 2^-45 (n <= 2^18: 2^-27 in the
    worst case, 2^-36 for errors of either sign): a row whose draw is nearer to a border than that would say nothing, and none
    may be."""
    rows = logits.shape[0]
    dev = lambda a, dt: None if a is None else torch.as_tensor(a, dtype=dt, device="cuda")
    args = dict(temperature=dev(t, torch.float32), top_k=dev(k, torch.int32), top_p=dev(p, torch.float32), min_p=dev(m, torch.float32))
    uu = dev(u, torch.float32)
    got = kv.sample(logits, uu, **args).cpu().numpy()
    x = logits.double().cpu().numpy()
    at = lambda key, i, off: off if args[key] is None else float(args[key][i])
    for i in range(rows):
        want, gap = plain_row(x[i], at("temperature", i, 1.0), int(at("top_k", i, 0)), at("top_p", i, 1.0), at("min_p", i, 0.0), float(uu[i]))
        assert gap > near, ("borders too near", i, gap)
        assert got[i] == want, (i, int(got[i]), want)
    return got


check = checked


def model_logits(seed, rows, n, io="f32", pad=0, spread=2.2):
    g = np.random.Generator(np.random.Philox(key=seed))
    x = g.standard_normal((rows, n + pad)).astype(np.float32) * np.float32(spread)
    for r in range(rows):
        x[r, g.integers(0, n, 20)] += 3 + 9 * g.random(20).astype(np.float32)
    return torch.from_numpy(x).cuda().to(TORCH[io])[:, :n], g


MODES = {"plain": {}, "top_k": dict(k=40), "top_p": dict(p=0.9), "min_p": dict(m=0.05), "k_p": dict(k=60, p=0.85), "k_m": dict(k=30, m=0.02),
         "p_m": dict(p=0.95, m=0.01), "all": dict(k=100, p=0.97, m=0.004)}


@pytest.mark.parametrize("mode", list(MODES))
@pytest.mark.parametrize("io,rows,n,pad", [("f32", 1, 1, 0), ("f32", 3, 2, 1), ("bf16", 2, 33, 7), ("f32", 5, 1000, 0), ("f16", 4, 2049, 0),
                                           ("f32", 2, 8193, 3), ("bf16", 3, 50257, 7), ("f32", 3, 128256, 0), ("f16", 2, 200000, 0),
                                           ("f32", 2, 300001, 0), ("bf16", 1, 524288, 0)])
def test_modes_types_and_sizes(kv, mode, io, rows, n, pad):
    x, g = model_logits(n + rows, rows, n, io, pad)
    t = 0.4 + g.random(rows)
    full = lambda v, dt: None if v is None else np.full(rows, v, dt)
    kw = MODES[mode]
    check(kv, x, g.random(rows), t, full(kw.get("k"), np.int32), full(kw.get("p"), np.float32), full(kw.get("m"), np.float32))


@pytest.mark.parametrize("rows,n", [(300, 700), (160, 40000), (700, 9000)])
def test_many_rows_with_settings_of_their_own(kv, rows, n):
    x, g = model_logits(rows + n, rows, n)
    kind = g.integers(0, 8, rows)
    t = np.where(kind == 7, 0.0, 0.3 + 1.2 * g.random(rows))
    k = np.where(np.isin(kind, (1, 4, 6)), g.integers(1, 300, rows), 0)
    p = np.where(np.isin(kind, (2, 4, 5, 6)), 0.3 + 0.69 * g.random(rows), 1.0)
    m = np.where(np.isin(kind, (3, 5, 6)), 0.3 * g.random(rows) ** 3 + 1e-4, 0.0)
    got = check(kv, x, g.random(rows), t, k.astype(np.int32), p, m)
    greedy = kv.argmax(x.float().contiguous()).cpu().numpy()
    assert (got[kind == 7] == greedy[kind == 7]).all()


@pytest.mark.parametrize("mode", ["plain", "top_p", "top_k", "k_p"])
@pytest.mark.parametrize("spread,temperature", [(0.02, 1.0), (2.0, 30.0), (1.0, 1.0), (6.0, 0.05)])
@pytest.mark.parametrize("rows", [3, 200])
def test_flat_and_peaked_rows(kv, mode, spread, temperature, rows):
    # flat rows keep more tokens than are gathered, peaked ones a single one
    n = 30000
    g = np.random.Generator(np.random.Philox(key=7))
    x = torch.from_numpy((g.standard_normal((rows, n)) * spread).astype(np.float32)).cuda()
    kw = dict(plain={}, top_p=dict(p=np.full(rows, 0.97)), top_k=dict(k=np.full(rows, 12345)), k_p=dict(k=np.full(rows, 20000), p=np.full(rows, 0.6)))[mode]
    check(kv, x, g.random(rows), np.full(rows, temperature), **kw)


@pytest.mark.parametrize("copies", [1, 50])
def test_equal_logits_are_taken_by_rising_index(kv, copies):
    n = 9000
    six = lambda a: np.tile(np.asarray(a), copies)
    check = lambda kv, x, u, **kw: checked(kv, x.repeat(copies, 1), six(u), **{k: six(v) for k, v in kw.items()})[:len(u)]
    x = torch.full((6, n), -1.0, device="cuda")
    x[:, 5::7] = 2.0  # 1285 equal maxima
    x[:, 3::7] = 1.5
    u = np.array([0.0, 0.1, 0.5, 0.9, 0.999, 0.3])
    firsts = np.arange(5, n, 7)
    got = check(kv, x, u, k=np.full(6, 10))  # of the equal ones the first ten
    assert (got == firsts[(u.astype(np.float32).astype(np.float64) * 10).astype(int)]).all()
    check(kv, x, u, p=np.full(6, 0.25, np.float32))
    check(kv, x, u, k=np.full(6, 1300), p=np.full(6, 0.999, np.float32))
    check(kv, x, u, k=np.full(6, 100), p=np.full(6, 0.5, np.float32))
    flat = torch.zeros((6, 40000), device="cuda")
    check(kv, flat, u, k=np.full(6, 7))
    check(kv, flat, u, p=np.full(6, 0.3, np.float32))
    # positive and negative zero are the same logit
    zero = torch.zeros((1, 100), device="cuda")
    zero[0, ::2] = -0.0
    assert check(kv, zero, [0.0], k=[1])[0] == 0
    assert check(kv, zero, [0.6], k=[5])[0] == 3


@pytest.mark.parametrize("copies", [1, 40])  # few rows, many rows
def test_infinities_nan_and_empty_rows(kv, copies):
    inf, nan = float("inf"), float("nan")
    n = 5000
    x = torch.randn((8, n), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    x[0, :] = -inf
    x[1, :] = nan
    x[2, 100:] = -inf            # masked vocabulary
    x[3, [7, 4000]] = inf        # infinite logits share the row
    x[4, 1::2] = nan
    x[5, :] = -inf
    x[5, 4321] = -80.0           # one token left
    x[6, :] = torch.finfo(torch.float32).min  # masks of the type's lowest value: a row of them is flat
    x[7, :] = torch.finfo(torch.float32).min
    x[7, 17] = 1.0
    x = x.repeat(copies, 1)
    rows = 8 * copies
    u = np.full(rows, 0.71)
    for kw in ({}, dict(k=np.full(rows, 20)), dict(p=np.full(rows, 0.9, np.float32)), dict(m=np.full(rows, 0.1, np.float32)),
               dict(k=np.full(rows, 2500), p=np.full(rows, 0.8, np.float32)), dict(k=np.full(rows, 4990))):
        got = check(kv, x, u, **kw)
        assert got[0] == 0 and got[1] == 0 and got[2] < 100 and got[3] == 4000 and got[4] % 2 == 0 and got[5] == 4321 and got[7] == 17


def test_settings_at_their_ends(kv):
    x, g = model_logits(11, 4, 3001)
    u = g.random(4)
    best = torch.argmax(x, 1).cpu().numpy()
    one = lambda v, dt=np.float32: np.full(4, v, dt)
    for kw in (dict(k=one(1, np.int32)), dict(p=one(0.0)), dict(p=one(-1.0)), dict(p=one(1e-30)), dict(m=one(1.0)), dict(m=one(5.0)), dict(t=one(0.0)),
               dict(t=one(-2.0)), dict(t=one(float("nan"))), dict(t=one(1e-38))):
        assert (check(kv, x, u, **kw) == best).all(), kw
    plain = check(kv, x, u)
    for kw in (dict(k=one(0, np.int32)), dict(k=one(-5, np.int32)), dict(k=one(3001, np.int32)), dict(k=one(2 ** 31 - 1, np.int32)), dict(p=one(1.0)),
               dict(p=one(2.0)), dict(m=one(0.0)), dict(m=one(-1.0)), dict(m=one(1e-38))):
        assert (check(kv, x, u, **kw) == plain).all(), kw
    dev = lambda a: torch.as_tensor(a, dtype=torch.float32, device="cuda")
    assert (kv.sample(x, dev(u), top_p=dev(one(float("nan"))), min_p=dev(one(float("nan")))).cpu().numpy() == plain).all()
    # the ends of the draw, and what lies outside
    for kw in ({}, dict(top_k=torch.full((4,), 50, dtype=torch.int32, device="cuda"))):
        first, last = kv.sample(x, dev(one(0.0)), **kw), kv.sample(x, dev(one(np.nextafter(np.float32(1), np.float32(0)))), **kw)
        assert torch.equal(kv.sample(x, dev(one(-3.0)), **kw), first) and torch.equal(kv.sample(x, dev(one(float("nan"))), **kw), first)
        assert bool((kv.sample(x, dev(one(7.0)), **kw) >= last).all())
    for t in (1e-3, 1e-5, 1e-7, 1e-9, 1e-12, 1e-30):  # down to where neighbouring floats are far apart
        near = torch.full((2, 5000), 9.0, device="cuda")
        near[:, 7::3] = float(np.nextafter(np.float32(10), np.float32(0)))
        near[:, 9::11] = 10.0
        for kw in (dict(), dict(p=np.full(2, 0.7, np.float32)), dict(k=np.full(2, 900, np.int32))):
            check(kv, near, [0.31, 0.87], np.full(2, t), **kw)
    inf_t = kv.sample(x, dev(one(0.5)), temperature=dev(one(float("inf"))))  # a uniform draw
    assert (inf_t.cpu().numpy() == 1500).all()


def test_every_draw_lands_in_its_share(kv):
    # one distribution, many draws: the tokens follow from the draws alone and come in rising order
    n, rows = 517, 4000
    x, g = model_logits(3, 1, n)
    u = np.sort(g.random(rows)).astype(np.float32)
    for kw in ({}, dict(p=np.full(rows, 0.8, np.float32)), dict(k=np.full(rows, 9))):
        got = check(kv, x.expand(rows, n).contiguous(), u, np.full(rows, 0.9), **kw)
        assert (np.diff(got) >= 0).all()


def test_repeats_strides_streams_and_graphs(kv):
    x, g = model_logits(5, 6, 128256, pad=5)
    dev = lambda a, dt=torch.float32: torch.as_tensor(a, dtype=dt, device="cuda")
    args = dict(temperature=dev(np.full(6, 0.8)), top_k=dev([0, 50, 0, 0, 20, 0], torch.int32), top_p=dev([0.9, 0.95, 1, 1, 1, 0.99]), min_p=dev([0, 0, 0.05, 0, 0, 0]))
    u = dev(g.random(6))
    want = kv.sample(x, u, **args)
    for _ in range(5):
        assert torch.equal(kv.sample(x, u, **args), want)
    assert torch.equal(kv.sample(x.contiguous(), u, **args), want)
    shifted = torch.empty(6 * 128256 + 1, device="cuda")[1:].view(6, 128256)  # rows off the 16-byte grid
    shifted.copy_(x)
    assert torch.equal(kv.sample(shifted, u, **args), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(kv.sample(x, u, **args), want)
    # two graphs, a workspace each, replayed side by side on new inputs
    graphs = []
    for i in range(2):
        out, scratch, xi = torch.empty(6, dtype=torch.int32, device="cuda"), kv.sample_scratch(6, 128256), x.clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kv.sample(xi, u, **args, out=out, scratch=scratch)
        graphs.append((graph, xi, out, scratch, torch.cuda.Stream()))
    y, _ = model_logits(6, 6, 128256, pad=5)
    graphs[1][1].copy_(y)
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, _, _, _, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][2], want) and torch.equal(graphs[1][2], kv.sample(y, u, **args))


def test_refusals(kv):
    x, u = torch.zeros((2, 100), device="cuda"), torch.zeros(2, device="cuda")
    L = kv.lib()
    out, scratch = torch.full((2,), -7, dtype=torch.int32, device="cuda"), kv.sample_scratch(2, 300000)
    assert scratch.numel() >= 2 * 300000 * 4 and kv.sample_scratch(2, 262144).numel() == 0
    call = lambda logits=x.data_ptr(), stride=100, dtype=0, rows=2, n=100, uniform=u.data_ptr(), o=out.data_ptr(), s=scratch.data_ptr(): L.b200kv_sample(
        logits, stride, dtype, rows, n, None, None, None, None, uniform, o, s, None)
    for kw, why in ((dict(logits=None), b"null"), (dict(uniform=None), b"null"), (dict(o=None), b"null"), (dict(s=None, n=300000, stride=300000), b"workspace"), (dict(rows=0), b"positive"),
                    (dict(n=0), b"positive"), (dict(dtype=3), b"dtype"), (dict(stride=99), b"apart"), (dict(s=scratch.data_ptr() + 8), b"aligned"),
                    (dict(n=524289, stride=524289), b"at most"), (dict(rows=70000), b"at most")):
        assert call(**kw) == 1 and why in L.b200kv_last_error(), kw
    torch.cuda.synchronize()
    assert bool((out == -7).all())
    assert L.b200kv_sample_scratch_bytes(0, 5) == -1 and L.b200kv_sample_scratch_bytes(5, 0) == -1
    with pytest.raises(kv.B200KvError, match="uniform"):
        kv.sample(x, None)
    with pytest.raises(kv.B200KvError, match="dtype"):
        kv.sample(x.double(), u)


def test_rows_past_two_to_the_31st_logit(kv):
    # rows of a wide matrix: the last ones begin 2^31 elements and more behind the first
    n, stride, rows = 1000, 2 ** 28, 9
    wide = torch.zeros(rows * stride - (stride - n), dtype=torch.bfloat16, device="cuda").as_strided((rows, n), (stride, 1))
    x, g = model_logits(77, rows, n, "bf16")
    wide.copy_(x)
    check(kv, wide, g.random(rows), 0.5 + g.random(rows), np.full(rows, 50, np.int32), np.full(rows, 0.9, np.float32), None)


def test_two_graphs_of_one_decode_loop(kv):
    # captured with buffers of their own, replayed in turn with new logits and numbers
    x, g = model_logits(5, 6, 50257)
    y, _ = model_logits(6, 6, 50257)
    u = torch.from_numpy(g.random((4, 6)).astype(np.float32)).cuda()
    k = torch.full((6,), 40, dtype=torch.int32, device="cuda")
    want = [[kv.sample(t, u[j], top_k=k) for t in (x, y)] for j in range(4)]
    outs, uu, graphs = [torch.empty(6, dtype=torch.int32, device="cuda") for _ in range(2)], torch.zeros(6, device="cuda"), []
    torch.cuda.synchronize()
    for t, out in zip((x, y), outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kv.sample(t, uu, top_k=k, out=out)
        graphs.append(graph)
    for j in (2, 0, 3, 1):
        uu.copy_(u[j])
        for graph in graphs:
            graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(outs, want[j]))
