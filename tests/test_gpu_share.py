"""Sequences that share pages (fork_shared) and the attention that reads shared pages once (attend_shared): contents bit for
bit, attention against a plain implementation in 64 bits over what the cache exports."""
import numpy as np
import pytest

from util import normal

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

NP = {"f32": np.float32, "f16": np.float16, "bf16": np.float32}
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
FORMATS = [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("q8_1", "f16"), ("q4_0", "bf16")]


@pytest.fixture(scope="module")
def kv():
    import tract_b200

    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    tract_b200.lib()
    return tract_b200


def rows(seed, shape, io, scale=1.0):
    return torch.from_numpy(normal(seed, shape, scale=scale)).cuda().to(TORCH[io])


def add(cache, seqs, seed, n, io):
    k, v = (rows(seed + i, (len(seqs), cache.n_kv_heads, n, cache.head_dim), io) for i in (0, 1))
    cache.append(seqs, k, v)


def held(cache, seq, io):
    """What a sequence holds, bit for bit: its exported tensors, and the codes and scales of the block formats."""
    if cache.seq_len(seq) == 0:
        return []
    got = list(cache.export(seq, TORCH[io]))
    if cache.fmt in (3, 4):
        got += [t for which in (0, 1) for t in cache.export_codes(seq, which)]
    return [t.clone() for t in got]


def same(a, b):
    return len(a) == len(b) and all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))


def reference(cache, seqs, q, scale=None):
    """(attention in 64 bits, sum of weight x |value|) of each query over everything its sequence holds."""
    out, size = [], []
    dt = torch.float32 if cache.fmt in (0, 3, 4) else TORCH[{1: "f16", 2: "bf16"}[cache.fmt]]
    for i, s in enumerate(seqs):
        k, v = (t.double() for t in cache.export(s, dt))
        Hkv, n, D = k.shape
        qi = q[i, :, 0].double().reshape(Hkv, -1, D)
        w = qi @ k.transpose(1, 2) * (scale or D ** -0.5)
        w = torch.exp(w - w.amax(-1, keepdim=True))
        w = w / w.sum(-1, keepdim=True)
        out.append((w @ v).reshape(-1, 1, D))
        size.append((w @ v.abs()).reshape(-1, 1, D))
    return torch.stack(out), torch.stack(size)


def assert_close(got, ref, size, io):
    """A result is off by its own rounding (half a step, relative to the value) and by what rounding the weights and the
    dequantised values to 16 bits can add: at most half an f16 step each, relative to sum weight x |value|.  The sums and
    exponentials in 32 bits add less than 2^-15 of that size (scores up to 2^5 with an error of 2^-22 each, 2^-21 of the
    exponential, sums of at most 2^16 terms in trees and chains of 64); f32 results have nothing else."""
    if io == "f32":
        bound = 2.0 ** -24 * ref.abs() + 2.0 ** -17 * size
    else:
        bound = torch.finfo(TORCH[io]).eps / 2 * ref.abs() + (2 * 2.0 ** -11 + 2.0 ** -15) * size
    bad = (got.double() - ref).abs() > bound
    assert torch.isfinite(got).all()
    assert not bad.any(), (int(bad.sum()), float(((got.double() - ref).abs() / bound).max()), bad.nonzero()[0].tolist())


# ---- page sharing ----------------------------------------------------------------------------------------

@pytest.mark.parametrize("fmt,io", FORMATS)
@pytest.mark.parametrize("D,n", [(128, 1), (64, 63), (128, 64), (128, 65), (64, 130), (128, 191)])
def test_children_hold_the_parent_and_go_their_own_way(kv, fmt, io, D, n):
    cache = kv.KvCache(fmt, 3, D, max_seqs=6, max_seq_tokens=512)
    a, b = cache.new_seq(), cache.new_seq()
    add(cache, [a], 1, n, io)
    add(cache, [b], 3, 77, io)
    free = cache.free_pages()
    kids = cache.fork_shared([a, b, a, a])
    assert cache.free_pages() == free - (4 if n % 64 else 1)  # the partly filled pages only
    want_a, want_b = held(cache, a, io), held(cache, b, io)
    for kid, want in zip(kids, (want_a, want_b, want_a, want_a)):
        assert cache.seq_len(kid) == (n if want is want_a else 77) and same(held(cache, kid, io), want)
    # everybody goes on: one batch of different tokens, then more for one child across a page border
    everyone = [a, b, *kids]
    add(cache, everyone, 10, 3, io)
    add(cache, [kids[2]], 20, 70, io)
    after = [held(cache, s, io) for s in everyone]
    for i, s in enumerate(everyone):  # a sequence of its own that was given the same tokens holds the same
        lone = kv.KvCache(fmt, 3, D, max_seqs=1, max_seq_tokens=512)
        t = lone.new_seq()
        parent = b if s in (b, kids[1]) else a
        add(lone, [t], 3 if parent == b else 1, 77 if parent == b else n, io)
        k, v = (rows(10 + j, (len(everyone), 3, 3, D), io)[i:i + 1] for j in (0, 1))
        lone.append([t], k, v)
        if s == kids[2]:
            add(lone, [t], 20, 70, io)
        assert same(held(lone, t, io), after[i]), i
        lone.close()
    cache.check()
    cache.free_seqs(everyone)
    fresh = kv.KvCache(fmt, 3, D, max_seqs=6, max_seq_tokens=512)
    assert cache.free_pages() == fresh.free_pages()
    cache.close(), fresh.close()


def test_pages_go_back_with_their_last_holder(kv):
    cache = kv.KvCache("f16", 2, 64, max_seqs=5, max_seq_tokens=640)
    total = cache.free_pages()
    a = cache.new_seq()
    add(cache, [a], 1, 300, "f16")  # 4 full pages and 44 tokens
    kids = cache.fork_shared([a, a])
    assert cache.free_pages() == total - 5 - 2
    want = held(cache, a, "f16")
    cache.free_seq(a)  # its own last page only
    assert cache.free_pages() == total - 4 - 2
    grandkid = cache.fork_shared([kids[0]])[0]
    cache.trim(kids[0], 100)  # tokens 200 ..: gives back its hold on three shared pages
    cache.truncate(kids[1], 128)
    assert cache.free_pages() == total - 4 - 2  # kids[0] and the grandchild hold a tail each; kids[1] dropped its own; grandkid took one
    assert same(held(cache, grandkid, "f16"), want)
    # the freed slot and pages serve the next sequence without touching the shared ones
    b = cache.new_seq()
    add(cache, [b], 9, 400, "f16")
    assert same(held(cache, grandkid, "f16"), want)
    cache.free_seqs([kids[0], kids[1], b])
    assert cache.free_pages() == total - 5
    deep = cache.fork(grandkid)  # a deep copy of shared pages
    assert cache.free_pages() == total - 10 and same(held(cache, deep, "f16"), want)
    cache.free_seqs([grandkid, deep])
    assert cache.free_pages() == total
    cache.check()
    cache.close()


@pytest.mark.parametrize("fmt,io", FORMATS)
@pytest.mark.parametrize("many", [False, True])
def test_append_into_a_shared_page_copies_it_first(kv, fmt, io, many):
    cache = kv.KvCache(fmt, 2, 128, max_seqs=4, max_seq_tokens=512)
    a = cache.new_seq()
    add(cache, [a], 1, 192, io)
    kids = cache.fork_shared([a, a])
    before = held(cache, kids[1], io)
    cache.truncate_many([a, kids[0]], [100, 70])  # both inside a page that kids[1] holds full
    half = held(cache, a, io)
    if many:
        add(cache, [a, kids[0], kids[1]], 30, 5, io)
    else:
        for i, s in enumerate((a, kids[0], kids[1])):
            k, v = (rows(30 + j, (3, 2, 5, 128), io)[i:i + 1] for j in (0, 1))
            cache.append([s], k, v)
    assert [cache.seq_len(s) for s in (a, *kids)] == [105, 75, 197]
    got = [held(cache, s, io) for s in (a, *kids)]
    for parts, full, n in ((got[0], before, 100), (got[1], before, 70), (got[2], before, 192)):
        for x, y in zip(parts, full):
            assert torch.equal(x[:, :n].contiguous().view(torch.uint8), y[:, :n].contiguous().view(torch.uint8))
    lone = kv.KvCache(fmt, 2, 128, max_seqs=3, max_seq_tokens=512)
    for i, (n, parts) in enumerate(zip((100, 70, 192), got)):
        t = lone.new_seq()
        add(lone, [t], 1, 192, io)
        lone.truncate(t, n)
        k, v = (rows(30 + j, (3, 2, 5, 128), io)[i:i + 1] for j in (0, 1))
        lone.append([t], k, v)
        assert same(held(lone, t, io), parts)
    assert len(half) == len(before)
    cache.check()
    cache.close(), lone.close()


def test_append_without_a_page_for_the_copy_changes_nothing(kv):
    cache = kv.KvCache("f16", 1, 64, max_seqs=2, max_seq_tokens=256, pool_tokens=128)  # 2 + 2 pages
    a = cache.new_seq()
    add(cache, [a], 1, 128, "f16")
    kid = cache.fork_shared([a])[0]
    cache.truncate(a, 100)
    add(cache, [kid], 5, 128, "f16")  # takes the two free pages
    want = [held(cache, s, "f16") for s in (a, kid)]
    assert cache.free_pages() == 0
    with pytest.raises(kv.B200KvError, match="page of its own"):
        add(cache, [a], 7, 1, "f16")
    assert cache.seq_len(a) == 100 and all(same(held(cache, s, "f16"), w) for s, w in zip((a, kid), want))
    cache.truncate(kid, 192)  # one page back
    with pytest.raises(kv.B200KvError, match="exhausted"):
        add(cache, [a, kid], 7, 1, "f16")  # two needed: the copy, and a page for the other one
    assert cache.free_pages() == 1 and cache.seq_len(a) == 100 and cache.seq_len(kid) == 192
    assert same(held(cache, a, "f16"), want[0])
    add(cache, [a], 7, 1, "f16")
    assert cache.free_pages() == 0 and cache.seq_len(a) == 101
    assert torch.equal(cache.export(kid, torch.float16)[0], want[1][0][:, :192])
    cache.check()
    cache.close()


def test_fork_shared_refusals_change_nothing(kv):
    cache = kv.KvCache("f16", 1, 64, max_seqs=3, max_seq_tokens=128, pool_tokens=64)  # 1 + 3 pages
    a = cache.new_seq()
    add(cache, [a], 1, 70, "f16")
    free = cache.free_pages()
    for seqs, why in (([a, a, a], "slots are free"), ([7], "not live"), ([a, 2], "not live"), ([], "at least one")):
        with pytest.raises(kv.B200KvError, match=why):
            cache.fork_shared(seqs)
    assert cache.free_pages() == free
    b = cache.new_seq()
    add(cache, [b], 1, 70, "f16")
    with pytest.raises(kv.B200KvError, match="exhausted"):
        cache.fork_shared([a])
    assert cache.free_pages() == 0
    with pytest.raises(kv.B200KvError, match="not live"):
        cache.free_seqs([a, 2])
    with pytest.raises(kv.B200KvError, match="twice"):
        cache.free_seqs([a, a])
    assert cache.seq_len(a) == 70
    cache.free_seq(b)
    empty = cache.new_seq()
    kid = cache.fork_shared([empty])[0]  # an empty parent: an empty child, no page
    assert cache.seq_len(kid) == 0 and cache.free_pages() == 2
    cache.close()
    kivi = kv.KvCache("kivi8", 1, 64, max_seqs=2, max_seq_tokens=128)
    s = kivi.new_seq()
    add(kivi, [s], 1, 70, "f16")
    with pytest.raises(kv.B200KvError, match="KIVI"):
        kivi.fork_shared([s])
    with pytest.raises(kv.B200KvError, match="KIVI"):
        kivi.attend_shared([s], rows(2, (1, 1, 1, 64), "f16"))
    kivi.close()


# ---- attention over shared pages ---------------------------------------------------------------------------

def family(kv, fmt, io, Hkv, D, prompts, per_prompt, own, hq):
    """A cache with `per_prompt` continuations of each prompt, own[i % len(own)] tokens behind it; the sequences in order."""
    n = len(prompts) * per_prompt
    cache = kv.KvCache(fmt, Hkv, D, max_seqs=n + len(prompts) + 2, max_seq_tokens=max(prompts) + max(own) + 64, max_q_heads=hq)
    seqs = []
    for i, length in enumerate(prompts):
        parent = cache.new_seq()
        add(cache, [parent], 100 + 2 * i, length, io)
        seqs += cache.fork_shared([parent] * per_prompt)
        cache.free_seq(parent)
    for i, s in enumerate(seqs):
        if own[i % len(own)]:
            add(cache, [s], 200 + 2 * i, own[i % len(own)], io)
    return cache, seqs


@pytest.mark.parametrize("fmt,io", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("q8_1", "f16"), ("q8_1", "bf16"), ("q8_1", "f32"), ("q4_0", "f16"),
                                    ("q4_0", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("D,Hkv,G,prompts,per_prompt,own", [
    (128, 2, 4, [64], 2, [1]),               # one shared page, one token each
    (128, 8, 4, [2048], 8, [0, 1, 63, 64, 65, 200]),
    (64, 2, 7, [515, 700, 64], 5, [40, 1]),  # rows that fill no tile, three prompts
    (128, 1, 1, [1000], 3, [0]),             # nothing but the prompt, no grouped heads
    (64, 1, 16, [640], 9, [7]),              # 144 rows: two tiles
    (128, 2, 24, [4100], 12, [3, 90]),       # 288 rows: two CTAs of two tiles
])
@pytest.mark.parametrize("way", [0, 1, 2])  # the one that the sizes choose, and both others whatever they are
def test_attend_shared_against_64_bits(kv, fmt, io, D, Hkv, G, prompts, per_prompt, own, way):
    if fmt == "f16" and io == "f32":  # a bit-copy cache takes its own type; its queries may be f32
        cache, seqs = family(kv, fmt, "f16", Hkv, D, prompts, per_prompt, own, Hkv * G)
    else:
        cache, seqs = family(kv, fmt, io, Hkv, D, prompts, per_prompt, own, Hkv * G)
    cache.profile(False, shared_way=way)
    q = rows(5, (len(seqs), Hkv * G, 1, D), io, scale=1.3)
    out = cache.attend_shared(seqs, q)
    cache.check()
    ref, size = reference(cache, seqs, q)
    assert_close(out, ref, size, io)
    again = cache.attend_shared(seqs, q)  # the same bits every time
    assert torch.equal(out, again)
    cache.close()


@pytest.mark.parametrize("fmt,io", FORMATS)
@pytest.mark.parametrize("way", [0, 1, 2])
def test_attend_shared_over_a_mixed_batch(kv, fmt, io, way):
    # neighbours that share much, little and nothing, a trimmed sequence, branches of branches, an order that is not that of
    # the sequence ids
    Hkv, D, G = 2, 128, 4
    cache = kv.KvCache(fmt, Hkv, D, max_seqs=24, max_seq_tokens=3000, max_q_heads=Hkv * G)
    a, b, lone, cut = (cache.new_seq() for _ in range(4))
    for s, n, seed in ((a, 1500, 1), (b, 900, 3), (lone, 333, 5), (cut, 700, 7)):
        add(cache, [s], seed, n, io)
    kids = cache.fork_shared([a] * 4)
    add(cache, kids, 20, 600, io)
    deep = cache.fork_shared([kids[0]] * 3)  # share 2100 tokens with kids[0], 1500 with the others
    more = cache.fork_shared([b] * 2)
    add(cache, deep, 30, 65, io)
    add(cache, more, 40, 1, io)
    gone = cache.fork_shared([cut] * 2)
    cache.trim(gone[0], 300)
    batch = [more[1], b, more[0], lone, deep[2], deep[0], kids[0], deep[1], a, kids[3], kids[1], gone[1], cut]
    q = rows(9, (len(batch), Hkv * G, 1, D), io)
    cache.profile(False, shared_way=way)
    out = cache.attend_shared(batch, q)
    cache.check()
    ref, size = reference(cache, batch, q)
    assert_close(out, ref, size, io)
    # the trimmed one beside its sibling sees what regular attention shows it
    pair = [gone[0], gone[1]]
    got = cache.attend_shared(pair, q[:2])
    assert torch.equal(got, cache.attend(pair, q[:2]))
    # a batch in which nothing is shared: regular attention, bit for bit
    apart = [lone, a, b, cut]
    assert torch.equal(cache.attend_shared(apart, q[:4]), cache.attend(apart, q[:4]))
    cache.check()
    cache.close()


@pytest.mark.parametrize("fmt,io,D", [("f16", "f16", 128), ("bf16", "bf16", 64), ("q8_1", "bf16", 128), ("f32", "f32", 64)])
@pytest.mark.parametrize("way", [0, 1, 2])
def test_attend_shared_strides_rope_scale_and_quantised_result(kv, fmt, io, D, way):
    Hkv, G = 2, 4
    cache, seqs = family(kv, fmt, io, Hkv, D, [1300], 6, [5, 70], Hkv * G)
    cache.profile(False, shared_way=way)
    n, Hq = len(seqs), Hkv * G
    qkv = rows(5, (n, (Hq + 3) * D), io)  # the query heads of a fused projection: rows of a wider matrix
    q = qkv[:, D:D + Hq * D].unflatten(1, (Hq, 1, D))
    dense = q.contiguous()
    want = cache.attend_shared(seqs, dense)
    assert torch.equal(cache.attend_shared(seqs, q), want)
    wide = torch.full((n, 2 * Hq, 1, D), 7.0, dtype=q.dtype, device="cuda")
    cache.attend_shared(seqs, q, out=wide[:, ::2])
    assert torch.equal(wide[:, ::2], want) and bool((wide[:, 1::2] == 7.0).all())
    # rows that are not 16-byte aligned: the decode kernels alone
    odd = torch.empty(n * Hq * D + 1, dtype=q.dtype, device="cuda")[1:].view(n, Hq, 1, D)
    odd.copy_(dense)
    ref, size = reference(cache, seqs, q)
    assert_close(cache.attend_shared(seqs, odd), ref, size, io)
    ref, size = reference(cache, seqs, q, scale=0.03)
    assert_close(cache.attend_shared(seqs, q, scale=0.03), ref, size, io)
    # rotary embedding on the query load: the bits of a separate rope
    cos, sin = rows(21, (n, 1, D), io), rows(22, (n, 1, D), io)
    rot = kv.rope(dense, cos, sin)
    want = cache.attend_shared(seqs, rot)
    assert torch.equal(cache.attend_shared(seqs, q, cos=cos, sin=sin), want)
    # the result as the quantised activation of the following GEMM: the bits of quantising the result
    blocks = torch.randint(0, 256, (64, Hq * D // 32, 18), dtype=torch.uint8, device="cuda")
    blocks[:, :, :2] = torch.full((64, Hq * D // 32), 0.01, device="cuda").half().view(torch.uint8).reshape(64, -1, 2)
    lin = kv.Q40Linear(blocks, max_m=n)
    expect = lin.gemm(want.reshape(n, -1))
    scratch = torch.empty_like(lin.scratch)
    out = torch.empty_like(want)
    cache.attend_shared(seqs, q, cos=cos, sin=sin, scratch=scratch, out=out)
    assert torch.equal(out, want) and torch.equal(lin.gemm_quantized(n, scratch=scratch), expect)
    scratch.zero_()
    assert cache.attend_shared(seqs, q, cos=cos, sin=sin, scratch=scratch) is None
    assert torch.equal(lin.gemm_quantized(n, scratch=scratch), expect)
    lin.check(scratch)
    cache.check()
    cache.close()


@pytest.mark.parametrize("way", [0, 1, 2])
def test_attend_shared_more_than_256_sequences(kv, way):
    Hkv, D, G, n = 1, 64, 2, 300
    cache, seqs = family(kv, "f16", "f16", Hkv, D, [640], n, [3], Hkv * G)
    cache.profile(False, shared_way=way)
    q = rows(5, (n, Hkv * G, 1, D), "f16")
    cos, sin = rows(21, (n, 1, D), "f16"), rows(22, (n, 1, D), "f16")
    ref, size = reference(cache, seqs, kv.rope(q, cos, sin))
    assert_close(cache.attend_shared(seqs, q, cos=cos, sin=sin), ref, size, "f16")
    scratch = torch.empty(kv.Q40Linear.scratch_bytes(Hkv * G * D, n), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    cache.attend_shared(seqs, q, cos=cos, sin=sin, scratch=scratch, out=out)
    assert_close(out, ref, size, "f16")
    cache.check()
    cache.close()


@pytest.mark.parametrize("way", [0, 1, 2])
def test_attend_shared_in_a_small_workspace(kv, way):
    # a cache that announced one query head per kv head: the partials of the natural split do not fit, longer runs do
    Hkv, D, G = 2, 128, 16
    cache = kv.KvCache("f16", Hkv, D, max_seqs=34, max_seq_tokens=9000, max_q_heads=Hkv)
    cache.profile(False, shared_way=way)
    parent = cache.new_seq()
    add(cache, [parent], 1, 8000, "f16")
    seqs = cache.fork_shared([parent] * 32)
    add(cache, seqs, 3, 300, "f16")
    q = rows(5, (32, Hkv * G, 1, D), "f16")
    out = cache.attend_shared(seqs, q)
    cache.check()
    ref, size = reference(cache, seqs, q)
    assert_close(out, ref, size, "f16")
    cache.close()


@pytest.mark.parametrize("way", [0, 1, 2])
def test_attend_shared_peaked_scores(kv, way):
    # weights that sit on single keys of the shared pages, of the own ones, and maxima that rise page by page
    Hkv, D, G = 1, 128, 4
    cache = kv.KvCache("f16", Hkv, D, max_seqs=6, max_seq_tokens=1024, max_q_heads=G)
    cache.profile(False, shared_way=way)
    parent = cache.new_seq()
    k, v = rows(1, (1, Hkv, 640, D), "f16"), rows(2, (1, Hkv, 640, D), "f16")
    k *= torch.linspace(0.1, 12.0, 640, device="cuda").half()[None, None, :, None]
    cache.append([parent], k, v)
    seqs = cache.fork_shared([parent] * 4)
    add(cache, seqs, 7, 9, "f16")
    q = rows(5, (4, G, 1, D), "f16", scale=3.0)
    out = cache.attend_shared(seqs, q)
    # scores of up to some hundreds: their 32-bit error is up to 2^-13 in the exponent; one key carries nearly all of the weight
    ref, size = reference(cache, seqs, q)
    assert torch.isfinite(out).all()
    bound = 2.0 ** -11 * ref.abs() + (2 * 2.0 ** -11 + 2.0 ** -12) * size
    assert bool(((out.double() - ref).abs() <= bound).all())
    cache.check()
    cache.close()


def test_attend_shared_refusals_enqueue_nothing(kv):
    cache, seqs = family(kv, "f16", "f16", 2, 64, [130], 3, [2], 8)
    empty = cache.new_seq()
    q, out = rows(5, (3, 8, 1, 64), "f16"), torch.full((3, 8, 1, 64), 3.25, dtype=torch.float16, device="cuda")
    for call, why in ((lambda: cache.attend_shared([seqs[0], seqs[1], empty], q, out=out), "is empty"),
                      (lambda: cache.attend_shared([seqs[0], seqs[1], seqs[0]], q, out=out), "twice"),
                      (lambda: cache.attend_shared([seqs[0], seqs[1], 99], q, out=out), "not live"),
                      (lambda: cache.attend_shared(seqs, q[:, :7], out=out[:, :7]), "multiple of n_kv_heads"),
                      (lambda: cache.attend_shared(seqs, q.double(), out=out.double()), "unsupported dtype")):
        with pytest.raises(kv.B200KvError, match=why):
            call()
    torch.cuda.synchronize()
    assert bool((out == 3.25).all())
    keys = kv.KvCache("f16", 2, 64, max_seqs=1, max_seq_tokens=64, has_values=False)
    s = keys.new_seq()
    keys.append([s], rows(1, (1, 2, 5, 64), "f16"))
    with pytest.raises(kv.B200KvError, match="one tensor only"):
        keys.attend_shared([s], q[:1])
    cache.check()
    cache.close(), keys.close()


def test_fork_shared_without_values_and_on_another_stream(kv):
    cache = kv.KvCache("f16", 2, 128, max_seqs=4, max_seq_tokens=512, has_values=False)
    a = cache.new_seq()
    side = torch.cuda.Stream()
    k = rows(1, (1, 2, 200, 128), "f16")
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.append([a], k)
        kids = cache.fork_shared([a, a, a])
        cache.append(kids, k[:, :, :1].expand(3, 2, 1, 128).contiguous())
        got = [cache.export(s, torch.float16)[0] for s in kids]
    side.synchronize()
    for g in got:
        assert torch.equal(g[:, :200], k[0]) and torch.equal(g[:, 200:], k[0, :, :1])
    cache.check()
    cache.close()


def test_many_steps_of_branching(kv):
    # a small beam search: every step re-parents the beams, appends and attends; against caches without any sharing
    Hkv, D, G, B = 2, 64, 2, 4
    cache = kv.KvCache("q8_1", Hkv, D, max_seqs=2 * B, max_seq_tokens=512, max_q_heads=Hkv * G)
    lone = kv.KvCache("q8_1", Hkv, D, max_seqs=2 * B, max_seq_tokens=512, max_q_heads=Hkv * G)
    total = cache.free_pages()
    root, plain = cache.new_seq(), lone.new_seq()
    add(cache, [root], 1, 250, "f16")
    add(lone, [plain], 1, 250, "f16")
    beams, copies = cache.fork_shared([root] * B), [lone.fork(plain) for _ in range(B)]
    cache.free_seq(root), lone.free_seq(plain)
    g = np.random.default_rng(3)
    for step in range(20):
        k, v, q = (rows(50 + 3 * step + j, (B, h, 1, D), "f16") for j, h in enumerate((Hkv, Hkv, Hkv * G)))
        cache.append(beams, k, v), lone.append(copies, k, v)
        ref, size = reference(lone, copies, q)
        assert_close(cache.attend_shared(beams, q), ref, size, "f16")
        parents = [int(x) for x in g.integers(0, B, B)]
        kids = cache.fork_shared([beams[p] for p in parents])
        twins = [lone.fork(copies[p]) for p in parents]
        cache.free_seqs(beams), lone.free_seqs(copies)
        beams, copies = kids, twins
        if step % 7 == 6:  # a rejected draft
            n = cache.seq_len(beams[0]) - 5
            cache.truncate_many(beams, [n] * B), lone.truncate_many(copies, [n] * B)
    for s, t in zip(beams, copies):
        assert same(held(cache, s, "f16"), held(lone, t, "f16"))
    cache.check()
    cache.free_seqs(beams)
    assert cache.free_pages() == total
    cache.close(), lone.close()


@pytest.mark.parametrize("way", [0, 1, 2])
@pytest.mark.parametrize("fmt,io,D", [("f16", "f16", 128), ("q8_1", "bf16", 64), ("f32", "f32", 128)])
def test_attend_shared_captured_and_replayed(kv, fmt, io, D, way):
    # two graphs over one cache, replayed one after the other with new queries each time
    Hkv, G = 2, 4
    cache, seqs = family(kv, fmt, io, Hkv, D, [700], 6, [5, 70], Hkv * G)
    cache.profile(False, shared_way=way)
    qs = [rows(5 + j, (6, Hkv * G, 1, D), io) for j in range(4)]
    want = [cache.attend_shared(seqs, q) for q in qs]
    half = [cache.attend_shared(seqs[:3], q[:3]) for q in qs]
    q, out, part = qs[0].clone(), torch.empty_like(qs[0]), torch.empty_like(qs[0][:3])
    side = torch.cuda.Stream()
    graphs = []
    torch.cuda.synchronize()
    for call in (lambda: cache.attend_shared(seqs, q, out=out), lambda: cache.attend_shared(seqs[:3], q[:3], out=part)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            call()
        graphs.append(g)
    for j in (3, 1, 2, 0):
        q.copy_(qs[j])
        for g in graphs:
            g.replay()
        assert torch.equal(out, want[j]) and torch.equal(part, half[j])
    cache.check()
    cache.close()


@pytest.mark.parametrize("way", [0, 1, 2])
@pytest.mark.parametrize("fmt,io", [("f16", "f16"), ("q4_0", "f16"), ("f32", "f32")])
def test_attend_shared_many_calls_in_flight(kv, fmt, io, way):
    # the own pages run beside the shared ones, the next call's kernels are scheduled before this one has ended: 60 calls of two
    # batches without a synchronisation give the bits of the first, on either of two streams
    Hkv, G, D = 4, 4, 128
    cache, seqs = family(kv, fmt, io, Hkv, D, [1500, 200], 12, [3, 130, 64, 1], Hkv * G)
    cache.profile(False, shared_way=way)
    a, b = rows(5, (24, Hkv * G, 1, D), io), rows(6, (9, Hkv * G, 1, D), io)
    batches = [(seqs, a), (seqs[4:13], b)]
    want = [cache.attend_shared(*x) for x in batches]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), side):
        with torch.cuda.stream(stream):
            got = [cache.attend_shared(*batches[i % 2]) for i in range(60)]
        stream.synchronize()
        assert all(torch.equal(x, want[i % 2]) for i, x in enumerate(got))
    cache.check()
    cache.close()


@pytest.mark.parametrize("fmt,io", [("f16", "f16"), ("f32", "f32")])
def test_pages_past_four_gigabytes(kv, fmt, io):
    # a filler takes the first pages of the pool: what is shared, copied and read lies behind 2^32 bytes
    Hkv, G, D = 8, 4, 128
    size = 4 if fmt == "f32" else 2
    fill = (2 ** 32 // (2 * Hkv * D * size) + 63) // 64 * 64
    cache = kv.KvCache(fmt, Hkv, D, max_seqs=8, max_seq_tokens=fill, pool_tokens=fill + 8 * 640, max_q_heads=Hkv * G)
    filler = cache.new_seq()
    one = rows(1, (1, Hkv, 1, D), io)
    for at in range(0, fill, 2 ** 18):
        wide = one.expand(1, Hkv, min(2 ** 18, fill - at), D)
        cache.append([filler], wide, wide)
    parent = cache.new_seq()
    add(cache, [parent], 3, 400, io)
    seqs = cache.fork_shared([parent] * 4)
    add(cache, seqs, 5, 30, io)
    q = rows(7, (4, Hkv * G, 1, D), io)
    ref, size = reference(cache, seqs, q)
    for way in (0, 1, 2):
        cache.profile(False, shared_way=way)
        assert_close(cache.attend_shared(seqs, q), ref, size, io)
    cache.check()
    cache.close()


def test_children_of_empty_and_trimmed_parents(kv):
    Hkv, G, D = 2, 4, 128
    cache = kv.KvCache("f16", Hkv, D, max_seqs=12, max_seq_tokens=1024, max_q_heads=Hkv * G)
    empty, cut = cache.new_seq(), cache.new_seq()
    add(cache, [cut], 1, 700, "f16")
    cache.trim(cut, 250)
    kids = cache.fork_shared([empty, cut, empty, cut, cut])
    assert [cache.seq_len(s) for s in kids] == [0, 700, 0, 700, 700]
    add(cache, kids, 3, 70, "f16")
    q = rows(5, (5, Hkv * G, 1, D), "f16")
    for way in (0, 1, 2):
        cache.profile(False, shared_way=way)
        got = cache.attend_shared(kids, q)
        for i in (0, 2):  # nothing shared
            ref, size = reference(cache, [kids[i]], q[i:i + 1])
            assert_close(got[i:i + 1], ref, size, "f16")
        assert torch.equal(got, cache.attend(kids, q))  # the front of a trimmed sequence is gone: regular attention
    cache.check()
    cache.close()


@pytest.mark.parametrize("fmt,io", [("f16", "f16"), ("q8_1", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("way", [0, 1, 2])
def test_truncated_children_share_what_is_left(kv, fmt, io, way):
    # rolled back to different lengths, into pages that the others hold, and then on again: all in one call, twice
    Hkv, G, D = 2, 4, 128
    cache = kv.KvCache(fmt, Hkv, D, max_seqs=12, max_seq_tokens=1024, max_q_heads=Hkv * G)
    parent = cache.new_seq()
    add(cache, [parent], 1, 640, io)
    kids = cache.fork_shared([parent] * 6)
    for s, n in zip(kids, (640, 639, 321, 320, 64, 1)):
        cache.truncate(s, n)
    cache.profile(False, shared_way=way)
    batch = [parent] + kids
    for step in range(2):
        q = rows(5 + step, (7, Hkv * G, 1, D), io)
        ref, size = reference(cache, batch, q)
        assert_close(cache.attend_shared(batch, q), ref, size, io)
        add(cache, batch, 7 + 2 * step, 3, io)
    q = rows(9, (7, Hkv * G, 1, D), io)
    ref, size = reference(cache, batch, q)
    assert_close(cache.attend_shared(batch, q), ref, size, io)
    assert [cache.seq_len(s) for s in batch] == [646, 646, 645, 327, 326, 70, 7]
    cache.check()
    cache.close()


@pytest.mark.parametrize("way", [0, 1, 2])
def test_quantised_result_of_130_sequences(kv, way):
    # from 128 rows on the activation is laid out in tiles
    Hkv, G, D, n = 2, 2, 64, 130
    cache, seqs = family(kv, "f16", "f16", Hkv, D, [200], n, [3, 1], Hkv * G)
    cache.profile(False, shared_way=way)
    q = rows(5, (n, Hkv * G, 1, D), "f16")
    blocks = torch.randint(0, 256, (128, Hkv * G * D // 32, 18), dtype=torch.uint8, device="cuda")
    blocks[:, :, :2] = torch.full((128, Hkv * G * D // 32), 0.01, device="cuda").half().view(torch.uint8).reshape(128, -1, 2)
    lin = kv.Q40Linear(blocks, max_m=n)
    out, scratch = torch.empty_like(q), torch.empty_like(lin.scratch)
    cache.attend_shared(seqs, q, scratch=scratch, out=out)
    got = lin.gemm_quantized(n, scratch=scratch)
    assert torch.equal(got, lin.gemm(out.reshape(n, -1)))
    lin.check(scratch)
    cache.check()
    cache.close()


@pytest.mark.parametrize("fmt,io,D", [("f16", "f16", 128), ("bf16", "bf16", 64), ("q8_1", "f16", 128), ("f32", "f32", 64)])
@pytest.mark.parametrize("way", [0, 1, 2])
def test_what_lies_beyond_the_tokens_and_in_other_rows_stays_out(kv, fmt, io, D, way):
    # pages that held NaN and infinities before; a neighbour whose own keys, values or query are not numbers
    Hkv, G = 2, 4
    cache = kv.KvCache(fmt, Hkv, D, max_seqs=8, max_seq_tokens=1024, max_q_heads=Hkv * G, pool_tokens=1024)
    cache.profile(False, shared_way=way)
    dirty = cache.new_seq()
    bad = torch.full((1, Hkv, 1000, D), float("nan"), dtype=rows(1, (1,), io).dtype, device="cuda")
    if fmt != "q8_1":
        cache.append([dirty], bad, bad)
        bad.fill_(float("inf"))
        cache.truncate(dirty, 500)
    cache.append([dirty], bad[:, :, :500], bad[:, :, :500])
    cache.free_seq(dirty)
    parent = cache.new_seq()
    add(cache, [parent], 3, 330, io)
    kids = cache.fork_shared([parent] * 4)
    add(cache, kids, 5, 7, io)
    q = rows(7, (4, Hkv * G, 1, D), io)
    ref, size = reference(cache, kids, q)
    assert_close(cache.attend_shared(kids, q), ref, size, io)
    # one neighbour's query, then its newest token
    spoilt = q.clone()
    spoilt[1, 3] = float("inf")
    got = cache.attend_shared(kids, spoilt)
    others = [i for i in range(4) if i != 1]
    assert_close(got[others], ref[others], size[others], io)
    heads = [h for h in range(Hkv * G) if h != 3]
    assert_close(got[1, heads], ref[1, heads], size[1, heads], io)
    assert bool(got[1, 3].isnan().all())
    if fmt != "q8_1":
        add_bad = bad[:, :, :1]
        cache.append([kids[1]], add_bad, add_bad)
        got = cache.attend_shared(kids, q)
        assert_close(got[others], ref[others], size[others], io)
    cache.check()
    cache.close()


@pytest.mark.parametrize("way,kernels", [(1, {"decode", "combine"}), (2, {"prefix", "decode", "combine"})])
def test_timed_launches(kv, way, kernels):
    # an event pair around every launch stands between those that otherwise overlap: the same bits, and the records say what ran
    cache, seqs = family(kv, "f16", "f16", 2, 128, [700], 6, [5, 70], 8)
    q = rows(5, (6, 8, 1, 128), "f16")
    cache.profile(False, shared_way=way)
    want = cache.attend_shared(seqs, q)
    cache.profile(True, shared_way=way)
    assert torch.equal(cache.attend_shared(seqs, q), want)
    cache.fork_shared(seqs[:1])
    names = [name for name, ms in cache.profile_read() if ms > 0]
    assert set(names) == kernels | {"share"}
    cache.check()
    cache.close()


@pytest.mark.parametrize("fmt,io,D", [("f16", "f16", 64), ("q8_1", "f16", 128), ("f32", "f32", 64)])
@pytest.mark.parametrize("way", [0, 1, 2])
def test_thousands_of_rows_share_a_page(kv, fmt, io, D, way):
    n, G = 200, 40
    cache, seqs = family(kv, fmt, io, 1, D, [330], n, [2, 1], G)
    cache.profile(False, shared_way=way)
    q = rows(5, (n, G, 1, D), io)
    out = cache.attend_shared(seqs, q)
    ref, size = reference(cache, seqs, q)
    assert_close(out, ref, size, io)
    cache.check()
    cache.close()
