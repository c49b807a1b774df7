"""attend_shared where its ways could part: scores far from 0, the range of bf16 queries over quantised pages;
the distance from regular attention; waits that run out; refusals."""
import pytest

from test_gpu_share import assert_close, family, kv, reference, rows  # noqa: F401 (kv is a fixture)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("way", [1, 2])
@pytest.mark.parametrize("fmt,io,size", [("f16", "f16", 2000.0), ("f16", "f16", 9000.0), ("bf16", "bf16", 1e8), ("q8_1", "f16", 9000.0), ("q4_0", "f16", 9000.0),
                                         ("f32", "f32", 1e8)])
@pytest.mark.parametrize("D", [64, 128])
def test_scores_far_from_zero(kv, fmt, io, size, D, way):
    # A step of a score is a millionth and less of what the two largest scores of a row lie apart (by about a tenth of their
    # size over the rows of a few hundred keys, a thousandth in the worst of 200 rows): one key has all of the weight.
    Hkv, G, n = 2, 7, 6
    cache = kv.KvCache(fmt, Hkv, D, max_seqs=2 * n + 2, max_seq_tokens=1024, max_q_heads=Hkv * G)
    cache.profile(False, shared_way=way)
    k, v = rows(11, (1, Hkv, 640, D), io, scale=size), rows(12, (1, Hkv, 640, D), io)
    k_own, v_own = rows(13, (n, Hkv, 30, D), io, scale=size), rows(14, (n, Hkv, 30, D), io)
    q = rows(5, (n, Hkv * G, 1, D), io, scale=size)
    below = (q.abs(), -k.abs(), -k_own.abs())  # no score near 0
    for queries, keys, own in ((q, k, k_own), below):
        parent = cache.new_seq()
        cache.append([parent], keys, v)
        seqs = cache.fork_shared([parent] * n)
        cache.append(seqs, own, v_own)
        ref, weight = reference(cache, seqs, queries)
        assert_close(cache.attend_shared(seqs, queries), ref, weight, io)
        cache.free_seqs([parent, *seqs])
    cache.check()
    cache.close()


@pytest.mark.parametrize("fmt", ["q8_1", "q4_0"])
@pytest.mark.parametrize("D,own,way", [(64, [5, 70], 1), (64, [5, 70], 2), (64, [0], 2), (128, [0], 2)])
def test_bf16_queries_of_any_magnitude_over_quantised_pages(kv, fmt, D, own, way):
    # the scale of the call brings the scores back, so that the bound of the ordinary magnitudes holds for all of them.  (At
    # head_dim 128 nothing goes through the decode kernel, which takes f16 queries over such pages.)
    cache, seqs = family(kv, fmt, "bf16", 2, D, [640], 6, own, 14)
    cache.profile(False, shared_way=way)
    q = rows(5, (6, 14, 1, D), "bf16", scale=1.3)
    for size in (1e6, 1e20, 1e35, 1e-7, 1e-20, 1e-35):
        far = (q.float() * size).bfloat16()
        scale = D ** -0.5 / size
        ref, weight = reference(cache, seqs, far, scale=scale)
        assert_close(cache.attend_shared(seqs, far, scale=scale), ref, weight, "bf16")
    # one channel far above the others, one row far above its neighbours; a row of zeros
    mixed = q.clone()
    mixed[:, :, :, 3] *= 300.0
    mixed[2] *= 2.0 ** 40
    mixed[4, 1] = 0
    ref, weight = reference(cache, seqs, mixed, scale=2.0 ** -10)
    out = cache.attend_shared(seqs, mixed, scale=2.0 ** -10)
    others = [0, 1, 3, 4, 5]
    assert_close(out[others], ref[others], weight[others], "bf16")
    assert torch.isfinite(out).all()  # (row 2 sees one key alone or a tie)
    # ordinary magnitudes keep their bits when the power of two is another one
    assert torch.equal(cache.attend_shared(seqs, q, scale=0.125), cache.attend_shared(seqs, q * 2, scale=0.0625))
    cache.check()
    cache.close()


@pytest.mark.parametrize("fmt,io", [("f16", "f16"), ("bf16", "bf16"), ("q8_1", "f16"), ("q8_1", "bf16"), ("q4_0", "f16"), ("q8_1", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("way", [1, 2])
def test_distance_from_regular_attention(kv, fmt, io, D, way):
    # Both are off from the exact result by no more than assert_close allows, of which half a step of the result and two of the
    # weights and values are counted twice here; a flat row (many weights of the same size) beside peaked ones.
    cache, seqs = family(kv, fmt, io, 2, D, [1300], 8, [5, 70], 8)
    q = rows(5, (8, 8, 1, D), io, scale=1.3)
    q[0] = 0
    q[1] *= 4
    want = cache.attend(seqs, q)
    cache.profile(False, shared_way=way)
    got = cache.attend_shared(seqs, q)
    cache.check()
    ref, size = reference(cache, seqs, q)
    if io == "f32":
        bound = 2 * (2.0 ** -24 * ref.abs() + 2.0 ** -17 * size)
    else:
        bound = torch.finfo(got.dtype).eps * ref.abs() + 2 * (2.0 ** -10 + 2.0 ** -15) * size
    assert bool(((got.double() - want.double()).abs() <= bound).all())
    cache.close()


@pytest.mark.parametrize("fmt,io,D,n", [("f16", "f16", 128, 6), ("bf16", "bf16", 64, 6), ("q8_1", "f16", 128, 6), ("q4_0", "bf16", 64, 40), ("f16", "f16", 128, 40),
                                        ("f32", "f32", 128, 6), ("f32", "f32", 64, 40)])
@pytest.mark.parametrize("way", [0, 1, 2])
def test_a_wait_that_runs_out_is_reported_and_the_cache_stays_usable(kv, fmt, io, D, n, way):
    # one CTA of kv head 0 issues none of its copies and gives up after 1 ms: what the others hold is not touched by it
    Hkv, G = 2, 4
    cache, seqs = family(kv, fmt, io, Hkv, D, [1500], n, [5, 70, 130], Hkv * G)
    cache.profile(False, shared_way=way)
    q = rows(5, (n, Hkv * G, 1, D), io)
    good = cache.attend_shared(seqs, q)
    cache.check()
    cache.profile(False, shared_way=way, stall_next_decode=True)
    short = cache.attend_shared(seqs, q)  # about 1 ms longer; a run of pages is missing from some rows of kv head 0
    with pytest.raises(kv.B200KvError, match="bounded wait expired"):
        cache.check()
    cache.check()  # reported once
    assert torch.equal(short[:, G:], good[:, G:]) and torch.isfinite(short[:, :G]).all() and not torch.equal(short[:, :G], good[:, :G])
    for _ in range(2):  # the hook is spent
        assert torch.equal(cache.attend_shared(seqs, q), good)
        cache.check()
    ref, size = reference(cache, seqs, q)
    assert_close(cache.attend(seqs, q), ref, size, io)
    cache.check()
    cache.close()


@pytest.mark.parametrize("way", [0, 1, 2])
def test_a_batch_with_an_empty_sequence_is_refused_whole(kv, way):
    # more than 256 sequences are served in parts: nothing of the first part is written when a later one holds the empty sequence
    n = 280
    cache, seqs = family(kv, "f16", "f16", 1, 64, [130], n, [3], 2)
    cache.profile(False, shared_way=way)
    empty = cache.new_seq()
    q, out = rows(5, (n + 1, 2, 1, 64), "f16"), torch.full((n + 1, 2, 1, 64), 3.25, dtype=torch.float16, device="cuda")
    for at in (n, 256, 255, 0):
        with pytest.raises(kv.B200KvError, match="is empty"):
            cache.attend_shared(seqs[:at] + [empty] + seqs[at:], q, out=out)
    torch.cuda.synchronize()
    assert bool((out == 3.25).all())
    cache.check()
    cache.close()
