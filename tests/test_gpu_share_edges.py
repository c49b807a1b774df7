"""attend_shared where its ways could part: scores far from 0."""
import pytest

from test_gpu_share import assert_close, kv, reference, rows  # noqa: F401 (kv is a fixture)

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
