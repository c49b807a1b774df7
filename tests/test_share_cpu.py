"""Page sharing, attention over shared pages and sampling without a device: what the C entries refuse before they enqueue anything."""
import ctypes as C

import numpy as np
import pytest


@pytest.fixture(scope="module")
def kv():
    import tract_b200

    tract_b200.lib()
    return tract_b200


def refused(kv, rc, why):
    assert rc == 1 and why in kv.lib().b200kv_last_error(), (rc, kv.lib().b200kv_last_error())


def test_calls_without_a_cache(kv):
    L = kv.lib()
    ids, out = (C.c_int32 * 2)(0, 1), (C.c_int32 * 2)(-7, -7)
    strides = (C.c_int64 * 3)(1, 1, 1)
    refused(kv, L.b200kv_fork_shared(None, 2, ids, out, None), b"null")
    assert list(out) == [-7, -7]
    refused(kv, L.b200kv_seq_free_many(None, 2, ids), b"null")
    refused(kv, L.b200kv_attend_shared(None, 2, ids, 8, None, strides, None, None, 0, None, strides, None, 0, 0.0, None), b"null")


def test_sampling_arguments(kv):
    # host buffers stand in for tensors: every case is refused before a pointer is followed
    L = kv.lib()
    logits, uniform, out = (np.zeros(64, t) for t in (np.float32, np.float32, np.int32))
    p = lambda a: a.ctypes.data

    def call(logits=p(logits), stride=16, dtype=0, rows=4, n=16, uniform=p(uniform), out=p(out), scratch=None):
        return L.b200kv_sample(logits, stride, dtype, rows, n, None, None, None, None, uniform, out, scratch, None)

    for kw, why in ((dict(logits=None), b"null"), (dict(uniform=None), b"null"), (dict(out=None), b"null"), (dict(rows=0), b"positive"),
                    (dict(rows=-1), b"positive"), (dict(n=0), b"positive"), (dict(n=-5), b"positive"), (dict(rows=65536), b"at most 65535"),
                    (dict(n=2 ** 19 + 1, stride=2 ** 20), b"at most 524288"), (dict(dtype=-1), b"dtype"), (dict(dtype=3), b"dtype"),
                    (dict(stride=15), b"apart"), (dict(stride=-16), b"apart"), (dict(n=262145, stride=2 ** 19), b"workspace"),
                    (dict(scratch=8), b"aligned")):
        refused(kv, call(**kw), why)


def test_sampling_workspace_sizes(kv):
    L = kv.lib()
    size = L.b200kv_sample_scratch_bytes
    assert size(1, 1) == size(256, 128256) == size(65535, 262144) == 0
    for rows, n in ((1, 262145), (7, 300001), (100, 2 ** 19)):
        assert 4 * rows * n <= size(rows, n) <= 4 * rows * (n + 8 * 64)  # a row and little more
    for rows, n in ((0, 5), (5, 0), (-1, 5), (5, -1), (5, 2 ** 19 + 1)):
        assert size(rows, n) == -1
    with pytest.raises(kv.B200KvError, match="positive"):
        kv.sample_scratch(0, 5)


def test_marshalling_of_sequence_ids(kv):
    assert list(kv._ids([3, 1])) == [3, 1] and list(kv._ids(np.array([3, 1]))) == [3, 1]
    assert list(kv._ids([np.int64(5)])) == [5] and list(kv._ids((2,))) == [2]
    for ids in ([3, 1], np.array([3, 1]), (np.int64(3), 1), [3.0, 1.0]):
        assert np.frombuffer(kv._id_bytes(ids), np.int32).tolist() == [3, 1]
    assert kv._id_bytes([]) == b""
    with pytest.raises(OverflowError):
        kv._id_bytes([2 ** 31])


def test_marshalling_of_strides(kv):
    import torch

    t = torch.empty((2, 3, 5, 8))
    assert np.frombuffer(kv._stride_bytes(t), np.int64).tolist() == [120, 40, 8] == list(kv._strides(t, 3))
    assert np.frombuffer(kv._stride_bytes(t[:, ::2].expand(2, 2, 5, 8)), np.int64).tolist() == [120, 80, 8]
    with pytest.raises(kv.B200KvError, match="contiguous"):
        kv._stride_bytes(t.transpose(2, 3))
    assert np.frombuffer(kv._stride_bytes(t[..., :1]), np.int64).tolist() == [120, 40, 8]
