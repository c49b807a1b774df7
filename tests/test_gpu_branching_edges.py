"""The decode loop's branch() and set_sampling() where they are refused."""
import numpy as np
import pytest

from test_gpu_branching import small

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("use_graphs", [False, True])
def test_a_refused_branch_changes_nothing(use_graphs):
    # The rows were rolled back into a page that all of them hold: each new continuation needs a copy, none of the dropped ones
    # gives a page back, and the last layer has too few.
    import tract_b200 as kv

    dec, twin = (small(4, max_tokens=320, kv_format="f16", seed=21, use_graphs=use_graphs) for _ in range(2))
    cache = kv.KvCache("f16", 2, 128, max_seqs=8, max_seq_tokens=320, pool_tokens=64)  # 1 + 8 pages
    dec.layers[1]["cache"].close()
    dec.layers[1]["cache"], dec.seqs[1] = cache, [cache.new_seq() for _ in range(4)]
    prompt = torch.from_numpy(np.random.default_rng(3).integers(0, 640, 130).astype(np.int32))
    for d in (dec, twin):
        d.set_sampling(temperature=1.3, seed=4)
        d.prefill_shared(prompt)
        d.truncate(100)
    filler = cache.new_seq()
    x = torch.zeros((1, 2, 320, 128), dtype=torch.float16, device="cuda")
    cache.append([filler], x, x)
    free = [L["cache"].free_pages() for L in dec.layers]
    assert free[1] == 2
    before = ([list(s) for s in dec.seqs], list(dec.lengths), dec.tokens.clone(), dec.pos.clone())
    for parents in ([0, 0, 0, 0], [2, 2, 2, 2]):
        with pytest.raises(kv.B200KvError, match="exhausted"):
            dec.branch(parents)
        assert dec.seqs == before[0] and dec.lengths == before[1]
        assert torch.equal(dec.tokens, before[2]) and torch.equal(dec.pos, before[3])
        assert [L["cache"].free_pages() for L in dec.layers] == free
    cache.free_seq(filler)
    for parents in (None, [3, 3, 3, 3], [1, 0, 1, 2], None):  # and on, as if nothing had been tried
        for d in (dec, twin):
            if parents:
                d.branch(parents)
            d.step()
        assert torch.equal(dec.logits, twin.logits) and torch.equal(dec.tokens, twin.tokens)
    for d in (dec, twin):
        d.check()
        d.close()


def test_refused_settings_leave_the_draws_alone():
    dec, twin = (small(4, max_tokens=64, kv_format="f16", seed=22, use_graphs=True) for _ in range(2))
    prompt = torch.from_numpy(np.random.default_rng(5).integers(0, 640, (4, 9)).astype(np.int32))
    for d in (dec, twin):
        d.set_sampling(temperature=1.5, seed=6)
        d.prefill(prompt)
    for _ in range(3):
        with pytest.raises(AssertionError):
            dec.set_sampling(temperature=[1.0, 1.0], seed=6)  # two settings for four sequences
        for d in (dec, twin):
            d.step()
        assert torch.equal(dec.sampling["uniform"], twin.sampling["uniform"]) and torch.equal(dec.tokens, twin.tokens)
    for d in (dec, twin):
        d.check()
        d.close()
