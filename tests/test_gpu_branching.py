"""Several continuations of one prompt through the decode loop: the prompt's pages shared, attended to together, the next tokens
drawn."""
import numpy as np
import pytest

from test_gpu_decoder import OracleDecoder
from test_gpu_sample import plain_row
from util import rel_err

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def small(n_seqs, **kw):
    from tract_b200.decoder import Decoder, Shape

    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    sh = Shape(hidden=256, n_layers=2, n_q_heads=4, n_kv_heads=2, head_dim=128, ffn=512, vocab=640, rope_theta=10000.0)
    return Decoder(sh, n_seqs=n_seqs, **kw)


SETTINGS = dict(temperature=[0.9, 1.3, 0.0, 0.7], top_k=[0, 50, 0, 40], top_p=[0.95, 1.0, 1.0, 0.9], min_p=[0.0, 0.02, 0.0, 0.0])


def drawn(dec):
    """The tokens that the settings, the last draws and the logits say, in 64 bits."""
    x, u, c = dec.logits.double().cpu().numpy(), dec.sampling["uniform"].cpu().numpy(), dec.sampling
    out = []
    for i in range(dec.B):
        token, gap = plain_row(x[i], float(c["temperature"][i]), int(c["top_k"][i]), float(c["top_p"][i]), float(c["min_p"][i]), float(u[i]))
        assert gap > 2.0 ** -36  # see checked() of the sampling tests
        out.append(token)
    return np.array(out, np.int32)


@pytest.mark.parametrize("way", [0, 1, 2])
@pytest.mark.parametrize("use_graphs", [False, True])
def test_continuations_of_one_prompt_against_the_oracle(way, use_graphs):
    dec = small(4, max_tokens=256, kv_format="f16", seed=11, use_graphs=use_graphs)
    for L in dec.layers:
        L["cache"].profile(False, shared_way=way)
    ref = OracleDecoder(dec)
    dec.set_sampling(seed=5, **SETTINGS)
    prompt = np.random.default_rng(4).integers(0, dec.shape.vocab, 150).astype(np.int32)
    free = dec.layers[0]["cache"].free_pages()
    dec.prefill_shared(torch.from_numpy(prompt))
    assert free - dec.layers[0]["cache"].free_pages() == 2 + 4  # two full pages once, the third for each

    def compare(want):
        got = dec.logits.cpu().numpy()
        # the bars of the decode-step test of test_gpu_decoder.py, for its reasons
        assert np.abs(got - want).mean() / np.sqrt((want ** 2).mean()) <= 1.2e-2 and rel_err(got, want) <= 0.06
        tokens = dec.tokens.cpu().numpy()
        assert np.array_equal(tokens, drawn(dec))
        return tokens

    for t in prompt:
        want = ref.step(np.full(4, t))
    tokens = compare(want)
    assert len(set(tokens.tolist())) > 1  # every row draws for itself
    for step in range(8):
        if step == 4:  # rows 0 and 1 go on from what row 1 holds, row 2 from row 0, row 3 stays
            parents = [1, 1, 0, 3]
            dec.branch(parents)
            tokens = tokens[parents]
            ref.K, ref.V = [k[parents] for k in ref.K], [v[parents] for v in ref.V]
            assert np.array_equal(dec.tokens.cpu().numpy(), tokens)
        want = ref.step(tokens)
        dec.step()
        tokens = compare(want)
    assert dec.lengths == [158] * 4 and dec.pos.tolist() == [158] * 4
    dec.check()
    dec.close()


@pytest.mark.parametrize("kv_format", ["f16", "bf16", "q8_1", "q4_0"])
def test_shared_pages_and_copies_give_the_same_bits(kv_format):
    # a short prompt is attended to by the regular kernels, whose split follows from the lengths alone: sharing changes no bit
    shared, copied = (small(4, max_tokens=300, kv_format=kv_format, seed=12, use_graphs=True) for _ in range(2))
    pages = shared.layers[0]["cache"].free_pages()
    prompt = torch.from_numpy(np.random.default_rng(6).integers(0, shared.shape.vocab, 130).astype(np.int32))
    for dec in (shared, copied):
        dec.set_sampling(seed=8, **SETTINGS)
        dec.prefill_shared(prompt)
    for i, L in enumerate(copied.layers):
        cache = L["cache"]
        for r in range(1, 4):
            cache.free_seq(copied.seqs[i][r])
            copied.seqs[i][r] = cache.fork(copied.seqs[i][0])
    copied.shared = False
    assert torch.equal(shared.tokens, copied.tokens)
    for step in range(70):  # the third page fills and a fourth begins
        for dec in (shared, copied):
            dec.step()
        assert torch.equal(shared.logits, copied.logits) and torch.equal(shared.tokens, copied.tokens), step
    for dec in (shared, copied):  # back into the prompt, and on with another one
        dec.truncate(100)
        dec.prefill(prompt[:9].expand(4, 9))
        dec.step()
    assert torch.equal(shared.logits, copied.logits)
    for dec in (shared, copied):
        dec.check()
        dec.reset()
        assert dec.layers[0]["cache"].free_pages() == pages
        dec.close()


def test_greedy_settings_and_the_way_back():
    prompt = torch.from_numpy(np.random.default_rng(7).integers(0, 640, (4, 20)).astype(np.int32))
    runs = {}
    for how in ("as made", "temperature 0", "top 1", "back"):
        dec = small(4, max_tokens=64, kv_format="f16", seed=13, use_graphs=how != "top 1")
        if how == "back":
            dec.set_sampling(temperature=3.0)
            dec.prefill(prompt)
            dec.step()
            dec.reset()
            dec.set_greedy()
        elif how != "as made":
            dec.set_sampling(**(dict(temperature=0.0) if how == "temperature 0" else dict(top_k=1)))
        dec.prefill(prompt)
        tokens = [dec.tokens.clone()]
        for _ in range(6):
            dec.step()
            tokens.append(dec.tokens.clone())
        runs[how] = torch.stack(tokens)
        dec.check()
        dec.close()
    for how in runs:
        assert torch.equal(runs[how], runs["as made"]), how


def test_beam_search_keeps_within_its_pages():
    # re-parenting at every step in caches that hold no page to spare: what nobody goes on from is given back first
    dec = small(4, max_tokens=128, kv_format="q8_1", seed=14, use_graphs=True)
    dec.set_sampling(seed=1, temperature=1.2)
    dec.prefill_shared(torch.from_numpy(np.random.default_rng(9).integers(0, 640, 64).astype(np.int32)))
    g = np.random.default_rng(10)
    for _ in range(60):
        dec.branch(g.integers(0, 4, 4))
        dec.step()
        assert torch.isfinite(dec.logits).all()
    dec.check()
    with pytest.raises(AssertionError):
        dec.branch([0, 1, 2])
    with pytest.raises(AssertionError):
        dec.branch([0, 1, 2, 4])
    dec.close()
