"""Measured cases of the operators that run several continuations of one prompt.

    fork_shared    sequences that hold the pages of their parent by reference (copied where a page is partly filled)
    attend_shared  decode attention of a batch whose sequences begin with the same cached tokens
    sample         the next token from logits: temperature, top-k, top-p, min-p, a given uniform number per row

A case of kind "attend" is one attention call, "branch" is the first step of new continuations (fork, append one token,
attend, free the continuations again), "sample" is one sampling call.
"""
import math

import numpy as np
import torch

own = False

KV_BYTES = {"f32": lambda d: 4 * d, "f16": lambda d: 2 * d, "bf16": lambda d: 2 * d,
            "q8_1": lambda d: d + d // 16, "q4_0": lambda d: d // 2 + d // 16}  # one row of one head
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def attend_case(fmt, io, groups, per_group, prefix, own_max, hq, hkv, d):
    return dict(kind="attend", fmt=fmt, io=io, groups=groups, per_group=per_group, prefix=prefix, own_max=own_max, hq=hq, hkv=hkv, d=d)


def branch_case(fmt, io, groups, per_group, prefix, hq, hkv, d):
    return dict(kind="branch", fmt=fmt, io=io, groups=groups, per_group=per_group, prefix=prefix, own_max=1, hq=hq, hkv=hkv, d=d)


def sample_case(io, rows, n, pad, mode):
    return dict(kind="sample", io=io, rows=rows, n=n, pad=pad, mode=mode)


def listed():
    return [
        # four short conversations behind a system prompt of odd length, f32 cache, small heads: latency
        dict(name="attend-f32-4x515", **attend_case("f32", "f32", 1, 4, 515, 40, 8, 2, 64)),
        # eight samples of one 2048-token prompt
        dict(name="attend-f16-8x2048", **attend_case("f16", "f16", 1, 8, 2048, 128, 32, 8, 128)),
        # a full serving batch behind one 8k document
        dict(name="attend-bf16-64x8192", **attend_case("bf16", "bf16", 1, 64, 8192, 512, 32, 8, 128)),
        # 32 questions to one long context, int8 cache
        dict(name="attend-q8-32x32768", **attend_case("q8_1", "f16", 1, 32, 32768, 256, 32, 8, 128)),
        # three prompts of odd length with five continuations each, 4-bit cache, seven query heads per kv head, head_dim 64
        dict(name="attend-q4-3x5x5003", **attend_case("q4_0", "f16", 3, 5, 5003, 200, 14, 2, 64)),
        # a prompt pass has ended: four first tokens are drawn and continued
        dict(name="branch-f16-4x1000", **branch_case("f16", "f16", 1, 4, 1000, 32, 8, 128)),
        # eight beams of each of four prompts
        dict(name="branch-bf16-4x8x2085", **branch_case("bf16", "bf16", 4, 8, 2085, 32, 8, 128)),
        # sixteen branches of a long int8 context
        dict(name="branch-q8-16x16421", **branch_case("q8_1", "f16", 1, 16, 16421, 32, 8, 128)),
        # one conversation, nucleus sampling
        dict(name="sample-f32-1-top_p", **sample_case("f32", 1, 128256, 0, "top_p")),
        # eight samples of one prompt, the usual combination of filters
        dict(name="sample-f32-8-top_k_p", **sample_case("f32", 8, 128256, 0, "top_k_p")),
        # half-precision logits of an odd vocabulary in padded rows, min-p
        dict(name="sample-bf16-48-min_p", **sample_case("bf16", 48, 50257, 7, "min_p")),
        # a large serving batch in which every request brings settings of its own
        dict(name="sample-f32-256-mixed", **sample_case("f32", 256, 128256, 0, "mixed")),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "branch", "sample", "sample"])
    if kind == "sample":
        io, mode = rng.choice(["f32", "f32", "f16", "bf16"]), rng.choice(["top_p", "top_k", "top_k_p", "min_p", "plain", "greedy", "mixed"])
        return sample_case(io, _log(rng, 1, 256), _log(rng, 1000, 128256), rng.choice([0, 0, 1, 8, 13]), mode)
    fmt = rng.choice(["f32", "f16", "f16", "bf16", "q8_1", "q4_0"])
    io = fmt if fmt in DTYPES else rng.choice(["f16", "f16", "bf16"])
    hq, hkv, d = rng.choice([(32, 8, 128), (32, 8, 128), (8, 2, 64), (14, 2, 64), (16, 16, 128), (24, 3, 128)])
    seqs = _log(rng, 2, 64)
    groups = rng.choice([1, 1, 2, 4]) if seqs >= 8 else 1
    prefix = _log(rng, 64, 32768 if kind == "attend" else 16384)
    prefix = min(prefix, 64 * 8192 * 32 * 128 // (seqs * hq * d), 32768 // groups)  # no more than the largest listed case
    if kind == "branch":
        return branch_case(fmt, io, groups, max(1, seqs // groups), prefix, hq, hkv, d)
    return attend_case(fmt, io, groups, max(1, seqs // groups), prefix, _log(rng, 1, 512), hq, hkv, d)


def own_lengths(case):
    """Tokens of its own that each sequence holds: spread over 1 .. own_max."""
    return [1 + (i * 7919 + 13) % case["own_max"] for i in range(case["groups"] * case["per_group"])]


# ---- inputs ---------------------------------------------------------------------------------------------

def _quantise_q8_1(x):
    """Blocks of 32 channels: the value of largest magnitude over 127 as the scale, codes rounded half away from zero."""
    b = x.float().unflatten(-1, (-1, 32))
    big = b.gather(-1, b.abs().argmax(-1, keepdim=True))
    scale = big / 127.0
    r = torch.where(scale == 0, torch.zeros_like(scale), 1.0 / scale)
    v = b * r
    code = torch.where(v < 0, torch.ceil(v - 0.5), torch.floor(v + 0.5)).clamp(-128, 127)
    return code.to(torch.int8).flatten(-2), scale.squeeze(-1).half()


def _quantise_q4_0(x):
    """Blocks of 32 channels: the value of largest magnitude over -8 as the scale, codes 0 .. 15 (stored here minus 8)."""
    b = x.float().unflatten(-1, (-1, 32))
    big = b.gather(-1, b.abs().argmax(-1, keepdim=True))
    scale = big / -8.0
    r = torch.where(scale == 0, torch.zeros_like(scale), 1.0 / scale)
    code = torch.trunc(b * r + 8.5).clamp(max=15) - 8
    return code.to(torch.int8).flatten(-2), scale.squeeze(-1).half()


def _store(fmt, x):
    """What a cache of this format holds for the rows x: the rows themselves, or codes and scales."""
    if fmt == "q8_1":
        return _quantise_q8_1(x)
    if fmt == "q4_0":
        return _quantise_q4_0(x)
    return (x,)


def _rows(case, seed):
    """Keys and values of the prompts and of each continuation, and the queries, as a model gives them to the cache."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    g, n, hkv, d, dt = case["groups"], case["per_group"], case["hkv"], case["d"], DTYPES[case["io"]]
    longest = max(own_lengths(case))

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    # a few channels of the keys are large, as in trained models; queries that attend to some keys more than to others
    loud = torch.where(torch.rand((1, hkv, 1, d), generator=gen, device="cuda") < 0.03, 4.0, 1.0)
    k_prefix, v_prefix = (normal(g, hkv, case["prefix"], d) * loud).to(dt), normal(g, hkv, case["prefix"], d).to(dt)
    k_own, v_own = (normal(g * n, hkv, longest, d) * loud).to(dt), normal(g * n, hkv, longest, d).to(dt)
    q = (normal(g * n, case["hq"], 1, d) * 1.25).to(dt)
    return k_prefix, v_prefix, k_own, v_own, q


def _logits(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, n = case["rows"], case["n"]

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device="cuda")

    # the bulk of a vocabulary around zero, some dozens of tokens that fit the context well above it
    x = torch.randn((rows, n + case["pad"]), generator=gen, device="cuda") * 2.2
    fits = torch.randint(0, n, (rows, 48), generator=gen, device="cuda")
    x.scatter_add_(1, fits, 3.0 + 9.0 * uniform(rows, 48) * uniform(rows, 48))
    logits = x.to(DTYPES[case["io"]])[:, :n]
    # random numbers away from 0: the token of a number of exactly 0 is the first one whose weight is not 0 at all
    u = (uniform(rows) * 0.99999 + 5e-6).float()
    mode = torch.full((rows,), {"plain": 0, "top_p": 1, "top_k": 2, "top_k_p": 3, "min_p": 4, "greedy": 5, "mixed": 0}[case["mode"]], device="cuda")
    if case["mode"] == "mixed":
        mode = torch.randint(0, 6, (rows,), generator=gen, device="cuda")
    temperature = torch.where(mode == 5, 0.0, 0.5 + 0.7 * uniform(rows)).float()
    top_k = torch.where((mode == 2) | (mode == 3), torch.randint(2, 200, (rows,), generator=gen, device="cuda"), 0).to(torch.int32)
    top_p = torch.where((mode == 1) | (mode == 3), 0.6 + 0.39 * uniform(rows), 1.0).float()
    min_p = torch.where(mode == 4, 0.02 + 0.1 * uniform(rows), 0.0).float()
    return dict(logits=logits, uniform=u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)


def prepare(case, seed):
    if case["kind"] == "sample":
        state = dict(case=case, **_logits(case, seed))
        state["out"] = torch.empty(case["rows"], dtype=torch.int32, device="cuda")
        if own:
            import tract_b200 as kv
            state["scratch"] = kv.sample_scratch(case["rows"], case["n"])
        return state
    k_prefix, v_prefix, k_own, v_own, q = _rows(case, seed)
    n, lens = case["per_group"], own_lengths(case)
    state = dict(case=case, q=q, lens=torch.tensor(lens, device="cuda"))
    if case["kind"] == "branch":
        state.update(k_new=k_own, v_new=v_own)
    if not own:  # the tensors that hold what the cache holds
        state.update(k_prefix=_store(case["fmt"], k_prefix), v_prefix=_store(case["fmt"], v_prefix))
        if case["kind"] == "attend":
            state.update(k_own=_store(case["fmt"], k_own), v_own=_store(case["fmt"], v_own))
        return state
    import tract_b200 as kv
    total = len(lens)
    cache = kv.KvCache(case["fmt"], case["hkv"], case["d"], max_seqs=total + case["groups"], max_seq_tokens=case["prefix"] + max(lens) + 1,
                       pool_tokens=case["groups"] * (case["prefix"] + 64) + total * (max(lens) + 128), max_q_heads=case["hq"])
    parents = [cache.new_seq() for _ in range(case["groups"])]
    cache.append(parents, k_prefix, v_prefix)
    state.update(cache=cache, parents=[p for p in parents for _ in range(n)])
    if case["kind"] == "attend":  # the continuations are under way: each has its own tokens behind the prompt's
        seqs = cache.fork_shared(state["parents"])
        for i, s in enumerate(seqs):
            cache.append([s], k_own[i:i + 1, :, :lens[i]], v_own[i:i + 1, :, :lens[i]])
        state["out"] = torch.empty_like(q)
        state["step"] = cache.prepared_attend_shared(seqs, q, state["out"])
    return state


# ---- one pass -------------------------------------------------------------------------------------------

def _values(stored):
    if len(stored) == 1:
        return stored[0].float()
    codes, scales = stored
    return (codes.float().unflatten(-1, (-1, 32)) * scales.float().unsqueeze(-1)).flatten(-2)


def _attend_plain(case, q, k_prefix, v_prefix, k_own, v_own, lens):
    g, n, hkv, d = case["groups"], case["per_group"], case["hkv"], case["d"]
    h = case["hq"] // hkv
    kp, vp, ko, vo = _values(k_prefix), _values(v_prefix), _values(k_own), _values(v_own)
    rows = q.float().reshape(g, n, hkv, h, d)
    scale = 1.0 / math.sqrt(d)
    # against the prompt: all rows of a kv head at once; against the own tokens: each sequence for itself
    by_head = rows.permute(0, 2, 1, 3, 4).reshape(g, hkv, n * h, d)
    s_prefix = (by_head @ kp.transpose(-1, -2)) * scale
    s_prefix = s_prefix.reshape(g, hkv, n, h, -1).permute(0, 2, 1, 3, 4).reshape(g * n, hkv, h, -1)
    s_own = (rows.reshape(g * n, hkv, h, d) @ ko.transpose(-1, -2)) * scale
    hidden = torch.arange(s_own.shape[-1], device=q.device) >= lens[:, None]
    s_own = s_own.masked_fill(hidden[:, None, None, :], -math.inf)
    s = torch.cat([s_prefix, s_own], -1)
    w = torch.exp(s - s.amax(-1, keepdim=True))
    total = w.sum(-1, keepdim=True)
    w_prefix, w_own = w[..., :s_prefix.shape[-1]], w[..., s_prefix.shape[-1]:]
    w_by_head = w_prefix.reshape(g, n, hkv, h, -1).permute(0, 2, 1, 3, 4).reshape(g, hkv, n * h, -1)
    o = (w_by_head @ vp).reshape(g, hkv, n, h, d).permute(0, 2, 1, 3, 4).reshape(g * n, hkv, h, d) + w_own @ vo
    return (o / total).reshape(q.shape).to(q.dtype)


def _sample_plain(logits, uniform, temperature, top_k, top_p, min_p, out):
    """Weights, their sums and the comparisons with them in 64 bits: a token lies next to its neighbours' borders."""
    x = logits.double()
    w = torch.exp((x - x.amax(-1, keepdim=True)) / temperature.double().clamp_min(1e-30)[:, None])
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    sorted_w = w.gather(-1, order)
    rank = torch.arange(x.shape[1], device=x.device)[None, :]
    in_k = (rank < top_k[:, None]) | (top_k <= 0)[:, None]
    sorted_k = sorted_w * in_k
    before = torch.cumsum(sorted_k, -1) - sorted_k
    # kept as long as the mass before it has not reached p; the first one always
    in_p = (before < top_p.double()[:, None] * sorted_k.sum(-1, keepdim=True)) | (top_p >= 1)[:, None] | (rank == 0)
    keep_sorted = in_k & in_p & (sorted_w >= min_p.double()[:, None])
    kept = w * torch.zeros_like(keep_sorted).scatter(-1, order, keep_sorted)
    cdf = torch.cumsum(kept, -1)
    token = (cdf <= uniform.double()[:, None] * cdf[:, -1:]).sum(-1)
    out.copy_(torch.where(temperature > 0, token, order[:, 0]))
    return out


def run(state):
    case = state["case"]
    if case["kind"] == "sample":
        args = [state[k] for k in ("logits", "uniform", "temperature", "top_k", "top_p", "min_p")]
        if own:
            import tract_b200 as kv
            return kv.sample(*args, out=state["out"], scratch=state["scratch"])
        return _sample_plain(*args, state["out"])
    if case["kind"] == "attend":
        if own:
            state["step"]()
            return state["out"]
        return _attend_plain(case, state["q"], *(state[k] for k in ("k_prefix", "v_prefix", "k_own", "v_own", "lens")))
    if own:
        cache = state["cache"]
        seqs = cache.fork_shared(state["parents"])
        cache.append(seqs, state["k_new"], state["v_new"])
        out = cache.attend_shared(seqs, state["q"])
        cache.free_seqs(seqs)
        return out
    k_new, v_new = _store(case["fmt"], state["k_new"]), _store(case["fmt"], state["v_new"])
    return _attend_plain(case, state["q"], state["k_prefix"], state["v_prefix"], k_new, v_new, state["lens"])


def work(case):
    if case["kind"] == "sample":
        n = case["rows"] * case["n"]
        return {"bytes": n * (4 if case["io"] == "f32" else 2) + 24 * case["rows"], "flops": 4 * n}
    lens, hkv, d = own_lengths(case), case["hkv"], case["d"]
    token = 2 * hkv * KV_BYTES[case["fmt"]](d)
    elem = 4 if case["io"] == "f32" else 2
    moved = 2 * len(lens) * case["hq"] * d * elem + (case["groups"] * case["prefix"] + sum(lens)) * token
    if case["kind"] == "branch":  # the new tokens come in, and each continuation gets the last, partly filled page of its own
        moved += len(lens) * (2 * hkv * d * elem + (case["prefix"] % 64) * token)
    return {"bytes": moved, "flops": 4 * case["hq"] * d * (len(lens) * case["prefix"] + sum(lens))}


def exact(case, seed):
    if case["kind"] == "sample":
        return None  # whole numbers
    k_prefix, v_prefix, k_own, v_own, q = _rows(case, seed)
    fmt, n, lens = case["fmt"], case["per_group"], own_lengths(case)

    def held(x):
        s = _store(fmt, x)
        if len(s) == 1:
            return x.double()
        return (s[0].double().reshape(*x.shape[:-1], -1, 32) * s[1].double()[..., None]).reshape(x.shape)

    h = case["hq"] // case["hkv"]
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    for i, length in enumerate(lens):  # one sequence after the other over all its tokens
        k = held(torch.cat([k_prefix[i // n], k_own[i, :, :length]], 1))
        v = held(torch.cat([v_prefix[i // n], v_own[i, :, :length]], 1))
        s = torch.einsum("hgd,htd->hgt", q[i, :, 0].double().reshape(case["hkv"], h, -1), k) / np.sqrt(case["d"])
        p = torch.softmax(s, -1)
        out[i, :, 0] = torch.einsum("hgt,htd->hgd", p, v).reshape(case["hq"], -1)
    return out
