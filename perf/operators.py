"""What is measured of the paged key/value cache and of the attention that reads it.

Three operators, as a program that serves ragged batches of sequences calls them:

  append   the keys and values of new tokens are written into the pages of a cache, as they are or as 8-bit integers with
           a scale for each token and head, and read back
  read     whole sequences are read back from the cache, packed one after another
  attend   attention of each sequence's newest tokens over all of its cached ones (a chunk of a prompt, or one token)

A sequence b holds kv_lens[b] tokens, token t of it in page page_table[b, t // page] at place t % page. Its new tokens are
the last cu_new[b + 1] - cu_new[b] of them; new tokens of all sequences are packed one after another.
"""
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _case(name, op, batch, new, kv, heads, d, dtype, cache, page, causal=True, lens=1):
    """`new` and `kv` are (least, most) of the new and of the earlier tokens of a sequence, `heads` (query, key) heads."""
    return {"name": name, "op": op, "batch": batch, "new_lo": new[0], "new_hi": new[1], "kv_lo": kv[0], "kv_hi": kv[1],
            "heads_q": heads[0], "heads_kv": heads[1], "d": d, "dtype": dtype, "cache": cache, "page": page,
            "causal": causal, "lens": lens}


def listed():
    return [
        # one decoding step of a few sequences: four tokens are written, latency is all there is
        _case("append_step_int8", "append", 4, (1, 1), (100, 900), (32, 8), 128, "bf16", "int8", 16),
        # the prompt chunks of a busy batch, quantised as they are written
        _case("append_chunk_int8", "append", 16, (700, 2048), (0, 3000), (32, 8), 128, "bf16", "int8", 16),
        # a large ragged prefill written unquantised, every head its own keys
        _case("append_prefill_fp16", "append", 8, (1000, 4096), (0, 0), (16, 16), 64, "fp16", "same", 64),
        # sequences handed to another worker: all of their tokens out of an 8-bit cache
        _case("read_int8", "read", 8, (0, 0), (4000, 16384), (32, 8), 128, "bf16", "int8", 16),
        # one short sequence out of a 16-bit cache
        _case("read_short_fp16", "read", 1, (0, 0), (513, 513), (16, 16), 64, "fp16", "same", 64),
        # a lone user's next token, short context: latency
        _case("attend_lone_token", "attend", 1, (1, 1), (128, 128), (32, 8), 128, "bf16", "same", 16),
        # a decoding step of a full batch of ragged contexts
        _case("attend_tokens_bf16", "attend", 32, (1, 1), (200, 4095), (32, 8), 128, "bf16", "same", 16),
        # a decoding step over long contexts in an 8-bit cache
        _case("attend_tokens_int8", "attend", 16, (1, 1), (2000, 16383), (32, 8), 128, "bf16", "int8", 64),
        # decoding where every query head has its own keys
        _case("attend_tokens_fp16_d64", "attend", 8, (1, 1), (300, 2047), (16, 16), 64, "fp16", "same", 64),
        # a mixed step: new prompts, chunks of older ones and a few tokens, together
        _case("attend_mixed_fp16", "attend", 12, (1, 1500), (0, 6000), (16, 4), 128, "fp16", "same", 32),
        # chunks of two long prompts over an 8-bit cache
        _case("attend_chunk_int8", "attend", 2, (1023, 2048), (5000, 9000), (32, 8), 128, "bf16", "int8", 16),
        # the largest: a chunk of a long prompt
        _case("attend_chunk_bf16", "attend", 1, (4096, 4096), (12288, 12288), (32, 8), 128, "bf16", "same", 16),
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["append", "read", "attend", "attend"])
    dtype, cache = rng.choice(["fp16", "bf16"]), rng.choice(["same", "int8"])
    d, page = rng.choice([64, 128]), rng.choice([16, 32, 64, 128])
    heads = rng.choice([(32, 8), (16, 16), (16, 4), (8, 1), (12, 4), (20, 4)])
    if op == "append":
        new = _between(rng, 1, 2048)
        return _case("", op, rng.randint(1, 16), (max(1, new // 2), new), (0, _between(rng, 1, 4096)), heads, d, dtype,
                     cache, page, lens=rng.randrange(1 << 20))
    if op == "read":
        kv = _between(rng, 100, 16384)
        return _case("", op, rng.randint(1, 8), (0, 0), (max(1, kv // 3), kv), heads, d, dtype, cache, page,
                     lens=rng.randrange(1 << 20))
    if rng.random() < 0.5:  # single tokens
        kv = _between(rng, 64, 16384)
        batch = max(1, min(32, (1 << 17) // kv, rng.randint(1, 32)))
        return _case("", op, batch, (1, 1), (kv // 4, kv), heads, d, dtype, cache, page, lens=rng.randrange(1 << 20))
    new, kv, most = _between(rng, 2, 4096), _between(rng, 16, 12288), 32 * 4096 * 16384  # `most`: the largest listed case's
    kv = min(kv, most // (heads[0] * new) - new)
    batch = rng.randint(1, max(1, min(8, most // (heads[0] * new * (new + kv)))))
    return _case("", op, batch, (max(1, new // 3), new), (kv // 4, kv), heads, d, dtype, cache, page,
                 causal=rng.random() < 0.8, lens=rng.randrange(1 << 20))


def _lengths(case):
    """(new tokens, all tokens) of each sequence."""
    rng = random.Random(case["lens"])
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["batch"])]
    old = [rng.randint(case["kv_lo"], case["kv_hi"]) for _ in range(case["batch"])]
    return new, [a + b for a, b in zip(new, old)]


# ------------------------------------------------------------------------------------------------ plain forms


def _quantise(x):
    """8-bit integers and scales of x (..., d) in 32 bits: x ~ q * scale with scale = max|x| / 127 over d, at least 2^-100."""
    top = x.abs().amax(-1, keepdim=True).clamp_min(127.0 * 2.0 ** -100)
    return torch.round(x * 127.0 / top).to(torch.int8), (top / 127.0).squeeze(-1)


def _gather(state, cache, scale, b, pos):
    """The cached vectors of all heads at the positions `pos` of the sequences `b`, in 32 bits."""
    page = cache.shape[2]
    ids, place = state["page_table"][b, (pos // page).long()].long(), (pos % page).long()
    x = cache[ids, :, place].float()
    return x if scale is None else x * scale[ids, :, place][..., None]


def _places(state):
    """(sequence, position in it) of each of the packed new tokens."""
    i = torch.arange(state["total"], device=state["cu_new"].device, dtype=torch.int32)
    b = torch.searchsorted(state["cu_new"][1:].contiguous(), i, right=True)
    return b, state["kv_lens"][b] - state["cu_new"][b + 1] + i


def _plain_append(state):
    b, pos = _places(state)
    page = state["k_cache"].shape[2]
    ids, place = state["page_table"][b, (pos // page).long()].long(), (pos % page).long()
    for x, cache, scale in ((state["k"], state["k_cache"], state["k_scale"]), (state["v"], state["v_cache"], state["v_scale"])):
        if scale is None:
            cache[ids, :, place] = x
        else:
            cache[ids, :, place], scale[ids, :, place] = _quantise(x.float())
    return _plain_read(state)


def _plain_read(state):
    b, pos = _places(state)
    return tuple(_gather(state, state[c], state[s], b, pos).to(state["dtype"]) for c, s in (("k_cache", "k_scale"), ("v_cache", "v_scale")))


def _plain_attend(state):
    hq, d = state["q"].shape[1:]
    hkv = state["k_cache"].shape[1]
    batch, n, dev = state["kv_lens"].shape[0], state["max_new"], state["q"].device
    b, pos = _places(state)
    start = state["kv_lens"] - (state["cu_new"][1:] - state["cu_new"][:-1])
    # the new tokens padded to (batch, most of them), the query heads of one key head beside each other
    q = torch.zeros(batch, n, hq, d, device=dev)
    q[b, (pos - start[b]).long()] = state["q"].float()
    rows = q.view(batch, n, hkv, hq // hkv, d).transpose(1, 2).reshape(batch, hkv, -1, d)
    t = torch.arange(state["max_kv"], device=dev)
    inside = t < state["kv_lens"][:, None]
    k, v = (_gather(state, state[c], state[s], torch.arange(batch, device=dev)[:, None], torch.where(inside, t, 0)).transpose(1, 2)
            for c, s in (("k_cache", "k_scale"), ("v_cache", "v_scale")))
    s = (rows @ k.transpose(-1, -2)).mul_(d ** -0.5).view(batch, hkv, n, hq // hkv, -1)
    seen = inside[:, None]
    if state["causal"]:
        seen = seen & (t <= start[:, None, None] + torch.arange(n, device=dev)[:, None])
    s.masked_fill_(~seen[:, None, :, None], float("-inf"))
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    o = (s.view(batch, hkv, n * (hq // hkv), -1) @ v).view(batch, hkv, n, hq // hkv, d) / s.sum(-1, keepdim=True)
    return o.transpose(1, 2).reshape(batch, n, hq, d)[b, (pos - start[b]).long()].to(state["dtype"])


# ------------------------------------------------------------------------------------------------ what is measured


def prepare(case, seed):
    dev, dtype = torch.device("cuda"), DTYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    new, kv = _lengths(case)
    if case["op"] == "read":
        new = kv
    page, h, d = case["page"], case["heads_kv"], case["d"]
    need = [-(-n // page) for n in kv]
    table = torch.full((case["batch"], max(need) + 1), -1, dtype=torch.int32)
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    def cache(loud):
        # one vector in a hundred is eight times as long, as keys are met with
        x = normal(pages, h, page, d)
        if loud:
            x *= torch.where(torch.rand(pages, h, page, 1, device=dev, generator=g) < 0.01, 8.0, 1.0)
        if case["cache"] == "same":
            return x.to(dtype), None
        return _quantise(x.to(dtype).float())

    k_cache, k_scale = cache(True)
    v_cache, v_scale = cache(False)
    total = sum(new)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    state = {"op": case["op"], "dtype": dtype, "causal": case["causal"], "max_new": max(new), "max_kv": max(kv), "total": total,
             "k_cache": k_cache, "k_scale": k_scale, "v_cache": v_cache, "v_scale": v_scale, "page_table": table.to(dev),
             "kv_lens": torch.tensor(kv, dtype=torch.int32, device=dev), "cu_new": torch.tensor(cu, dtype=torch.int32, device=dev)}
    if case["op"] == "append":
        state["k"], state["v"] = normal(total, h, d).to(dtype), normal(total, h, d).to(dtype)
    if case["op"] == "attend":
        state["q"] = normal(total, case["heads_q"], d).to(dtype)
    return state


def run(state):
    if not own:
        return {"append": _plain_append, "read": _plain_read, "attend": _plain_attend}[state["op"]](state)
    cuda_attn = _package()
    where = (state["k_cache"], state["v_cache"], state["page_table"], state["kv_lens"], state["cu_new"])
    scales = {"k_scale": state["k_scale"], "v_scale": state["v_scale"]}
    if state["op"] == "attend":
        return cuda_attn.paged_attn(state["q"], *where, **scales, causal=state["causal"], max_new=state["max_new"])
    if state["op"] == "append":
        cuda_attn.paged_append(state["k"], state["v"], *where, **scales)
    return cuda_attn.paged_read(*where, state["total"], dtype=state["dtype"], **scales)


def _package():
    import sys
    if "phantom-a100_b200" not in sys.path:
        sys.path.insert(0, "phantom-a100_b200")
    import cuda_attn
    return cuda_attn


def work(case):
    new, kv = _lengths(case)
    if case["op"] == "read":
        new = kv
    h, d = case["heads_kv"], case["d"]
    held = 2 * h * (2 * d if case["cache"] == "same" else d + 4)  # a token's keys and values in the cache
    plain = 2 * h * 2 * d                                         # and as 16-bit vectors
    if case["op"] == "append":
        return {"bytes": sum(new) * 2 * (plain + held), "flops": 0}
    if case["op"] == "read":
        return {"bytes": sum(new) * (plain + held), "flops": 0}
    pairs = sum(n * (t - n) + n * (n + 1) // 2 if case["causal"] else n * t for n, t in zip(new, kv))
    return {"bytes": sum(kv) * held + sum(new) * 2 * case["heads_q"] * 2 * d, "flops": 4 * d * case["heads_q"] * pairs}


# ------------------------------------------------------------------------------------------------ the definition, in 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    new, kv = _lengths(case)
    if case["op"] == "read":
        new = kv
    if case["op"] == "attend" and case["heads_q"] * max(a * b for a, b in zip(new, kv)) > 1 << 31:
        return None  # the products of one sequence would take tens of gigabytes
    page = case["page"]
    out, keys, values, at = [], [], [], 0
    for b, (n, t) in enumerate(zip(new, kv)):
        ids = state["page_table"][b, :-(-t // page)].long()

        def sequence(name):
            x = state[name + "_cache"][ids].double()
            if case["cache"] == "int8":
                x = x * state[name + "_scale"][ids].double().unsqueeze(-1)
            return x.transpose(0, 1).flatten(1, 2)[:, :t]  # (heads, tokens, d)

        if case["op"] == "append":
            for name, into in (("k", keys), ("v", values)):
                x = state[name][at:at + n].double()
                if case["cache"] == "int8":
                    top = torch.clamp(x.abs().max(-1, keepdim=True).values, min=127 * 2.0 ** -100)
                    x = torch.round(127 * x / top) * top / 127
                into.append(x)
        elif case["op"] == "read":
            keys.append(sequence("k").transpose(0, 1))
            values.append(sequence("v").transpose(0, 1))
        else:
            share = case["heads_q"] // case["heads_kv"]
            k, v = (sequence(name).repeat_interleave(share, 0) for name in ("k", "v"))
            w = torch.einsum("ihd,hjd->hij", state["q"][at:at + n].double(), k) / case["d"] ** 0.5
            if case["causal"]:
                last = torch.arange(t - n, t, device=w.device)[:, None]
                w = w.masked_fill(torch.arange(t, device=w.device) > last, -torch.inf)
            out.append(torch.einsum("hij,hjd->ihd", torch.softmax(w, -1), v))
        at += n
    return torch.cat(out) if case["op"] == "attend" else (torch.cat(keys), torch.cat(values))
