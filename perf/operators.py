"""What the cache-shrinking operators cost: decode attention that adds up the weight every
cached token receives, eviction by those weights, and the latent cache (append, absorbed
attention over it, expanded attention for prompts).

``listed()`` names the measured cases, ``draw()`` gives more of the same ranges.  ``run()``
computes a case in its plain form, or through flashspec_b200 where ``own`` is true; both
take what ``prepare()`` makes.  ``work()`` is what a pass cannot do without, ``exact()`` the
result in 64 bits.
"""

import math

import torch

own = False


# ----------------------------------------------------------------------------- the cases


def listed():
    return [
        # One short request of a small model on one GPU: the latency of a step.
        {"name": "weights_one", "op": "weights", "batch": 1, "q_heads": 8, "kv_heads": 2, "dim": 64, "page": 16,
         "longest": 129, "shortest": 129, "format": "affine", "dtype": "bfloat16"},
        # A serving batch with grouped heads, lengths falling from 8192 to 128.
        {"name": "weights_ragged", "op": "weights", "batch": 64, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "longest": 8192, "shortest": 128, "format": "affine", "dtype": "float16"},
        # Two very long contexts, eight query heads a kv head.
        {"name": "weights_long", "op": "weights", "batch": 2, "q_heads": 64, "kv_heads": 8, "dim": 128, "page": 16,
         "longest": 131072, "shortest": 131072, "format": "symmetric", "dtype": "float16"},
        # The same serving batch cut to 1000 tokens a request: most requests shrink, the short ones stay.
        {"name": "evict_ragged", "op": "evict", "batch": 64, "kv_heads": 8, "dim": 128, "page": 16, "longest": 8192,
         "shortest": 128, "budget": 1000, "recent": 128, "sinks": 4, "format": "affine"},
        # The two long contexts cut to an eighth.
        {"name": "evict_long", "op": "evict", "batch": 2, "kv_heads": 8, "dim": 128, "page": 16, "longest": 131072,
         "shortest": 131072, "budget": 16384, "recent": 1024, "sinks": 16, "format": "symmetric"},
        # A decode step: one new token of each live request.
        {"name": "append_step", "op": "append", "batch": 64, "tokens": 1, "latent": 512, "rope": 64, "page": 64,
         "longest": 1024, "ragged": False, "dtype": "bfloat16"},
        # Prompts entering the cache, padded to the longest.
        {"name": "append_prompts", "op": "append", "batch": 8, "tokens": 4096, "latent": 512, "rope": 64, "page": 64,
         "longest": 100, "ragged": True, "dtype": "float16"},
        # One short request, the heads that one of eight GPUs holds.
        {"name": "latent_one", "op": "latent", "batch": 1, "tokens": 1, "heads": 16, "latent": 512, "rope": 64,
         "page": 64, "longest": 777, "shortest": 777, "dtype": "float16"},
        # The ragged serving batch over a latent cache.
        {"name": "latent_ragged", "op": "latent", "batch": 64, "tokens": 1, "heads": 16, "latent": 512, "rope": 64,
         "page": 64, "longest": 8192, "shortest": 128, "dtype": "bfloat16"},
        # Two query tokens a request (a drafted one beside the last) and every head on one GPU.
        {"name": "latent_wide", "op": "latent", "batch": 16, "tokens": 2, "heads": 64, "latent": 512, "rope": 64,
         "page": 64, "longest": 8192, "shortest": 4096, "dtype": "float16"},
        # Short chunks behind a cached prefix.
        {"name": "prompt_chunks", "op": "prompt", "batch": 3, "heads": 8, "nope": 64, "rope": 32, "value": 64,
         "longest": 130, "shortest": 1, "prefix": 200, "dtype": "float16"},
        # Whole prompts of different lengths, packed.
        {"name": "prompt_packed", "op": "prompt", "batch": 4, "heads": 16, "nope": 128, "rope": 64, "value": 128,
         "longest": 4096, "shortest": 500, "prefix": 0, "dtype": "bfloat16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["weights", "evict", "append", "latent", "prompt"])
    kinds = ["float16", "bfloat16"]
    if op == "weights":
        kv, group = rng.choice([1, 2, 8, 32]), rng.choice([1, 2, 3, 4, 8])
        batch = _log(rng, 1, 64)
        longest = _log(rng, 16, max(64, min(131072, 2000000 // (batch * kv * group))))
        dim, page = rng.choice([(128, 16), (128, 16), (64, 16), (64, 32), (32, 16), (256, 32)])
        return {"op": op, "batch": batch, "q_heads": kv * group, "kv_heads": kv, "dim": dim, "page": page,
                "longest": longest, "shortest": rng.randint(0, longest), "format": rng.choice(["affine", "symmetric"]),
                "dtype": rng.choice(kinds)}
    if op == "evict":
        batch, kv = _log(rng, 1, 64), rng.choice([1, 2, 8, 32])
        longest = _log(rng, 64, max(128, min(131072, 2000000 // (batch * kv))))
        budget = rng.randint(longest // 16 + 1, longest)
        recent = rng.randint(0, budget)
        dim, page = rng.choice([(128, 16), (128, 16), (64, 16), (64, 32), (256, 32)])
        return {"op": op, "batch": batch, "kv_heads": kv, "dim": dim, "page": page, "longest": longest,
                "shortest": rng.randint(0, longest), "budget": budget, "recent": recent,
                "sinks": rng.randint(0, min(64, budget - recent)), "format": rng.choice(["affine", "symmetric"])}
    latent, rope = rng.choice([(512, 64), (512, 64), (256, 32), (128, 64)])
    page = rng.choice([16, 32, 64])
    if op == "append":
        batch = _log(rng, 1, 64)
        tokens = _log(rng, 1, 32768 // batch)
        return {"op": op, "batch": batch, "tokens": tokens, "latent": latent, "rope": rope, "page": page,
                "longest": _log(rng, 1, 2000), "ragged": rng.random() < 0.5, "dtype": rng.choice(kinds)}
    if op == "latent":
        batch, heads, tokens = _log(rng, 1, 64), _log(rng, 1, 128), rng.choice([1, 1, 1, 2, 3])
        rows = heads * tokens
        longest = _log(rng, 16, max(32, min(65536, 500000 // batch, 12000000 // (batch * rows))))
        return {"op": op, "batch": batch, "tokens": tokens, "heads": heads, "latent": latent, "rope": rope,
                "page": page, "longest": longest, "shortest": rng.randint(0, longest), "dtype": rng.choice(kinds)}
    nope, rope, value = rng.choice([(128, 64, 128), (128, 64, 128), (64, 32, 64), (128, 32, 64), (64, 64, 128)])
    batch, heads = _log(rng, 1, 6), rng.choice([1, 4, 7, 16])
    longest = _log(rng, 1, 4096)
    return {"op": op, "batch": batch, "heads": heads, "nope": nope, "rope": rope, "value": value, "longest": longest,
            "shortest": rng.randint(1, longest), "prefix": rng.choice([0, 0, rng.randint(1, 1000)]),
            "dtype": rng.choice(kinds)}


def _lengths(case):
    """Lengths falling evenly from the longest to the shortest."""
    b, hi, lo = case["batch"], case["longest"], case["shortest"]
    return [hi if b == 1 else int(round(hi - (hi - lo) * i / (b - 1))) for i in range(b)]


def _counts(case):
    """New tokens of each request of an append: all, or falling to a few."""
    b, t = case["batch"], case["tokens"]
    return [t if not case["ragged"] else max(1, t - (t * i) // b) for i in range(b)]


# ------------------------------------------------------------------------------- inputs


def _table(lengths, page, gen):
    """A block table with pages of the pool in random order, -1 behind a request's pages."""
    need = [(n + page - 1) // page for n in lengths]
    total = max(1, sum(need))
    perm = torch.randperm(total, generator=gen, device="cuda")
    cols = max(1, max(need))
    col = torch.arange(cols, device="cuda")
    need_t = torch.tensor(need, device="cuda")
    first = torch.cumsum(need_t, 0) - need_t
    at = (first[:, None] + col).clamp_max(total - 1)
    return torch.where(col < need_t[:, None], perm[at], torch.full_like(at, -1)), total


def _pool(pages, heads, page, dim, form, gen):
    """int8 pages of normal values with their scales (and zero points)."""
    values = torch.empty((pages, heads, page, dim), dtype=torch.int8, device="cuda")
    scale = torch.empty((pages, heads, page if form == "symmetric" else 1), device="cuda")
    zero = torch.zeros((pages, heads), dtype=torch.int16, device="cuda")
    step = max(1, (1 << 25) // (heads * page * dim))
    for i in range(0, pages, step):
        x = torch.randn(values[i:i + step].shape, generator=gen, device="cuda")
        if form == "symmetric":
            s = (x.abs().amax(-1) / 127.0).clamp_min(1e-8)
            values[i:i + step] = (x / s[..., None]).round().clamp(-127, 127).to(torch.int8)
            scale[i:i + step] = s
        else:
            lo, hi = x.amin((2, 3)), x.amax((2, 3))
            s = ((hi - lo) / 255.0).clamp_min(1e-8)
            z = (-lo / s).round().clamp(0, 255)
            u = (x / s[..., None, None] + z[..., None, None]).round().clamp(0, 255)
            values[i:i + step] = (u - 128).to(torch.int8)
            scale[i:i + step, :, 0] = s
            zero[i:i + step] = z.to(torch.int16)
    return {"values": values, "scale": scale, "zero": zero}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, case.get("dtype", "float32"))

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda").to(dtype)

    s = {"case": case}
    if case["op"] in ("weights", "evict"):
        lengths = _lengths(case)
        s["table"], pages = _table(lengths, case["page"], gen)
        s["lengths"] = torch.tensor(lengths, device="cuda")
        for kv in ("k", "v"):
            s[kv] = _pool(pages, case["kv_heads"], case["page"], case["dim"], case["format"], gen)
        shape = (pages, case["kv_heads"], case["page"])
        # weights received so far: a few heavy tokens, many light ones
        s["weights"] = torch.randn(shape, generator=gen, device="cuda").mul_(2).sub_(5).exp_()
        if case["op"] == "weights":
            s["q"] = normal(case["batch"], case["q_heads"], case["dim"])
        else:  # tokens that no step has looked at yet have weight zero
            s["weights"] *= torch.rand(shape, generator=gen, device="cuda") > 0.02
            s["moved"] = torch.zeros_like(s["weights"])
        return s
    if case["op"] == "append":
        b, t, page = case["batch"], case["tokens"], case["page"]
        held = [max(0, case["longest"] - 3 * i) for i in range(b)]
        counts = _counts(case)
        s["table"], pages = _table([h + c for h, c in zip(held, counts)], page, gen)
        s["lengths"], s["counts"] = torch.tensor(held, device="cuda"), torch.tensor(counts, device="cuda")
        s["latent"], s["rope"] = normal(b, t, case["latent"]), normal(b, t, case["rope"])
        s["values"] = torch.zeros((pages, page, case["latent"]), dtype=torch.int8, device="cuda")
        s["scale"] = torch.zeros((pages, page), device="cuda")
        s["ropes"] = torch.zeros((pages, page, case["rope"]), dtype=dtype, device="cuda")
        return s
    if case["op"] == "latent":
        lengths = _lengths(case)
        s["table"], pages = _table(lengths, case["page"], gen)
        s["lengths"] = torch.tensor(lengths, device="cuda")
        pool = _pool(pages, 1, case["page"], case["latent"], "symmetric", gen)
        s["values"], s["scale"] = pool["values"][:, 0], pool["scale"][:, 0].contiguous()
        s["ropes"] = normal(pages, case["page"], case["rope"])
        s["q"] = normal(case["batch"], case["tokens"], case["heads"], case["latent"])
        s["q_rope"] = normal(case["batch"], case["tokens"], case["heads"], case["rope"])
        s["sm_scale"] = (case["latent"] + case["rope"]) ** -0.5
        return s
    lens = _lengths(case)
    keys = [n + case["prefix"] for n in lens]
    s["longest_q"], s["longest_k"] = max(lens), max(keys)

    def offsets(n):
        return torch.cumsum(torch.tensor([0] + n, device="cuda"), 0)

    s["q_offsets"], s["k_offsets"] = offsets(lens), offsets(keys)
    s["q"] = normal(sum(lens), case["heads"], case["nope"] + case["rope"])
    s["kv"] = normal(sum(keys), case["heads"], case["nope"] + case["value"])
    s["k_rope"] = normal(sum(keys), case["rope"])
    s["sm_scale"] = (case["nope"] + case["rope"]) ** -0.5
    return s


# --------------------------------------------------------------------------- plain forms


def _softmax(scores, seen):
    """Softmax over the last axis of the scores that are seen; rows that see nothing give zeros."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, torch.ones_like(total))


def _values(pool, pages):
    """The fp32 values of the listed pages: [..., heads, page, dim]."""
    x = pool["values"][pages].float()
    if pool["scale"].shape[-1] > 1:
        return x * pool["scale"][pages][..., None]
    return (x + 128.0 - pool["zero"][pages].float()[..., None, None]) * pool["scale"][pages][..., None]


def _plain_weights(s):
    q, table = s["q"], s["table"]
    b, hq, d = q.shape
    hkv, page = s["weights"].shape[1:]
    pages = table.clamp_min(0)
    tokens = table.shape[1] * page
    k = _values(s["k"], pages).transpose(1, 2).reshape(b, hkv, tokens, d)
    seen = torch.arange(tokens, device="cuda") < s["lengths"][:, None]
    scores = (q.float().view(b, hkv, hq // hkv, d) @ k.transpose(2, 3)) * d ** -0.5
    del k
    p = _softmax(scores, seen[:, None, None])
    del scores
    v = _values(s["v"], pages).transpose(1, 2).reshape(b, hkv, tokens, d)
    out = (p @ v).view(b, hq, d).to(q.dtype)
    got = p.sum(2).view(b, hkv, -1, page).transpose(1, 2)
    s["weights"].index_add_(0, pages.reshape(-1), got.reshape(-1, hkv, page))  # zeros behind a request's pages
    return {"out": out, "weights": s["weights"]}


def _plain_evict(s):
    case, table, lengths = s["case"], s["table"], s["lengths"]
    b, cols = table.shape
    hkv, page, budget = case["kv_heads"], case["page"], case["budget"]
    pages = table.clamp_min(0)
    tokens = cols * page
    w = s["weights"][pages].transpose(1, 2).reshape(b, hkv, tokens)
    pos = torch.arange(tokens, device="cuda")
    n = lengths[:, None]
    always = (pos < case["sinks"]) | (pos >= n - case["recent"]) | (n <= budget)
    key = w.masked_fill(always[:, None], math.inf).masked_fill((pos >= n)[:, None], -1.0)
    slots = torch.arange(budget, device="cuda")
    best = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :budget]
    count = lengths.clamp_max(budget)
    valid = (slots[: best.shape[-1]] < count[:, None])[:, None]  # as many as there are
    best = torch.sort(best.masked_fill(~valid, tokens), dim=-1).values
    kept = torch.full((b, hkv, budget), -1, dtype=torch.int32, device="cuda")
    kept[..., : best.shape[-1]] = torch.where(best < tokens, best, torch.full_like(best, -1)).int()

    npg = (budget + page - 1) // page  # the pages that may be rewritten
    fill = torch.full((b, hkv, npg * page), -1, dtype=torch.int64, device="cuda")
    fill[..., :budget] = kept
    live = fill >= 0
    at = fill.clamp_min(0)
    src_page = torch.gather(pages[:, None].expand(b, hkv, cols), 2, at // page)
    heads = torch.arange(hkv, device="cuda")[None, :, None].expand_as(at)
    row = at % page
    stays = ((fill == torch.arange(npg * page, device="cuda")) | ~live).view(b, hkv, npg, page).all(-1)
    write = (~stays).nonzero(as_tuple=True)
    dst = pages[write[0], write[2]], write[1]
    for kv in ("k", "v"):
        pool = s[kv]
        x = pool["values"][src_page, heads, row]
        if case["format"] == "symmetric":
            x = x.masked_fill(~live[..., None], 0)
            sc = pool["scale"][src_page, heads, row].masked_fill(~live, 1e-8)
            pool["values"][dst] = x.view(b, hkv, npg, page, -1)[write]
            pool["scale"][dst] = sc.view(b, hkv, npg, page)[write]
            continue
        z = pool["zero"][src_page, heads].float()[..., None]
        x = ((x.float() + 128.0 - z) * pool["scale"][src_page, heads]).masked_fill(~live[..., None], 0.0)
        x = x.view(b, hkv, npg, page, -1)[write]
        lo, hi = x.amin((1, 2)), x.amax((1, 2))
        sc = ((hi - lo) / torch.full_like(hi, 255.0)).clamp_min(1e-8)
        z = (-lo / sc).round().clamp(0, 255)
        u = (x / sc[:, None, None] + z[:, None, None]).round().clamp(0, 255)
        pool["values"][dst] = (u - 128).to(torch.int8)
        pool["scale"][dst] = sc[:, None]
        pool["zero"][dst] = z.to(torch.int16)
    moved = torch.zeros((b, hkv, tokens), device="cuda")
    moved[..., : min(tokens, npg * page)] = torch.gather(w, 2, at).masked_fill(~live, 0.0)[..., :tokens]
    held = table >= 0
    s["moved"][table[held]] = moved.view(b, hkv, cols, page).transpose(1, 2)[held]
    # codes move (or are computed again) bit for bit by the format's rule: whole numbers
    return {"kept": kept, "weights": s["moved"], "k": s["k"]["values"], "k_scale": s["k"]["scale"],
            "k_zero": s["k"]["zero"], "v": s["v"]["values"], "v_scale": s["v"]["scale"], "v_zero": s["v"]["zero"]}


def _plain_append(s):
    x = s["latent"].float()
    b, t, _ = x.shape
    page = s["values"].shape[1]
    top = x.abs().amax(-1)
    scale = (top / torch.full_like(top, 127.0)).clamp_min(1e-8)
    codes = (x / scale[..., None]).round().clamp(-127, 127)
    step = torch.arange(t, device="cuda")
    new = step < s["counts"][:, None]
    pos = (s["lengths"][:, None] + step)[new]
    row = torch.arange(b, device="cuda")[:, None].expand(b, t)[new]
    at = s["table"][row, pos // page], pos % page
    s["values"][at] = codes[new].to(torch.int8)
    s["scale"][at] = scale[new]
    s["ropes"][at] = s["rope"][new]
    held = (codes * scale[..., None]).masked_fill(~new[..., None], 0.0).to(s["latent"].dtype)
    return {"held": held, "scale": s["scale"], "rope": s["ropes"]}


def _plain_latent(s):
    q, q_rope = s["q"].float(), s["q_rope"].float()
    b, t, h, dc = q.shape
    pages = s["table"].clamp_min(0)
    c = (s["values"][pages].float() * s["scale"][pages][..., None]).flatten(1, 2)
    r = s["ropes"][pages].float().flatten(1, 2)
    scores = (q.view(b, t * h, dc) @ c.mT + q_rope.view(b, t * h, -1) @ r.mT) * s["sm_scale"]
    last = s["lengths"][:, None] - t + 1 + torch.arange(t, device="cuda")  # tokens that query t sees
    seen = torch.arange(c.shape[1], device="cuda") < last.repeat_interleave(h, 1)[..., None]
    return (_softmax(scores, seen) @ c).view(b, t, h, dc).to(s["q"].dtype)


def _plain_prompt(s):
    q, kv, dn = s["q"].float(), s["kv"].float(), s["case"]["nope"]
    qo, ko = s["q_offsets"], s["k_offsets"]
    nq, nk = qo[1:] - qo[:-1], ko[1:] - ko[:-1]
    i, j = torch.arange(s["longest_q"], device="cuda"), torch.arange(s["longest_k"], device="cuda")
    in_q, in_k = i < nq[:, None], j < nk[:, None]
    qi = (qo[:-1, None] + i).clamp_max(q.shape[0] - 1)
    kj = (ko[:-1, None] + j).clamp_max(kv.shape[0] - 1)
    qp, kvp, rp = q[qi].transpose(1, 2), kv[kj].transpose(1, 2), s["k_rope"].float()[kj]
    scores = qp[..., :dn] @ kvp[..., :dn].mT + qp[..., dn:] @ rp[:, None].mT
    seen = (j <= i[:, None] + (nk - nq)[:, None, None]) & in_k[:, None]
    out = _softmax(scores * s["sm_scale"], seen[:, None]) @ kvp[..., dn:]
    return out.transpose(1, 2)[in_q].to(s["q"].dtype)


_PLAIN = {"weights": _plain_weights, "evict": _plain_evict, "append": _plain_append, "latent": _plain_latent,
          "prompt": _plain_prompt}


# ------------------------------------------------------------------------ the framework's


def _paged_cache(fs, s):
    """The cache handle a program keeps; built on the first pass over a state."""
    if "cache" not in s:
        case = s["case"]

        def pool(p):
            pages, heads, page, dim = p["values"].shape
            if case["format"] == "symmetric":
                return fs.SymQuantizedTensor(p["values"], p["scale"], page, (pages, heads, page, dim))
            one = (pages, heads, 1, 1, 1)
            return fs.QuantizedTensor(p["values"].view(pages, heads, 1, page, dim), p["scale"].view(one),
                                      p["zero"].view(one), page, (pages, heads, page, dim))

        s["cache"] = fs.PagedKVCache(pool(s["k"]), pool(s["v"]), s["table"], s["lengths"], case["page"],
                                     case["longest"])
    return s["cache"]


def _own(s):
    import flashspec_b200 as fs

    case = s["case"]
    if case["op"] == "weights":
        out = fs.paged_quant_attention_weights_cuda(s["q"], _paged_cache(fs, s), s["weights"])
        return {"out": out, "weights": s["weights"]}
    if case["op"] == "evict":
        _, kept = fs.evict_tokens_cuda(_paged_cache(fs, s), s["weights"], case["budget"], recent=case["recent"],
                                       sinks=case["sinks"], weights_out=s["moved"])
        return {"kept": kept, "weights": s["moved"], "k": s["k"]["values"], "k_scale": s["k"]["scale"],
                "k_zero": s["k"]["zero"], "v": s["v"]["values"], "v_scale": s["v"]["scale"],
                "v_zero": s["v"]["zero"]}
    if case["op"] == "prompt":
        return fs.latent_prefill_attention_cuda(s["q"], s["kv"], s["k_rope"], s["q_offsets"], s["k_offsets"],
                                                sm_scale=s["sm_scale"])
    if "cache" not in s:
        longest = case["longest"] + (case["tokens"] if case["op"] == "append" else 0)
        s["cache"] = fs.LatentKVCache(s["values"], s["scale"], s["ropes"], s["table"], s["lengths"], longest)
    if case["op"] == "append":
        _, held = s["cache"].append(s["latent"], s["rope"], s["counts"], return_held=True)
        return {"held": held, "scale": s["scale"], "rope": s["ropes"]}
    return fs.latent_attention_cuda(s["q"], s["q_rope"], s["cache"], sm_scale=s["sm_scale"])


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------- work


def work(case):
    op = case["op"]
    if op == "prompt":
        lens = _lengths(case)
        h, dn, dr, dv = case["heads"], case["nope"], case["rope"], case["value"]
        pairs = sum(n * case["prefix"] + n * (n + 1) // 2 for n in lens)
        nq, nk = sum(lens), sum(lens) + case["prefix"] * len(lens)
        return {"bytes": 2 * (nq * h * (dn + dr + dv) + nk * (h * (dn + dv) + dr)),
                "flops": 2 * pairs * h * (dn + dr + dv)}
    if op == "append":
        tokens, dc, dr = sum(_counts(case)), case["latent"], case["rope"]
        return {"bytes": tokens * (2 * dc + 2 * dr + dc + 4 + 2 * dr + 2 * dc), "flops": 4 * tokens * dc}
    lens = _lengths(case)
    if op == "latent":
        dc, dr, rows = case["latent"], case["rope"], case["tokens"] * case["heads"]
        return {"bytes": sum(lens) * (dc + 4 + 2 * dr) + 2 * len(lens) * rows * (2 * dc + dr),
                "flops": 2 * sum(lens) * rows * (2 * dc + dr)}
    hkv, d = case["kv_heads"], case["dim"]
    per_token = 4 if case["format"] == "symmetric" else 6 / case["page"]  # scale (and zero point)
    if op == "weights":
        return {"bytes": sum(lens) * hkv * (2 * (d + per_token) + 8) + 4 * len(lens) * case["q_heads"] * d,
                "flops": 4 * sum(lens) * case["q_heads"] * d}
    cut = [n for n in lens if n > case["budget"]]
    moved = len(cut) * hkv * case["budget"]
    return {"bytes": sum(lens) * hkv * 4 + moved * (2 * 2 * (d + per_token) + 8), "flops": 4 * moved * d}


# -------------------------------------------------------------------------- in 64 bits


def _attend64(q, k, v, seen, sm_scale):
    """softmax(q k^T) and its product with v, rows [R, D] over tokens [N, D], in 64 bits."""
    a = torch.einsum("...rd,...nd->...rn", q, k) * sm_scale
    a = torch.where(seen, a, torch.tensor(-math.inf, dtype=torch.float64, device="cuda"))
    p = torch.nan_to_num(torch.softmax(a, -1), nan=0.0)
    return p, torch.einsum("...rn,...nd->...rd", p, v)


def _tokens64(pool, pages, n):
    """The first n tokens of a request's pages, [heads, n, dim]."""
    x = pool["values"][pages].double()
    if pool["scale"].shape[-1] > 1:
        x = x * pool["scale"][pages].double()[..., None]
    else:
        x = (x + 128 - pool["zero"][pages].double()[..., None, None]) * pool["scale"][pages].double()[..., None]
    return x.transpose(0, 1).flatten(1, 2)[:, :n]


def _exact_weights(s, case):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    weights = s["weights"].double()
    hkv, page, d = case["kv_heads"], case["page"], case["dim"]
    for b, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        pages = s["table"][b, : (n + page - 1) // page]
        k, v = (_tokens64(s[kv], pages, n) for kv in ("k", "v"))
        seen = torch.ones(n, dtype=torch.bool, device="cuda")
        p, o = _attend64(s["q"][b].double().view(hkv, -1, d), k, v, seen, 1 / math.sqrt(d))
        out[b] = o.reshape(-1, d)
        got = torch.zeros((hkv, len(pages) * page), dtype=torch.float64, device="cuda")
        got[:, :n] = p.sum(1)
        weights[pages] += got.view(hkv, -1, page).transpose(0, 1)
    return {"out": out, "weights": weights}


def _exact_evict(s, case):
    """The kept tokens' weights where they belong; codes and scales follow from the format's own rounding."""
    moved = s["moved"].double()
    page, budget = case["page"], case["budget"]
    for b, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        pages = s["table"][b, : (n + page - 1) // page]
        w = s["weights"][pages].double().transpose(0, 1).flatten(1)
        place = torch.zeros_like(w)
        for h in range(w.shape[0]):
            keep = list(range(n))
            if n > budget:
                mid = w[h, case["sinks"]: n - case["recent"]].tolist()
                order = sorted(range(len(mid)), key=lambda i: (-mid[i], i))
                chosen = sorted(i + case["sinks"] for i in order[: budget - case["sinks"] - case["recent"]])
                keep = keep[: case["sinks"]] + chosen + keep[n - case["recent"]:]
            place[h, : len(keep)] = w[h, torch.tensor(keep, dtype=torch.int64, device="cuda")]
        moved[pages] = place.view(w.shape[0], -1, page).transpose(0, 1)
    return {"kept": None, "weights": moved, "k": None, "k_scale": None, "k_zero": None, "v": None, "v_scale": None,
            "v_zero": None}


def _exact_append(s, case):
    held = torch.zeros(s["latent"].shape, dtype=torch.float64, device="cuda")
    scale, ropes = s["scale"].double(), s["ropes"].double()
    page = case["page"]
    for b, (n, at) in enumerate(zip(_counts(case), s["lengths"].tolist())):
        x = s["latent"][b, :n].double()
        sc = (x.abs().max(1).values / 127).clamp(min=1e-8)
        pos = torch.arange(at, at + n, device="cuda")
        where = s["table"][b, pos // page], pos % page
        scale[where], ropes[where] = sc, s["rope"][b, :n].double()
        # a code is rounded from the 32-bit quotient that the format defines
        sc32 = sc.float()
        code = torch.clamp(torch.round(s["latent"][b, :n].float() / sc32[:, None]), -127, 127).double()
        held[b, :n] = code * sc32.double()[:, None]
    return {"held": held, "scale": scale, "rope": ropes}


def _exact_latent(s, case):
    q = torch.cat([s["q"], s["q_rope"]], -1).double()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    page = case["page"]
    for b, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        pages = s["table"][b, : (n + page - 1) // page]
        c = (s["values"][pages].double() * s["scale"][pages].double()[..., None]).flatten(0, 1)[:n]
        r = s["ropes"][pages].double().flatten(0, 1)[:n]
        for t in range(case["tokens"]):
            seen = torch.arange(n, device="cuda") <= n - case["tokens"] + t
            out[b, t] = _attend64(q[b, t], torch.cat([c, r], -1), c, seen, s["sm_scale"])[1]
    return out


def _exact_prompt(s, case):
    out = torch.zeros((s["q"].shape[0], case["heads"], case["value"]), dtype=torch.float64, device="cuda")
    qo, ko, dn = s["q_offsets"].tolist(), s["k_offsets"].tolist(), case["nope"]
    for b in range(case["batch"]):
        nq, nk = qo[b + 1] - qo[b], ko[b + 1] - ko[b]
        rope = s["k_rope"][ko[b]: ko[b + 1]].double()
        seen = torch.ones((nq, nk), dtype=torch.bool, device="cuda").tril(nk - nq)
        for h in range(case["heads"]):
            kv = s["kv"][ko[b]: ko[b + 1], h].double()
            q = s["q"][qo[b]: qo[b + 1], h].double()
            out[qo[b]: qo[b + 1], h] = _attend64(q, torch.cat([kv[:, :dn], rope], 1), kv[:, dn:], seen,
                                                 s["sm_scale"])[1]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"weights": _exact_weights, "evict": _exact_evict, "append": _exact_append, "latent": _exact_latent,
            "prompt": _exact_prompt}[case["op"]](s, case)
