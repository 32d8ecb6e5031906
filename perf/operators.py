"""Operators of 8-bit serving, each as one call: the matrix product of tokens and weights in 8-bit integers, the write of
a step's keys and values into a cache held in 8 bits, and the attention over that cache.

A number held in 8 bits is a code in [-127, 127] times a float32 scale: one scale a token (activations), an output channel
(weights), or a page of tokens and key/value head (cache).  Scales and codes are defined in float32 arithmetic, each step
rounded once: scale = max|x| * (1 / 127), code = rint(x / scale), 0 where the scale is 0.

``run`` computes the plain form with elementary torch operations in 32 bits; with ``own`` set, the framework's calls.
"""

import torch

own = False

_DT = {"bfloat16": torch.bfloat16, "float32": torch.float32}
DEV = "cuda"


# ------------------------------------------------------------------------------------------------ cases
def _linear(name, tokens, k, n, dtype="bfloat16", gated=False, wide=False):
    """``wide``: the result leaves as float32 (logits)."""
    return dict(name=name, op="linear", tokens=tokens, k=k, n=n, dtype=dtype, gated=gated, wide=wide)


def _step(name, op, singles, lo, hi, portions, q, past, heads, kv_heads, dim, page=16, window=0, dtype="bfloat16"):
    """A step's tokens: ``singles`` requests that bring one token at contexts between ``lo`` and ``hi``, and ``portions``
    prompt portions of up to ``q`` tokens (the later ones shorter) behind ``past`` cached ones."""
    return dict(name=name, op=op, singles=singles, lo=lo, hi=hi, portions=portions, q=q, past=past, heads=heads,
                kv_heads=kv_heads, dim=dim, page=page, window=window, dtype=dtype)


def listed():
    return [
        # one request decoding at 1B sizes: the gate and up projections with the SiLU gate
        _linear("linear_1_gated", 1, 2048, 16384, gated=True),
        # a decode step of eight requests at 1B sizes: the down projection
        _linear("linear_8_down", 8, 8192, 2048),
        # a decode step of 64 requests at 8B sizes: the stacked q|k|v projection
        _linear("linear_64_qkv", 64, 4096, 6144),
        # a prompt of 2,048 tokens at 1B sizes: the gate and up projections with the SiLU gate
        _linear("linear_2048_gated", 2048, 2048, 16384, gated=True),
        # a check run in float32 with sizes that fill no tile: odd token count, odd width, the tiny test vocabulary
        _linear("linear_333_odd_f32", 333, 1001, 509, dtype="float32"),
        # a prompt of 4,096 tokens at 8B sizes, gate and up projections: the largest product
        _linear("linear_4096_gated_8b", 4096, 4096, 28672, gated=True),
        # 64 decoding requests at 1B sizes append their token to pages that are part full
        _step("write_64_single", "write", 64, 1025, 2300, 0, 0, 0, 32, 8, 64),
        # ragged prompts at 8B sizes, 8,000 tokens in all, one of them going on inside a page
        _step("write_prompts_8b", "write", 0, 0, 0, 4, 3200, 7, 32, 8, 128),
        # eight decoding requests at 1B sizes beyond 2,048 keys
        _step("attend_8_at_2k", "attend", 8, 2049, 2304, 0, 0, 0, 32, 8, 64),
        # 64 requests at context 8,192 at 8B sizes: the largest cache
        _step("attend_64_at_8k_8b", "attend", 64, 8192, 8192, 0, 0, 0, 32, 8, 128),
        # a prompt of 2,048 tokens at 1B sizes
        _step("attend_prompt_2048", "attend", 0, 0, 0, 1, 2048, 0, 32, 8, 64),
        # tiny model in float32 under chunked prefill: portions of 24 tokens beside decoding requests, a window of 50 keys
        _step("attend_mixed_odd_f32", "attend", 3, 1, 100, 2, 24, 37, 3, 1, 32, page=8, window=50, dtype="float32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "write", "attend", "attend", "attend"])
    dtype = "float32" if rng.random() < 0.2 else "bfloat16"
    if kind == "linear":
        while True:
            m, k, n = _log(rng, 1, 8192), _log(rng, 64, 8192), _log(rng, 64, 28672)
            if m * k * n <= 4096 * 4096 * 28672:
                break
        gated = rng.random() < 0.3
        return _case_only(_linear("", m, k, max(16, n // 16 * 16) if gated else n, dtype, gated,
                                  wide=not gated and rng.random() < 0.2))
    kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 6, 8])
    dim = rng.choice([16, 32, 64, 64, 80, 96, 128, 128])
    page = rng.choice([8, 16, 16, 16, 32, 64])
    singles = rng.choice([0, _log(rng, 1, 128)])
    portions = rng.choice([0, 1, rng.randint(2, 6)]) if singles else rng.randint(1, 6)
    hi = _log(rng, 1, 8192)
    lo = max(1, int(hi * rng.random()))
    q, past = _log(rng, 2, 3000), rng.choice([0, _log(rng, 1, 3000)])
    window = rng.choice([0, 0, _log(rng, 8, 4096)])
    # no more cached numbers and no more tokens than the largest listed cases hold
    singles = min(singles, 64 * 8192 * 1024 // (hi * kv_heads * dim))
    q = max(2, min(q, 8000 // max(1, portions)))
    if kind == "write":
        window = 0
    else:
        # the plain form's scores stay within a few GB
        while portions and (singles + portions) * q * max(hi, q + past) * kv_heads * group > 6e8:
            q = max(2, q // 2)
            if singles > portions and q < 64:
                singles //= 2
            past //= 2
            hi = max(1, hi // 2)
            lo = min(lo, hi)
    if singles == 0:
        lo = hi = 0
        portions = max(1, portions)
    return _case_only(_step("", kind, singles, lo, hi, portions, q if portions else 0, past if portions else 0,
                            kv_heads * group, kv_heads, dim, page, window, dtype))


def _case_only(case):
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------------ what a step holds
def _lengths(case):
    """(tokens brought, keys afterwards) of every request: the single tokens first."""
    n, lo, hi = case["singles"], case["lo"], case["hi"]
    out = [(1, lo + (hi - lo) * (i * 7919 % n) // max(1, n - 1)) for i in range(n)]
    for j in range(case["portions"]):
        q = max(2, case["q"] * (case["portions"] - j) // case["portions"])
        out.append((q, q + max(0, case["past"] - j)))
    return out


def _visible(case):
    """(keys that some query of the request sees, sum over its queries of the keys seen) of every request."""
    out = []
    for q, kv in _lengths(case):
        w = case["window"] or kv
        first = max(0, kv - q - w + 1)
        full = max(0, min(q, kv - w + 1)) if w < kv else 0  # queries whose window is full
        short = q - full
        p0 = kv - q  # position of the first query
        out.append((kv - first, full * w + short * (p0 + 1) + short * (short - 1) // 2))
    return out


def work(case):
    size = 2 if case["dtype"] == "bfloat16" else 4
    if case["op"] == "linear":
        m, k, n = case["tokens"], case["k"], case["n"]
        cols = n // 2 if case["gated"] else n
        return {"bytes": m * k * size + n * k + 4 * n + m * cols * (4 if case["wide"] else size), "flops": 2 * m * n * k}
    kvh, d, page = case["kv_heads"], case["dim"], case["page"]
    lengths = _lengths(case)
    tokens = sum(q for q, _ in lengths)
    if case["op"] == "write":
        blocks = sum((kv - 1) // page - (kv - q) // page + 1 for q, kv in lengths)
        # the tokens' keys and values; each touched block's codes and scale out, and its values as they are read back
        return {"bytes": 2 * tokens * kvh * d * size + 2 * blocks * kvh * (page * d * 5 + 4), "flops": 4 * tokens * kvh * d}
    seen = _visible(case)
    keys = sum(s for s, _ in seen)
    return {"bytes": 2 * keys * kvh * d + 8 * keys // page * kvh + 2 * tokens * case["heads"] * d * size,
            "flops": 4 * d * case["heads"] * sum(p for _, p in seen)}


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed * 2654435761 % (1 << 62) + 1)
    dt = _DT[case["dtype"]]
    randn = lambda *shape: torch.randn(*shape, generator=g, device=DEV)  # noqa: E731
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    if case["op"] == "linear":
        m, k, n = case["tokens"], case["k"], case["n"]
        # activations with a few channels far larger than the rest, as the streams of language models have
        x = (randn(m, k) * (1 + 15 * (torch.rand(k, generator=g, device=DEV) < 0.01).float())).to(dt)
        w = randn(n, k) * 0.02
        w_scale = w.abs().amax(1) / 127
        store = torch.zeros(n, (k + 15) // 16 * 16, dtype=torch.int8, device=DEV)  # rows on 16-byte boundaries
        store[:, :k] = torch.round(w / w_scale[:, None]).to(torch.int8)
        return dict(case=case, x=x, w=store[:, :k], w_scale=w_scale, status=status)
    heads, kvh, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    lengths = _lengths(case)
    need = [(kv + page - 1) // page for _, kv in lengths]
    pool = sum(need) + 3
    ids = torch.randperm(pool, generator=g, device=DEV)[: sum(need)].to(torch.int32)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    starts, first = [0], [0]
    for (q, _), p in zip(lengths, need):
        starts.append(starts[-1] + q)
        first.append(first[-1] + p)
    tokens = starts[-1]
    q_len, kv_len = i32([q for q, _ in lengths]), i32([kv for _, kv in lengths])
    seq = torch.repeat_interleave(torch.arange(len(lengths), device=DEV), q_len.long())
    pos = torch.arange(tokens, device=DEV) - i32(starts).long()[seq] + (kv_len - q_len).long()[seq]
    codes = [torch.empty(pool, kvh, page, d, dtype=torch.int8, device=DEV) for _ in range(2)]
    for c in codes:
        for part in c.split(max(1, (1 << 27) // (kvh * page * d))):
            part.copy_((randn(*part.shape) * 40).clamp_(-127, 127).round_())
    scales = [torch.exp(0.5 * randn(pool, kvh)) * (2 / 127) for _ in range(2)]
    width = heads if case["op"] == "attend" else heads + 2 * kvh
    rows = randn(tokens, width * d).to(dt)
    # the blocks that the step's tokens touch, in order of the tokens, for the plain form and for reading them back
    slot_of = i32(first).long()[seq] + pos // page
    blocks, where = torch.unique_consecutive(slot_of, return_inverse=True)
    return dict(case=case, rows=rows, kcache=codes[0], vcache=codes[1], k_scale=scales[0], v_scale=scales[1],
                positions=pos.to(torch.int32), token_seq=seq.to(torch.int32), q_start=i32(starts[:-1]), q_len=q_len,
                kv_len=kv_len, page_indptr=i32(first), page_ids=ids, status=status, touched=ids[blocks],
                block_of=where, slot=pos % page, fresh=torch.zeros(blocks.numel(), dtype=torch.bool, device=DEV).index_fill_(
                    0, where[pos % page == 0], True),
                max_q=max(q for q, _ in lengths), max_kv=max(kv for _, kv in lengths))


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return {"linear": _own_linear, "write": _own_write, "attend": _own_attend}[op](state)
    return {"linear": _plain_linear, "write": _plain_write, "attend": _plain_attend}[op](state)


def _own_linear(s):
    from tokasaurus_b200.kernels import int8

    c = s["case"]
    return int8.linear_int8(s["x"], s["w"], s["w_scale"], s["status"], gated=c["gated"],
                            out_dtype=torch.float32 if c["wide"] else None)


def _own_write(s):
    from tokasaurus_b200.kernels import int8

    c = s["case"]
    int8.rope_kv8_write(s["rows"], s["positions"], s["token_seq"], s["page_indptr"], s["page_ids"], None, s["kcache"],
                        s["vcache"], s["k_scale"], s["v_scale"], c["heads"], c["kv_heads"], c["dim"], 0, c["page"], True,
                        s["status"])
    return int8.read_kv8(s["kcache"], s["vcache"], s["k_scale"], s["v_scale"], s["touched"], s["status"])


def _own_attend(s):
    from tokasaurus_b200.kernels import int8

    c = s["case"]
    out = torch.empty_like(s["rows"])
    int8.attn_kv8(s["rows"], out, s["kcache"], s["vcache"], s["k_scale"], s["v_scale"], s["q_start"], s["q_len"],
                  s["kv_len"], s["page_indptr"], s["page_ids"], c["heads"], c["kv_heads"], c["dim"], c["page"],
                  c["dim"] ** -0.5, c["window"] or None, s["status"], max_q_len=s["max_q"], max_kv_len=s["max_kv"],
                  single_tokens=c["singles"])
    return out


def _plain_linear(s):
    c = s["case"]
    x = s["x"].float()
    scale = x.abs().amax(1, keepdim=True) * (1 / 127)
    codes = torch.where(scale > 0, torch.round(x / scale), 0).clamp(-127, 127)
    y = (codes @ s["w"].float().t()) * (scale * s["w_scale"])
    if c["gated"]:
        z = y.view(y.shape[0], -1, 2, 8)  # gate and up features in groups of eight
        gate, up = z[:, :, 0], z[:, :, 1]
        y = (gate / (1 + torch.exp(-gate)) * up).reshape(y.shape[0], -1)
    return y if c["wide"] else y.to(s["x"].dtype)


def _plain_write(s):
    c = s["case"]
    heads, kvh, d, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    kv = s["rows"][:, heads * d:].float().view(-1, 2, kvh, d)
    pages = s["touched"].long()
    out = []
    for i, (cache, scales) in enumerate(((s["kcache"], s["k_scale"]), (s["vcache"], s["v_scale"]))):
        new = torch.zeros(pages.numel(), page, kvh, d, device=DEV)
        new[s["block_of"], s["slot"]] = kv[:, i]
        new = new.transpose(1, 2)
        written = torch.zeros(pages.numel(), page, dtype=torch.bool, device=DEV)
        written[s["block_of"], s["slot"]] = True
        old_scale = torch.where(s["fresh"][:, None], 0, scales[pages])
        scale = torch.maximum(old_scale, new.abs().amax((2, 3)) * (1 / 127))
        kept = cache[pages].float() * old_scale[:, :, None, None]
        codes = torch.where(written[:, None, :, None], new, kept) / scale[:, :, None, None]
        codes = torch.where(scale[:, :, None, None] > 0, torch.round(codes), 0).clamp(-127, 127)
        cache[pages] = codes.to(torch.int8)
        scales[pages] = scale
        out.append(codes * scale[:, :, None, None])
    return tuple(out)


def _plain_attend(s):
    c = s["case"]
    heads, kvh, d, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    n, length, most = s["kv_len"].numel(), s["max_kv"], s["max_q"]
    at = torch.arange(length, device=DEV)
    inside = at < s["kv_len"][:, None]
    place = s["page_indptr"][:-1, None] + at // page
    pages = s["page_ids"][torch.where(inside, place, 0).long()].long()
    k = s["kcache"][pages, :, at % page].float() * s["k_scale"][pages][..., None]  # [requests, keys, kv heads, d]
    v = s["vcache"][pages, :, at % page].float() * s["v_scale"][pages][..., None]
    j = torch.arange(most, device=DEV)
    real = j < s["q_len"][:, None]
    token = torch.where(real, s["q_start"][:, None] + j, 0).long()
    q = s["rows"].float()[token].view(n, most, kvh, heads // kvh, d)
    scores = torch.einsum("sqhgd,skhd->shgqk", q, k) * d ** -0.5
    pos = (s["kv_len"] - s["q_len"])[:, None] + j
    see = (at <= pos[:, :, None]) & inside[:, None]
    if c["window"]:
        see &= at > pos[:, :, None] - c["window"]
    scores.masked_fill_(~see[:, None, None], float("-inf"))
    scores -= scores.amax(-1, keepdim=True).clamp_min(-1e30)
    p = scores.exp_()
    o = torch.einsum("shgqk,skhd->sqhgd", p / p.sum(-1, keepdim=True).clamp_min(1e-30), v)
    return o.reshape(n, most, heads * d)[real].to(s["rows"].dtype)


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """The codes go by the definition's float32 steps, what is computed from them is in 64 bits."""
    s = prepare(case, seed)
    f8 = torch.float64
    if case["op"] == "linear":
        x = s["x"].to(torch.float32)
        t = x.abs().max(dim=1).values * torch.tensor(1 / 127, dtype=torch.float32, device=DEV)
        codes = torch.nan_to_num(x / t[:, None], nan=0.0).round().clamp(-127, 127)
        y = torch.mm(codes.to(f8), s["w"].to(f8).t()) * t.to(f8)[:, None] * s["w_scale"].to(f8)[None]
        if case["gated"]:
            y = y.reshape(y.shape[0], -1, 16)
            y = (y[:, :, :8] * torch.sigmoid(y[:, :, :8]) * y[:, :, 8:]).flatten(1)
        return y
    heads, kvh, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    lengths = _lengths(case)
    starts, first = s["q_start"].tolist(), s["page_indptr"].tolist()
    ids = s["page_ids"].long()
    if case["op"] == "write":
        out = []
        for i, (cache, scales) in enumerate(((s["kcache"], s["k_scale"]), (s["vcache"], s["v_scale"]))):
            parts = []
            for r, (q, kv) in enumerate(lengths):
                rows = s["rows"][starts[r]:starts[r] + q, (heads + i * kvh) * d:(heads + (i + 1) * kvh) * d]
                rows = rows.to(torch.float32).reshape(q, kvh, d)
                p0 = kv - q
                b0, b1 = p0 // page, (kv - 1) // page
                pg = ids[first[r] + b0:first[r] + b1 + 1]
                old = scales[pg].clone()
                if p0 % page == 0:
                    old[0] = 0
                old[1:] = 0
                width = (b1 - b0 + 1) * page
                flat = torch.zeros(width, kvh, d, device=DEV)
                lead = p0 - b0 * page
                flat[lead:lead + q] = rows
                flat = flat.reshape(-1, page, kvh, d)
                most = flat.abs().permute(0, 2, 1, 3).flatten(2).max(dim=2).values
                new = torch.fmax(old, most * torch.tensor(1 / 127, dtype=torch.float32, device=DEV))
                kept = cache[pg].permute(0, 2, 1, 3).to(torch.float32) * old[:, None, :, None]
                fill = torch.zeros(width, dtype=torch.bool, device=DEV)
                fill[lead:lead + q] = True
                val = torch.where(fill.reshape(-1, page, 1, 1), flat, kept)
                codes = torch.nan_to_num(val / new[:, None, :, None], nan=0.0).round().clamp(-127, 127)
                parts.append((codes.to(f8) * new.to(f8)[:, None, :, None]).permute(0, 2, 1, 3))
            out.append(torch.cat(parts))
        return tuple(out)
    out = torch.empty(s["rows"].shape, dtype=f8, device=DEV)
    group = heads // kvh
    for r, (q, kv) in enumerate(lengths):
        pg = ids[first[r]:first[r + 1]]
        qs = s["rows"][starts[r]:starts[r] + q].to(f8).reshape(q, heads, d)
        pos = torch.arange(kv - q, kv, device=DEV)
        at = torch.arange(kv, device=DEV)
        hide = at[None] > pos[:, None]
        if case["window"]:
            hide |= at[None] <= pos[:, None] - case["window"]
        for h in range(kvh):
            kk = (s["kcache"][pg, h].to(f8) * s["k_scale"][pg, h].to(f8)[:, None, None]).reshape(-1, d)[:kv]
            vv = (s["vcache"][pg, h].to(f8) * s["v_scale"][pg, h].to(f8)[:, None, None]).reshape(-1, d)[:kv]
            for u in range(h * group, (h + 1) * group):
                score = (qs[:, u] @ kk.t() / d ** 0.5).masked_fill_(hide, -torch.inf)
                out[starts[r]:starts[r] + q, u * d:(u + 1) * d] = torch.softmax(score, -1) @ vv
    return out
