"""The 8-bit latent cache of the MLA layers and the attention over it: cases, plain forms, exact values.

Three operators share one paged cache.  A cached token is a latent ``c`` of ``KVL`` channels held as 8-bit
floating-point codes (e4m3), an optional rope key of ``DR`` channels held in 16 bits, and one power-of-two
scale ``s`` for both::

    e = max(least e1 with amax|c| <= 448 * 2^e1, least e2 with amax|k_rope| <= 2^15 * 2^e2, -100)
    s = 2^e  (NaN when a value of the token is not finite),  code = e4m3(c / s),  rope = 16 bits of k_rope / s

Sequence ``b`` has ``lens[b]`` tokens, its last ``n_b`` of them new; token ``i`` of the new ones sits at
position ``p = lens[b] - n_b + i`` (page ``block_table[b, p // page]``, slot ``p % page``).

* append: quantises the new tokens into their slots (a token with ``p < 0`` is skipped);
* read: the new tokens back in 16 bits (zeros where ``p < 0``);
* attend: ``softmax(scale * (q_lat . c + q_rope . k_rope))`` over the positions ``0 .. p`` of the sequence,
  weighing the latents themselves; the result and the natural logarithm of the softmax's sum (zeros and
  ``-inf`` where a row sees nothing).
"""

import math

import torch

own = False

E4M3_MAX = 448.0
ROPE_MAX = 32768.0
MIN_EXP = -100


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _case(name, op, B, L, n, H=16, KVL=512, DR=0, page=64, dtype="bf16", ragged=False, idle=False):
    """``L``: the longest sequence, its new tokens included; ``n``: the most new tokens of a sequence;
    ``ragged``: lengths (and, above eight, new tokens) differ; ``idle``: some slots hold no sequence."""
    return dict(name=name, op=op, B=B, L=L, n=n, H=H, KVL=KVL, DR=DR, page=page, dtype=dtype,
                ragged=ragged, idle=idle)


def listed():
    return [
        # one decode step of the 1.5B configuration's batch of four: four rows are quantised (latency)
        _case("append_step", "append", 4, 8193, 1, dtype="f16"),
        # a ragged mix of prompts with a rope part and small pages being written
        _case("append_ragged_rope", "append", 7, 5000, 5000, DR=64, page=16, ragged=True),
        # the 1.5B configuration's prompt: 4 x 8192 tokens
        _case("append_prompt", "append", 4, 8192, 8192, dtype="f16"),
        # a short shared prefix read back, narrow latents
        _case("read_short", "read", 3, 77, 77, KVL=256, DR=64, page=16, ragged=True),
        # prefixes read back for a prompt chunk's expanded attention
        _case("read_prefix", "read", 4, 8192, 8192, page=128, ragged=True),
        # one sequence at the start of its answer: a single token against a short context (latency)
        _case("decode_one", "attend", 1, 200, 1, dtype="f16"),
        # the 1.5B configuration's decode step: four sequences past a prompt of 8192
        _case("decode_4x8k", "attend", 4, 8193, 1, dtype="f16"),
        # a full serving batch, ragged, with idle slots
        _case("decode_64_ragged", "attend", 64, 8192, 1, ragged=True, idle=True),
        # long contexts, small batch
        _case("decode_8x32k", "attend", 8, 32768, 1, page=128),
        # four tokens verified at once, with a rope part
        _case("verify_16_rope", "attend", 16, 6001, 4, DR=64, ragged=True),
        # a prompt's chunk of 512 tokens on top of what is cached
        _case("chunk_512", "attend", 1, 8704, 512, page=128, dtype="bf16"),
        # whole ragged prompts at once through the cache, f16
        _case("prompts_ragged", "attend", 4, 1500, 1500, page=32, dtype="f16", ragged=True),
    ]


def _cost(case):
    """Microseconds at nominal rates, for keeping the drawn cases below the largest listed one."""
    w = work(case)
    return max(w["bytes"] / 6.5e6, w["flops"] / 1.6e9)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "read", "attend", "attend"])
    case = dict(
        op=op, B=_log(rng, 1, 64), L=_log(rng, 1, 32768), n=1,
        H=rng.choice([1, 4, 8, 12, 16, 16, 16, 32, 64, 128]) if op == "attend" else 16,
        KVL=rng.choice([128, 256, 384, 512, 512, 512]), DR=rng.choice([0, 0, 64]),
        page=rng.choice([16, 32, 64, 128, 256]), dtype=rng.choice(["f16", "bf16"]),
        ragged=rng.random() < 0.7, idle=rng.random() < 0.3)
    kind = rng.random()
    if op == "attend":
        case["n"] = 1 if kind < 0.5 else rng.randint(2, 8) if kind < 0.7 else _log(rng, 9, 1024)
    else:
        case["n"] = 1 if kind < 0.3 else _log(rng, 2, 8192)
    case["n"] = min(case["n"], case["L"])
    top = max(_cost(c) for c in listed() if c["op"] == op)
    while _cost(case) > top or case["B"] * case["L"] > 600000 \
            or case["B"] * case["n"] * case["H"] * case["L"] > 150000000 * (1 if op == "attend" else 1000):
        k = rng.choice(["B", "L", "n"])
        case[k] = max(1, int(case[k] * 0.8))
        case["n"] = min(case["n"], case["L"])
    if case["L"] % 1024 == 0 and case["L"] > 1024:
        case["L"] -= 1
        case["n"] = min(case["n"], case["L"])
    return case


def _lengths(case):
    """``(lens, news)`` of a case: plain lists, the same for every seed."""
    B, L, n = case["B"], case["L"], case["n"]
    lens, news = [], []
    for b in range(B):
        f = (b * 0.6180339887498949) % 1.0 if case["ragged"] else 0.0
        length = max(1, L - int(f * (L - 1)))
        new = min(length, n if n <= 8 else max(1, n - int(((b * 0.7548776662466927) % 1.0) * (n - 1)))
                  if case["ragged"] else n)
        if case["op"] == "read" and n == L:
            new = length
        if case["idle"] and b % 13 == 5:
            length = 0            # the slot's new tokens (if any) belong to nobody
            new = new if n <= 8 else 0
        lens.append(length)
        news.append(new)
    return lens, news


def work(case):
    lens, news = _lengths(case)
    N, KVL, DR, H = sum(news), case["KVL"], case["DR"], case["H"]
    token8, token16 = KVL + 4 + 2 * DR, 2 * (KVL + DR)
    if case["op"] != "attend":
        return {"bytes": N * (token8 + token16), "flops": 0}
    pairs = sum(sum(max(0, length - new + i + 1) for i in range(new)) for length, new in zip(lens, news))
    return {"bytes": sum(lens) * token8 + N * H * (token16 + 2 * KVL + 4),
            "flops": 2 * pairs * H * (2 * KVL + DR)}


# ---------------------------------------------------------------------------
# what a program has in hand
# ---------------------------------------------------------------------------
def _dtype(case):
    return {"f16": torch.float16, "bf16": torch.bfloat16}[case["dtype"]]


def _pow2(e):
    """``2 ** e`` in 32 bits for whole ``e``."""
    return torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)


def _least_exp(amax, top):
    """Least whole ``e`` with ``amax <= top * 2 ** e`` (``amax`` > 0; for zero, a value below any other)."""
    m, x = torch.frexp(amax)
    tm, tx = math.frexp(top)
    e = x - tx + (m > tm).to(x.dtype)
    return torch.where(amax > 0, e, torch.full_like(e, -1000))


def _quantise(c, k_rope):
    """``(codes, rope, scale)`` of latents ``c`` [N, KVL] and rope keys [N, DR] or None."""
    x = c.float()
    amax = x.abs().amax(-1)
    e = _least_exp(amax, E4M3_MAX)
    fine = torch.isfinite(amax)
    if k_rope is not None:
        y = k_rope.float()
        ramax = y.abs().amax(-1)
        e = torch.maximum(e, _least_exp(ramax, ROPE_MAX))
        fine = fine & torch.isfinite(ramax)
    e = torch.where(fine, e.clamp(min=MIN_EXP), torch.zeros_like(e))
    nan = torch.full_like(amax, float("nan"))
    s = torch.where(fine, _pow2(e), nan)
    inv = torch.where(fine, _pow2(-e), nan)[:, None]
    codes = (x * inv).to(torch.float8_e4m3fn)
    return codes, None if k_rope is None else (y * inv).to(k_rope.dtype), s


def _positions(state):
    """For every new token: its sequence, its position, whether it has one, and its slot in the pool."""
    q_start, lens = state["q_start"].long(), state["lens"].long()
    tok = torch.arange(state["N"], device=lens.device)
    b = torch.searchsorted(q_start[1:].contiguous(), tok, right=True)
    pos = lens[b] - (q_start[b + 1] - tok)
    ok = pos >= 0
    p = pos.clamp(min=0)
    page = state["page"]
    slot = state["block_table"].long()[b, p // page] * page + p % page
    return b, pos, ok, slot


def _latents(gen, n, case, dev):
    """Latents as a norm layer leaves them: channels of unequal gain, some tokens louder than others."""
    KVL = case["KVL"]
    gain = torch.exp(0.4 * torch.randn(KVL, generator=gen, device=dev))
    loud = torch.exp(0.3 * torch.randn(n, 1, generator=gen, device=dev))
    return torch.randn(n, KVL, generator=gen, device=dev) * gain * loud


def prepare(case, seed):
    dev, dt, page = torch.device("cuda"), _dtype(case), case["page"]
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    lens, news = _lengths(case)
    B, N, KVL, DR, H = case["B"], sum(news), case["KVL"], case["DR"], case["H"]
    need = [-(-length // page) for length in lens]
    width = max(1, max(need))
    pages = sum(need) + 3
    perm = torch.randperm(pages, generator=gen, device=dev).int()
    # rows of the table: a sequence's own pages, then pages of other sequences (never to be looked at)
    starts = torch.tensor([sum(need[:b]) for b in range(B)], device=dev)
    table = perm[(starts[:, None] + torch.arange(width, device=dev)) % pages].contiguous()
    state = dict(
        spare=perm[-1].long() * page, op=case["op"], N=N, page=page, H=H, KVL=KVL, DR=DR,
        block_table=table, lens=torch.tensor(lens, dtype=torch.int32, device=dev),
        q_start=torch.tensor([sum(news[:b]) for b in range(B + 1)], dtype=torch.int32, device=dev),
        uniform=len(set(news)) == 1, most=max(1, max(news)), dtype=dt, scale=(128 + DR) ** -0.5)
    # the pool as it comes: memory that nothing has been written to reads as NaN
    codes = torch.full((pages * page, KVL), 0x7F, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
    scales = torch.full((pages * page,), float("nan"), device=dev)
    rope = torch.full((pages * page, DR), float("nan"), dtype=dt, device=dev) if DR else None
    # the tokens that are in the cache already
    old = [length - new if case["op"] == "append" else length for length, new in zip(lens, news)]
    M = sum(max(0, o) for o in old)
    if M:
        cached = torch.tensor([max(0, o) for o in old], device=dev)
        b = torch.repeat_interleave(torch.arange(B, device=dev), cached)
        first = torch.cumsum(cached, 0) - cached
        pos = torch.arange(M, device=dev) - first[b]
        slot = table.long()[b, pos // page] * page + pos % page
        c = _latents(gen, M, case, dev)
        # every sequence's first token draws attention from all heads
        c[first[cached > 0], : KVL // 8] += 4.0
        k = torch.randn(M, DR, generator=gen, device=dev).mul_(2.0).to(dt) if DR else None
        q8, qr, s = _quantise(c.to(dt), k)
        codes[slot] = q8
        scales[slot] = s
        if DR:
            rope[slot] = qr
    state.update(codes=codes.view(pages, page, KVL), scales=scales.view(pages, page),
                 rope=None if rope is None else rope.view(pages, page, DR))
    if case["op"] == "append":
        state["c_kv"] = _latents(gen, N, case, dev).to(dt)
        state["k_rope"] = torch.randn(N, DR, generator=gen, device=dev).mul_(2.0).to(dt) if DR else None
    elif case["op"] == "attend":
        q = torch.randn(N, H, KVL, generator=gen, device=dev) * (0.6 * (512 / KVL) ** 0.5)
        q[..., : KVL // 8] += 0.25
        state["q_lat"] = q.to(dt)
        state["q_rope"] = torch.randn(N, H, DR, generator=gen, device=dev).to(dt) if DR else None
    if own:
        import importlib
        kb = importlib.import_module("-kimi-linear-_b200")
        state["kb"] = kb
        state["cache"] = kb.LatentCache.from_tensors(state["codes"], state["scales"], state["rope"], dtype=dt)
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    op = state["op"]
    if own:
        kb, cache, table, lens = state["kb"], state["cache"], state["block_table"], state["lens"]
        q_start = None if state["uniform"] else state["q_start"]
        if op == "append":
            kb.latent_append(cache, state["c_kv"], table, lens, q_start=q_start, k_rope=state["k_rope"])
            return [cache.codes, cache.scales, cache.rope]
        if op == "read":
            return list(kb.latent_read(cache, table, lens, state["N"], q_start=q_start))
        return list(kb.latent_attention(state["q_lat"], cache, table, lens, state["scale"], q_start=q_start,
                                        q_rope=state["q_rope"], return_lse=True))
    if op == "append":
        return _append(state)
    return _read(state) if op == "read" else _attend(state)


def _append(state):
    _, _, ok, slot = _positions(state)
    fresh = _quantise(state["c_kv"], state["k_rope"])
    # a token without a position writes back what a slot of no sequence holds
    slot = torch.where(ok, slot, state["spare"])
    for pool, value in zip((state["codes"], state["rope"], state["scales"]), fresh):
        if value is not None:
            pool = pool.view(-1, *value.shape[1:])
            kept = pool[slot]
            pool[slot] = torch.where(ok.view(-1, *[1] * (value.dim() - 1)), value.to(kept.dtype), kept)
    return [state["codes"], state["scales"], state["rope"]]


def _read(state):
    _, _, ok, slot = _positions(state)
    s = state["scales"].view(-1)[slot]
    dt = state["dtype"]
    c = state["codes"].view(-1, state["KVL"])[slot].float() * s[:, None]
    c = torch.where(ok[:, None], c, torch.zeros_like(c)).to(dt)
    if not state["DR"]:
        return [c, None]
    k = state["rope"].view(-1, state["DR"])[slot].float() * s[:, None]
    return [c, torch.where(ok[:, None], k, torch.zeros_like(k)).to(dt)]


def _attend(state):
    N, H, KVL, page = state["N"], state["H"], state["KVL"], state["page"]
    table, lens = state["block_table"].long(), state["lens"].long()
    B, dev = table.shape[0], table.device
    L = table.shape[1] * page
    at = torch.arange(L, device=dev)
    held = at[None, :] < lens[:, None]                                        # [B, L]
    slot = table[:, at // page] * page + at % page
    s = state["scales"].view(-1)[slot]
    c = state["codes"].view(-1, KVL)[slot].float() * s[..., None]
    c = torch.where(held[..., None], c, torch.zeros_like(c))                  # [B, L, KVL]
    # the queries, padded to the most new tokens of a sequence
    b, pos, _, _ = _positions(state)
    i = torch.arange(N, device=dev) - state["q_start"].long()[b]
    n = state["most"]
    q = c.new_zeros(B, n, H, KVL)
    q[b, i] = state["q_lat"].float()
    score = torch.matmul(q.view(B, n * H, KVL), c.transpose(1, 2))            # [B, n H, L]
    if state["DR"]:
        k = state["rope"].view(-1, state["DR"])[slot].float() * s[..., None]
        k = torch.where(held[..., None], k, torch.zeros_like(k))
        qr = c.new_zeros(B, n, H, state["DR"])
        qr[b, i] = state["q_rope"].float()
        score += torch.matmul(qr.view(B, n * H, -1), k.transpose(1, 2))
    score = score.mul_(state["scale"]).view(B, n, H, L)
    last = torch.full((B, n), -1, device=dev)
    last[b, i] = pos
    score.masked_fill_(at > last[:, :, None, None], float("-inf"))
    m = score.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    w = score.sub_(m).exp_()
    total = w.sum(-1, keepdim=True)                                           # [B, n, H, 1]
    out = torch.matmul(w.view(B, n * H, L), c).view(B, n, H, KVL)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    lse = (m + total.log()).squeeze(-1)
    return [out[b, i].to(state["q_lat"].dtype), lse[b, i]]


# ---------------------------------------------------------------------------
# the same from the definition, in 64 bits
# ---------------------------------------------------------------------------
def _token64(x, y):
    """Codes, rope part and scale of one call's tokens in 64 bits; ``y`` [N, 0] where there is no rope."""
    def least(a, top):
        e = torch.ceil(torch.log2(a / top))
        e = torch.where(a > top * torch.exp2(e), e + 1, e)
        return torch.where(a <= top * torch.exp2(e - 1), e - 1, e)
    a = x.abs().amax(-1)
    e = torch.where(a > 0, least(a, 448.0), torch.full_like(a, -1000.0))
    if y.shape[1]:
        r = y.abs().amax(-1)
        e = torch.maximum(e, torch.where(r > 0, least(r, 32768.0), torch.full_like(r, -1000.0)))
    s = torch.exp2(e.clamp(min=-100.0))[:, None]
    v = x / s
    # e4m3: three bits after the leading one, steps of 2^-9 below 2^-6
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step, y / s, s[:, 0]


def exact(case, seed):
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    lens, news = _lengths(case)
    page, KVL, DR, H, dev = case["page"], case["KVL"], case["DR"], case["H"], state["lens"].device
    table = state["block_table"].long()
    codes, scales = state["codes"].double(), state["scales"].double()
    rope = state["rope"].double() if DR else None
    outs, lses, ks, first = [], [], [], 0
    for b, (length, new) in enumerate(zip(lens, news)):
        at = torch.arange(length, device=dev)
        pg, sl = table[b, at // page], at % page
        mine = slice(first, first + new)
        first += new
        known = length > 0
        if case["op"] == "append":
            if known and new:
                x = state["c_kv"][mine].double()
                y = state["k_rope"][mine].double() if DR else x[:, :0]
                q, r, s = _token64(x, y)
                w = slice(length - new, length)
                codes[pg[w], sl[w]], scales[pg[w], sl[w]] = q, s
                if DR:
                    rope[pg[w], sl[w]] = r
            continue
        c = codes[pg, sl] * scales[pg, sl][:, None]
        k = rope[pg, sl] * scales[pg, sl][:, None] if DR else None
        if case["op"] == "read":
            outs.append(c[length - new:] if known else c.new_zeros(new, KVL))
            if DR:
                ks.append(k[length - new:] if known else c.new_zeros(new, DR))
            continue
        if not known:
            outs.append(c.new_zeros(new, H, KVL))
            lses.append(c.new_full((new, H), float("-inf")))
            continue
        for t in range(0, new, 64):
            rows = slice(first - new + t, min(first - new + t + 64, first))
            q = state["q_lat"][rows].double()
            z = torch.einsum("nhc,lc->nhl", q, c)
            if DR:
                z += torch.einsum("nhr,lr->nhl", state["q_rope"][rows].double(), k)
            z *= state["scale"]
            p = length - new + t + torch.arange(q.shape[0], device=dev)
            z.masked_fill_(at[None, None, :] > p[:, None, None], float("-inf"))
            lse = torch.logsumexp(z, -1)
            outs.append(torch.einsum("nhl,lc->nhc", torch.exp(z - lse[..., None]), c))
            lses.append(lse)
    if case["op"] == "append":
        return [codes, scales, rope]
    if case["op"] == "read":
        return [torch.cat(outs), torch.cat(ks) if DR else None]
    return [torch.cat(outs), torch.cat(lses)]
