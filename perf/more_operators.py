"""The gated linear recurrence and the norm-and-rotation of queries and keys: cases, plain forms, exact values.

* scan: ``h_t = a_t h_{t-1} + w_t x_t`` per channel with ``a_t = exp(g_t)``, ``w_t = 1`` or ``1 - a_t``, from
  an initial state, over a batch ``[B, T, D]`` or over sequences packed one behind the other (``[N, D]``, sequence
  ``s`` owns rows ``q_start[s] .. q_start[s + 1] - 1``; rows of no sequence give zeros); all ``h`` and every
  sequence's last one;
* scan_train: the same and the gradients of ``x``, ``g`` and the initial state;
* step: one token for each row of a serving batch, the old states taken from a pool;
* norm: queries and keys normalised per head (root mean square with a weight, length one, or not at all), then
  their first channels rotated by the token's position;
* norm_train: the same and the gradients of queries, keys and weights.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _scan(name, op, B, T, D, x="bf16", g="f32", complement=False, seqs=0):
    """``seqs``: 0 for a batch [B, T, D]; else T tokens of that many packed sequences (B is 1)."""
    return dict(name=name, op=op, B=B, T=T, D=D, x=x, g=g, complement=complement, seqs=seqs)


def _step(name, B, D, x="bf16", g="f32", complement=False, pool=0):
    """``pool``: states in the pool (0: row i has state i)."""
    return dict(name=name, op="step", B=B, D=D, x=x, g=g, complement=complement, pool=pool)


def _norm(name, op, B, T, H, HK, D, R, x="bf16", norm="rms", weight="head_dim", interleaved=False,
          positions="first"):
    """``weight``: none, head_dim ([D]) or heads ([H, D]); ``positions``: first (one a sequence, [B]), each
    (one a token, [B, T]) or none (0, 1, ...)."""
    return dict(name=name, op=op, B=B, T=T, H=H, HK=HK, D=D, R=R, x=x, norm=norm, weight=weight,
                interleaved=interleaved, positions=positions)


def listed():
    return [
        # a short prompt of one sequence at the 1.5B configuration's width (latency)
        _scan("scan_short", "scan", 1, 77, 2048),
        # the 1.5B configuration's prompt: 4 x 8192 tokens
        _scan("scan_prompt", "scan", 4, 8192, 2048, x="f16", complement=True),
        # one long context, gates in 16 bits as a projection leaves them
        _scan("scan_long", "scan", 1, 32768, 2048, g="bf16"),
        # a small model's training step in 32 bits, a length that no tile divides
        _scan("train_small", "scan_train", 2, 251, 60, x="f32"),
        # one sequence of the training length of the chunkwise benchmark
        _scan("train_4k", "scan_train", 1, 4096, 2048, complement=True),
        # documents of unequal length packed into one row
        _scan("train_packed", "scan_train", 1, 16000, 2048, x="f16", seqs=23),
        # one decode step of four sequences (latency)
        _step("step_4", 4, 2048),
        # a large serving batch with idle rows, its states in a pool
        _step("step_pool", 1024, 2048, x="f16", pool=1200),
        # the rope part of an attention layer's decode step: rotation alone, 16 heads and one shared key (latency)
        _norm("rope_step", "norm", 4, 1, 16, 1, 64, 64, norm="none", weight="none", interleaved=True),
        # the 1.5B configuration's prompt, one weight for all heads, every channel rotated
        _norm("norm_prompt", "norm", 4, 8192, 16, 16, 128, 128, x="f16"),
        # a short batch: grouped keys, an odd head size, a part rotated, weights of their own for every head
        _norm("norm_train_odd", "norm_train", 3, 333, 12, 3, 90, 30, weight="heads", positions="each"),
        # a training step's queries and keys
        _norm("norm_train_8k", "norm_train", 2, 8192, 16, 16, 128, 64, positions="none"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["scan", "scan", "scan_train", "scan_train", "step", "norm", "norm_train"])
    x = rng.choice(["f32", "f16", "bf16", "bf16"])
    if op == "step":
        B = _log(rng, 1, 1024)
        case = dict(op=op, B=B, D=_log(rng, 16, 4096), x=x, g=rng.choice(["f32", x]),
                    complement=rng.random() < 0.4, pool=rng.choice([0, B + _log(rng, 1, 300)]))
    elif op.startswith("scan"):
        case = dict(op=op, B=_log(rng, 1, 64), T=_log(rng, 1, 32768), D=_log(rng, 16, 4096), x=x,
                    g=rng.choice(["f32", x]), complement=rng.random() < 0.4, seqs=0)
        if rng.random() < 0.35:
            case["T"] *= case["B"]
            case["B"], case["seqs"] = 1, case["B"]
        if rng.random() < 0.5:
            case["D"] = max(16, case["D"] // 8 * 8)
    else:
        D = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 192, 256, 2 * rng.randint(8, 128)])
        R = rng.choice([0, D, D, D // 4 * 2, 2 * rng.randint(1, D // 2)])
        H = rng.choice([1, 4, 8, 12, 16, 16, 20, 32])
        norm = rng.choice(["rms", "rms", "l2", "none"]) if R else "rms"
        case = dict(op=op, B=_log(rng, 1, 64), T=_log(rng, 1, 8192), H=H,
                    HK=rng.choice([h for h in (1, 2, 4, 8, H) if H % h == 0]), D=D, R=R, x=x, norm=norm,
                    weight="none" if norm == "none" else rng.choice(["none", "head_dim", "head_dim", "heads"]),
                    interleaved=rng.random() < 0.4, positions=rng.choice(["first", "each", "none"]))
    top = max(work(c)["bytes"] for c in listed() if c["op"] == op)
    while work(case)["bytes"] > top:
        k = rng.choice(["B", "T"] if "T" in case else ["B", "D"])
        case[k] = max(1, int(case[k] * 0.8))
        if case.get("seqs"):
            case["B"] = 1
            case["seqs"] = min(case["seqs"], case["T"])
        if case.get("pool"):
            case["pool"] = max(case["pool"], case["B"])
    return case


def _sizes(case):
    """Bytes of a value of x and of g."""
    b = {"f32": 4, "f16": 2, "bf16": 2}
    return b[case["x"]], b[case.get("g", "f32")]


def work(case):
    es, gs = _sizes(case)
    if case["op"] == "step":
        live = sum(1 for i in _slots(case) if i >= 0)
        n = live * case["D"]
        return {"bytes": n * (es + gs + 4) + case["B"] * case["D"] * (es + 4), "flops": 2 * n}
    if case["op"].startswith("scan"):
        n, s = case["B"] * case["T"] * case["D"], (case["seqs"] or case["B"]) * case["D"]
        if case["op"] == "scan":
            return {"bytes": n * (2 * es + gs) + 8 * s, "flops": 2 * n}
        return {"bytes": n * (4 * es + 2 * gs) + 16 * s, "flops": 8 * n}
    n = case["B"] * case["T"] * (case["H"] + case["HK"]) * case["D"]
    train = case["op"] == "norm_train"
    return {"bytes": n * es * (4 if train else 2), "flops": n * (18 if train else 8)}


def _starts(case):
    """Where the packed sequences of a case start: the same for every seed.  Some are empty, and a few rows
    behind the last one (a batch padded to a fixed length) belong to none."""
    n, s = case["T"], case["seqs"]
    pad = min(n - 1, 5) if s > 2 else 0
    parts = [0.15 + (i * 0.6180339887498949) % 1.0 if not (s > 4 and i % 7 == 3) else 0.0 for i in range(s)]
    ends, total, acc = [0], sum(parts), 0.0
    for p in parts:
        acc += p
        ends.append(int((n - pad) * acc / total))
    ends[-1] = n - pad
    return ends


def _slots(case):
    """The pool's place of every row of a step: all different; some rows are idle (-1) where there is a pool."""
    B, pool = case["B"], case["pool"]
    if not pool:
        return list(range(B))
    m = next(m for m in (211, 223, 227, 229, 233) if pool % m)
    return [-1 if i % 11 == 7 else (i * m + 3) % pool for i in range(B)]


# ---------------------------------------------------------------------------
# what a program has in hand
# ---------------------------------------------------------------------------
def _gates(gen, shape, dev):
    """Log decays of the KDA gate: -exp(A_log) softplus(x + dt_bias), per-channel rates from slow to fast."""
    D = shape[-1]
    rate = torch.empty(D, device=dev).uniform_(1.0, 16.0, generator=gen)
    dt = torch.empty(D, device=dev).uniform_(1e-3, 0.1, generator=gen)
    bias = torch.log(torch.expm1(dt))
    x = torch.randn(shape, generator=gen, device=dev)
    return -rate * torch.log1p(torch.exp(x + bias))


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    op, dt = case["op"], DTYPES[case["x"]]
    state = dict(case=case, op=op)
    if op == "step":
        B, D = case["B"], case["D"]
        state.update(
            x=torch.randn(B, D, generator=gen, device=dev).to(dt),
            g=_gates(gen, (B, D), dev).to(DTYPES[case["g"]]),
            pool=torch.randn(case["pool"] or B, D, generator=gen, device=dev),
            slots=torch.tensor(_slots(case), dtype=torch.int32, device=dev) if case["pool"] else None)
    elif op.startswith("scan"):
        shape = (case["B"], case["T"], case["D"])
        rows = case["B"]
        if case["seqs"]:
            shape, rows = shape[1:], case["seqs"]
            state["q_start"] = torch.tensor(_starts(case), dtype=torch.int32, device=dev)
        else:
            state["q_start"] = None
        state.update(
            x=torch.randn(shape, generator=gen, device=dev).to(dt),
            g=_gates(gen, shape, dev).to(DTYPES[case["g"]]),
            s0=torch.randn(rows, case["D"], generator=gen, device=dev))
        if op == "scan_train":
            state.update(dh=torch.randn(shape, generator=gen, device=dev).to(dt),
                         dS=torch.randn(rows, case["D"], generator=gen, device=dev))
    else:
        B, T, H, HK, D, R = (case[k] for k in ("B", "T", "H", "HK", "D", "R"))
        def heads(n):
            loud = torch.exp(0.5 * torch.randn(n, 1, generator=gen, device=dev))
            return torch.randn(B, T, n, D, generator=gen, device=dev) * loud
        if op == "norm":
            # queries and keys as they stand side by side in the output of one projection
            both = torch.cat([heads(H), heads(HK)], 2).to(dt)
            state.update(q=both[:, :, :H], k=both[:, :, H:])
        else:
            state.update(q=heads(H).to(dt), k=heads(HK).to(dt), dq=heads(H).to(dt), dk=heads(HK).to(dt))
        for name, n in (("wq", H), ("wk", HK)):
            size = {"none": None, "head_dim": (D,), "heads": (n, D)}[case["weight"]]
            state[name] = None if size is None else 1 + 0.2 * torch.randn(size, generator=gen, device=dev)
        first = torch.randint(0, 131072, (B,), generator=gen, device=dev, dtype=torch.int32)
        state["positions"] = {
            "first": first, "none": None,
            "each": torch.arange(T, device=dev, dtype=torch.int32)[None, :] + first[:, None]}[case["positions"]]
        freq = 10000.0 ** (-torch.arange(0, R, 2, device=dev, dtype=torch.float64) / max(R, 1))
        state["inv_freq"] = freq.float() if R else None
        state["eps"] = 1e-6
    if own:
        import importlib
        state["kb"] = importlib.import_module("-kimi-linear-_b200")
        if op == "scan_train":
            state["leaves"] = [state[n].requires_grad_(True) for n in ("x", "g", "s0")]
        elif op == "norm_train":
            state["leaves"] = [state[n].requires_grad_(True) for n in ("q", "k", "wq", "wk")
                               if state[n] is not None]
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    op = state["op"]
    if not own:
        return {"scan": _plain_scan, "scan_train": _plain_scan_train, "step": _plain_step, "norm": _plain_norm,
                "norm_train": _plain_norm_train}[op](state)
    kb, case = state["kb"], state["case"]
    if op == "step":
        return list(kb.gated_step(state["x"], state["g"], state["pool"], slots=state["slots"],
                                  complement=case["complement"]))
    if op.startswith("scan"):
        h, S = kb.gated_scan(state["x"], state["g"], state["s0"], q_start=state["q_start"],
                             complement=case["complement"])
        if op == "scan":
            return [h, S]
        return [h.detach(), S.detach(),
                *torch.autograd.grad([h, S], state["leaves"], [state["dh"], state["dS"]])]
    norm = None if case["norm"] == "none" else case["norm"]
    q, k = kb.qk_norm_rope(state["q"], state["k"], state["wq"], state["wk"], norm=norm, eps=state["eps"],
                           positions=state["positions"], inv_freq=state["inv_freq"],
                           interleaved=case["interleaved"])
    if op == "norm":
        return [q, k]
    grads = list(torch.autograd.grad([q, k], state["leaves"], [state["dq"], state["dk"]]))
    return [q.detach(), k.detach(), *grads, *[None] * (4 - len(grads))]


def _first_rows(state, like):
    """True for every row that starts a sequence (packed), and for every row that belongs to one."""
    n, q_start = like.shape[0], state["q_start"].long()
    row = torch.arange(n, device=like.device)
    seq = torch.searchsorted(q_start[1:].contiguous(), row, right=True)
    mine = (row >= q_start[0]) & (row < q_start[-1])
    seq = seq.clamp(max=q_start.shape[0] - 2)
    return (row == q_start[seq]) & mine, mine, seq


def _carry(a, b):
    """``h_t = a_t h_{t-1} + b_t`` from ``h_{-1} = 0`` along dimension 1, by doubling."""
    a, h, step, T = a.clone(), b.clone(), 1, b.shape[1]
    while step < T:
        last = 2 * step >= T
        tail = a[:, step:] * h[:, :-step]
        if not last:
            a[:, step:] = a[:, step:] * a[:, :-step]
        h[:, step:] += tail
        step *= 2
    return h


def _plain_gates(state):
    """Decays ``a``, inputs' weights ``w`` (or None), inputs, and ``a`` with the sequences cut apart and the
    initial states' part of the inputs."""
    x, g, s0 = state["x"].float(), state["g"].float(), state["s0"].float()
    a = torch.exp(g)
    w = -torch.expm1(g) if state["case"]["complement"] else None
    b = x if w is None else w * x
    if state["q_start"] is None:
        cut, b = a, b.clone()
        b[:, 0] += a[:, 0] * s0
        return x, a, w, cut, b, None
    first, mine, seq = _first_rows(state, x)
    b = torch.where(mine[:, None], b + torch.where(first[:, None], a * s0[seq], torch.zeros_like(a)),
                    torch.zeros_like(b))
    cut = torch.where(first[:, None] | ~mine[:, None], torch.zeros_like(a), a)
    return x[None], a[None], None if w is None else w[None], cut[None], b[None], (first, mine, seq)


def _last_states(state, h, rows):
    """Every sequence's last ``h`` in 32 bits (its initial state where it is empty)."""
    if rows is None:
        return h[:, -1].clone()
    q_start = state["q_start"].long()
    some = q_start[1:] > q_start[:-1]
    return torch.where(some[:, None], h[0][(q_start[1:] - 1).clamp(min=0)], state["s0"].float())


def _plain_scan(state):
    x, a, w, cut, b, rows = _plain_gates(state)
    h = _carry(cut, b)
    S = _last_states(state, h, rows)
    return [h.to(state["x"].dtype).view(state["x"].shape), S]


def _plain_scan_train(state):
    x, a, w, cut, b, rows = _plain_gates(state)
    h = _carry(cut, b)
    S = _last_states(state, h, rows)
    shape, dS, s0 = state["x"].shape, state["dS"].float(), state["s0"].float()
    dh = state["dh"].float().view(h.shape).clone()
    before = torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1)
    if rows is None:
        before[:, 0] = s0
        dh[:, -1] += dS
        after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    else:
        first, mine, seq = rows
        last = torch.cat([first[1:] | ~mine[1:], torch.ones_like(first[:1])]) & mine
        before = torch.where(first[None, :, None], s0[seq][None], before)
        dh = torch.where(mine[None, :, None], dh + torch.where(last[:, None], dS[seq], torch.zeros_like(x[0])),
                         torch.zeros_like(dh))
        after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
        after = torch.where((last | ~mine)[None, :, None], torch.zeros_like(after), after)
    d = _carry(after.flip(1), dh.flip(1)).flip(1)
    dx = d if w is None else w * d
    dg = a * (before if w is None else before - x) * d
    if rows is None:
        ds0 = a[:, 0] * d[:, 0]
    else:
        q_start = state["q_start"].long()
        some = q_start[1:] > q_start[:-1]
        at = q_start[:-1].clamp(max=shape[0] - 1)
        ds0 = torch.where(some[:, None], (a * d)[0][at], dS)
        dg = torch.where(mine[None, :, None], dg, torch.zeros_like(dg))
    return [h.to(state["x"].dtype).view(shape), S, dx.to(state["x"].dtype).view(shape),
            dg.to(state["g"].dtype).view(shape), ds0]


def _plain_step(state):
    x, g, s, slots = state["x"].float(), state["g"].float(), state["pool"], state["slots"]
    if slots is not None:
        s = s[slots.long().clamp(min=0)]
    S = torch.exp(g) * s + (x * -torch.expm1(g) if state["case"]["complement"] else x)
    if slots is not None:
        S = torch.where((slots >= 0)[:, None], S, torch.zeros_like(S))
    return [S.to(state["x"].dtype), S]


def _angles(state):
    """Cosines and sines [B, T, 1, R / 2]: far positions' angles need 64 bits."""
    case, dev = state["case"], state["q"].device
    t = torch.arange(case["T"], device=dev)
    p = {"first": lambda: state["positions"].long()[:, None] + t, "each": lambda: state["positions"].long(),
         "none": lambda: t[None, :].expand(case["B"], -1)}[case["positions"]]()
    angle = (p[..., None].double() * state["inv_freq"].double())[:, :, None, :]
    return torch.cos(angle).float(), torch.sin(angle).float()


def _split(x, state):
    """The two halves of the rotated pairs, as views."""
    R = state["case"]["R"]
    return (x[..., 0:R:2], x[..., 1:R:2]) if state["case"]["interleaved"] else (x[..., :R // 2], x[..., R // 2:R])


def _turn(x, cos, sin, state):
    out = x.clone()
    (u, v), (a, b) = _split(x, state), _split(out, state)
    a.copy_(u * cos - v * sin)
    b.copy_(v * cos + u * sin)
    return out


def _rate(x, state):
    """``r`` of ``n = x r``."""
    kind = state["case"]["norm"]
    if kind == "none":
        return None
    if kind == "rms":
        return torch.rsqrt((x * x).mean(-1, keepdim=True) + state["eps"])
    return torch.rsqrt((x * x).sum(-1, keepdim=True)).clamp(max=1.0 / state["eps"])


def _plain_norm(state):
    outs = []
    cos, sin = _angles(state) if state["case"]["R"] else (None, None)
    for name, w in (("q", state["wq"]), ("k", state["wk"])):
        x = state[name].float()
        r = _rate(x, state)
        z = x if r is None else x * r
        z = z if w is None else z * w.float()
        z = z if cos is None else _turn(z, cos, sin, state)
        outs.append(z.to(state[name].dtype))
    return outs


def _plain_norm_train(state):
    case = state["case"]
    cos, sin = _angles(state) if case["R"] else (None, None)
    grads, dws = [], []
    for name, w in (("q", state["wq"]), ("k", state["wk"])):
        x, dz = state[name].float(), state["d" + name].float()
        dz = dz if cos is None else _turn(dz, cos, -sin, state)
        r = _rate(x, state)
        if r is None:
            grads.append(dz.to(state[name].dtype))
            dws.append(None)
            continue
        n = x * r
        if w is not None:
            # long sums over the tokens
            along = (0, 1, 2) if w.dim() == 1 else (0, 1)
            dws.append((dz * n).double().sum(along).to(w.dtype))
            dz = dz * w.float()
        else:
            dws.append(None)
        dot = (dz * n).mean(-1, keepdim=True) if case["norm"] == "rms" else (dz * n).sum(-1, keepdim=True)
        dx = r * (dz - n * dot)
        if case["norm"] == "l2":
            dx = torch.where(r < 1.0 / state["eps"], dx, r * dz)
        grads.append(dx.to(state[name].dtype))
    dws = [d for d in dws if d is not None]
    return [*_plain_norm(state), *grads, *dws, *[None] * (2 - len(dws))]


# ---------------------------------------------------------------------------
# the same from the definition, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "step":
        return _exact_step(case, state)
    return _exact_scan(case, state) if case["op"].startswith("scan") else _exact_norm(case, state)


def _exact_step(case, state):
    pool = state["pool"].double()
    h = torch.zeros(state["x"].shape, dtype=torch.float64, device=pool.device)
    live = [(i, s) for i, s in enumerate(_slots(case)) if s >= 0]
    rows = torch.tensor([i for i, _ in live], device=pool.device)
    at = torch.tensor([s for _, s in live], device=pool.device)
    a = state["g"].double()[rows].exp()
    h[rows] = a * pool[at] + (1 - a if case["complement"] else 1) * state["x"].double()[rows]
    return [h, h.clone()]


def _exact_scan(case, state):
    """Token by token; packed sequences side by side, the longest first, so that those still running at a
    token are the first rows."""
    x, g, s0 = state["x"], state["g"], state["s0"].double()
    train = case["op"] == "scan_train"
    if case["seqs"]:
        q = _starts(case)
        spans = sorted(((q[i], q[i + 1] - q[i], i) for i in range(case["seqs"])), key=lambda s: -s[1])
        base = torch.tensor([s[0] for s in spans], device=x.device)
        order = torch.tensor([s[2] for s in spans], device=x.device)
        count = [s[1] for s in spans]
    else:
        B, T = case["B"], case["T"]
        x, g = x.reshape(B * T, -1), g.reshape(B * T, -1)
        base, order, count = torch.arange(B, device=x.device) * T, torch.arange(B, device=x.device), [T] * B
    dh = state["dh"].reshape(x.shape) if train else None
    h = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    now, alive, lives = s0[order].clone(), len(count), []
    for t in range(count[0]):
        while count[alive - 1] <= t:
            alive -= 1
        lives.append(alive)
        rows = base[:alive] + t
        a = g[rows].double().exp()
        b = x[rows].double()
        if case["complement"]:
            b = b * -torch.expm1(g[rows].double())
        now[:alive] = a * now[:alive] + b
        h[rows] = now[:alive]
    S = torch.empty_like(now)
    S[order] = now
    shape = state["x"].shape
    if not train:
        return [h.view(shape), S]
    dx, dg = torch.zeros_like(h), torch.zeros_like(h)
    u = state["dS"].double()[order].clone()
    for t in range(count[0] - 1, -1, -1):
        n = lives[t]
        rows = base[:n] + t
        gt = g[rows].double()
        a, d = gt.exp(), dh[rows].double() + u[:n]
        prev = h[rows - 1] if t else s0[order][:n]
        if case["complement"]:
            dx[rows] = -torch.expm1(gt) * d
            prev = prev - x[rows].double()
        else:
            dx[rows] = d
        dg[rows] = a * prev * d
        u[:n] = a * d
    ds0 = torch.empty_like(u)
    ds0[order] = u
    return [h.view(shape), S, dx.view(shape), dg.view(shape), ds0]


def _exact_norm(case, state):
    """The rotation as a product of complex numbers, the norm's gradient by its Jacobian's two terms."""
    T, R, D, eps = case["T"], case["R"], case["D"], state["eps"]
    dev = state["q"].device
    turn = None
    if R:
        at = torch.arange(T, device=dev, dtype=torch.float64)[None, :].repeat(case["B"], 1)
        if case["positions"] == "first":
            at = at + state["positions"][:, None].double()
        elif case["positions"] == "each":
            at = state["positions"].double()
        angle = at[:, :, None, None] * state["inv_freq"].double()
        turn = torch.complex(angle.cos(), angle.sin())

    def rotate(v, by):
        if by is None:
            return v
        head, tail = v[..., :R], v[..., R:]
        if case["interleaved"]:
            z = torch.view_as_complex(head.unflatten(-1, (R // 2, 2)).contiguous()) * by
            return torch.cat([torch.view_as_real(z).flatten(-2), tail], -1)
        z = torch.complex(head[..., :R // 2].contiguous(), head[..., R // 2:].contiguous()) * by
        return torch.cat([z.real, z.imag, tail], -1)

    outs, grads, dws = [], [], []
    for name, w in (("q", state["wq"]), ("k", state["wk"])):
        v = state[name].double()
        w64 = 1.0 if w is None else w.double()
        sq = (v * v).sum(-1, keepdim=True)
        if case["norm"] == "rms":
            r = (sq / D + eps) ** -0.5
            slope = r ** 3 / D
        elif case["norm"] == "l2":
            r = torch.clamp(sq ** -0.5, max=1.0 / eps)
            slope = torch.where(sq.sqrt() > eps, r ** 3, torch.zeros_like(r))
        else:
            r, slope = torch.ones_like(sq), torch.zeros_like(sq)
        outs.append(rotate(v * r * w64, turn))
        if case["op"] == "norm_train":
            dz = rotate(state["d" + name].double(), None if turn is None else turn.conj())
            if w is not None:
                dws.append((dz * v * r).sum((0, 1, 2) if w.dim() == 1 else (0, 1)))
            dn = dz * w64
            grads.append(r * dn - slope * (dn * v).sum(-1, keepdim=True) * v)
    if case["op"] == "norm":
        return outs
    return [*outs, *grads, *dws, *[None] * (2 - len(dws))]
