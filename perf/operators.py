"""The operators that are measured: rotary positions and sliding-window attention, in plain torch and as the framework's calls.

``run`` computes them in elementary torch operations, or, where ``own`` is true, through ``f5_tts_amd.ops``; ``exact`` computes the
definition in 64 bits.  Sizes: 24 kHz audio has 93.75 mel frames a second; 469 frames are a prompt of 5 s, 1406 frames a prompt and
10 s of speech, 8192 frames the longest utterance that the sampler's position table holds.  The base model has 16 heads of 64, and
its guided batch holds two sequences per utterance.
"""
import math

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _attention(name, batch, tq, tk, heads, kv_heads, dim, dtype, left, right, sinks, align, ragged):
    c = dict(op="attention", batch=batch, tq=tq, tk=tk, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, left=left, right=right,
             sinks=sinks, align=align, ragged=ragged)
    return dict(c, name=name) if name else c


def _rotary(name, batch, tokens, heads, kv_heads, dim, rot, half, dtype, rot_heads, scaling, factor, start, ragged):
    c = dict(op="rotary", batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, rot=rot, half=half, dtype=dtype,
             rot_heads=rot_heads, scaling=scaling, factor=factor, start=start, ragged=ragged)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one new token of one stream against its cache: the smallest call, all latency
        _attention("token", 1, 1, 1406, 16, 16, 64, "fp16", 255, 0, 4, "end", False),
        # one new token for each of many streams, caches of different lengths (one still empty), grouped heads
        _attention("tokens of 64 streams", 64, 1, 8192, 32, 8, 128, "bf16", 4095, 0, 16, "end", True),
        # a chunk of new tokens behind each of a few long caches
        _attention("chunks", 6, 200, 6000, 32, 8, 128, "bf16", 2047, 0, 64, "end", True),
        # one utterance of the sampler, guided: a window to both sides, the prompt stays visible
        _attention("utterance", 2, 1406, 1406, 16, 16, 64, "fp16", 256, 256, 469, "start", False),
        # the same in 32 bits: the sampler's exact mode
        _attention("utterance in 32 bits", 2, 1406, 1406, 16, 16, 64, "fp32", 256, 256, 469, "start", False),
        # a padded batch of utterances of different lengths, 12 heads as in the small model
        _attention("ragged utterances", 16, 1237, 1237, 12, 12, 64, "fp16", 200, 200, 300, "start", True),
        # the longest utterance that the sampler takes, guided
        _attention("long utterance", 2, 8192, 8192, 16, 16, 64, "fp16", 512, 512, 469, "start", False),
        # the positions of one new token, far into a stream
        _rotary("position of a token", 1, 1, 16, 16, 64, 64, False, "fp16", -1, "none", 1.0, 131071, False),
        # one utterance of the sampler, guided; interleaved pairs, every head
        _rotary("positions of an utterance", 2, 1406, 16, 16, 64, 64, False, "fp16", -1, "ntk", 2.0, 0, False),
        # the first head only, in 32 bits
        _rotary("positions in 32 bits", 2, 1406, 16, 16, 64, 64, False, "fp32", 1, "none", 1.0, 0, False),
        # long sequences, grouped heads, halves of three quarters of the head, frequencies scaled by parts
        _rotary("positions of long sequences", 4, 8192, 32, 8, 128, 96, True, "bf16", -1, "yarn", 8.0, 0, False),
        # new tokens of streams that stand at different places
        _rotary("positions of streams", 64, 7, 32, 8, 128, 128, True, "bf16", -1, "linear", 4.0, 0, True),
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["tokens", "chunks", "sequences", "sequences", "rotary", "rotary"])
    dtype = rng.choice(["fp16", "bf16", "fp16", "bf16", "fp32"])
    kv_heads = rng.choice([1, 2, 4, 8, 12, 16])
    group = rng.choice([1, 1, 2, 4]) if kv_heads > 8 else rng.choice([1, 2, 3, 4, 8])
    dim, size = rng.choice([64, 64, 128, 96, 40]), 4 if dtype == "fp32" else 2
    if kind == "rotary":
        batch, tokens = _log(rng, 1, 32), _log(rng, 1, 16384)
        rot = rng.choice([dim, dim, dim // 2, 16])
        heads = min(group * kv_heads, 32)
        while 2 * batch * tokens * (heads + kv_heads) * dim * size > 900 << 20:
            tokens = tokens // 2
        return _rotary(None, batch, tokens, heads, kv_heads, dim, rot, rng.random() < 0.5, dtype, rng.choice([-1, -1, 1]),
                       rng.choice(["none", "linear", "ntk", "yarn"]), rng.choice([2.0, 3.5, 8.0]), rng.choice([0, _log(rng, 1, 1000000)]),
                       rng.random() < 0.3)
    heads = min(group, max(1, 32 // kv_heads)) * kv_heads
    left, sinks = _log(rng, 16, 4096), rng.choice([0, 1, 4, _log(rng, 1, 512)])
    if kind == "sequences":
        batch, t = _log(rng, 1, 16), _log(rng, 17, 8192)
        while batch * heads * t * t > 1 << 31:
            batch, t = max(1, batch // 2), t if batch > 1 else t * 3 // 4
        right = rng.choice([left, left, 0])
        left = _fit(batch * heads * t, dim, left, sinks, right, dtype)
        right = min(left, right)
        return _attention(None, batch, t, t, heads, kv_heads, dim, dtype, left, right, sinks, "start", rng.random() < 0.4)
    batch, tk = _log(rng, 1, 64), _log(rng, 16, 16384)
    tq = rng.choice([1, 1, 2, 5]) if kind == "tokens" else _log(rng, 9, 512)
    tk = max(tk, tq)
    while batch * heads * tq * tk > 1 << 31 or 2 * batch * tk * kv_heads * dim * size > 900 << 20:
        batch, tk = max(1, batch // 2), tk if batch > 1 else max(tq, tk // 2)
    left = _fit(batch * heads * tq, dim, left, sinks, 0, dtype)
    return _attention(None, batch, tq, tk, heads, kv_heads, dim, dtype, left, 0, sinks, "end", rng.random() < 0.6)


def _fit(rows, dim, left, sinks, right, dtype):
    """A window no wider than the work of the largest listed case allows; 32 bits cost more."""
    most = (1 << 36) // (8 if dtype == "fp32" else 1)
    return max(16, min(left, (most // (4 * dim * rows) - sinks) // (2 if right else 1)))


def _lengths(case):
    """The sequences' key counts (a list): spread over [0, tk], the longest and, from three on, an empty one among them."""
    b, t = case["batch"], case["tk"]
    if not case["ragged"]:
        return [t] * b
    return [t if i == 0 else 0 if i == 2 else 1 + (i * 7919 * (t // 3 + 1)) % t for i in range(b)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t, e = TYPES[case["dtype"]], case["dim"]
    if case["op"] == "rotary":
        b, n, h, hk = case["batch"], case["tokens"], case["heads"], case["kv_heads"]
        # q and k as a fused projection leaves them: columns of one buffer, [q | k | v] for each token
        fused = torch.randn(b, n, h + 2 * hk, e, generator=g, device="cuda").to(t)
        s = {"case": case, "q": fused[:, :, :h], "k": fused[:, :, h:h + hk], "positions": None}
        if case["ragged"]:
            first = torch.randint(0, 200000, (b, 1), generator=g, device="cuda")
            s["positions"] = first + torch.arange(n, device="cuda")[None]
        f, s["amplitude"] = _frequencies(case)  # 64 bits; made once by a user's program
        s["freq"] = f.cuda()
        return s
    b, h, hk = case["batch"], case["heads"], case["kv_heads"]
    if case["align"] == "start":  # a fused projection's buffer, as above
        fused = torch.randn(b, case["tq"], h + 2 * hk, e, generator=g, device="cuda").to(t)
        q, k, v = fused[:, :, :h], fused[:, :, h:h + hk], fused[:, :, h + hk:]
    else:  # new queries and a cache
        q = torch.randn(b, case["tq"], h, e, generator=g, device="cuda").to(t)
        k = torch.randn(b, case["tk"], hk, e, generator=g, device="cuda").to(t)
        v = torch.randn(b, case["tk"], hk, e, generator=g, device="cuda").to(t)
    lens = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda") if case["ragged"] else None
    return {"case": case, "q": q, "k": k, "v": v, "kv_len": lens}


def _frequencies(case):
    """f_i = base^(-2 i / R), scaled for contexts `factor` times the trained 2048 positions, and the amplitude."""
    r, s = case["rot"], case["factor"]
    i = torch.arange(r // 2, dtype=torch.float64)
    base = 10000.0 * s ** (r / (r - 2)) if case["scaling"] == "ntk" else 10000.0
    f = base ** (-2 * i / r)
    if case["scaling"] == "linear":
        f = f / s
    if case["scaling"] == "yarn":  # turns within the trained length: below 1 the frequency is divided, above 32 kept, between them mixed
        g = ((2048 * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
        f = f * (g + (1 - g) / s)
    return f, 0.1 * math.log(s) + 1 if case["scaling"] == "yarn" else 1.0


def run(state):
    c = state["case"]
    if own:
        from f5_tts_amd import ops

        if c["op"] == "rotary":
            return ops.rotary(state["q"], state["k"], state["freq"], amplitude=state["amplitude"], positions=state["positions"], offset=c["start"],
                              layout="half" if c["half"] else "interleaved", rot_heads=None if c["rot_heads"] < 0 else c["rot_heads"])
        return ops.window_attention(state["q"], state["k"], state["v"], window=(c["left"], c["right"]), sinks=c["sinks"],
                                    kv_len=state["kv_len"], align=c["align"])
    return _rotate(state) if c["op"] == "rotary" else _attend(state)


def _rotate(state):
    c, r = state["case"], state["case"]["rot"]
    p = state["positions"]
    if p is None:
        p = torch.arange(c["start"], c["start"] + c["tokens"], device="cuda")[None]
    angle = p.double()[..., None] * state["freq"]  # [batch or 1, tokens, rot / 2], in 64 bits: far positions
    cos, sin = ((f(angle) * state["amplitude"]).float()[:, :, None] for f in (torch.cos, torch.sin))
    out = []
    for x in (state["q"], state["k"]):
        turned = x.shape[2] if c["rot_heads"] < 0 else min(c["rot_heads"], x.shape[2])
        y = x.float()
        z = y[:, :, :turned, :r]
        a, b = (z[..., :r // 2], z[..., r // 2:]) if c["half"] else (z[..., 0::2], z[..., 1::2])
        z = torch.cat([a * cos - b * sin, a * sin + b * cos], -1) if c["half"] else torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
        y = torch.cat([z, y[:, :, :turned, r:]], -1) if turned == x.shape[2] else \
            torch.cat([torch.cat([z, y[:, :, :turned, r:]], -1), y[:, :, turned:]], 2)
        out.append(y.to(x.dtype))
    return tuple(out)


def _visible(c, lens):
    """[batch or 1, tq, tk]: which keys each query sees."""
    n = torch.full((1,), c["tk"], device="cuda") if lens is None else lens.long()
    i, j = torch.arange(c["tq"], device="cuda"), torch.arange(c["tk"], device="cuda")
    p = (i[None] if c["align"] == "start" else n[:, None] - c["tq"] + i[None])[..., None]
    return (j < n[:, None, None]) & (j <= p + c["right"]) & ((j >= p - c["left"]) | (j < c["sinks"]))


def _attend(state):
    c, q = state["case"], state["q"]
    b, tq, h, e = q.shape
    hk = c["kv_heads"]
    q = q.float().reshape(b, tq, hk, h // hk, e).permute(0, 2, 3, 1, 4)          # [b, hk, group, tq, e]
    k = state["k"].float().permute(0, 2, 3, 1)[:, :, None]                       # [b, hk, 1, e, tk]
    v = state["v"].float().permute(0, 2, 1, 3)[:, :, None]                       # [b, hk, 1, tk, e]
    seen = _visible(c, state["kv_len"])[:, None, None]
    s = torch.matmul(q, k) * e ** -0.5
    s = torch.where(seen, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    w = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w, v) / torch.where(total == 0, 1.0, total)                 # a row that sees nothing is zero
    return o.permute(0, 3, 1, 2, 4).reshape(b, tq, h, e).to(state["q"].dtype)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    h, hk, e = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "rotary":
        n = case["batch"] * case["tokens"]
        turned = sum(x if case["rot_heads"] < 0 else min(case["rot_heads"], x) for x in (h, hk))
        return {"bytes": 2 * size * n * (h + hk) * e + 4 * case["rot"] + (8 * n if case["ragged"] else 0), "flops": 3 * n * turned * case["rot"]}
    pairs = keys = 0
    for n in _lengths(case):
        first = 0 if case["align"] == "start" else n - case["tq"]
        low, high = n, 0  # the windows' union: they move by one key a row
        for p in range(first, first + case["tq"]):
            end = max(0, min(n, p + case["right"] + 1))
            begin = min(max(0, p - case["left"]), end)
            pairs += end - begin + min(case["sinks"], begin)
            if end > begin:
                low, high = min(low, begin), max(high, end)
        keys += max(0, high - low) + min(case["sinks"], low, high)
    q = case["batch"] * case["tq"] * h * e
    return {"bytes": size * (2 * q + 2 * keys * hk * e) + (4 * case["batch"] if case["ragged"] else 0), "flops": 4 * e * h * pairs}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        r = case["rot"]
        p = torch.arange(case["start"], case["start"] + case["tokens"], device="cuda")[None] if s["positions"] is None else s["positions"]
        # as a product of complex numbers: (x + i y) a e^(i angle)
        turn = torch.polar(torch.full((), s["amplitude"], dtype=torch.float64, device="cuda"), p.double()[:, :, None, None] * s["freq"])
        out = []
        for x in (s["q"], s["k"]):
            y = x.double().clone()
            turned = x.shape[2] if case["rot_heads"] < 0 else case["rot_heads"]
            pairs = (slice(0, r // 2), slice(r // 2, r)) if case["half"] else (slice(0, r, 2), slice(1, r, 2))
            z = torch.complex(*(y[:, :, :turned, at].contiguous() for at in pairs)) * turn
            y[:, :, :turned, pairs[0]], y[:, :, :turned, pairs[1]] = z.real, z.imag
            out.append(y)
        return tuple(out)
    b, tq, h, e = s["q"].shape
    o = torch.zeros(b, tq, h, e, dtype=torch.float64, device="cuda")
    lens = _lengths(case)
    rows = max(1, (1 << 26) // case["tk"])  # queries at a time
    for i in range(b):
        n = lens[i]
        for at in range(0, tq if n else 0, rows):
            p = torch.arange(at, min(at + rows, tq), device="cuda")[:, None] + (0 if case["align"] == "start" else n - tq)
            j = torch.arange(n, device="cuda")[None]
            away = (j > p + case["right"]) | ((j < p - case["left"]) & (j >= case["sinks"]))
            for head in range(h):
                group = head // (h // case["kv_heads"])
                x = s["q"][i, at:at + rows, head].double() @ s["k"][i, :n, group].double().T / math.sqrt(e)
                x = x.masked_fill(away, -math.inf)
                x = torch.softmax(x, -1).masked_fill(away.all(-1, keepdim=True), 0.0)
                o[i, at:at + rows, head] = x @ s["v"][i, :n, group].double()
    return o
