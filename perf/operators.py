"""Timed cases of bounded-visibility attention and of the 4-bit KV cache.

Three operators that long-context fine-tuning and generation use together:

* ``attention`` -- causal GQA attention over a packed qkv projection in which a query sees the last
  ``window`` keys and the first ``sinks`` keys of its sequence; forward (prefill) and forward +
  backward (training).
* ``cache`` -- K / V rows quantised to 4 bits as they are written into a cache, and read back.
* ``decode`` -- one new token per sequence: its K / V row is written into the 4-bit cache and its
  query heads attend over the cache (whole length, or window + sinks).

4-bit values: groups of 32 along the head dimension share one bf16 scale ``s``; with ``e`` the
group's element of largest magnitude (the positive one if both signs have it) ``s = -e / 8``, a value
is held as ``c = clamp(round_half_even(x / s), -8, 7)`` and stands for ``s * c``.  A group whose
largest magnitude is under 2^-100 is held as zeros.

``own = False`` computes the plain form with elementary torch operations in 32 bits; ``own = True``
calls ``finetune_controller_amd.ops``.
"""
import math

import torch

own = False

GROUP = 32  # values that share a scale
TINY = 2.0 ** -100  # groups below this magnitude are held as zeros


# ---------------------------------------------------------------- cases
def _attn(name, B, S, H, KV, D, window, sinks, grad):
    return {"name": name, "op": "attention", "B": B, "S": S, "H": H, "KV": KV, "D": D, "window": window,
            "sinks": sinks, "grad": grad}


def _cache(name, B, n, H, KV, D, start):
    return {"name": name, "op": "cache", "B": B, "n": n, "H": H, "KV": KV, "D": D, "start": start}


def _decode(name, B, L, H, KV, D, window, sinks, ragged):
    return {"name": name, "op": "decode", "B": B, "L": L, "H": H, "KV": KV, "D": D, "window": window, "sinks": sinks,
            "ragged": ragged}


def listed():
    return [
        # a prompt of odd length read by a small grouped model with a short window
        _attn("prefill-1001", 1, 1001, 8, 2, 128, 256, 4, False),
        # a 16k-token prompt at the 8B / 7B head layout, 4096-key window (the 7B preset's)
        _attn("prefill-16k", 1, 16384, 32, 8, 128, 4096, 4, False),
        # a fine-tuning step's attention: the headline batch with a quarter-length window
        _attn("train-4x4096", 4, 4096, 32, 8, 128, 1024, 4, True),
        # ordinary multi-head layout, head_dim 64, odd length, one sink
        _attn("train-2x2049-d64", 2, 2049, 8, 8, 64, 300, 1, True),
        # one decode step's rows of a batch of 32, appended and read back (latency)
        _cache("append-32", 32, 1, 32, 8, 128, 777),
        # one 8192-token prompt written and read back
        _cache("prompt-8192", 1, 8192, 32, 8, 128, 0),
        # a batch of 16 continued by 4001 tokens each from an odd position, head_dim 64
        _cache("extend-16x4001-d64", 16, 4001, 16, 8, 64, 95),
        # interactive use: one sequence, short context
        _decode("decode-1x2000", 1, 2000, 32, 8, 128, 0, 0, False),
        # the generation batch (32 sequences of differing lengths around 4k)
        _decode("decode-32x4096", 32, 4096, 32, 8, 128, 0, 0, True),
        # long contexts, 64 sequences: bound by the cache bytes
        _decode("decode-64x16384", 64, 16384, 32, 8, 128, 0, 0, True),
        # 32k contexts under a 4096-key window with sinks
        _decode("decode-16x32768-w4096", 16, 32768, 32, 8, 128, 4096, 4, True),
        # eight query heads per kv head, head_dim 64
        _decode("decode-8x8191-g8-d64", 8, 8191, 16, 2, 64, 0, 0, True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("attention", "cache", "decode"))
    D = rng.choice((64, 128))
    if op == "attention":
        KV = rng.choice((1, 2, 4, 8))
        H = KV * rng.choice((1, 2, 4))
        grad = rng.random() < 0.5
        S = _log_int(rng, 1, 8192)
        B = rng.randint(1, max(1, min(4, 16384 // S)))
        window = _log_int(rng, 1, 4096)
        return {k: v for k, v in _attn("", B, S, H, KV, D, window, rng.randint(1, 64), grad).items() if k != "name"}
    if op == "cache":
        KV = rng.choice((1, 2, 4, 8))
        n = _log_int(rng, 1, 8192)
        B = max(1, min(_log_int(rng, 1, 64), 65536 // n))
        start = rng.randint(0, 300)
        return {k: v for k, v in _cache("", B, n, KV * rng.choice((1, 4)), KV, D, start).items() if k != "name"}
    KV = rng.choice((1, 2, 4, 8))
    H = KV * rng.choice((1, 2, 3, 4, 7, 8))
    L = _log_int(rng, 1, 32768)
    B = max(1, min(_log_int(rng, 1, 64), 524288 // L))
    window, sinks = (_log_int(rng, 16, 8192), rng.randint(0, 64)) if rng.random() < 0.4 else (0, 0)
    return {k: v for k, v in _decode("", B, L, H, KV, D, window, sinks, rng.random() < 0.7).items() if k != "name"}


def _lens(case):
    """Lengths of the sequences of a decode case, the new token included."""
    B, L = case["B"], case["L"]
    if not case["ragged"]:
        return [L] * B
    return [max(1, L - (b * 997) % max(1, L // 3)) for b in range(B)]


# ---------------------------------------------------------------- inputs
def _gen(seed, part=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + part)
    return g


def _rows(case, seed, part, n, width):
    """n rows of K (or V, or q) as projections give them: channels of differing size around zero."""
    g = _gen(seed, 2 * part)
    x = torch.randn(n, width, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(width, generator=_gen(seed, 1), device="cuda"))
    return x.to(torch.bfloat16)


def _inputs(case, seed):
    B, H, KV, D = case["B"], case["H"], case["KV"], case["D"]
    W = (H + 2 * KV) * D
    if case["op"] == "attention":
        st = {"qkv": _rows(case, seed, 0, B * case["S"], W)}
        if case["grad"]:
            st["do"] = torch.randn(B * case["S"], H * D, generator=_gen(seed, 3), device="cuda").to(torch.bfloat16)
        return st
    if case["op"] == "cache":
        return {"qkv": _rows(case, seed, 0, B * case["n"], W)}
    return {"qkv": _rows(case, seed, 0, B, W)}


def _past(case, seed, b):
    """K, V rows [L, KV*D] that sequence b of a decode case already holds (the last one is the new token's)."""
    kv = case["KV"] * case["D"]
    x = _rows(case, seed, 10 + b, case["L"], 2 * kv)
    return x[:, :kv], x[:, kv:]


def prepare(case, seed):
    st = {"case": case, **_inputs(case, seed)}
    if case["op"] == "attention":
        if own:
            from finetune_controller_amd import ops  # noqa: F401  (loads the kernels)
        return st
    B, KV, D = case["B"], case["KV"], case["D"]
    dev = st["qkv"].device
    cap = case["start"] + case["n"] if case["op"] == "cache" else case["L"]
    if case["op"] == "cache":
        st["start"] = torch.full((B,), case["start"], dtype=torch.int32, device=dev)
    else:
        lens = _lens(case)
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        st["last"] = st["lens"] - 1
        st["host_lens"] = lens
    if own:
        from finetune_controller_amd import ops

        st["data"] = ops.kv4_alloc(B, cap, KV, D, device=dev)
        if case["op"] == "decode":
            zero = torch.zeros(1, dtype=torch.int32, device=dev)
            for b in range(B):
                k, v = _past(case, seed, b)
                ops.kv4_store(st["data"][b:b + 1], k.unsqueeze(0), v.unsqueeze(0), zero)
        return st
    # the plain cache: two values to a byte and a scale for each group, [B, cap, KV, ...]
    for t in ("k", "v"):
        st[t + "q"] = torch.zeros(B, cap, KV, D // 2, dtype=torch.uint8, device=dev)
        st[t + "s"] = torch.zeros(B, cap, KV, D // GROUP, dtype=torch.bfloat16, device=dev)
    if case["op"] == "decode":
        for b in range(B):
            for t, x in zip("kv", _past(case, seed, b)):
                st[t + "q"][b], st[t + "s"][b] = _quantise(x, KV, D)
    return st


# ---------------------------------------------------------------- plain forms
def _quantise(x, KV, D):
    """[..., KV*D] -> codes packed two to a byte [..., KV, D/2], scales [..., KV, D/GROUP]."""
    g = x.float().reshape(*x.shape[:-1], KV, D // GROUP, GROUP)
    hi, lo = g.amax(-1), g.amin(-1)
    s = torch.where(hi >= -lo, hi, lo) / -8.0
    s = torch.where(s.abs() * 8.0 < TINY, torch.zeros_like(s), s)
    c = torch.where(s[..., None] != 0, g / s[..., None], torch.zeros_like(g))
    c = torch.round(c).clamp_(-8, 7).to(torch.int16).reshape(*x.shape[:-1], KV, D) + 8
    return (c[..., 0::2] | (c[..., 1::2] << 4)).to(torch.uint8), s.to(torch.bfloat16)


def _values(q, s):
    """fp32 values [..., D] that packed codes [..., D/2] with scales [..., D/GROUP] stand for."""
    c = torch.stack((q & 15, q >> 4), -1).reshape(*q.shape[:-1], s.shape[-1], GROUP).float() - 8.0
    return (c * s.float()[..., None]).reshape(*q.shape[:-1], s.shape[-1] * GROUP)


def _split(qkv, H, KV, D):
    return qkv[:, :H * D], qkv[:, H * D:(H + KV) * D], qkv[:, (H + KV) * D:]


def _plain_attention(st):
    c = st["case"]
    B, S, H, KV, D = c["B"], c["S"], c["H"], c["KV"], c["D"]
    G, scale = H // KV, 1.0 / math.sqrt(D)
    q, k, v = _split(st["qkv"].float(), H, KV, D)
    q = q.reshape(B, S, H, D).transpose(1, 2).reshape(B * H, S, D)
    k = k.reshape(B, S, KV, D).transpose(1, 2).reshape(B * KV, S, D)
    v = v.reshape(B, S, KV, D).transpose(1, 2).reshape(B * KV, S, D)
    i = torch.arange(S, device=q.device)
    seen = (i[None, :] <= i[:, None]) & ((i[:, None] - i[None, :] < c["window"]) | (i[None, :] < c["sinks"]))
    if c["grad"]:
        do = st["do"].float().reshape(B, S, H, D).transpose(1, 2).reshape(B * H, S, D)
        dq, dk, dv = torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)
    o = torch.empty_like(q)
    step = max(1, min(B * H, (1 << 28) // (S * S)))
    for h0 in range(0, B * H, step):
        hs = torch.arange(h0, min(B * H, h0 + step), device=q.device)
        kvs = hs // G  # (b*H + h) // G == b*KV + h // G
        qh, kh, vh = q[hs], k[kvs], v[kvs]
        s = (qh @ kh.transpose(1, 2)) * scale
        s = torch.where(seen, s, torch.full_like(s, float("-inf")))
        p = torch.exp(s - s.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        oh = p @ vh
        o[hs] = oh
        if c["grad"]:
            doh = do[hs]
            dv.index_add_(0, kvs, p.transpose(1, 2).contiguous() @ doh)
            ds = p * (doh @ vh.transpose(1, 2) - (doh * oh).sum(-1, keepdim=True)) * scale
            dq[hs] = ds @ kh
            dk.index_add_(0, kvs, ds.transpose(1, 2).contiguous() @ qh)

    def flat(t, n):
        return t.reshape(B, n, S, D).transpose(1, 2).reshape(B * S, n * D)

    out = {"o": flat(o, H).to(torch.bfloat16)}
    if c["grad"]:
        out["dqkv"] = torch.cat([flat(dq, H), flat(dk, KV), flat(dv, KV)], 1).to(torch.bfloat16)
    return out


def _plain_cache(st):
    c = st["case"]
    B, n, H, KV, D, s0 = c["B"], c["n"], c["H"], c["KV"], c["D"], c["start"]
    _, k, v = _split(st["qkv"], H, KV, D)
    out = {}
    for t, x in (("k", k), ("v", v)):
        q, s = _quantise(x.reshape(B, n, KV * D), KV, D)
        st[t + "q"][:, s0:s0 + n], st[t + "s"][:, s0:s0 + n] = q, s
        out[t] = _values(st[t + "q"][:, s0:s0 + n], st[t + "s"][:, s0:s0 + n]).reshape(B, n, KV * D).to(torch.bfloat16)
    return out


def _plain_decode(st):
    c = st["case"]
    B, H, KV, D, L = c["B"], c["H"], c["KV"], c["D"], c["L"]
    G, scale = H // KV, 1.0 / math.sqrt(D)
    q, kn, vn = _split(st["qkv"], H, KV, D)
    rows, last = torch.arange(B, device=q.device), st["last"].long()
    out = {}
    for t, x in (("k", kn), ("v", vn)):
        st[t + "q"][rows, last], st[t + "s"][rows, last] = _quantise(x, KV, D)
        out[t] = _values(st[t + "q"][rows, last], st[t + "s"][rows, last]).reshape(B, 1, KV * D).to(torch.bfloat16)
    qf = q.float().reshape(B, KV, G, D)
    pos, n = torch.arange(L, device=q.device), st["lens"].long()[:, None]
    seen = pos[None] < n
    if c["window"] > 0:
        seen &= (pos[None] >= n - c["window"]) | (pos[None] < c["sinks"])
    o = torch.empty(B, KV, G, D, device=q.device)
    step = max(1, (1 << 27) // (L * KV * D))
    for b in range(0, B, step):
        e = min(B, b + step)
        k = _values(st["kq"][b:e], st["ks"][b:e]).transpose(1, 2).contiguous()  # [b, KV, L, D]
        s = (qf[b:e] @ k.transpose(2, 3)) * scale
        s = torch.where(seen[b:e, None, None], s, torch.full_like(s, float("-inf")))
        p = torch.exp(s - s.amax(-1, keepdim=True))
        v = _values(st["vq"][b:e], st["vs"][b:e]).transpose(1, 2).contiguous()
        o[b:e] = (p @ v) / p.sum(-1, keepdim=True)
    out["o"] = o.reshape(B, H * D).to(torch.bfloat16)
    return out


# ---------------------------------------------------------------- the framework's calls
def _own_attention(st):
    from finetune_controller_amd import ops

    c = st["case"]
    kw = dict(window=c["window"], sinks=c["sinks"])
    dims = (c["B"], c["S"], c["H"], c["KV"], c["D"])
    if not c["grad"]:
        with torch.no_grad():
            return {"o": ops.attention_packed(st["qkv"], *dims, **kw)}
    x = st["qkv"].detach().requires_grad_()
    o = ops.attention_packed(x, *dims, **kw)
    (dx,) = torch.autograd.grad(o, x, st["do"])
    return {"o": o.detach(), "dqkv": dx}


def _own_cache(st):
    from finetune_controller_amd import ops

    c = st["case"]
    B, n, H, KV, D = c["B"], c["n"], c["H"], c["KV"], c["D"]
    _, k, v = _split(st["qkv"], H, KV, D)
    ops.kv4_store(st["data"], k.unflatten(0, (B, n)), v.unflatten(0, (B, n)), st["start"])
    k, v = ops.kv4_load(st["data"], st["start"], n, D)
    return {"k": k, "v": v}


def _own_decode(st):
    from finetune_controller_amd import ops

    c = st["case"]
    o = ops.decode_attention_kv4(st["qkv"], st["data"], st["lens"], max(st["host_lens"]), c["H"], c["KV"], c["D"],
                                 window=c["window"], sinks=c["sinks"])
    k, v = ops.kv4_load(st["data"], st["last"], 1, c["D"])  # the row that the step wrote
    return {"k": k, "v": v, "o": o}


_PLAIN = {"attention": _plain_attention, "cache": _plain_cache, "decode": _plain_decode}
_OWN = {"attention": _own_attention, "cache": _own_cache, "decode": _own_decode}


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


# ---------------------------------------------------------------- definitions in 64 bits
def _held(x, D):
    """fp64 values [rows, width] that bf16 rows stand for once held in 4 bits."""
    g = x.double().reshape(-1, GROUP)
    big = g.abs().max(dim=1, keepdim=True).values
    sign = torch.where((g == big).any(dim=1, keepdim=True), 1.0, -1.0).double()
    s = -(big * sign) / 8.0
    live = big >= TINY
    code = torch.where(live, g / torch.where(live, s, torch.ones_like(s)), torch.zeros_like(g))
    return (torch.clamp(torch.round(code), -8.0, 7.0) * torch.where(live, s, torch.zeros_like(s))).reshape(x.shape)


def _exact_attention(case, seed):
    B, S, H, KV, D, w, n = (case[t] for t in ("B", "S", "H", "KV", "D", "window", "sinks"))
    if B * H * S * min(S, w + n + 512) * D > 6e12:
        return None
    st = _inputs(case, seed)
    x = st["qkv"].double().reshape(B, S, H + 2 * KV, D)
    o = torch.zeros(B, S, H, D, dtype=torch.float64, device=x.device)
    dx = torch.zeros_like(x)
    do = st["do"].double().reshape(B, S, H, D) if case["grad"] else None
    r = D ** -0.5
    for q0 in range(0, S, 512):
        q1 = min(S, q0 + 512)
        lo = max(0, q0 - w + 1)
        keys = torch.cat([torch.arange(0, min(n, lo)), torch.arange(lo, q1)]).to(x.device)
        qi = torch.arange(q0, q1, device=x.device)
        dist = qi[:, None] - keys[None, :]
        hide = (dist < 0) | ((dist >= w) & (keys[None, :] >= n))
        for b in range(B):
            for h in range(H):
                kvh = H + h // (H // KV)
                Q, K, V = x[b, q0:q1, h], x[b, keys, kvh], x[b, keys, kvh + KV]
                P = torch.softmax((r * (Q @ K.T)).masked_fill(hide, -math.inf), dim=1)
                o[b, q0:q1, h] = P @ V
                if do is not None:
                    dO = do[b, q0:q1, h]
                    dP = dO @ V.T
                    dS = r * P * (dP - (P * dP).sum(dim=1, keepdim=True))
                    dx[b, q0:q1, h] = dS @ K
                    dx[b, :, kvh].index_add_(0, keys, dS.T @ Q)
                    dx[b, :, kvh + KV].index_add_(0, keys, P.T @ dO)
    out = {"o": o.reshape(B * S, H * D)}
    if do is not None:
        out["dqkv"] = dx.reshape(B * S, (H + 2 * KV) * D)
    return out


def _exact_cache(case, seed):
    B, n, H, KV, D = (case[t] for t in ("B", "n", "H", "KV", "D"))
    x = _inputs(case, seed)["qkv"]
    cols = {"k": x[:, H * D:(H + KV) * D], "v": x[:, (H + KV) * D:]}
    return {t: _held(c, D).reshape(B, n, KV * D) for t, c in cols.items()}


def _exact_decode(case, seed):
    B, H, KV, D, w, n = (case[t] for t in ("B", "H", "KV", "D", "window", "sinks"))
    x = _inputs(case, seed)["qkv"]
    o = torch.zeros(B, KV, H // KV, D, dtype=torch.float64, device=x.device)
    new = {"k": _held(x[:, H * D:(H + KV) * D], D), "v": _held(x[:, (H + KV) * D:], D)}
    for b, length in enumerate(_lens(case)):
        k, v = _past(case, seed, b)
        idx = torch.arange(length, device=x.device)
        if w > 0:
            idx = idx[(idx >= length - w) | (idx < n)]
        K, V = _held(k[idx], D), _held(v[idx], D)
        at = (idx == length - 1).nonzero().flatten()
        K[at], V[at] = new["k"][b], new["v"][b]
        K, V = (t.reshape(-1, KV, D).transpose(0, 1) for t in (K, V))
        Q = x[b, :H * D].double().reshape(KV, H // KV, D)
        o[b] = torch.softmax(torch.matmul(Q, K.transpose(1, 2)) * D ** -0.5, dim=2) @ V
    return {**{t: r.reshape(B, 1, KV * D) for t, r in new.items()}, "o": o.reshape(B, H * D)}


def exact(case, seed):
    return {"attention": _exact_attention, "cache": _exact_cache, "decode": _exact_decode}[case["op"]](case, seed)


# ---------------------------------------------------------------- work
def _seen(length, window, sinks):
    """Keys that the last query of a sequence of this length sees."""
    if window <= 0 or window >= length:
        return length
    return window + min(sinks, length - window)


def work(case):
    B, H, KV, D = case["B"], case["H"], case["KV"], case["D"]
    held = 2 * KV * (D // 2 + D // GROUP * 2)  # bytes of one token's K and V in the cache
    if case["op"] == "attention":
        S, w, n = case["S"], case["window"], case["sinks"]
        pairs = sum(_seen(i + 1, w, n) for i in range(S))
        rows = B * S
        qkv, o = rows * (H + 2 * KV) * D * 2, rows * H * D * 2
        if case["grad"]:
            return {"bytes": 2 * qkv + 2 * o, "flops": 14.0 * B * H * D * pairs}
        return {"bytes": qkv + o, "flops": 4.0 * B * H * D * pairs}
    if case["op"] == "cache":
        tokens = B * case["n"]
        # rows in, cache out; cache in, rows out
        return {"bytes": tokens * (2 * 2 * KV * D * 2 + 2 * held), "flops": 6.0 * tokens * 2 * KV * D}
    seen = sum(_seen(length, case["window"], case["sinks"]) for length in _lens(case))
    io = B * ((H + 2 * KV) * D * 2 + H * D * 2 + held + 2 * KV * D * 2)
    return {"bytes": seen * held + io, "flops": 4.0 * H * D * seen}
