"""Operators of the 4-bit KV cache whose speed is watched: writing and reading it, and the attention over it.

  write    keys and values of new tokens, rotated by their position, quantised to 4 bits into the cache, and read back
           (``KVCache4.append`` and ``KVCache4.read``): what a decode step, a prompt or a batch of prompts does in every layer.
  attend   attention of one to many new tokens per sequence over the cache (``KVCache4.attend``), causal, optionally with a sliding
           window and a few first slots that stay visible.

The format.  A group is 64 neighbouring channels of one slot of one KV head: x = (c - z) * s with a code c in 0..15, a bf16 scale s and
an fp16 zero point z, from the group's minimum and maximum.  A tile is 32 slots of one KV head in one piece of 36 * dim bytes (G = dim / 64):

  K codes   [G][32 slots][32 bytes]                               channel 2 b in the low half of byte b, 2 b + 1 in the high half
  V codes   [G][16 pairs of slots][8 chunks][2 slots][4 bytes]    chunk = 8 channels; chunk g of pair p lies at place g ^ ((p & 2) << 1)
  K         [32 slots][G] {fp16 zero, bf16 scale}
  V scale   [32 slots][G] bf16,  V zero [G][32 slots] fp16

A cache is [sequences][KV heads][tiles][36 * dim] bytes.  Shapes are those of a Mistral-7B block (32 / 8 heads of 128), a Gemma-3-27B
block (32 / 16 heads of 128, a window of 1024) and heads of 64 and 256.  All data is synthetic and seeded.
"""
import math

import torch

own = False
DEV = "cuda"
GROUP = 64
TILE = 32


# ----------------------------------------------------------------------------- the cases
def _write(name, seqs, tokens, start, heads, kv, dim, slots, rope=True):
    return {"name": name, "op": "write", "seqs": seqs, "tokens": tokens, "start": start, "heads": heads, "kv": kv, "dim": dim,
            "slots": slots, "rope": rope}


def _attend(name, seqs, tokens, shortest, longest, heads, kv, dim, slots, window=0, sinks=0):
    """``shortest`` .. ``longest``: slots in use (the new tokens' among them) of the sequences, spread evenly."""
    return {"name": name, "op": "attend", "seqs": seqs, "tokens": tokens, "shortest": shortest, "longest": longest, "heads": heads,
            "kv": kv, "dim": dim, "slots": slots, "window": window, "sinks": sinks}


def listed():
    return [
        # one layer of a chat's decode step: the smallest call, latency alone
        _write("write_1tok", 1, 1, 1000, 32, 8, 128, 2048),
        # a batch of prompts of a served 27B block that end inside tiles, keys already rotated by the caller
        _write("write_8x200", 8, 200, 0, 32, 16, 128, 512, rope=False),
        # a long prompt of a 7B block
        _write("write_prompt_8191", 1, 8191, 0, 32, 8, 128, 8192),
        # a chat's decode step
        _attend("attend_1seq_1001", 1, 1, 1001, 1001, 32, 8, 128, 2048),
        # eight conversations of a 27B block's sliding layer, lengths apart
        _attend("attend_8seq_window", 8, 1, 90, 4000, 32, 16, 128, 4096, window=1024),
        # sixteen long documents of a 7B block: the largest cache
        _attend("attend_16seq_32k", 16, 1, 15000, 32768, 32, 8, 128, 32768),
        # an endless conversation: a window and four first tokens out of 64k slots
        _attend("attend_64k_sinks", 4, 1, 60001, 65535, 32, 8, 128, 65536, window=4000, sinks=4),
        # wide heads that share one KV head
        _attend("attend_dim256", 4, 1, 1111, 9000, 8, 1, 256, 9000),
        # five proposed tokens of eight sequences checked at once, heads of 64
        _attend("attend_5tok_dim64", 8, 5, 700, 6000, 16, 4, 64, 6144),
        # time to first token: a prompt of a 7B block
        _attend("prompt_2048", 1, 2048, 2048, 2048, 32, 8, 128, 2048),
        # pieces of two long prompts of a 27B block's sliding layer
        _attend("prompt_2x500_window", 2, 500, 5000, 6001, 32, 16, 128, 6144, window=1024, sinks=4),
    ]


def _log_int(rng, lo, hi):
    return min(max(int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))), lo), hi)


def draw(rng):
    kind = rng.choice(["write", "decode", "decode", "few", "prompt"])
    dim = rng.choice([64, 128, 128, 128, 192, 256])
    kv = rng.choice([1, 2, 4, 8, 16])
    heads = kv * rng.choice([1, 2, 3, 4, 8])
    if kind == "write":
        seqs = _log_int(rng, 1, 16)
        tokens = _log_int(rng, 1, 8192 // seqs)
        while tokens * seqs * (heads + kv) * dim > 8191 * 40 * 128:
            tokens = max(1, tokens // 2)
        start = rng.choice([0, rng.randint(1, 4000)])
        case = _write("", seqs, tokens, start, heads, kv, dim, start + tokens + rng.randint(0, 500), rng.random() < 0.7)
    else:
        seqs = _log_int(rng, 1, 16)
        tokens = 1 if kind == "decode" else rng.randint(2, 16) if kind == "few" else _log_int(rng, 17, 2048)
        longest = max(tokens, _log_int(rng, 30, 32768 if tokens <= 16 else 4096))
        while seqs > 1 and (seqs * longest * kv * dim > 16 * 24000 * 8 * 128 or seqs * tokens * longest * heads * dim > 2048 * 2048 * 32 * 128):
            seqs //= 2
        while tokens * longest * heads * dim > 2048 * 2048 * 32 * 128:
            tokens = max(1, tokens // 2)
        shortest = rng.randint(tokens, longest)
        window = rng.choice([0, 0, _log_int(rng, 16, 4096)])
        case = _attend("", seqs, tokens, shortest, longest, heads, kv, dim, longest + rng.randint(0, 100), window,
                       rng.choice([0, 4, rng.randint(1, 40)]) if window else 0)
    del case["name"]
    return case


def _lengths(case):
    n, a, b = case["seqs"], case["shortest"], case["longest"]
    return [b if n == 1 else a + (b - a) * i // (n - 1) for i in range(n)]


def _visible(length, tokens, window, sinks):
    """(slots that some token of the sequence sees, (token, slot) pairs) of the last ``tokens`` of ``length`` slots."""
    pairs = 0
    for p in range(length - tokens, length):
        pairs += p + 1 if not window else min(window, p + 1) + min(sinks, max(0, p + 1 - window))
    first = max(0, length - tokens - window + 1) if window else 0
    return length - first + min(sinks, first), pairs


def work(case):
    kv, dim, heads = case["kv"], case["dim"], case["heads"]
    slot = kv * dim * 9 // 8                                               # 4-bit codes, scales and zeros of K and V
    if case["op"] == "write":
        n = case["seqs"] * case["tokens"]
        q = 4 * heads * dim if case["rope"] else 0
        return {"bytes": n * (q + 4 * kv * dim + slot + 4 * kv * dim + 8), "flops": n * (2 * kv * 8 + (heads + kv) * 6 * case["rope"]) * dim}
    seen = [_visible(n, case["tokens"], case["window"], case["sinks"]) for n in _lengths(case)]
    return {"bytes": sum(s for s, _ in seen) * slot + case["seqs"] * case["tokens"] * (heads * dim * 4 + 8),
            "flops": 4 * dim * heads * sum(p for _, p in seen)}


# ----------------------------------------------------------------------------- the format, in torch operations
def _quantise(x):
    """bf16 ``[..., dim]`` -> codes uint8, scale bf16 and zero fp16 ``[..., G]``."""
    g = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1), g.amax(-1)
    s = ((hi - lo) / torch.full_like(lo, 15.0)).bfloat16()
    s = torch.where(s == 0, (lo.abs() * 2.0 ** -8).bfloat16(), s)          # a constant group
    z = torch.where(s == 0, torch.zeros_like(lo), -lo / s.float()).half()
    c = (torch.where(s == 0, 0.0, 1.0).unsqueeze(-1) * g / torch.where(s == 0, 1.0, s.float()).unsqueeze(-1) + z.float().unsqueeze(-1)).round()
    return c.clamp(0, 15).to(torch.uint8).flatten(-2), s, z


def _values(c, s, z):
    return ((c.unflatten(-1, (-1, GROUP)).float() - z.float().unsqueeze(-1)) * s.float().unsqueeze(-1)).flatten(-2)


def _pack(k, v):
    """bf16 ``[..., slots, dim]`` (slots a multiple of 32) -> tiles ``[..., slots / 32, 36 * dim]``."""
    lead, dim = k.shape[:-2], k.shape[-1]
    G, n = dim // GROUP, k.shape[-2] // TILE
    parts = []
    for x, keys in ((k, True), (v, False)):
        c, s, z = _quantise(x.reshape(-1, TILE, dim))
        c, s, z = c.view(-1, TILE, G, 32, 2), s.view(torch.int16), z.view(torch.int16)
        b = c[..., 0] | (c[..., 1] << 4)                                   # [tile, slot, G, 32 bytes]
        if keys:
            parts += [b.transpose(1, 2).flatten(1), torch.stack([z, s], -1).flatten(1).view(torch.uint8)]
        else:
            b = b.view(-1, 4, 2, 2, 2, G, 8, 4).permute(0, 5, 1, 2, 3, 6, 4, 7)        # [tile, G, p / 4, p bit 1, p bit 0, chunk, parity, 4]
            b = torch.stack([b[:, :, :, 0], b[:, :, :, 1].roll(4, -3)], 3)
            parts += [b.flatten(1), s.flatten(1).view(torch.uint8), z.transpose(1, 2).flatten(1).view(torch.uint8)]
    return torch.cat([parts[0], parts[2], parts[1], parts[3], parts[4]], 1).view(*lead, n, 36 * dim)


def _unpack(tiles, dim):
    """fp32 keys and values ``[sequences, kv, slots, dim]`` of tiles."""
    G, (B, H, n, _) = dim // GROUP, tiles.shape
    t = tiles.reshape(-1, 36 * dim)
    kc, vc, km, vs, vz = t.split([16 * dim, 16 * dim, 2 * dim, dim, dim], 1)
    km = km.contiguous().view(torch.int16).view(-1, TILE, G, 2)
    vc = vc.reshape(-1, G, 4, 2, 2, 8, 2, 4)
    vc = torch.stack([vc[:, :, :, 0], vc[:, :, :, 1].roll(4, -3)], 3).permute(0, 2, 3, 4, 6, 1, 5, 7).reshape(-1, TILE, dim // 2)
    out = []
    for b, s, z in ((kc.reshape(-1, G, TILE, 32).transpose(1, 2).reshape(-1, TILE, dim // 2), km[..., 1], km[..., 0]),
                    (vc, vs.contiguous().view(torch.int16).view(-1, TILE, G), vz.contiguous().view(torch.int16).view(-1, G, TILE).transpose(1, 2))):
        c = torch.stack([b & 15, b >> 4], -1).flatten(-2)
        out.append(_values(c, s.contiguous().view(torch.bfloat16), z.contiguous().view(torch.float16)).view(B, H, n * TILE, dim))
    return out


def _rotate(x, positions, inv_freq):
    """``x [seqs, tokens, heads, dim]``: half-split rotation; angle, cosine and sine in fp32, tables and products rounded to bf16 as the
    model's own cache holds them."""
    ang = positions.float().unsqueeze(-1) * inv_freq                       # [seqs, tokens, dim / 2]
    c, s = ang.cos().bfloat16().float().unsqueeze(2), ang.sin().bfloat16().float().unsqueeze(2)
    a, b = x.float().chunk(2, -1)
    r = lambda t: t.bfloat16().float()  # noqa: E731
    return torch.cat([r(a * c) + r(-b * s), r(b * c) + r(a * s)], -1).bfloat16()


# ----------------------------------------------------------------------------- preparation
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(1_000_003 * (seed % 1_000_003) + 17)


def _keys(g, *shape):
    """Keys as projections make them: channels of unequal spread and mean, the same for every slot."""
    gain = torch.exp(0.5 * torch.randn(*shape[:-2], 1, shape[-1], generator=g, device=DEV))
    mean = 0.5 * torch.randn(*shape[:-2], 1, shape[-1], generator=g, device=DEV)
    return ((torch.randn(*shape, generator=g, device=DEV) + mean) * gain).bfloat16()


def prepare(case, seed):
    g = _gen(seed)
    B, T, H, kv, D = case["seqs"], case["tokens"], case["heads"], case["kv"], case["dim"]
    tiles = -(-case["slots"] // TILE)
    q = torch.randn(B, T, H * D, generator=g, device=DEV).bfloat16()
    state = {"op": case["op"], "dim": D, "kv": kv, "slots": case["slots"], "q": q}
    if case["op"] == "write":
        state["k"] = _keys(g, B, kv, T, D).transpose(1, 2).reshape(B, T, kv * D)
        state["v"] = torch.randn(B, T, kv * D, generator=g, device=DEV).bfloat16()
        state["tiles"] = torch.zeros(B, kv, tiles, 36 * D, dtype=torch.uint8, device=DEV)
        state["positions"] = case["start"] + torch.arange(T, device=DEV).expand(B, T).contiguous()
        state["inv_freq"] = 1.0 / (1e6 ** (torch.arange(0, D, 2, dtype=torch.float32, device=DEV) / D)) if case["rope"] else None
        return state
    # every slot holds something: what an earlier, longer sequence left lies behind the last one in use
    state["tiles"] = torch.stack([_pack(_keys(g, kv, tiles * TILE, D), torch.randn(kv, tiles * TILE, D, generator=g, device=DEV).bfloat16())
                                  for _ in range(B)])
    state["positions"] = torch.tensor([[n - T + i for i in range(T)] for n in _lengths(case)], device=DEV)
    state["window"], state["sinks"] = case["window"], case["sinks"]
    return state


# ----------------------------------------------------------------------------- one pass
def _run_own(st):
    from cobalt_b200 import KVCache4
    cache = KVCache4.wrap(st["tiles"], st["dim"], st["slots"])
    if st["op"] == "write":
        if st["inv_freq"] is None:
            cache.append(st["k"], st["v"], st["positions"])
            return cache.read(st["positions"])
        q = cache.append(st["k"], st["v"], st["positions"], q=st["q"], inv_freq=st["inv_freq"])
        return (q, *cache.read(st["positions"]))
    return cache.attend(st["q"], st["positions"], window=st["window"], sinks=st["sinks"])


def run(st):
    if own:
        return _run_own(st)
    D, kv, q, pos = st["dim"], st["kv"], st["q"], st["positions"]
    B, T, W = q.shape
    if st["op"] == "write":
        k, v = st["k"].view(B, T, kv, D), st["v"].view(B, T, kv, D)
        if st["inv_freq"] is not None:
            k = _rotate(k, pos, st["inv_freq"])
        back = _values(*_quantise(k)).bfloat16(), _values(*_quantise(v)).bfloat16()
        return back if st["inv_freq"] is None else (_rotate(q.view(B, T, W // D, D), pos, st["inv_freq"]).view(B, T, W), *back)
    k, v = _unpack(st["tiles"], D)
    rep = W // D // kv
    S = k.shape[2]
    qs = q.float().view(B, T, kv, rep, D).permute(0, 2, 3, 1, 4).reshape(B, kv, rep * T, D)
    x = (torch.matmul(qs, k.transpose(-1, -2)) * D ** -0.5).view(B, kv, rep, T, S)
    j, p = torch.arange(S, device=q.device), pos[..., None]
    see = (j <= p) & (j < st["slots"])
    if st["window"]:
        see &= (j > p - st["window"]) | (j < st["sinks"])
    x = x.masked_fill_(~see[:, None, None], float("-inf"))
    x = torch.exp(x.sub_(x.amax(-1, keepdim=True)))
    x = x.div_(x.sum(-1, keepdim=True)).view(B, kv, rep * T, S)
    return torch.matmul(x, v).view(B, kv, rep, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, W).bfloat16()


# ----------------------------------------------------------------------------- the definition in 64 bits
def _slot_values(tiles, dim, keys):
    """One head's tiles ``[n, 36 * dim]`` -> fp64 ``[n * 32, dim]``, byte by byte from the format's description."""
    G, n = dim // GROUP, tiles.shape[0]
    slot = torch.arange(TILE, device=tiles.device)[:, None]
    ch = torch.arange(dim, device=tiles.device)[None]
    g, i = ch // GROUP, ch % GROUP
    if keys:
        at = g * 1024 + slot * 32 + i // 2
        zero = 32 * dim + (slot * G + g) * 4
        scale = zero + 2
    else:
        pair, chunk = slot // 2, i // 8
        at = 16 * dim + g * 1024 + pair * 64 + (chunk ^ ((pair & 2) << 1)) * 8 + (slot % 2) * 4 + (i % 8) // 2
        scale = 34 * dim + (slot * G + g) * 2
        zero = 35 * dim + (g * TILE + slot) * 2
    byte = lambda a: tiles[:, a.expand(TILE, dim)].to(torch.int32)  # noqa: E731
    half = lambda a: (byte(a) | byte(a + 1) << 8).to(torch.int16)  # noqa: E731
    code = byte(at) >> (4 * (ch & 1)) & 15
    x = (code.double() - half(zero).view(torch.float16).double()) * half(scale).view(torch.bfloat16).double()
    return x.view(n * TILE, dim)


def exact(case, seed):
    st = prepare(case, seed)
    D, kv, q, pos = st["dim"], st["kv"], st["q"].double(), st["positions"]
    B, T, W = q.shape
    if st["op"] == "write":
        back, turned = [], []
        for x, turn in ((q, True), (st["k"].double(), True), (st["v"].double(), False)):
            x = x.view(B, T, -1, D)
            if turn and st["inv_freq"] is not None:                        # tables and products are bf16 by definition, the angle fp32
                ang = (pos.float()[..., None] * st["inv_freq"]).double()
                cs, sn = (f(ang).bfloat16().double()[:, :, None] for f in (torch.cos, torch.sin))
                a, b = x[..., :D // 2], x[..., D // 2:]
                x = torch.cat([(a * cs).bfloat16().double() - (b * sn).bfloat16().double(),
                               (b * cs).bfloat16().double() + (a * sn).bfloat16().double()], -1).bfloat16().double()
            turned.append(x)
        for x in turned[1:]:
            for_group = []
            for c0 in range(0, D, GROUP):
                y = x[..., c0:c0 + GROUP]
                lo = y.min(-1, keepdim=True).values
                s = ((y.max(-1, keepdim=True).values - lo) / 15).bfloat16().double()
                s = torch.where(s > 0, s, (lo.abs() / 256).bfloat16().double()).clamp_min(1e-300)
                z = (-lo / s).half().double()
                for_group.append(((y / s + z).round().clamp(0, 15) - z) * s)
            back.append(torch.cat(for_group, -1))
        return tuple(back) if st["inv_freq"] is None else (turned[0].reshape(B, T, W), *back)
    rep = W // D // kv
    if B * kv * case["slots"] * (rep * T + 64) > 2 ** 32:                  # about 20 seconds of fp64
        return None
    out = torch.zeros(B, T, kv * rep, D, dtype=torch.float64, device=DEV)
    slots = torch.arange(st["slots"], device=DEV)
    for b in range(B):
        for h in range(kv):
            K, V = (_slot_values(st["tiles"][b, h], D, keys)[:st["slots"]] for keys in (True, False))
            for t0 in range(0, T, 256):
                p = pos[b, t0:t0 + 256, None]
                hidden = slots > p
                if st["window"]:
                    hidden = hidden | ((slots <= p - st["window"]) & (slots >= st["sinks"]))
                for r in range(rep):
                    qh = q[b, t0:t0 + 256, (h * rep + r) * D:(h * rep + r + 1) * D]
                    out[b, t0:t0 + 256, h * rep + r] = torch.softmax((qh @ K.T / math.sqrt(D)).masked_fill(hidden, -math.inf), -1) @ V
    return out.view(B, T, W)
