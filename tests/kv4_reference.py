"""The 4-bit KV cache in plain torch, from the format's description: quantiser (fp32 operations on the CPU, which are the kernels' bit for
bit), a byte-by-byte reader of the tiles, and attention in fp64."""
import torch

GROUP, TILE = 64, 32


def quantise(x):
    """bf16 ``[..., D]`` (CPU) -> codes uint8 ``[..., D]``, scale bf16, zero fp16 ``[..., D / 64]``."""
    g = x.float().reshape(*x.shape[:-1], -1, GROUP)
    lo, hi = g.amin(-1), g.amax(-1)
    s = ((hi - lo) / torch.tensor(15.0)).bfloat16().float()
    bad = ~torch.isfinite(s) | ~torch.isfinite(g).all(-1)
    s = torch.where(s == 0, (lo.abs() * 2.0 ** -8).bfloat16().float(), s)
    empty = s == 0
    z = torch.where(empty | bad, 0.0, -lo / torch.where(empty | bad, 1.0, s)).half()
    c = (g / torch.where(empty | bad, 1.0, s)[..., None] + z.float()[..., None]).round().clamp(0, 15)
    c = torch.where((empty | bad)[..., None], 0.0, c).to(torch.uint8).reshape(x.shape)
    return c, torch.where(bad, float("nan"), s).bfloat16(), z


def rotate(x, positions, inv_freq):
    """``x [n, T, heads, D]`` bf16 on the CPU, rounding points of the bf16 cache's rotation."""
    ang = positions.float()[..., None] * inv_freq
    c, s = ang.cos().bfloat16().float()[:, :, None], ang.sin().bfloat16().float()[:, :, None]
    a, b = x.float().chunk(2, -1)
    r = lambda t: t.bfloat16().float()
    return torch.cat([r(a * c) + r(-b * s), r(b * c) + r(a * s)], -1).bfloat16()


def head_norm(x, w, eps):
    f = x.float()
    r = torch.rsqrt((f * f).mean(-1, keepdim=True) + eps)
    return (f * r * (1.0 + w.float())).bfloat16()


def tile_parts(tiles, D):
    """uint8 ``[..., 36 * D]`` -> (codes, scale, zero) of keys and of values: ``[..., 32, D]``, ``[..., 32, D / 64]``."""
    G = D // GROUP
    slot, ch = torch.arange(TILE)[:, None], torch.arange(D)[None]
    g, i = ch // GROUP, ch % GROUP
    pair, chunk = slot // 2, i // 8
    k_at = g * 1024 + slot * 32 + i // 2
    v_at = 16 * D + g * 1024 + pair * 64 + (chunk ^ ((pair & 2) << 1)) * 8 + (slot % 2) * 4 + (i % 8) // 2
    gg = torch.arange(G)[None]
    out = []
    for at, zero, scale in ((k_at, 32 * D + (slot * G + gg) * 4, 32 * D + (slot * G + gg) * 4 + 2),
                            (v_at, 35 * D + (gg * TILE + slot) * 2, 34 * D + (slot * G + gg) * 2)):
        byte = lambda a: tiles[..., a.to(tiles.device)].to(torch.int32)
        half = lambda a: (byte(a) | byte(a + 1) << 8).to(torch.int16)
        out.append(((byte(at) >> (4 * (ch & 1)).to(tiles.device)) & 15, half(scale).view(torch.bfloat16), half(zero).view(torch.float16)))
    return out


def values(c, s, z):
    """fp64 ``[..., D]`` of codes, scales and zeros."""
    d = c.double().reshape(*c.shape[:-1], -1, GROUP)
    return ((d - z.double()[..., None]) * s.double()[..., None]).reshape(c.shape)


def cache_values(tiles, D):
    """fp64 ``(k, v) [n_seq, n_kv, slots, D]``."""
    n_seq, n_kv, n_tiles, _ = tiles.shape
    return [values(*p).reshape(n_seq, n_kv, n_tiles * TILE, D) for p in tile_parts(tiles, D)]


def visible(positions, slots, window, sinks):
    j = torch.arange(slots, device=positions.device)
    see = j <= positions[..., None]
    if window:
        see &= (j > positions[..., None] - window) | (j < sinks)
    return see


def attend(q, k, v, positions, slots, n_heads, scale, window=0, sinks=0):
    """fp64 ``[n, T, n_heads * D]``, per element the largest visible |value| of its channel's head, and per element what bounds of
    roundings need: sum p |v|, and the largest visible scale * |q k| (2-norm of the products) of the row."""
    n, T, _ = q.shape
    D, n_kv = k.shape[-1], k.shape[1]
    rep = n_heads // n_kv
    see = visible(positions, slots, window, sinks)                                     # [n, T, slots]
    out = torch.zeros(n, T, n_heads, D, dtype=torch.float64, device=q.device)
    top = torch.zeros(n, T, n_heads, 1, dtype=torch.float64, device=q.device)
    more = torch.zeros(2, n, T, n_heads, D, dtype=torch.float64, device=q.device)
    qh = q.double().view(n, T, n_heads, D)
    for h in range(n_heads):
        kh, vh = k[:, h // rep, :slots], v[:, h // rep, :slots]
        s = (qh[:, :, h] @ torch.nan_to_num(kh).transpose(1, 2) * scale).masked_fill(~see, float("-inf"))
        p = torch.nan_to_num(torch.softmax(s, -1))                                      # a row without slots: zeros
        out[:, :, h] = p @ torch.nan_to_num(vh)
        more[0, :, :, h] = p @ torch.nan_to_num(vh).abs()
        qk = (qh[:, :, h].square() @ torch.nan_to_num(kh).square().transpose(1, 2)).sqrt() * abs(scale)
        more[1, :, :, h] = torch.where(see, qk, 0.0).amax(-1, keepdim=True)
        top[:, :, h] = torch.where(see[..., None], torch.nan_to_num(vh).abs().amax(-1)[:, None, :, None], 0.0).amax(2)
    return out.view(n, T, -1), top.expand(-1, -1, -1, D).reshape(n, T, -1), more.view(2, n, T, -1)


def spread(q, k, v, positions, slots, n_heads, scale, window=0, sinks=0):
    """fp64 ``[n, T, n_heads * D]``: roots of sum p^2 v^2 and of sum p^2, what independent errors of weights or values, or of the same size in
    every slot, add up to per unit of error."""
    n, T, _ = q.shape
    D, rep = k.shape[-1], n_heads // k.shape[1]
    see = visible(positions, slots, window, sinks)
    out, even = (torch.zeros(n, T, n_heads, D, dtype=torch.float64, device=q.device) for _ in range(2))
    qh = q.double().view(n, T, n_heads, D)
    for h in range(n_heads):
        kh, vh = torch.nan_to_num(k[:, h // rep, :slots]), torch.nan_to_num(v[:, h // rep, :slots])
        s = (qh[:, :, h] @ kh.transpose(1, 2) * scale).masked_fill(~see, float("-inf"))
        p2 = torch.nan_to_num(torch.softmax(s, -1)).square()
        out[:, :, h] = (p2 @ vh.square()).sqrt()
        even[:, :, h] = p2.sum(-1, keepdim=True).sqrt()
    return out.view(n, T, -1), even.view(n, T, -1)


def form(cache, n, T, heads, window=0, sinks=0):
    """Which kernel an attention call takes (``_lib.KV4_HEADS``, ``KV4_LIST`` or ``KV4_PROMPT``)."""
    from cobalt_b200 import _lib
    with torch.cuda.device(cache.device):
        return _lib.load().cobalt_kv4_attend_form(n, T, heads, cache.n_kv_heads, cache.head_dim, cache.slots, window, sinks)
