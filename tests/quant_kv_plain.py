"""A key/value cache held in 4 bits, plainly and in 64 bits: quantised numbers, the place of every code, attention over them."""
import math

import torch


def down(a):
    """The largest number of 8 significant bits (bf16's, range aside) that is not above a."""
    m, e = torch.frexp(a)
    return torch.ldexp(torch.floor(m * 256), e - 8)


def quantised(x, group):
    """x [..., dim] -> codes, scales and offsets [..., groups], all in 64 bits."""
    x = x.double().unflatten(-1, (-1, group))
    z = down(x.amin(-1))
    s = -down((z - x.amax(-1)) / torch.full_like(z, 15.0))
    c = torch.round((x - z[..., None]) / torch.where(s > 0, s, 1.0)[..., None]).clamp(0, 15)
    return torch.where(s[..., None] > 0, c, 0.0).flatten(-2), s, z


def values(c, s, z, group):
    return (c.unflatten(-1, (-1, group)) * s[..., None] + z[..., None]).flatten(-2)


def read_back(x, group):
    """What a cache holds of x."""
    return values(*quantised(x, group), group)


def cache_at(cache, page, off):
    """Keys and values [n, heads, dim] in 64 bits at (page, offset) of a 4-bit cache, every code by its address."""
    pool = cache.pool.cpu()
    _, H, blocks, size = pool.shape
    D, G = cache.dim, cache.dim // cache.group
    flat = pool.reshape(-1)
    base = ((page[:, None] * H + torch.arange(H)) * blocks + (off // 16)[:, None])[:, :, None] * size
    t, d = (off % 16)[:, None, None], torch.arange(D)
    k_at = t * (D // 2) + ((d // 8 % 4) * (D // 32) + d // 32) * 4 + d % 8 // 2
    v_at = (d // 64) * 512 + (d % 8) * 64 + (t // 4) * 16 + (d // 16 % 4) * 4 + t % 2 * 2 + t // 2 % 2
    out = []
    for start, at, nib in ((0, k_at, d % 2), (size // 2, v_at, d // 8 % 2)):
        c = (flat[base + start + at].int() >> (4 * nib)) & 15
        w = base + start + 8 * D + t * 4 * G + 2 * (d // cache.group)
        number = lambda a: ((flat[a].int() | flat[a + 1].int() << 8) << 16).view(torch.float32).double()  # noqa: E731
        out.append(number(w + 2 * G) + number(w) * c)
    return out


def attention(q, k, v, at, *, scale, window=0, keep_first=0, softcap=0.0, sink=None):
    """Rows q [n, heads, dim] at positions `at` [n] over keys and values [m, kv_heads, dim], in 64 bits; also sum_j p_j |v_j| and the
    largest |score|."""
    n, Q, _ = q.shape
    rep = Q // k.shape[1]
    k, v = (x.repeat_interleave(rep, 1) for x in (k, v))
    z = torch.einsum("nhd,mhd->hnm", q.double(), k) * scale
    if softcap:
        z = softcap * torch.tanh(z / softcap)
    j = torch.arange(k.shape[0])
    seen = j <= at[:, None]
    if window:
        seen = seen & ((j > at[:, None] - window) | (j < keep_first))
    z = z.masked_fill(~seen, -math.inf)
    most = z.masked_fill(~seen, 0.0).abs().amax().item() if z.numel() else 0.0
    if sink is not None:
        z = torch.cat([z, sink.double().view(Q, 1, 1).expand(Q, n, 1)], 2)
    p = torch.softmax(z, 2)[:, :, :k.shape[0]]
    p = torch.nan_to_num(p)             # (a row that sees nothing)
    return torch.einsum("hnm,mhd->nhd", p, v), torch.einsum("hnm,mhd->nhd", p, v.abs()), most
