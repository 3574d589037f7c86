"""The E8 key/value cache and the attention over it in 64 bits, on the CPU, written from the definitions."""
import math

import torch


def scales_of(x, bits):
    """bf16-valued scales [...] of the vectors x [..., D] (fp64): max|x| / C rounded up, 0 below 2^-64, NaN above 2^64
    or where x is not finite."""
    C = 7 - 2.0 ** -19 if bits == 4 else 127 - 2.0 ** -15
    top = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1) | (top > 2.0 ** 64)
    b = torch.where(bad, torch.ones_like(top), top) / C
    m, e = torch.frexp(b)
    up = torch.ldexp(torch.ceil(m * 256) / 256, e)
    up = torch.where(top < 2.0 ** -64, torch.zeros_like(up), up)
    return torch.where(bad, torch.full_like(up, math.nan), up)


def points_of(x, beta):
    """The E8 points [..., D/8, 8] nearest to x / beta (fp64), vectors of scale 0 or NaN at the origin; equal distances
    to the integers, equal remainders to the first coordinate."""
    ok = beta > 0
    b = torch.where(ok, beta, torch.ones_like(beta))[..., None, None]
    x = torch.where(ok[..., None], x, torch.zeros_like(x)).unflatten(-1, (-1, 8))
    lane = torch.arange(8)

    def even(p, shift, far):
        """The nearest values p + shift, the furthest coordinate moved to its second nearest where sum p is odd."""
        k = torch.where(far == far.amax(-1, keepdim=True), lane, torch.full_like(lane, 8)).amin(-1, keepdim=True)
        d = x - (p + shift) * b
        q = p + torch.where(d >= 0, 1.0, -1.0) * (lane == k)
        p = torch.where(p.sum(-1, keepdim=True) % 2 != 0, q, p) + shift
        return p, ((x - p * b) ** 2).sum(-1, keepdim=True)

    f = torch.round(x / b)
    away = (x - f * b).abs()
    g = torch.where(x < f * b, f - 1, f)
    (pi, di), (ph, dh) = even(f, 0.0, away), even(g, 0.5, b / 2 - away)
    return torch.where(dh < di * (1 - 1e-12), ph, pi)


def words_of(points, bits):
    """points [..., nb, 8] -> int32 words [..., nb, bits / 4]."""
    half = (points[..., :1] % 1 != 0).long()
    n = torch.floor(points).long() + (1 << (bits - 1))
    n[..., 7:] = n[..., 7:] - n[..., 7:] % 2 + half
    per = 32 // bits
    words = []
    for i in range(bits // 4):
        u = sum(n[..., i * per + j] << (bits * j) for j in range(per))
        words.append(u - ((u >> 31) << 32))
    return torch.stack(words, -1).int()


def points_from(words, bits):
    """int32 words [..., nb, bits / 4] -> fp64 points [..., nb * 8]."""
    u = words.long() & 0xffffffff
    per = 32 // bits
    n = torch.stack([(u[..., j // per] >> (bits * (j % per))) % (1 << bits) for j in range(8)], -1)
    half = n[..., 7] % 2
    n[..., 7] = n[..., 7] - half + n[..., :7].sum(-1) % 2
    return (n - (1 << (bits - 1)) + 0.5 * half[..., None].double()).flatten(-2)


def row_words(cache, page, head, off):
    """The key's and the value's words [nb, w] and scales of one row, by the stated layout."""
    w = cache.bits // 4
    k = cache.k[page, head, off].reshape(-1, w)
    v = cache.v[page, head, off // 4, :, off % 4]
    return k, v, cache.scales[page, head, off]


def dense(cache, pages, length):
    """Keys and values [kv heads, length, D] in fp64 of the rows of `pages` (CPU copies)."""
    nb, w = cache.head_dim // 8, cache.bits // 4
    k = cache.k[pages].cpu().transpose(0, 1).flatten(1, 2)[:, :length].unflatten(-1, (nb, w))
    v = cache.v[pages].cpu().permute(1, 0, 2, 4, 3, 5).flatten(1, 3)[:, :length]
    s = cache.scales[pages].cpu().double().transpose(0, 1).flatten(1, 2)[:, :length]
    return points_from(k, cache.bits) * s[..., :1], points_from(v, cache.bits) * s[..., 1:]


def attend(q, cache, table, lengths, starts, mask, scale):
    """out [n, heads, D], lse [n, heads], reach [n, heads, D] = sum p |v| and size [n, heads] = the largest
    scale sum |q| |k| of a seen token, in fp64 on the CPU."""
    q = q.detach().cpu().double()
    n, heads, D = q.shape
    group = heads // cache.kv_heads
    out = torch.zeros(n, heads, D, dtype=torch.float64)
    lse = torch.full((n, heads), -math.inf, dtype=torch.float64)
    reach = torch.zeros_like(out)
    size = torch.zeros(n, heads, dtype=torch.float64)
    for b, length in enumerate(lengths.tolist()):
        new = starts[b + 1] - starts[b]
        if length == 0 or new == 0:
            continue
        used = table[b, :-(-length // cache.page_size)].cpu().long()
        k, v = dense(cache, used.to(cache.k.device), length)
        for t in range(new):
            i = starts[b] + t
            seen = torch.zeros(length, dtype=torch.bool)
            for at in range(max(0, length - new), length):
                d = at - (length - new)
                if mask is None:
                    seen[at] = d <= t
                else:
                    seen[at] = d < 64 * mask.shape[1] and bool(int(mask[i, d // 64]) >> (d % 64) & 1)
            seen[:max(0, length - new)] = True
            if not seen.any():
                continue
            for h in range(heads):
                kk, vv = k[h // group][seen], v[h // group][seen]
                s = scale * (kk @ q[i, h])
                lse[i, h] = torch.logsumexp(s, 0)
                p = torch.softmax(s, 0)
                out[i, h] = p @ vv
                reach[i, h] = p @ vv.abs()
                size[i, h] = abs(scale) * (kk.abs() @ q[i, h].abs()).max()
    return out, lse, reach, size
