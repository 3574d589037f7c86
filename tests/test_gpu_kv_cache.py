"""Rows of the E8 key/value cache written and read back, against the nearest-point definition in 64 bits.

Inputs of 8 to 11 significant bits leave no near ties: there the words, the
scales and the values read back are equal bit for bit."""
import pytest
import torch

import kv_oracle as O

pytestmark = pytest.mark.gpu


def _cache(ca, pages, page, heads, dim, bits):
    c = ca.E8KVCache.empty(pages, page, heads, dim, bits)
    assert c.nbytes() == pages * page * heads * (2 * dim * bits // 8 + 4)
    return c


def _inputs(n, heads, dim, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(n, heads, dim, generator=g) * torch.exp(2 * torch.randn(n, heads, 1, generator=g))
    v = torch.randn(n, heads, dim, generator=g)
    k[:, :, 3] *= 6.0
    if dtype == torch.float32:   # few bits, so that no tie is near
        k, v = k.bfloat16().float(), v.half().float()
    return k.to(dtype), v.to(dtype)


def _check_rows(cache, slots, k, v, bits):
    """Words, scales and read-back of every row in `slots` that lies in the cache."""
    import coset_amd as ca
    rows = cache.pages * cache.page_size
    for name, x, which in (("k", k, 0), ("v", v, 1)):
        xd = x.cpu().double()
        beta = O.scales_of(xd, bits)
        pts = O.points_of(xd, beta)
        words = O.words_of(pts, bits)
        for i, s in enumerate(slots.tolist()):
            if not 0 <= s < rows:
                continue
            for h in range(cache.kv_heads):
                got = O.row_words(cache, s // cache.page_size, h, s % cache.page_size)
                assert torch.equal(got[which].cpu(), words[i, h]), (name, i, h)
                assert torch.equal(got[2][which].cpu().view(torch.int16), beta[i, h].bfloat16().view(torch.int16)), (name, i, h)
        for dtype in (torch.float32, torch.bfloat16, torch.float16):
            back = ca.kv_read(cache, slots, dtype)[which].cpu()
            # beta (8 bits) times a point (9 at most) is exact in fp32
            want = (pts.flatten(-2) * beta[..., None]).float().to(dtype)
            out = (slots < 0) | (slots >= rows)
            want[out.cpu()] = 0
            assert torch.equal(torch.nan_to_num(back.float(), nan=-7.0), torch.nan_to_num(want.float(), nan=-7.0)), (name, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,heads,dim,bits,page", [
    (1, 1, 32, 4, 16), (1, 8, 128, 8, 32), (5, 3, 64, 4, 48), (33, 2, 96, 8, 16), (70, 1, 160, 4, 64),
    (17, 4, 256, 8, 16), (19, 2, 256, 4, 128), (3, 5, 128, 4, 16), (6, 2, 224, 8, 32)])
def test_rows_match_the_definition(n, heads, dim, bits, page, dtype):
    import coset_amd as ca
    print(f"rows n={n} heads={heads} dim={dim} bits={bits} page={page} {dtype}", flush=True)
    pages = -(-n // page) + 2
    cache = _cache(ca, pages, page, heads, dim, bits)
    k, v = _inputs(n, heads, dim, dtype, n + dim)
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(1))[:n]
    ca.kv_write(cache, k.cuda(), v.cuda(), slots.cuda())
    _check_rows(cache, slots.cuda(), k, v, bits)
    # the other rows stay as they were: zero words and scales
    rest = torch.ones(pages * page, dtype=torch.bool)
    rest[slots] = False
    assert int(cache.scales.cpu().float().transpose(1, 2).reshape(pages * page, -1)[rest].abs().sum()) == 0
    assert int((cache.k.cpu().transpose(1, 2).reshape(pages * page, -1)[rest] != 0).sum()) == 0
    vs = cache.v.cpu().permute(0, 2, 4, 1, 3, 5).reshape(pages * page, -1)
    assert int((vs[rest] != 0).sum()) == 0


@pytest.mark.parametrize("bits", [4, 8])
def test_unusual_vectors(bits):
    """Zeros, the smallest and largest kept, infinities and NaN, one value alone, equal values, exact ties."""
    import coset_amd as ca
    D = 64
    rows = [torch.zeros(D), torch.full((D,), -0.0), torch.full((D,), 2.0 ** -65), torch.full((D,), 2.0 ** -64),
            torch.full((D,), 2.0 ** 64), torch.full((D,), 2.0 ** 65), torch.full((D,), 3e38)]
    for bad in (float("inf"), float("-inf"), float("nan")):
        x = torch.ones(D)
        x[D - 1] = bad
        rows.append(x)
    for sign in (1.0, -1.0):
        x = torch.zeros(D)
        x[5] = sign
        rows.append(x)
        rows.append(torch.full((D,), sign * 0.3125))
    C = 7 if bits == 4 else 127
    # beta = 2^-3 (1 + 2^-7): halves of it, all alike, alternating and one short of a tie
    beta = 2.0 ** -3 * (1 + 2.0 ** -7)
    j = torch.arange(D)
    for h in (0.5, 1.5, 2.5, 0.25):
        x = torch.full((D,), h * beta)
        x[0] = C * 2.0 ** -3
        rows.append(x)
        rows.append(x * torch.where(j % 2 == 0, 1.0, -1.0))
        rows.append(torch.where(j % 8 < 3, x, torch.zeros(D)))
    x = torch.stack(rows)[:, None, :]
    cache = _cache(ca, 3, 16, 1, D, bits)
    slots = torch.arange(len(rows))
    ca.kv_write(cache, x.cuda(), -x.flip(0).cuda(), slots.cuda())
    _check_rows(cache, slots.cuda(), x, -x.flip(0), bits)


@pytest.mark.parametrize("bits", [4, 8])
def test_fp32_is_nearest_to_rounding(bits):
    """Inputs of 24 bits: the point's squared distance is the least, in units of beta^2, to
    2^-20: the roundings of the two compared sides (four sums below beta, two below 2 beta, one below 4 beta, three
        of the sides themselves: 4 2^-25 + 2 2^-24 + 2^-23 + 2 2^-24 + 2^-25 < 2^-20), plus
    2^-21 (4 bits) or 2^-17 (8 bits): a quotient that rounds across a half, off by half an ulp 2^-22 or 2^-18, twice."""
    import coset_amd as ca
    g = torch.Generator().manual_seed(3)
    x = torch.randn(500, 2, 128, generator=g)
    cache = _cache(ca, 32, 16, 2, 128, bits)
    slots = torch.arange(500)
    ca.kv_write(cache, x.cuda(), x.cuda(), slots.cuda())
    k, v = ca.kv_read(cache, slots.cuda(), torch.float32)
    assert torch.equal(k, v)
    xd = x.double()
    beta = O.scales_of(xd, bits)
    best = O.points_of(xd, beta).flatten(-2) * beta[..., None]
    d = lambda y: ((y - xd) ** 2).unflatten(-1, (-1, 8)).sum(-1)  # noqa: E731
    tol = 2.0 ** -20 + (2.0 ** -21 if bits == 4 else 2.0 ** -17)
    assert float(((d(k.cpu().double()) - d(best)) / beta[..., None] ** 2).max()) <= tol
    # and the error is below that of rounding each value at this scale
    plain = (torch.round(xd / beta[..., None]) * beta[..., None] - xd).square().sum()
    assert float((k.cpu().double() - xd).square().sum()) < 0.93 * float(plain)


def test_strides_slots_and_types():
    """Views of one projection, unaligned rows, heads apart, int32 slots, rows outside the cache, nothing to do."""
    import coset_amd as ca
    n, heads, dim = 9, 2, 64
    g = torch.Generator().manual_seed(5)
    for off in (0, 1, 8):
        buf = torch.randn(n, 2 * heads * dim + 24, generator=g).bfloat16().cuda()
        k = buf[:, off:off + heads * dim].view(n, heads, dim)
        v = buf[:, off + heads * dim:off + 2 * heads * dim].view(n, heads, dim)
        cache = _cache(ca, 2, 16, heads, dim, 4)
        slots = torch.tensor([3, -1, 31, 32, 0, 1 << 40, 17, -(1 << 50), 8], device="cuda")
        ca.kv_write(cache, k, v, slots)
        _check_rows(cache, slots, k, v, 4)
    flipped = torch.randn(heads, n, dim, generator=g).cuda().transpose(0, 1)
    wide = torch.randn(n, heads, 2 * dim, generator=g).cuda()[..., ::2]
    flipped, wide = flipped.bfloat16().float(), wide.bfloat16().float()
    cache = _cache(ca, 2, 16, heads, dim, 8)
    slots = torch.arange(n, device="cuda", dtype=torch.int32)
    ca.kv_write(cache, flipped, wide, slots)
    _check_rows(cache, slots.long(), flipped, wide, 8)
    before = cache.k.clone()
    ca.kv_write(cache, flipped[:0], wide[:0], slots[:0])
    k, v = ca.kv_read(cache, slots[:0])
    assert k.shape == (0, heads, dim) and torch.equal(before, cache.k)


def test_another_stream():
    import coset_amd as ca
    cache = _cache(ca, 8, 16, 2, 128, 4)
    k, v = (t.cuda() for t in _inputs(100, 2, 128, torch.bfloat16, 9))
    slots = torch.arange(100, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ca.kv_write(cache, k, v, slots)
        kk, vv = ca.kv_read(cache, slots)
    torch.cuda.current_stream().wait_stream(s)
    _check_rows(cache, slots, k, v, 4)
    assert torch.equal(kk, ca.kv_read(cache, slots)[0]) and torch.equal(vv, ca.kv_read(cache, slots)[1])


def test_offsets_beyond_32_bits():
    """The last rows of a cache of 2^31 words and more in each of k and v."""
    import coset_amd as ca
    heads, dim, page = 8, 256, 64
    pages = (1 << 31) // (heads * page * dim // 4) + 2
    cache = ca.E8KVCache.empty(pages, page, heads, dim, 8)
    assert cache.k.numel() > 1 << 31
    k, v = _inputs(5, heads, dim, torch.bfloat16, 2)
    rows = pages * page
    slots = torch.tensor([rows - 1, rows - page, rows - 2 * page + 5, 0, 7], device="cuda")
    ca.kv_write(cache, k.cuda(), v.cuda(), slots)
    _check_rows(cache, slots, k, v, 8)


def test_refusals():
    import coset_amd as ca
    cache = _cache(ca, 2, 16, 2, 64, 4)
    k = torch.randn(3, 2, 64, device="cuda")
    s = torch.arange(3, device="cuda")
    for args in ((k[:, :1], k[:, :1], s), (k[..., :32], k[..., :32], s), (k, k[:2], s), (k, k.half(), s),
                 (k.double(), k.double(), s), (k, k, s[:2]), (k, k, s.float()), (k, k, s[None]),
                 (k.cpu(), k, s), (k, k, s.cpu())):
        with pytest.raises(ValueError):
            ca.kv_write(cache, *args)
    with pytest.raises(ValueError):
        ca.kv_read(cache, s, torch.float64)
    with pytest.raises(ValueError):
        ca.kv_read(cache, s.cpu())
    for bad in (dict(page_size=8), dict(page_size=24), dict(head_dim=48), dict(head_dim=288), dict(bits=5)):
        with pytest.raises(ValueError):
            ca.E8KVCache.empty(**{**dict(pages=2, page_size=16, kv_heads=1, head_dim=64), **bad})
