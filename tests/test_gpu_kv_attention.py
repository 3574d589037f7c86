"""Attention over the E8 key/value cache against its definition in 64 bits on the cache's own words.

Tolerance per element, derived from the roundings:
  out   u |out| + (w + 2 ds) sum p |v|   u: half an ulp of the output type (2^-8 bf16, 2^-11 fp16), 2^-22 for fp32, whose last steps round too;
        w: of a weight in fp16 parts (2^-11 in one part, 2^-21 in two and fp32 sums); ds: of a score
  lse   2 ds + 2^-21 max(1, |lse|)
  ds = e max(scale sum |q| |k|), e = 2^-17: products of exact points with queries of 11 bits or two parts of 11 (2^-22
       of the row's largest), sums of the offset points (at most 24 / 7 or 640 / 127 of the keys' largest) in fp32 over
       up to 256 terms and a few roundings of exp2's argument
"""
import math

import pytest
import torch

import kv_oracle as O

pytestmark = pytest.mark.gpu

_U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -22}
_W = {torch.bfloat16: 2.0 ** -11, torch.float16: 2.0 ** -19, torch.float32: 2.0 ** -19}


def _fill(ca, pages, page, kv, dim, bits, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    cache = ca.E8KVCache.empty(pages, page, kv, dim, bits)
    n = pages * page
    k = torch.randn(n, kv, dim, generator=g)
    v = torch.randn(n, kv, dim, generator=g) * torch.exp(spread * torch.randn(n, kv, 1, generator=g))
    ca.kv_write(cache, k.cuda(), v.cuda(), torch.arange(n, device="cuda"))
    return cache


def _table(seqs, most, pages, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(pages, generator=g)[:seqs * most].view(seqs, most).int()


def _check(got, lse, ref, dtype):
    out, want_lse, reach, size = ref
    ds = 2.0 ** -17 * size
    tol = _U[dtype] * out.abs().clamp(min=torch.finfo(dtype).tiny) + (_W[dtype] + 2 * ds[..., None]) * reach + 1e-30
    err = (got.cpu().double() - out).abs()
    assert torch.isfinite(got).all()
    assert bool((err <= tol).all()), (float((err / tol).max()), out[err > tol].abs().tolist()[:5], err[err > tol].tolist()[:5])
    none = want_lse == -math.inf
    assert bool((lse.cpu()[none] == -math.inf).all()) and bool((got.cpu()[none] == 0).all())
    err = (lse.cpu().double() - want_lse)[~none].abs()
    assert bool((err <= (2 * ds + 2.0 ** -21 * want_lse.abs().clamp(min=1))[~none]).all()), float(err.max())


def _run(ca, cache, lengths, counts, heads, dtype, table, mask=None, scale=None, q=None, seed=0):
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c)
    if q is None:
        g = torch.Generator().manual_seed(seed)
        q = torch.randn(starts[-1], heads, cache.head_dim, generator=g).to(dtype).cuda()
    lengths = torch.tensor(lengths, dtype=torch.int32)
    same = len(set(counts)) == 1
    out, lse = ca.kv_attention(q, cache, table.cuda(), lengths.cuda(), scale=scale, return_lse=True,
                               cu_queries=None if same else torch.tensor(starts, dtype=torch.int32, device="cuda"),
                               tree_mask=None if mask is None else mask.cuda())
    sc = cache.head_dim ** -0.5 if scale is None else scale
    _check(out, lse, O.attend(q, cache, table, lengths, starts, mask, sc), dtype)
    return q, out, lse


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dim,bits,page", [(32, 4, 16), (64, 8, 32), (64, 4, 64), (96, 4, 48), (128, 8, 16), (128, 4, 32),
                                           (160, 8, 64), (256, 4, 16), (256, 8, 128), (224, 4, 32)])
def test_one_token(dim, bits, page, dtype):
    """Decoding: one new token a sequence, lengths from one token to several steps of 128, one past each border."""
    import coset_amd as ca
    lengths = [1, 15, 16, 17, 33, 127, 128, 129, 300]
    most = -(-300 // page)
    for heads, kv in ((4, 2), (3, 3), (7, 1)):
        print(f"one token dim={dim} bits={bits} page={page} heads={heads}/{kv} {dtype}", flush=True)
        cache = _fill(ca, len(lengths) * most + 1, page, kv, dim, bits, dim + bits)
        _run(ca, cache, lengths, [1] * len(lengths), heads, dtype, _table(len(lengths), most, cache.pages, 1))


@pytest.mark.parametrize("dtype,dim,bits", [(torch.bfloat16, 128, 4), (torch.float16, 64, 8), (torch.float32, 128, 8),
                                            (torch.bfloat16, 256, 8), (torch.float32, 256, 4), (torch.float16, 96, 4)])
@pytest.mark.parametrize("heads,kv,counts", [(4, 1, [5, 5, 5]), (8, 2, [1, 9, 3]), (2, 2, [40, 17, 64]), (12, 1, [70, 1, 0]),
                                             (5, 1, [0, 0, 3])])
def test_chunks(heads, kv, counts, dtype, dim, bits):
    """Several new tokens a sequence, each seeing itself and what precedes it; sequences with none, new tokens only."""
    import coset_amd as ca
    print(f"chunk dim={dim} bits={bits} heads={heads}/{kv} counts={counts} {dtype}", flush=True)
    page = 32
    lengths = [counts[0], counts[1] + 130, counts[2] + 31]
    most = -(-max(lengths) // page)
    cache = _fill(ca, 3 * most, page, kv, dim, bits, 7)
    _run(ca, cache, lengths, counts, heads, dtype, _table(3, most, cache.pages, 2))


@pytest.mark.parametrize("dtype,dim,bits", [(torch.bfloat16, 128, 4), (torch.float16, 256, 4), (torch.float32, 64, 8)])
@pytest.mark.parametrize("heads,kv", [(2, 2), (8, 1), (6, 2)])
def test_whole_prompts(heads, kv, dtype, dim, bits):
    """Prompts from their first token on, whose rows see from one token to all of them: many row tiles of a sequence,
    odd and even numbers of them, beside one behind a context and one with more new tokens than cached ones."""
    import coset_amd as ca
    print(f"whole prompts dim={dim} bits={bits} heads={heads}/{kv} {dtype}", flush=True)
    page = 32
    for counts, lengths in (([400, 129, 1, 257], [400, 129, 5, 300]), ([65], [65]), ([330], [400]), ([300, 40], [200, 40])):
        most = -(-max(lengths) // page)
        cache = _fill(ca, len(counts) * most, page, kv, dim, bits, 13)
        _run(ca, cache, lengths, counts, heads, dtype, _table(len(counts), most, cache.pages, 4))


@pytest.mark.parametrize("dtype,dim,bits", [(torch.bfloat16, 128, 8), (torch.float16, 128, 4), (torch.float32, 64, 4)])
def test_trees(dtype, dim, bits):
    """Trees of drafted tokens over a context, some with no context, some rows that see nothing, and two mask words."""
    import coset_amd as ca
    g = torch.Generator().manual_seed(4)
    counts, page, kv = [7, 70, 1, 20], 16, 2
    lengths = [7, 170, 40, 20]
    rows = []
    for c in counts:
        parents = [int(torch.randint(-1, t, (1,), generator=g)) if t else -1 for t in range(c)]
        m = ca.draft_tree_mask(parents)
        rows.append(torch.nn.functional.pad(m, (0, 2 - m.shape[1])))
    mask = torch.cat(rows)
    mask[3] = 0           # the first sequence has no context: these rows see nothing
    mask[5] = 1 << 20     # a bit of no token
    mask[80, 1] = -1      # all bits of the second word
    most = -(-max(lengths) // page)
    cache = _fill(ca, 4 * most, page, kv, dim, bits, 8)
    for heads in (2, 8, 10):
        print(f"tree heads={heads} {dtype}", flush=True)
        _run(ca, cache, lengths, counts, heads, dtype, _table(4, most, cache.pages, 3), mask=mask)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_long_and_ragged(dtype):
    """Long sequences split over many workgroups beside short and empty ones."""
    import coset_amd as ca
    page, kv, dim = 64, 2, 64
    lengths = [20011, 0, 3, 700, 128, 9000]
    most = -(-max(lengths) // page)
    cache = _fill(ca, 6 * most, page, kv, dim, 4, 11)
    print(f"long {dtype}", flush=True)
    _run(ca, cache, lengths, [1] * 6, 4, dtype, _table(6, most, cache.pages, 5))
    _run(ca, cache, lengths[:1], [2], 2, dtype, _table(1, most, cache.pages, 6))
    # more sequences than lanes
    many = [(37 * i) % 300 for i in range(150)]
    _run(ca, cache, many, [1] * 150, 2, dtype, _table(150, 5, cache.pages, 7))


def test_masked_places_do_not_matter():
    """NaN, infinities and the largest numbers in rows behind a sequence's end, in drafted tokens that are not seen and
    in other pages change nothing, bit for bit."""
    import coset_amd as ca
    page, kv, dim = 16, 2, 128
    cache = _fill(ca, 12, page, kv, dim, 4, 12)
    table = torch.tensor([[3, 5, 1], [7, 2, 9]], dtype=torch.int32)
    lengths = [37, 41]
    mask = ca.draft_tree_mask([[-1, 0, -1], [-1, 0, 1]]).flatten(0, 1)
    mask[4:] &= ~1                       # no row but its first sees the second sequence's first new token
    mask[3] = 0
    q, out, lse = _run(ca, cache, lengths, [3, 3], 4, torch.bfloat16, table, mask=mask)
    bad = torch.full((3, kv, dim), float("nan"))
    bad[1] = float("inf")
    bad[2] = 1e19
    # behind the ends (rows 37.. of page 1, 41.. of page 9), another page, and the unseen token at 38 of page 9
    slots = torch.tensor([1 * page + 5, 9 * page + 9, 4 * page], device="cuda")
    ca.kv_write(cache, bad.cuda(), bad.cuda(), slots)
    slots = torch.tensor([9 * page + 6, 1 * page + 15, 9 * page + 15], device="cuda")
    ca.kv_write(cache, bad.cuda(), bad.cuda(), slots)
    again, lse2 = ca.kv_attention(q, cache, table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                                  tree_mask=mask.cuda(), return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    # a seen NaN reaches its sequence's rows and key head's heads, and no other
    ca.kv_write(cache, bad[:1, :1].expand(1, kv, dim).cuda(), torch.zeros(1, kv, dim).cuda(), torch.tensor([3 * page], device="cuda"))
    again = ca.kv_attention(q, cache, table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"), tree_mask=mask.cuda())
    assert torch.isnan(again[:3]).all() and torch.equal(again[3:], out[3:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_extreme_scales(dtype):
    """Value scales over 20 decades, keys and queries of large and tiny size, zero vectors, peaked and flat softmaxes."""
    import coset_amd as ca
    page, kv, dim = 32, 1, 64
    g = torch.Generator().manual_seed(6)
    n = 640
    k = torch.randn(n, kv, dim, generator=g)
    v = torch.randn(n, kv, dim, generator=g) * 10.0 ** torch.randint(-6, 4, (n, kv, 1), generator=g)
    v[::7] = 0
    k[::11] = 0
    cache = ca.E8KVCache.empty(20, page, kv, dim, 8)
    table = torch.arange(20, dtype=torch.int32)[None]
    ca.kv_write(cache, k.cuda(), v.cuda(), torch.arange(n, device="cuda"))
    for size, scale in ((1.0, None), (1e-4, 1.0), (300.0, 1e-3), (30.0, 0.125), (1.0, 0.0), (1.0, -0.2)):
        q = (size * torch.randn(3, 2, dim, generator=g)).to(dtype).cuda()
        q[1] = 0
        print(f"scales size={size} scale={scale} {dtype}", flush=True)
        _run(ca, cache, [n], [3], 2, dtype, table, scale=scale, q=q)
    # all values zero: zeros, and a finite sum of weights
    ca.kv_write(cache, k.cuda(), torch.zeros_like(v).cuda(), torch.arange(n, device="cuda"))
    out, lse = ca.kv_attention(q, cache, table.cuda(), torch.tensor([n], dtype=torch.int32, device="cuda"), return_lse=True)
    assert float(out.abs().max()) == 0 and torch.isfinite(lse).all()


def test_layouts_streams_and_workspace():
    """Strided and unaligned queries, a wide block table, a kept workspace, another stream: the same bits."""
    import coset_amd as ca
    page, kv, dim, heads = 32, 2, 128, 4
    cache = _fill(ca, 80, page, kv, dim, 4, 15)
    table = _table(2, 40, 80, 1)
    lengths = torch.tensor([1201, 650], dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(2, heads * dim + 9, generator=g).bfloat16().cuda()
    q = wide[:, 1:1 + heads * dim].view(2, heads, dim)
    flat = q.contiguous()
    out = ca.kv_attention(flat, cache, table.cuda(), lengths)
    assert torch.equal(out, ca.kv_attention(q, cache, table.cuda(), lengths))
    turned = flat.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(out, ca.kv_attention(turned, cache, table.cuda(), lengths))
    spread = torch.randn(2, heads, dim, 2, generator=g).bfloat16().cuda()
    spread[..., 0] = flat
    assert torch.equal(out, ca.kv_attention(spread[..., 0], cache, table.cuda(), lengths))
    big = torch.zeros(2, 64, dtype=torch.int32, device="cuda")
    big[:, :40] = table.cuda()
    assert torch.equal(out, ca.kv_attention(flat, cache, big[:, :40], lengths))
    ws = torch.full((1 << 22,), float("nan"), device="cuda")
    for _ in range(3):
        assert torch.equal(out, ca.kv_attention(flat, cache, table.cuda(), lengths, workspace=ws))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = ca.kv_attention(flat, cache, table.cuda(), lengths)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, other)
    # lengths and pages beyond the tables are clamped, nothing is read outside the cache
    wild = table.clone()
    wild[0, 3], wild[1, 2] = 1 << 30, -5
    got = ca.kv_attention(flat, cache, wild.cuda(), torch.tensor([1 << 30, -3], dtype=torch.int32, device="cuda"))
    assert torch.isfinite(got).all() and float(got[1].abs().max()) == 0


def test_captured_in_a_graph():
    """Replayed with other lengths, table and queries in the same buffers, eager work in between."""
    import coset_amd as ca
    page, kv, dim, heads = 32, 2, 128, 8
    cache = _fill(ca, 100, page, kv, dim, 4, 16)
    table = _table(3, 30, 100, 4).cuda()
    lengths = torch.tensor([900, 200, 33], dtype=torch.int32, device="cuda")
    q = torch.randn(3, heads, dim, device="cuda").bfloat16()
    k, v = torch.randn(2, 3, kv, dim, device="cuda").bfloat16()
    slots = torch.empty(3, dtype=torch.int64, device="cuda")

    def rows():
        last = lengths.long() - 1
        slots.copy_(table[torch.arange(3, device="cuda"), last // page].long() * page + last % page)

    def step():
        ca.kv_write(cache, k, v, slots)
        return ca.kv_attention(q, cache, table, lengths)

    rows()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        lengths += 7
        q.copy_(torch.randn(3, heads, dim, device="cuda"))
        k.copy_(torch.randn(3, kv, dim, device="cuda"))
        rows()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, step()), i


def test_offsets_beyond_32_bits():
    """The last pages of a cache of more than 2^31 words in each of k and v."""
    import coset_amd as ca
    heads, dim, page = 8, 256, 64
    pages = (1 << 31) // (heads * page * dim // 4) + 2
    cache = ca.E8KVCache.empty(pages, page, heads, dim, 8)
    g = torch.Generator().manual_seed(1)
    used = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32)
    n = 3 * page
    slots = (used[0].long()[:, None] * page + torch.arange(page)).reshape(-1)
    ca.kv_write(cache, torch.randn(n, heads, dim, generator=g).cuda(), torch.randn(n, heads, dim, generator=g).cuda(), slots.cuda())
    _run(ca, cache, [n - 3], [2], heads, torch.bfloat16, used)


def test_refusals():
    import coset_amd as ca
    cache = _fill(ca, 4, 16, 2, 64, 4, 1)
    q = torch.randn(2, 4, 64, device="cuda")
    table = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    lengths = torch.ones(2, dtype=torch.int32, device="cuda")

    def no(q=q, table=table, lengths=lengths, kind=ValueError, **more):
        with pytest.raises(kind):
            ca.kv_attention(q, cache, table, lengths, **more)

    no(q=q[0])
    no(q=q[..., :32])
    no(q=q.double())
    no(q=q[:, :3])
    no(q=q.cpu())
    no(table=table.long())
    no(table=table[:1])
    no(table=table.cpu())
    no(table=table.t()[:, :2].t().repeat(1, 2)[:, ::2])
    no(lengths=lengths.long())
    no(lengths=lengths[:1])
    no(q=torch.randn(3, 4, 64, device="cuda"))
    no(cu_queries=torch.zeros(2, dtype=torch.int32, device="cuda"))
    no(cu_queries=torch.zeros(3, dtype=torch.int64, device="cuda"))
    no(cu_queries=torch.zeros(3, dtype=torch.int32))
    no(tree_mask=torch.zeros(2, dtype=torch.int64, device="cuda"))
    no(tree_mask=torch.zeros(3, 1, dtype=torch.int64, device="cuda"))
    no(tree_mask=torch.zeros(2, 1, dtype=torch.int32, device="cuda"))
    no(workspace=torch.empty(1 << 22, dtype=torch.float16, device="cuda"))
    # no tokens: an empty result
    out, lse = ca.kv_attention(q[:0], cache, table, lengths, return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)


@pytest.mark.parametrize("dtype,dim,bits", [(torch.bfloat16, 128, 8), (torch.float16, 256, 4), (torch.float32, 64, 4)])
@pytest.mark.parametrize("counts", [[20], [33, 17], [1, 90]])
def test_many_rows_of_few_long_sequences(counts, dtype, dim, bits):
    """Draft trees over long contexts: few segments, each left in many parts by many workgroups."""
    import coset_amd as ca
    print(f"few long counts={counts} dim={dim} bits={bits} {dtype}", flush=True)
    g = torch.Generator().manual_seed(6)
    page, lengths = 64, [9001, 517][:len(counts)]
    most = -(-max(lengths) // page)
    cache = _fill(ca, len(counts) * most, page, 1, dim, bits, 17)
    rows = []
    for c in counts:
        parents = [int(torch.randint(-1, t, (1,), generator=g)) if t else -1 for t in range(c)]
        m = ca.draft_tree_mask(parents)
        rows.append(torch.nn.functional.pad(m, (0, 2 - m.shape[1])))
    table = _table(len(counts), most, cache.pages, 5)
    _run(ca, cache, lengths, counts, 4, dtype, table, mask=torch.cat(rows))
    _run(ca, cache, lengths, counts, 8, dtype, table)
