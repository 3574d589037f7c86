"""The attention operators of a served model whose keys and values are kept as E8 lattice points.

A case is a dict of plain values; ``op`` names the operator:

  rope       RMS norm of each head's query and key and the position rotation, in one pass
  rope_grad  its backward pass: gradients of queries, keys and both norm weights, beside the outputs
  cache      keys and values written to a paged cache as E8 points, and the same rows read back
  read       rows of a cache read back
  attend     attention of new tokens over a cache: one token per sequence, a chunk of a prompt
             (each token sees itself and what precedes it), or a tree of drafted tokens

The cache (``bits`` 4 or 8).  A head's vector x of D values is stored as one scale and D/8 points of the
lattice E8 = D8 + {0, 1/2}^8 diagonal, x_hat = beta * lambda.  With C = 7 - 2^-19 (4 bits) or 127 - 2^-15:

  beta = max|x| / C rounded up to bf16; 0 where max|x| < 2^-64; NaN where it is above 2^64 or not finite
  f = round(x / beta) (halves to even), r = x - beta f, g = f - (r < 0), all in fp32 (r is exact)
  integers: f, where sum f is odd coordinate k = argmax |r| moved by +1 (r_k >= 0) or -1
  halves:   g + 1/2, where sum g is odd coordinate k = argmin |r| moved by +1 (r_k < 0) or -1
  lambda = halves where 2 beta - sum|r| + odd(g) 2 min|r| < odd(f) (beta - 2 max|r|), else integers
           (the nearer of the two: the squared distances' difference, over beta)

(|x| < C beta keeps every lambda inside c + h/2 with c in [-8, 7] or [-128, 127] and h in {0, 1}.)  A block is
held in 8 * bits bits: n_j = c_j + 8 (or + 128) in field j, and since sum c is even, the lowest bit of n_7
follows from the others and holds h instead.

  k       [pages, kv heads, page size, D/8 * w]         w = bits / 4 words of 32 bits for a block
  v       [pages, kv heads, page size / 4, D/8, 4, w]   four tokens' words of a block side by side
  scales  [pages, kv heads, page size, 2]               bf16, the key's and the value's
"""
import math

import torch

own = False

# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------


def listed():
    return [
        # one decoding step of 16 sequences, 32 query and 8 key heads: one small launch, bound by latency
        dict(name="rope_decode", op="rope", tokens=16, hq=32, hkv=8, dim=128, rot=128, axes=1, norm=True, pairs="half",
             dtype="bf16"),
        # four prompts of 4096 tokens
        dict(name="rope_prompt", op="rope", tokens=16384, hq=32, hkv=8, dim=128, rot=128, axes=1, norm=True,
             pairs="half", dtype="bf16"),
        # a training step on 32 sequences of 512 tokens, 12 heads of 64 (768 wide), time / height / width positions
        dict(name="rope_train", op="rope_grad", tokens=16384, hq=12, hkv=12, dim=64, rot=64, axes=3, norm=True,
             pairs="half", dtype="bf16"),
        # the same in fp32 on a ragged batch, a rotation of part of the head in neighbouring pairs
        dict(name="rope_train_f32", op="rope_grad", tokens=1999, hq=10, hkv=2, dim=96, rot=64, axes=1, norm=True,
             pairs="neighbours", dtype="f32"),
        # the new tokens of 16 sequences: latency
        dict(name="cache_decode", op="cache", tokens=16, hkv=8, dim=128, bits=4, page=32, dtype="bf16"),
        # a prompt of 16384 tokens
        dict(name="cache_prompt", op="cache", tokens=16384, hkv=8, dim=128, bits=4, page=64, dtype="bf16"),
        # a shared prefix of 60001 tokens handed to a dense path
        dict(name="read_prefix", op="read", tokens=60001, hkv=8, dim=128, bits=8, page=128, dtype="bf16"),
        # one sequence, 1000 tokens: latency
        dict(name="attend_1", op="attend", seqs=1, new=1, ragged=False, shortest=1000, longest=1000, hq=32, hkv=8,
             dim=128, bits=4, page=32, mask="causal", dtype="bf16"),
        # a serving batch of 64 sequences of 1000 to 8192 tokens
        dict(name="attend_64", op="attend", seqs=64, new=1, ragged=False, shortest=1000, longest=8192, hq=32, hkv=8,
             dim=128, bits=4, page=64, mask="causal", dtype="bf16"),
        # one long document, 12 heads of 64 without sharing, fp32
        dict(name="attend_long_f32", op="attend", seqs=1, new=1, ragged=False, shortest=100003, longest=100003, hq=12,
             hkv=12, dim=64, bits=8, page=16, mask="causal", dtype="f32"),
        # 16 sequences with a tree of up to 32 drafted tokens each
        dict(name="attend_tree", op="attend", seqs=16, new=32, ragged=True, shortest=500, longest=6000, hq=32, hkv=8,
             dim=128, bits=8, page=32, mask="tree", dtype="bf16"),
        # 512 tokens more of two prompts, half precision
        dict(name="attend_chunk", op="attend", seqs=2, new=512, ragged=False, shortest=2500, longest=4001, hq=16, hkv=2,
             dim=256, bits=4, page=64, mask="causal", dtype="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = [(32, 8), (12, 12), (16, 2), (10, 2), (8, 1), (16, 16), (24, 8), (6, 3)]


def draw(rng):
    op = rng.choice(["rope", "rope_grad", "cache", "read", "attend", "attend", "attend", "attend"])
    hq, hkv = rng.choice(_HEADS)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    dim = rng.choice([64, 96, 128, 128, 256])
    bits = rng.choice([4, 4, 8])
    page = rng.choice([16, 32, 64, 128])
    if op in ("rope", "rope_grad"):
        most = 16384 * 40 * 128 if op == "rope" else 16384 * 24 * 64
        tokens = _log(rng, 1 if op == "rope" else 30, max(64, most // ((hq + hkv) * dim * (2 if dtype == "f32" else 1))))
        return dict(op=op, tokens=tokens, hq=hq, hkv=hkv, dim=dim, rot=rng.choice([dim, dim, dim // 2]),
                    axes=rng.choice([1, 1, 3]), norm=rng.random() < 0.8, pairs=rng.choice(["half", "half", "neighbours"]),
                    dtype=dtype)
    if op in ("cache", "read"):
        most = (16384 if op == "cache" else 60000) * 8 * 128
        tokens = _log(rng, 1 if op == "cache" else 30, most // (hkv * dim * (2 if dtype == "f32" else 1)))
        return dict(op=op, tokens=tokens, hkv=hkv, dim=dim, bits=bits, page=page, dtype=dtype)
    mask, new = rng.choice([("causal", 1), ("causal", 1), ("tree", _log(rng, 2, 80)), ("causal", _log(rng, 2, 512))])
    longest = _log(rng, max(new, 20), 131072)
    # no more cached values and no more products than the largest listed cases have
    most = min(64 * 8192 * 8 * 128, 2 * 512 * 16 * 4001 * 256 * hkv // (new * hq))
    seqs = max(1, min(_log(rng, 1, 128), most // (longest * hkv * dim)))
    longest = max(new, min(longest, most // (seqs * hkv * dim)))
    return dict(op=op, seqs=seqs, new=new, ragged=new > 1 and rng.random() < 0.5,
                shortest=rng.choice([longest, max(new, longest // 8)]), longest=longest, hq=hq, hkv=hkv, dim=dim,
                bits=bits, page=page, mask=mask, dtype=dtype)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_EPS = 1e-6


def _randn(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


def _randint(g, lo, hi, shape):
    return torch.randint(lo, hi, shape, device="cuda", generator=g)


def _sections(case):
    """How many rotated pairs follow each axis's position (the first axis takes what three do not share evenly)."""
    half = case["rot"] // 2
    if case["axes"] == 1:
        return [half]
    rest = half * 3 // 8
    return [half - 2 * rest, rest, rest]


def _keys_values(case, g, n):
    """Keys, some channels of them several times the others' size, and values, as they leave a projection: views of
    one [tokens, 2 * kv heads * D] product."""
    hkv, dim = case["hkv"], case["dim"]
    both = _randn(g, n, 2 * hkv * dim)
    loud = 1 + 3 * (torch.rand(hkv * dim, device="cuda", generator=g) < 0.05).float()
    both[:, :hkv * dim] *= loud
    both = both.to(_DT[case["dtype"]])
    k, v = both.split(hkv * dim, dim=1)
    return k.view(n, hkv, dim), v.view(n, hkv, dim)


def _slots(case, g, n):
    """n cache rows: the tokens of whole pages, the pages in no order."""
    pages = -(-n // case["page"]) + 3
    order = torch.randperm(pages, device="cuda", generator=g)
    rows = order[:, None] * case["page"] + torch.arange(case["page"], device="cuda")
    return pages, rows.reshape(-1)[:n].contiguous()


def _empty(pages, case):
    w = case["bits"] // 4
    nb = case["dim"] // 8
    h, page = case["hkv"], case["page"]
    return dict(k=torch.zeros((pages, h, page, nb * w), dtype=torch.int32, device="cuda"),
                v=torch.zeros((pages, h, page // 4, nb, 4, w), dtype=torch.int32, device="cuda"),
                scales=torch.zeros((pages, h, page, 2), dtype=torch.bfloat16, device="cuda"))


def _filled(case, g, pages):
    """A cache whose rows are all written."""
    n = pages * case["page"]
    state = _empty(pages, case)
    k, v = _keys_values(case, g, n)
    _write(state, k, v, torch.arange(n, device="cuda"), case["bits"])
    return state


def _counts(case):
    """New tokens of each sequence: all of them, or (ragged) from half of them up."""
    seqs, new = case["seqs"], case["new"]
    return [new - (5 * b % (new - new // 2) if case["ragged"] else 0) for b in range(seqs)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DT[case["dtype"]]
    op = case["op"]
    if op in ("rope", "rope_grad"):
        n, hq, hkv, dim, rot = (case[i] for i in ("tokens", "hq", "hkv", "dim", "rot"))
        # queries, keys and values of one projection; keys and queries are read where they stand
        qkv = _randn(g, n, (hq + 2 * hkv) * dim).to(dt)
        q = qkv[:, :hq * dim].view(n, hq, dim)
        k = qkv[:, hq * dim:(hq + hkv) * dim].view(n, hkv, dim)
        length = 8192
        angle = torch.arange(length, dtype=torch.float64, device="cuda")[:, None] * torch.pow(
            10000.0, -torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
        table = torch.cat([angle.cos(), angle.sin()], dim=1).float()
        state = dict(case=case, q=q, k=k, table=table, positions=_randint(g, 0, length, (case["axes"], n)),
                     sections=_sections(case), wq=None, wk=None)
        if case["norm"]:
            state["wq"] = (1 + 0.2 * _randn(g, dim)).to(dt)
            state["wk"] = (1 + 0.2 * _randn(g, dim)).to(dt)
        if op == "rope_grad":
            state["gq"] = _randn(g, n, hq, dim).to(dt)
            state["gk"] = _randn(g, n, hkv, dim).to(dt)
            for name in ("q", "k", "wq", "wk"):
                if state[name] is not None:
                    state[name] = state[name].detach().requires_grad_()
        return state
    if op == "cache":
        pages, slots = _slots(case, g, case["tokens"])
        k, v = _keys_values(case, g, case["tokens"])
        return dict(case=case, slots=slots, kx=k, vx=v, **_empty(pages, case))
    if op == "read":
        pages, slots = _slots(case, g, case["tokens"])
        return dict(case=case, slots=slots, **_filled(case, g, pages))
    seqs, new, longest, page = case["seqs"], case["new"], case["longest"], case["page"]
    most = -(-longest // page)
    state = dict(case=case, **_filled(case, g, seqs * most))
    state["table"] = torch.randperm(seqs * most, device="cuda", generator=g).view(seqs, most).int()
    lengths = _randint(g, case["shortest"], longest + 1, (seqs,)).int()
    lengths[0] = longest
    state["lengths"] = lengths
    counts = torch.tensor(_counts(case), device="cuda")
    starts = torch.zeros(seqs + 1, dtype=torch.int32, device="cuda")
    starts[1:] = counts.cumsum(0)
    state["starts"] = starts
    state["q"] = _randn(g, sum(_counts(case)), case["hq"], case["dim"]).to(dt)
    state["mask"] = None
    if case["mask"] == "tree":
        # each drafted token follows an earlier one of its sequence, the first the context; bit j: token j is on its path
        seen = torch.eye(new, dtype=torch.bool, device="cuda").expand(seqs, new, new).contiguous()
        parent = (torch.rand((seqs, new), device="cuda", generator=g) * torch.arange(new, device="cuda")).long()
        at = torch.arange(seqs, device="cuda")
        for t in range(1, new):
            seen[:, t] |= seen[at, parent[:, t]]
        width = -(-new // 64)
        flat = torch.zeros((seqs, new, width * 64), dtype=torch.int64, device="cuda")
        flat[:, :, :new] = seen
        words = (flat.view(seqs, new, width, 64) << torch.arange(64, device="cuda")).sum(-1)
        state["mask"] = words[torch.arange(new, device="cuda")[None, :] < counts[:, None]].contiguous()
    return state


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------


def _quantise(x, bits):
    """fp32 [..., D] -> (c [..., D/8, 8] int32, h [..., D/8] bool, beta [...] fp32)."""
    top = 7 - 2.0 ** -19 if bits == 4 else 127 - 2.0 ** -15
    amax = x.abs().amax(-1)
    # divided by a tensor: by a Python number it is a product with the reciprocal
    up = (((amax / torch.full_like(amax, top)).view(torch.int32) + 0xffff) & -0x10000).view(torch.float32)
    small = amax < 2.0 ** -64
    fine = (amax >= 2.0 ** -64) & (amax <= 2.0 ** 64)
    beta = torch.where(fine, up, torch.where(small, 0.0, math.nan))
    unit = torch.where(fine, up, 1.0)[..., None]
    x = torch.where(fine[..., None], x, 0.0).unflatten(-1, (-1, 8))
    f = (x / unit[..., None]).round()
    r = x - unit[..., None] * f
    g = f - (r < 0).float()
    a = r.abs()
    s = a[..., :4] + a[..., 4:]
    s = s[..., :2] + s[..., 2:]
    s = s[..., 0] + s[..., 1]
    most, least = a.amax(-1), a.amin(-1)
    odd_f = f.sum(-1).remainder(2) == 1
    odd_g = g.sum(-1).remainder(2) == 1
    half = 2 * unit - s + torch.where(odd_g, 2 * least, 0.0) < torch.where(odd_f, unit - 2 * most, 0.0)
    lane = torch.arange(8, device=x.device)
    picked = torch.where(half, least, most)[..., None] == a
    first = torch.where(picked, lane, 8).amin(-1, keepdim=True) == lane
    step = torch.where((r < 0) == half[..., None], 1.0, -1.0)
    moved = first & torch.where(half, odd_g, odd_f)[..., None]
    c = torch.where(half[..., None], g, f) + torch.where(moved, step, 0.0)
    return c.int(), half, beta


def _pack(c, half, bits):
    """[..., nb, 8], [..., nb] -> words [..., nb, w] int32."""
    n = c + (8 if bits == 4 else 128)
    last = (n[..., 7:] & -2) | half[..., None].int()
    n = torch.cat([n[..., :7], last], dim=-1)
    per = 32 // bits
    n = n.unflatten(-1, (-1, per)) << (bits * torch.arange(per, device=c.device, dtype=torch.int32))
    return n.sum(-1, dtype=torch.int32)


def _points(words, bits):
    """words [..., nb, w] int32 -> lambda [..., nb * 8] fp32."""
    per = 32 // bits
    n = (words[..., None] >> (bits * torch.arange(per, device=words.device, dtype=torch.int32))) & ((1 << bits) - 1)
    n = n.flatten(-2)
    half = n[..., 7:] & 1
    odd = n[..., :7].sum(-1, keepdim=True, dtype=torch.int32) & 1
    c = torch.cat([n[..., :7], (n[..., 7:] & -2) | odd], dim=-1) - (8 if bits == 4 else 128)
    return (c.float() + 0.5 * half.float()).flatten(-2)


def _write(state, k, v, slots, bits):
    page = state["k"].shape[2]
    w = bits // 4
    at, off = slots // page, slots % page
    c, half, beta = _quantise(k.float(), bits)
    state["k"][at, :, off] = _pack(c, half, bits).flatten(-2)
    state["scales"][at, :, off, 0] = beta.to(torch.bfloat16)
    c, half, beta = _quantise(v.float(), bits)
    state["v"][at, :, off // 4, :, off % 4] = _pack(c, half, bits).view(*c.shape[:-1], w)
    state["scales"][at, :, off, 1] = beta.to(torch.bfloat16)


def _read(state, slots, bits, dtype):
    page = state["k"].shape[2]
    at, off = slots // page, slots % page
    scales = state["scales"][at, :, off].float()
    kw = state["k"][at, :, off].unflatten(-1, (-1, bits // 4))
    vw = state["v"][at, :, off // 4, :, off % 4]
    return ((_points(kw, bits) * scales[..., :1]).to(dtype), (_points(vw, bits) * scales[..., 1:]).to(dtype))


def _cos_sin(state):
    """[N, 1, rot/2] each: a pair's angle goes by the position on its own axis."""
    axis = torch.repeat_interleave(torch.arange(len(state["sections"]), device="cuda"),
                                   torch.tensor(state["sections"], device="cuda"))
    pos = state["positions"][axis].t()
    half = axis.numel()
    pair = torch.arange(half, device="cuda")
    return state["table"][pos, pair][:, None], state["table"][pos, half + pair][:, None]


def _pairs(x, case):
    rot = case["rot"]
    if case["pairs"] == "half":
        return x[..., :rot // 2], x[..., rot // 2:rot]
    return x[..., 0:rot:2], x[..., 1:rot:2]


def _joined(a, b, rest, case):
    if case["pairs"] == "half":
        return torch.cat([a, b, rest], dim=-1)
    return torch.cat([torch.stack([a, b], dim=-1).flatten(-2), rest], dim=-1)


def _rope(x, w, cos, sin, case):
    z = x.float()
    if w is not None:
        z = z * torch.rsqrt((z * z).mean(-1, keepdim=True) + _EPS) * w.float()
    a, b = _pairs(z, case)
    return _joined(a * cos - b * sin, b * cos + a * sin, z[..., case["rot"]:], case).to(x.dtype)


def _rope_grad(x, w, gy, cos, sin, case):
    gy = gy.float()
    a, b = _pairs(gy, case)
    gz = _joined(a * cos + b * sin, b * cos - a * sin, gy[..., case["rot"]:], case)
    if w is None:
        return gz.to(x.dtype), None
    z = x.float()
    r = torch.rsqrt((z * z).mean(-1, keepdim=True) + _EPS)
    u = z * r
    gw = (gz * u).sum((0, 1)).to(w.dtype)
    gu = gz * w.float()
    return (r * (gu - u * (gu * u).mean(-1, keepdim=True))).to(x.dtype), gw


def _attend(state):
    case = state["case"]
    bits, dim, hq, hkv = case["bits"], case["dim"], case["hq"], case["hkv"]
    table, lengths, starts = state["table"].long(), state["lengths"].long(), state["starts"].long()
    seqs, new = table.shape[0], case["new"]
    counts = starts[1:] - starts[:-1]
    t = torch.arange(new, device="cuda")
    there = t < counts[:, None]
    row = torch.where(there, starts[:-1, None] + t, 0)
    total = table.shape[1] * case["page"]
    scales = state["scales"][table].float().transpose(1, 2).flatten(2, 3)
    k = state["k"][table].unflatten(-1, (-1, bits // 4)).transpose(1, 2).flatten(2, 3)
    v = state["v"][table].permute(0, 2, 1, 3, 5, 4, 6).flatten(2, 4)
    j = torch.arange(total, device="cuda")
    inside = j < lengths[:, None]
    k = _points(k, bits) * torch.where(inside[:, None, :, None], scales[..., :1], 0.0)
    v = _points(v, bits) * torch.where(inside[:, None, :, None], scales[..., 1:], 0.0)
    q = state["q"].float()[row].view(seqs, new, hkv, hq // hkv, dim).permute(0, 2, 1, 3, 4).flatten(2, 3)
    s = torch.matmul(q, k.transpose(2, 3)) * dim ** -0.5
    draft = j - (lengths - counts)[:, None]
    if state["mask"] is None:
        seen = draft[:, None, :] <= t[:, None]
    else:
        at = draft.clamp(0, 64 * state["mask"].shape[1] - 1)
        words = state["mask"][row].gather(2, (at >> 6)[:, None].expand(-1, new, -1))
        seen = (draft < 0)[:, None] | ((words >> (at & 63)[:, None] & 1) == 1)
    seen = (seen & inside[:, None] & there[:, :, None]).repeat_interleave(hq // hkv, dim=1)[:, None]
    s = torch.where(seen, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(s - top)
    l = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(l == 0, 1.0, l)
    lse = top + torch.log(l)
    out = out.view(seqs, hkv, new, hq // hkv, dim).permute(0, 2, 1, 3, 4).reshape(seqs, new, hq, dim)
    lse = lse.view(seqs, hkv, new, hq // hkv).permute(0, 2, 1, 3).reshape(seqs, new, hq)
    return out[there].to(state["q"].dtype), lse[there]


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def _run_own(state):
    import coset_amd as ca

    case = state["case"]
    op = case["op"]
    if op in ("rope", "rope_grad"):
        q, k = ca.qk_norm_rope(state["q"], state["k"], state["table"], state["positions"], state["wq"], state["wk"],
                               eps=_EPS, sections=state["sections"], interleaved=case["pairs"] == "neighbours")
        if op == "rope":
            return q, k
        wanted = [state[name] for name in ("q", "k", "wq", "wk") if state[name] is not None]
        return (q.detach(), k.detach()) + torch.autograd.grad([q, k], wanted, [state["gq"], state["gk"]])
    cache = ca.E8KVCache(state["k"], state["v"], state["scales"], bits=case["bits"])
    if op == "attend":
        return ca.kv_attention(state["q"], cache, state["table"], state["lengths"],
                               cu_queries=state["starts"] if case["ragged"] else None, tree_mask=state["mask"],
                               return_lse=True)
    if op == "cache":
        ca.kv_write(cache, state["kx"], state["vx"], state["slots"])
    return ca.kv_read(cache, state["slots"], dtype=_DT[case["dtype"]])


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        case = state["case"]
        op = case["op"]
        if op in ("rope", "rope_grad"):
            cos, sin = _cos_sin(state)
            out = (_rope(state["q"], state["wq"], cos, sin, case), _rope(state["k"], state["wk"], cos, sin, case))
            if op == "rope":
                return out
            gq, gwq = _rope_grad(state["q"], state["wq"], state["gq"], cos, sin, case)
            gk, gwk = _rope_grad(state["k"], state["wk"], state["gk"], cos, sin, case)
            return out + ((gq, gk) if gwq is None else (gq, gk, gwq, gwk))
        if op == "attend":
            return _attend(state)
        if op == "cache":
            _write(state, state["kx"], state["vx"], state["slots"], case["bits"])
        return _read(state, state["slots"], case["bits"], _DT[case["dtype"]])


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    op, size, dim = case["op"], _SIZE[case["dtype"]], case["dim"]
    if op in ("rope", "rope_grad"):
        n, values = case["tokens"], case["tokens"] * (case["hq"] + case["hkv"]) * dim
        # a token's positions and its row of the table; the rotation 3 operations a value, the norm 4
        side = n * (8 * case["axes"] + 4 * case["rot"])
        if op == "rope":
            return {"bytes": 2 * values * size + side, "flops": 7 * values}
        return {"bytes": 4 * values * size + side, "flops": 20 * values}
    held = lambda n: n * case["hkv"] * 2 * (dim * case["bits"] // 8 + 2)  # noqa: E731
    if op in ("cache", "read"):
        n, values = case["tokens"], 2 * case["tokens"] * case["hkv"] * dim
        # the nearest point of a block about 10 operations a value; read back 2
        if op == "read":
            return {"bytes": held(n) + values * size + 8 * n, "flops": 2 * values}
        return {"bytes": 2 * held(n) + 2 * values * size + 8 * n, "flops": 12 * values}
    # lengths are even between the shortest and the longest
    tokens = case["longest"] + (case["seqs"] - 1) * (case["shortest"] + case["longest"]) / 2
    rows = sum(_counts(case))
    queries = rows * case["hq"] * dim
    pairs = tokens * rows / case["seqs"] - (0 if case["mask"] == "tree" else rows * case["new"] / 2)
    return {"bytes": held(tokens) + 2 * queries * size + 4 * rows * case["hq"], "flops": 4 * pairs * case["hq"] * dim}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------


def _exact_rope(case, state):
    """Pairs as complex numbers, the norm as written; gradients by automatic differentiation."""
    state = {name: t.detach().double() if isinstance(t, torch.Tensor) and t.is_floating_point() else t
             for name, t in state.items()}
    half = case["rot"] // 2
    unit = torch.complex(state["table"][:, :half], state["table"][:, half:])
    at = 0
    turns = []
    for axis, width in enumerate(state["sections"]):
        turns.append(unit[state["positions"][axis], at:at + width])
        at += width
    turn = torch.cat(turns, dim=1)[:, None]

    def one(x, w):
        if w is not None:
            x = x / ((x ** 2).sum(-1, keepdim=True) / case["dim"] + _EPS).sqrt() * w
        front, rest = x[..., :2 * half], x[..., 2 * half:]
        if case["pairs"] == "half":
            z = torch.complex(front[..., :half].contiguous(), front[..., half:].contiguous()) * turn
            return torch.cat([z.real, z.imag, rest], dim=-1)
        z = torch.view_as_complex(front.reshape(*front.shape[:-1], half, 2).contiguous()) * turn
        return torch.cat([torch.view_as_real(z).flatten(-2), rest], dim=-1)

    names = [name for name in ("q", "k", "wq", "wk") if state[name] is not None]
    if case["op"] == "rope":
        return one(state["q"], state["wq"]), one(state["k"], state["wk"])
    for name in names:
        state[name].requires_grad_()
    out = (one(state["q"], state["wq"]), one(state["k"], state["wk"]))
    grads = torch.autograd.grad(out, [state[name] for name in names], [state["gq"], state["gk"]])
    return tuple(o.detach() for o in out) + grads


def _exact_nearest(x, bits):
    """beta times the E8 point nearest to x / beta, by the distances to the nearest points of both cosets."""
    x = x.double()
    amax = x.abs().amax(-1, keepdim=True)
    beta = amax / (7 - 2.0 ** -19 if bits == 4 else 127 - 2.0 ** -15)
    # up to 8 significant bits: 45 of the 52 stored ones cleared
    rest = (1 << 45) - 1
    beta = ((beta.view(torch.int64) + rest) & ~rest).view(torch.float64)
    x, scale = x.unflatten(-1, (-1, 8)), beta[..., None]
    whole = torch.round(x / scale)
    away = (x - whole * scale).abs()
    ranks = torch.arange(8, 0, -1, device="cuda")
    best = []
    for shift, p, e in ((0.0, whole, away), (0.5, torch.where(x < whole * scale, whole - 1, whole), scale / 2 - away)):
        # the coordinate that is furthest from its nearest value, the first of equals
        k = ((e == e.amax(-1, keepdim=True)) * ranks).argmax(-1, keepdim=True)
        other = torch.where(x >= (p + shift) * scale, p + 1, p - 1)
        odd = p.sum(-1, keepdim=True) % 2 != 0
        p = torch.where(odd, p.scatter(-1, k, other.gather(-1, k)), p) + shift
        best.append((p, ((x - p * scale) ** 2).sum(-1, keepdim=True)))
    # equals, beyond the rounding of these sums, go to the integers
    point = torch.where(best[1][1] < best[0][1] * (1 - 1e-12), best[1][0], best[0][0])
    return point.flatten(-2) * beta


def _exact_values(words, beta, bits):
    """words [..., blocks, w] and a scale for each vector -> [..., 8 * blocks] fp64, by the fields' arithmetic."""
    fields = []
    for j in range(8):
        word, shift = words[..., j * bits // 32].long(), j * bits % 32
        fields.append(torch.div(word % (1 << 32), 1 << shift, rounding_mode="floor") % (1 << bits))
    half = fields[7] % 2
    fields[7] = fields[7] - half + sum(fields[:7]) % 2
    value = torch.stack(fields, dim=-1).double() - (1 << (bits - 1)) + half[..., None].double() / 2
    return value.flatten(-2) * beta.double()[..., None]


def _exact_attend(case, state):
    """Sequence by sequence and head by head."""
    bits, dim, group, page = case["bits"], case["dim"], case["hq"] // case["hkv"], case["page"]
    starts, lengths = state["starts"].tolist(), state["lengths"].tolist()
    outs, sums = [], []
    for b, length in enumerate(lengths):
        pages = state["table"][b, :-(-length // page)].long()
        rows = state["q"][starts[b]:starts[b + 1]].double()
        new = rows.shape[0]
        scales = state["scales"][pages].transpose(0, 1).flatten(1, 2)[:, :length]
        kw = state["k"][pages].transpose(0, 1).flatten(1, 2)[:, :length]
        k = _exact_values(kw.unflatten(-1, (dim // 8, bits // 4)), scales[..., 0], bits)
        vw = state["v"][pages].permute(1, 0, 2, 4, 3, 5).flatten(1, 3)[:, :length]
        v = _exact_values(vw, scales[..., 1], bits)
        drafts = torch.arange(length, device="cuda") - (length - new)
        if state["mask"] is None:
            hidden = drafts[None] > torch.arange(new, device="cuda")[:, None]
        else:
            words = state["mask"][starts[b]:starts[b + 1]]
            bit = torch.stack([(words[:, i // 64] >> (i % 64)) & 1 for i in range(new)], dim=1) == 0
            hidden = torch.zeros((new, length), dtype=torch.bool, device="cuda")
            hidden[:, length - new:] = bit
        heads = [torch.empty(0)] * case["hq"]
        tops = [torch.empty(0)] * case["hq"]
        for h in range(case["hq"]):
            s = rows[:, h] @ k[h // group].t().contiguous() / math.sqrt(dim)
            s = s.masked_fill(hidden, -math.inf)
            tops[h] = torch.logsumexp(s, dim=1)
            heads[h] = torch.softmax(s, dim=1) @ v[h // group]
        outs.append(torch.stack(heads, dim=1))
        sums.append(torch.stack(tops, dim=1))
    return torch.cat(outs), torch.cat(sums)


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op in ("rope", "rope_grad"):
        return _exact_rope(case, state)
    if op == "attend":
        return _exact_attend(case, state)
    if op == "cache":
        return _exact_nearest(state["kx"], case["bits"]), _exact_nearest(state["vx"], case["bits"])
    slots, page, bits = state["slots"], case["page"], case["bits"]
    at, off = slots // page, slots % page
    scales = state["scales"][at, :, off]
    kw = state["k"][at, :, off].unflatten(-1, (case["dim"] // 8, bits // 4))
    vw = state["v"][at, :, off // 4, :, off % 4]
    return _exact_values(kw, scales[..., 0], bits), _exact_values(vw, scales[..., 1], bits)
