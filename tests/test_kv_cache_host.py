"""Host side of the E8 key/value cache (no kernel): the tree masks, the constructor's checks, the C entry points'
refusals and the 64-bit oracle itself."""
import ctypes

import pytest
import torch

import kv_oracle as O


def test_draft_tree_mask():
    import coset_amd as ca
    m = ca.draft_tree_mask([-1, 0, 0, 1, -1, 4])
    assert m.shape == (6, 1) and m[:, 0].tolist() == [0b1, 0b11, 0b101, 0b1011, 0b10000, 0b110000]
    chain = ca.draft_tree_mask(torch.arange(-1, 129)[None].repeat(2, 1))
    assert chain.shape == (2, 130, 3)
    assert chain[1, 129].tolist() == [-1, -1, 3] and chain[0, 63].tolist() == [-1, 0, 0] and chain[0, 64].tolist() == [-1, 1, 0]
    for bad in ([0], [-1, 1], [[-1, 0], [-1, 2]]):
        with pytest.raises(ValueError):
            ca.draft_tree_mask(torch.tensor(bad))


def _tensors(pages=2, heads=3, page=16, dim=64, bits=4):
    w, nb = bits // 4, dim // 8
    return (torch.zeros(pages, heads, page, nb * w, dtype=torch.int32),
            torch.zeros(pages, heads, page // 4, nb, 4, w, dtype=torch.int32),
            torch.zeros(pages, heads, page, 2, dtype=torch.bfloat16))


def test_cache_constructor():
    import coset_amd as ca
    k, v, s = _tensors()
    c = ca.E8KVCache(k, v, s)
    assert (c.pages, c.page_size, c.kv_heads, c.head_dim, c.bits) == (2, 16, 3, 64, 4)
    k8, v8, s8 = _tensors(bits=8)
    assert ca.E8KVCache(k8, v8, s8, bits=8).head_dim == 64
    for args in ((k8, v8, s8, 4), (k, v, s, 8), (k, v, s, 3), (k.float(), v, s), (k, v, s.half()), (k, v[:1], s),
                 (k.transpose(0, 1).contiguous().transpose(0, 1), v, s), (k[0], v, s), (k, v, s[:, :, :8])):
        with pytest.raises(ValueError):
            ca.E8KVCache(*args)
    with pytest.raises(ca._lib.CosetError):   # tensors on the host: no kernel to run
        ca.kv_write(c, torch.zeros(1, 3, 64), torch.zeros(1, 3, 64), torch.zeros(1, dtype=torch.long))


def test_c_entry_points_refuse():
    """Argument checks come before any HIP call."""
    from coset_amd import _lib
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(buf) + 255) // 256 * 256
    good = dict(k=at, v=at, scales=at, pages=2, page_size=16, kv_heads=2, head_dim=64, bits=4)

    def cache(**more):
        return _lib.KvCacheStruct(**{**good, **more})

    def write(c, n=1, k=at, dtype=1):
        return lib.coset_kv_write(ctypes.addressof(c) if c else None, k, 128, 64, at, 128, 64, dtype, at, n, None)

    for c, rc in ((cache(bits=5), -1), (cache(page_size=8), -1), (cache(page_size=24), -1), (cache(head_dim=48), -2),
                  (cache(head_dim=288), -2), (cache(kv_heads=0), -1), (cache(pages=-1), -1), (cache(k=None), -1),
                  (cache(scales=at + 2), -1), (cache(pages=1 << 28), -2)):
        assert write(c) == rc, lib.coset_last_error()
    assert write(None) == -1 and write(cache(), n=-1) == -1 and write(cache(), k=None) == -1
    assert write(cache(), dtype=7) == -2 and write(cache(), k=at + 1) == -1

    def attend(c=None, n=4, heads=4, seqs=2, dtype=1, starts=None, pages=3, words=0, ws=at, floats=1 << 40, out=at, q=at):
        c = c or cache()
        return lib.coset_kv_attention(ctypes.addressof(c), q, 256, 64, dtype, n, heads, seqs, starts, at, at, pages, pages,
                                      None, words, 0.1, out, None, ws, floats, None)

    for more, rc in ((dict(heads=3), -1), (dict(heads=0), -1), (dict(n=5), -1), (dict(seqs=0), -1), (dict(dtype=3), -2),
                     (dict(words=1), -1), (dict(ws=None), -1), (dict(floats=10), -1), (dict(out=at + 8), -1),
                     (dict(q=None), -1), (dict(pages=1 << 30), -2), (dict(pages=0), -1), (dict(c=cache(pages=0)), -1),
                     (dict(n=-1), -1), (dict(words=-1), -1)):
        assert attend(**more) == rc, (more, lib.coset_last_error())
    assert attend(n=0) == 0   # nothing to do, nothing launched
    c = cache()
    assert lib.coset_kv_attention_workspace_floats(ctypes.addressof(c), 4, 2, 4, 1, 3) > 0
    assert lib.coset_kv_attention_workspace_floats(ctypes.addressof(c), 4, 2, 3, 1, 3) == 0

    def rope(side=None, **more):
        r = _lib.RopeStruct(**{**dict(table=at, positions=at, n=4, length=8, pos_stride=4, dim=64, rot=32, axes=1,
                                      norm=1, interleaved=0, dtype=1, w_dtype=1, eps=1e-6), **more})
        s = _lib.RopeSideStruct(**{**dict(x=at, out=at, token_stride=128, head_stride=64, heads=2), **(side or {})})
        return lib.coset_qk_norm_rope_fwd(ctypes.addressof(r), ctypes.addressof(s), ctypes.addressof(s), None)

    for more, rc in ((dict(dim=60), -2), (dict(dim=1024), -2), (dict(rot=36), -2), (dict(rot=72), -2), (dict(axes=0), -1),
                     (dict(axes=5), -1), (dict(n=-1), -1), (dict(length=0), -1), (dict(table=None), -1), (dict(eps=-1.0), -1),
                     (dict(dtype=9), -2), (dict(table=at + 4), -1), (dict(side=dict(x=None)), -1),
                     (dict(side=dict(out=at + 2)), -1), (dict(side=dict(heads=0)), -1)):
        assert rope(**more) == rc, (more, lib.coset_last_error())


@pytest.mark.parametrize("bits", [4, 8])
def test_oracle_point_is_nearest(bits):
    """The oracle's point against every move to a neighbour of E8 (the 240 shortest vectors), and its words' round trip."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(200, 32, generator=g, dtype=torch.float64)
    beta = O.scales_of(x, bits)
    p = O.points_of(x, beta)
    assert torch.equal(O.points_from(O.words_of(p, bits), bits), p.flatten(-2))
    assert float(p.floor().min()) >= -(1 << (bits - 1)) and float(p.floor().max()) < 1 << (bits - 1)
    short = []
    for i in range(8):
        for j in range(i):
            for a in (-1.0, 1.0):
                for b in (-1.0, 1.0):
                    e = [0.0] * 8
                    e[i], e[j] = a, b
                    short.append(e)
    for s in range(256):
        if bin(s).count("1") % 2 == 0:
            short.append([0.5 - (s >> i & 1) for i in range(8)])
    short = torch.tensor(short, dtype=torch.float64)
    assert short.shape == (240, 8)
    y = (x / beta[:, None]).unflatten(-1, (-1, 8))
    here = ((y - p) ** 2).sum(-1)
    there = ((y[:, :, None] - p[:, :, None] - short) ** 2).sum(-1).amin(-1)
    assert bool((here <= there + 1e-12).all())
