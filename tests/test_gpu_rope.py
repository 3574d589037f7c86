"""Head norms with the position rotation, and its gradient, against the definition in 64 bits.

Tolerance: the outputs are a handful of fp32 operations on values of size z (norm, weight, two products and a sum), so
16 units of 2^-24 on |z_a| + |z_b| and half an ulp of the output's type.  A gradient of x adds the mean over dim:
32 units on r (|du| + |u| mean |du u|).  A weight's gradient sums n * heads terms in fp32 in chains of at most a few
hundred and trees above: 2^-15 of sum |dz u|, and half an ulp of its type."""
import pytest
import torch

pytestmark = pytest.mark.gpu



def _half_ulp(x, dtype):
    """Of dtype at |x|; subnormals have the smallest normal number's."""
    f = torch.finfo(dtype)
    return 1.01 * f.eps / 2 * x.abs().clamp(min=f.tiny)



def _turn(z, cos, sin, rot, interleaved):
    z = z.clone()
    if interleaved:
        a, b = z[..., 0:rot:2].clone(), z[..., 1:rot:2].clone()
        z[..., 0:rot:2], z[..., 1:rot:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = z[..., :rot // 2].clone(), z[..., rot // 2:rot].clone()
        z[..., :rot // 2], z[..., rot // 2:rot] = a * cos - b * sin, b * cos + a * sin
    return z


def _angles(table, positions, sections):
    rot = table.shape[1]
    pos = positions.clamp(0, table.shape[0] - 1)
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections))
    p = pos[axis].t()
    i = torch.arange(rot // 2)
    return table[p, i][:, None].double(), table[p, rot // 2 + i][:, None].double()


def _make(n, hq, hk, dim, rot, axes, dtype, seed, length=512):
    import coset_amd as ca
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(n, hq, dim, generator=g).to(dtype)
    k = (3 * torch.randn(n, hk, dim, generator=g)).to(dtype)
    wq = (1 + 0.3 * torch.randn(dim, generator=g)).to(dtype)
    wk = (1 + 0.3 * torch.randn(dim, generator=g)).to(dtype)
    table = ca.rope_table(length, rot, device="cpu")
    pos = torch.randint(0, length, (axes, n), generator=g)
    half = rot // 2
    sections = [half] if axes == 1 else [half - 2 * (half // 3)] + [half // 3] * 2 if axes == 3 else [half - half // 4, half // 4]
    return q, k, wq, wk, table, pos, sections


CASES = [  # n, hq, hk, dim, rot, axes, interleaved
    (1, 1, 1, 8, 8, 1, False), (1, 32, 8, 128, 128, 1, False), (5, 3, 1, 64, 64, 3, False), (37, 2, 2, 96, 48, 1, True),
    (130, 6, 3, 128, 64, 2, False), (19, 4, 4, 256, 256, 3, True), (7, 2, 1, 40, 24, 1, False), (9, 1, 1, 512, 512, 1, False),
    (300, 5, 1, 80, 80, 1, True), (3, 2, 2, 64, 8, 1, False)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("normed", [True, False])
@pytest.mark.parametrize("n,hq,hk,dim,rot,axes,interleaved", CASES)
def test_forward_and_gradients(n, hq, hk, dim, rot, axes, interleaved, normed, dtype):
    import coset_amd as ca
    print(f"rope n={n} {hq}/{hk} dim={dim} rot={rot} axes={axes} near={interleaved} norm={normed} {dtype}", flush=True)
    q, k, wq, wk, table, pos, sections = _make(n, hq, hk, dim, rot, axes, dtype, n + dim)
    g = torch.Generator().manual_seed(1)
    gq, gk = torch.randn(q.shape, generator=g).to(dtype), torch.randn(k.shape, generator=g).to(dtype)
    cos, sin = _angles(table, pos, sections)
    leaves = [t.cuda().requires_grad_() for t in ((q, k, wq, wk) if normed else (q, k))]
    args = (leaves[2], leaves[3]) if normed else (None, None)
    oq, ok = ca.qk_norm_rope(leaves[0], leaves[1], table.cuda(), pos.cuda(), *args, eps=1e-5, sections=sections,
                             interleaved=interleaved)
    grads = torch.autograd.grad([oq, ok], leaves, [gq.cuda(), gk.cuda()])
    with torch.no_grad():
        fq, fk = ca.qk_norm_rope(leaves[0], leaves[1], table.cuda(), pos.cuda(), *args, eps=1e-5, sections=sections,
                                 interleaved=interleaved)
    assert torch.equal(fq, oq) and torch.equal(fk, ok)
    for i, (x, w, gy, out) in enumerate(((q, wq, gq, oq), (k, wk, gk, ok))):
        x, w, gy = x.double(), w.double(), gy.double()
        r = ((x * x).mean(-1, keepdim=True) + 1e-5) ** -0.5 if normed else torch.ones_like(x[..., :1])
        u = x * r
        z = u * w if normed else x
        want = _turn(z, cos, sin, rot, interleaved)
        room = _turn(z.abs(), cos.abs(), -sin.abs(), rot, interleaved).abs() + _turn(z.abs(), cos.abs(), sin.abs(), rot, interleaved).abs()
        err = (out.detach().cpu().double() - want).abs()
        assert bool((err <= 16 * 2.0 ** -24 * room + _half_ulp(want, dtype)).all()), ("out", i, float(err.max()))
        dz = _turn(gy, cos, -sin, rot, interleaved)
        dr = _turn(gy.abs(), cos.abs(), -sin.abs(), rot, interleaved).abs() + _turn(gy.abs(), cos.abs(), sin.abs(), rot, interleaved).abs()
        if normed:
            du = dz * w
            want = r * (du - u * (du * u).mean(-1, keepdim=True))
            room = r * (dr * w.abs() + u.abs() * (dr * w.abs() * u.abs()).mean(-1, keepdim=True))
            gw = (dz * u).sum((0, 1))
            err = (grads[2 + i].cpu().double() - gw).abs()
            assert bool((err <= 2.0 ** -15 * (dr * u.abs()).sum((0, 1)) + _half_ulp(gw, dtype)).all()), ("dw", i)
        else:
            want, room = dz, dr
        err = (grads[i].cpu().double() - want).abs()
        assert bool((err <= 32 * 2.0 ** -24 * room + _half_ulp(want, dtype)).all()), ("dx", i, float(err.max()))


def test_gradient_against_differences():
    """d/de of sum(g . f(x + e d)) in fp32 against the gradients' product with d.  Central differences at e = 2^-6 leave
    e^2 / 6 of the third derivative (below 60 here: |d|, |u|, |w| of order 1 over 4 * 64 values) and rounding 2^-24
    |sum| / e over a sum of 3 * 64 * 3 terms of order 1: 0.003 and 0.003."""
    import coset_amd as ca
    q, k, wq, wk, table, pos, sections = _make(3, 2, 1, 64, 32, 2, torch.float32, 5)
    leaves = [t.cuda() for t in (q, k, wq, wk)]
    g = torch.Generator().manual_seed(2)
    gq, gk = torch.randn(q.shape, generator=g).cuda(), torch.randn(k.shape, generator=g).cuda()

    def f(ts):
        oq, ok = ca.qk_norm_rope(ts[0], ts[1], table.cuda(), pos.cuda(), ts[2], ts[3], sections=sections)
        return float((oq.double() * gq.double()).sum() + (ok.double() * gk.double()).sum())

    live = [t.clone().requires_grad_() for t in leaves]
    oq, ok = ca.qk_norm_rope(live[0], live[1], table.cuda(), pos.cuda(), live[2], live[3], sections=sections)
    grads = torch.autograd.grad([oq, ok], live, [gq, gk])
    e = 2.0 ** -6
    for i in range(4):
        d = torch.randn(leaves[i].shape, generator=g).cuda()
        up, down = list(leaves), list(leaves)
        up[i], down[i] = leaves[i] + e * d, leaves[i] - e * d
        slope = (f(up) - f(down)) / (2 * e)
        assert abs(slope - float((grads[i].double() * d.double()).sum())) <= 0.01 * max(1.0, abs(slope)), i


def test_layouts_and_partial_gradients():
    """Views of one projection, unaligned and spread values, gradients that are broadcast, one weight, one output used,
    positions outside the table, no tokens."""
    import coset_amd as ca
    q, k, wq, wk, table, pos, sections = _make(11, 4, 2, 64, 64, 1, torch.bfloat16, 3)
    table, pos = table.cuda(), pos.cuda()
    want = ca.qk_norm_rope(q.cuda(), k.cuda(), table, pos, wq.cuda(), wk.cuda())
    for off in (0, 8, 1):
        buf = torch.zeros(11, 6 * 64 + 16, dtype=torch.bfloat16)
        buf[:, off:off + 256] = q.flatten(1)
        buf[:, off + 256:off + 384] = k.flatten(1)
        b = buf.cuda()
        got = ca.qk_norm_rope(b[:, off:off + 256].view(11, 4, 64), b[:, off + 256:off + 384].view(11, 2, 64), table, pos[0],
                              wq.cuda(), wk.cuda())
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    spread = torch.zeros(11, 4, 64, 2, dtype=torch.bfloat16, device="cuda")
    spread[..., 0] = q.cuda()
    got = ca.qk_norm_rope(spread[..., 0], k.cuda().transpose(0, 1).contiguous().transpose(0, 1), table, pos, wq.cuda(), wk.cuda())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # the sum's gradient is one value, broadcast; the keys' output is not used
    live = [t.cuda().requires_grad_() for t in (q, k, wq, wk)]
    oq, ok = ca.qk_norm_rope(live[0], live[1], table, pos, live[2], live[3])
    dense = torch.autograd.grad([oq], live, [torch.ones_like(oq)], retain_graph=True)
    oq.sum().backward()
    for t, d in zip(live, dense):
        assert torch.equal(t.grad, d)
    assert float(live[1].grad.abs().max()) == 0 and float(live[3].grad.abs().max()) == 0
    # one weight: the other side's is ones
    a = ca.qk_norm_rope(q.cuda(), k.cuda(), table, pos, wq.cuda(), None)
    b = ca.qk_norm_rope(q.cuda(), k.cuda(), table, pos, wq.cuda(), torch.ones(64, dtype=torch.bfloat16, device="cuda"))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    w = wq.cuda().requires_grad_()
    oq, _ = ca.qk_norm_rope(q.cuda(), k.cuda(), table, pos, w)
    (gw,) = torch.autograd.grad([oq], [w], [torch.ones_like(oq)])
    assert torch.equal(gw, dense[2])
    # positions are clamped
    far = pos.clone()
    far[0, 0], far[0, 1] = 1 << 40, -3
    near = pos.clone()
    near[0, 0], near[0, 1] = table.shape[0] - 1, 0
    assert torch.equal(ca.qk_norm_rope(q.cuda(), k.cuda(), table, far)[0], ca.qk_norm_rope(q.cuda(), k.cuda(), table, near)[0])
    live = [t[:0].cuda().requires_grad_() for t in (q, k)] + [wq.cuda().requires_grad_(), wk.cuda().requires_grad_()]
    oq, ok = ca.qk_norm_rope(live[0], live[1], table, pos[:, :0], live[2], live[3])
    grads = torch.autograd.grad([oq, ok], live, [oq, ok])
    assert oq.shape == (0, 4, 64) and float(grads[2].abs().max()) == 0 and float(grads[3].abs().max()) == 0


def test_special_values():
    """A zero vector has a finite norm; a NaN or an infinity stays in its own head."""
    import coset_amd as ca
    q, k, wq, wk, table, pos, _ = _make(4, 2, 2, 64, 64, 1, torch.float32, 4)
    q[0, 0] = 0
    want = ca.qk_norm_rope(q.cuda(), k.cuda(), table.cuda(), pos.cuda(), wq.cuda(), wk.cuda())
    assert float(want[0][0, 0].abs().max()) == 0 and torch.isfinite(want[0]).all()
    q[1, 1, 5], k[2, 0, 7] = float("nan"), float("inf")
    got = ca.qk_norm_rope(q.cuda(), k.cuda(), table.cuda(), pos.cuda(), wq.cuda(), wk.cuda())
    assert torch.isnan(got[0][1, 1]).all() and torch.isnan(got[1][2, 0]).any()
    q_rest = torch.ones(4, 2, dtype=torch.bool)
    q_rest[1, 1] = False
    k_rest = torch.ones(4, 2, dtype=torch.bool)
    k_rest[2, 0] = False
    assert torch.equal(got[0][q_rest.cuda()], want[0][q_rest.cuda()]) and torch.equal(got[1][k_rest.cuda()], want[1][k_rest.cuda()])


def test_refusals():
    import coset_amd as ca
    q, k, wq, wk, table, pos, _ = (t.cuda() if isinstance(t, torch.Tensor) else t for t in _make(4, 2, 2, 64, 32, 1, torch.float32, 4))

    def no(q=q, k=k, table=table, pos=pos, wq=wq, wk=wk, **more):
        with pytest.raises(ValueError):
            ca.qk_norm_rope(q, k, table, pos, wq, wk, **more)

    no(q=q[0])
    no(q=q[:2])
    no(k=k[..., :32])
    no(k=k.half())
    no(q=q.double(), k=k.double())
    no(table=table.half())
    no(table=table[:, :20].contiguous())
    no(table=torch.zeros(8, 128, device="cuda"))
    no(table=table.cpu())
    no(pos=pos.int())
    no(pos=pos[:, :2])
    no(pos=pos.repeat(2, 1))
    no(pos=pos.repeat(2, 1), sections=[8])
    no(pos=pos.repeat(2, 1), sections=[8, 9])
    no(pos=pos.repeat(5, 1), sections=[4, 4, 4, 2, 2])
    no(wq=wq[:32])
    no(wq=wq.half())
    no(wq=wq.cpu())
    no(norm=False)
    for bad in (0, 4, 12):
        with pytest.raises(ValueError):
            ca.rope_table(16, bad)
