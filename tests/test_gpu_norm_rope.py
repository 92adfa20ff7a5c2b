"""qk_norm_rope against its formula in float64, gradients against autograd of the
formula in float64 and against differences.

Bounds.  An output is rounded once: half a step of its type, eps / 2 relative.
Before that it carries fp32 arithmetic: the statistic (a sum of at most 128 squares,
rsqrt: below 16 steps of 2^-24 relative), three products and a sum of two; 32 *
2^-24 of the row's largest |y| covers it.  dx is rs (h - n mean(h n)): each of its
terms is bounded by rs max|h| (1 + max|n|^2 ...); the test takes 64 * 2^-24 of the
largest |dx| + rs max|h| of the row.  A weight gradient adds `rows` fp32 terms in a
tree of partial sums: its error is below 2^-24 * sqrt-free bound (rows per partial +
log) * sum |g n|; 256 * 2^-24 * sum |g n| holds for the row counts here (a lane adds
at most 128 rows).
"""
from __future__ import annotations

import pytest
import torch

import mtlflashattn_amd as mfa

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def formula(x, w, cos, sin, pos, eps, interleaved):
    """float64, differentiable; x [..., H, D], pos of the leading dims."""
    rot = 2 * cos.shape[1]
    n = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    y = n if w is None else n * w
    c, s = cos[pos].unsqueeze(-2), sin[pos].unsqueeze(-2)
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if interleaved else (y[..., :rot // 2], y[..., rot // 2:rot])
    u, v = a * c - b * s, b * c + a * s
    turned = torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)
    return torch.cat((turned, y[..., rot:]), -1)


def inputs(lead, Hq, Hkv, D, rot, dtype, wdtype=None, tdtype=torch.float32, top=50, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k = (torch.randn(*lead, h, D, generator=g).to(DEV, dtype) for h in (Hq, Hkv))
    qw, kw = ((1 + 0.3 * torch.randn(D, generator=g)).to(DEV, wdtype or dtype) for _ in range(2))
    ang = torch.rand(top, rot // 2, generator=g, dtype=torch.float64) * 6.28
    cos, sin = ang.cos().to(DEV, tdtype), ang.sin().to(DEV, tdtype)
    pos = torch.randint(0, top, lead, generator=g, dtype=torch.int32).to(DEV)
    return q, k, qw, kw, cos, sin, pos


def check_rows(got, ref, ulps=32):
    tol = torch.finfo(got.dtype).eps / 2 * ref.abs() + ulps * U * ref.abs().amax(-1, keepdim=True) + 1e-30
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25  # half a step of its subnormals
    err = (got.double().cpu() - ref).abs()
    assert bool((err <= tol).all()), f"max err / bound {float((err / tol).max()):.3f}"


def d64(*ts):
    return [None if t is None else t.detach().double().cpu() for t in ts]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot", [(128, 128), (128, 64), (64, 64), (64, 16), (96, 48), (80, 80), (32, 32), (8, 8),
                                   (40, 0), (36, 36), (36, 18), (80, 38), (127, 126), (1, 0), (2, 2), (5, 4), (128, 2)])
def test_forward(D, rot, interleaved, dtype):
    q, k, qw, kw, cos, sin, pos = inputs((2, 9), 5, 3, D, rot, dtype, seed=D + rot)
    oq, ok = mfa.qk_norm_rope(q, k, qw, kw, cos, sin, pos, interleaved=interleaved)
    assert oq.dtype == dtype and oq.is_contiguous() and ok.is_contiguous()
    q64, k64, qw64, kw64, c64, s64 = d64(q, k, qw, kw, cos, sin)
    check_rows(oq, formula(q64, qw64, c64, s64, pos.cpu().long(), 1e-6, interleaved))
    check_rows(ok, formula(k64, kw64, c64, s64, pos.cpu().long(), 1e-6, interleaved))


def reference_grads(q, k, qw, kw, cos, sin, pos, interleaved, gq, gk, eps=1e-6):
    """float64 gradients of (q, k, qw, kw), and sum |g n| per weight."""
    c64, s64 = d64(cos, sin)
    grads, mags = [], []
    for x, w, g in ((q, qw, gq), (k, kw, gk)):
        x64, w64, g64 = d64(x, w, g)
        x64.requires_grad_()
        if w64 is None:
            w64 = torch.ones(x64.shape[-1], dtype=torch.float64)
        w64.requires_grad_()
        y = formula(x64, w64, c64, s64, pos.cpu().long(), eps, interleaved)
        grads.append(torch.autograd.grad(y, (x64, w64), g64))
        # |g n| bounded by |g| |n| over the pair
        n = (x64 / torch.sqrt(x64.square().mean(-1, keepdim=True) + eps)).detach().abs()
        gm = g64.abs()
        rot = 2 * c64.shape[1]
        full = gm.clone()
        if rot:
            a, b = (gm[..., 0:rot:2], gm[..., 1:rot:2]) if interleaved else (gm[..., :rot // 2], gm[..., rot // 2:rot])
            t = a + b
            full[..., :rot] = torch.stack((t, t), -1).flatten(-2) if interleaved else torch.cat((t, t), -1)
        mags.append((full * n).flatten(0, -2).sum(0))
    return grads, mags


def check_grads(got, q, k, qw, kw, cos, sin, pos, interleaved, gq, gk):
    grads, mags = reference_grads(q, k, qw, kw, cos, sin, pos, interleaved, gq, gk)
    for i, x in enumerate((q, k)):
        ref, g = grads[i][0], got[i]
        rs = 1 / torch.sqrt(x.detach().double().cpu().square().mean(-1, keepdim=True) + 1e-6)
        up = (gq, gk)[i].double().cpu().abs().amax(-1, keepdim=True) * 2
        w = (qw, kw)[i]
        up = up * (1.0 if w is None else float(w.detach().abs().max()))
        n2 = (x.detach().double().cpu() * rs).abs().amax(-1, keepdim=True) ** 2 + 1
        tol = torch.finfo(g.dtype).eps / 2 * ref.abs() + 64 * U * rs * up * n2 + (2.0 ** -25 if g.dtype == torch.float16 else 0)
        err = (g.double().cpu() - ref).abs()
        assert bool((err <= tol).all()), f"d{'qk'[i]}: {float((err / tol).max()):.3f} of the bound"
        if w is not None and got[2 + i] is not None:
            gw, refw = got[2 + i], grads[i][1]
            tol = torch.finfo(gw.dtype).eps / 2 * refw.abs() + 256 * U * mags[i] + 1e-30
            err = (gw.double().cpu() - refw).abs()
            assert bool((err <= tol).all()), f"d{'qk'[i]}w: {float((err / tol).max()):.3f} of the bound"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot", [(128, 128), (64, 32), (96, 96), (32, 16), (36, 18), (80, 38), (40, 0), (7, 6)])
def test_backward(D, rot, interleaved, dtype):
    q, k, qw, kw, cos, sin, pos = inputs((2, 33), 4, 2, D, rot, dtype, seed=D)
    leaves = [t.clone().requires_grad_() for t in (q, k, qw, kw)]
    oq, ok = mfa.qk_norm_rope(*leaves, cos, sin, pos, interleaved=interleaved)
    g = torch.Generator().manual_seed(1)
    gq, gk = (torch.randn(t.shape, generator=g).to(DEV, dtype) for t in (q, k))
    got = torch.autograd.grad((oq, ok), leaves, (gq, gk))
    assert all(a.dtype == b.dtype and a.shape == b.shape for a, b in zip(got, leaves))
    check_grads(got, *leaves, cos, sin, pos, interleaved, gq, gk)


@pytest.mark.parametrize("rows", [1, 2, 31, 1000, 4097])
def test_weight_gradients_over_many_rows(rows):
    q, k, qw, kw, cos, sin, pos = inputs((rows,), 6, 1, 64, 64, torch.float32, seed=rows)
    leaves = [t.clone().requires_grad_() for t in (q, k, qw, kw)]
    g = torch.Generator().manual_seed(1)
    gq, gk = (torch.randn(t.shape, generator=g).to(DEV) for t in (q, k))
    got = []
    for _ in range(3):
        oq, ok = mfa.qk_norm_rope(*leaves, cos, sin, pos)
        got.append(torch.autograd.grad((oq, ok), leaves, (gq, gk)))
    check_grads(got[0], *leaves, cos, sin, pos, False, gq, gk)
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))


def test_gradients_against_differences():
    q, k, qw, kw, cos, sin, pos = inputs((3,), 2, 1, 16, 8, torch.float32, seed=5)
    leaves = [t.clone().requires_grad_() for t in (q, k, qw, kw)]
    u = [torch.randn_like(t) for t in (q, k)]
    f = lambda *xs: sum((o * w).double().sum() for o, w in zip(mfa.qk_norm_rope(*xs, cos, sin, pos), u))  # noqa: E731
    got = torch.autograd.grad(f(*leaves), leaves)
    h = 2.0 ** -8
    for i, x in enumerate(leaves):
        d = torch.randn_like(x)
        with torch.no_grad():
            hi = [t.detach() + h * d if j == i else t.detach() for j, t in enumerate(leaves)]
            lo = [t.detach() - h * d if j == i else t.detach() for j, t in enumerate(leaves)]
            num = float((f(*hi) - f(*lo)) / (2 * h))
        # third-order term h^2 / 6 * f''' (of order |f|) and fp32 rounding / 2h
        assert abs(num - float((got[i].double() * d.double()).sum())) <= 2e-3 * (1 + abs(num)), i


def test_positions_and_defaults():
    q, k, qw, kw, cos, sin, pos = inputs((2, 9), 5, 3, 64, 64, torch.bfloat16)
    base = mfa.qk_norm_rope(q, k, qw, kw, cos, sin, pos)
    for other in (pos.long(), pos.t().contiguous().t()):
        assert all(torch.equal(a, b) for a, b in zip(base, mfa.qk_norm_rope(q, k, qw, kw, cos, sin, other)))
    counted = mfa.qk_norm_rope(q, k, qw, kw, cos, sin)
    shared = mfa.qk_norm_rope(q, k, qw, kw, cos, sin, torch.arange(9, device=DEV))
    full = mfa.qk_norm_rope(q, k, qw, kw, cos, sin, torch.arange(9, device=DEV).expand(2, 9).contiguous())
    spread = mfa.qk_norm_rope(q, k, qw, kw, cos, sin, torch.arange(9, device=DEV).expand(2, 9))
    for other in (shared, full, spread):
        assert all(torch.equal(a, b) for a, b in zip(counted, other))
    ones = torch.ones(64, device=DEV, dtype=torch.bfloat16)
    assert all(torch.equal(a, b) for a, b in zip(mfa.qk_norm_rope(q, k, None, None, cos, sin, pos),
                                                 mfa.qk_norm_rope(q, k, ones, ones, cos, sin, pos)))
    one = mfa.qk_norm_rope(q, k, None, kw, cos, sin, pos)
    assert torch.equal(one[1], base[1])


@pytest.mark.parametrize("tdtype", [torch.float32, torch.bfloat16])
def test_types_of_weights_and_tables(tdtype):
    q, k, qw, kw, cos, sin, pos = inputs((9,), 5, 3, 64, 32, torch.bfloat16, wdtype=torch.float32, tdtype=tdtype)
    oq, ok = mfa.qk_norm_rope(q, k, qw, kw, cos, sin, pos)
    check_rows(oq, formula(*d64(q, qw, cos, sin), pos.cpu().long(), 1e-6, False))
    leaves = [t.clone().requires_grad_() for t in (q, k, qw, kw)]
    outs = mfa.qk_norm_rope(*leaves, cos, sin, pos)
    got = torch.autograd.grad(outs, leaves, [torch.ones_like(o) for o in outs])
    assert got[2].dtype == torch.float32
    check_grads(got, *leaves, cos, sin, pos, False, *[torch.ones_like(o) for o in outs])


@pytest.mark.parametrize("bad", [-1, 50, 1 << 30, -(1 << 31)])
def test_positions_outside_the_tables(bad):
    q, k, qw, kw, cos, sin, pos = inputs((9,), 5, 3, 64, 32, torch.bfloat16)
    ref = mfa.qk_norm_rope(q, k, qw, kw, cos, sin, pos)
    pos[4] = bad
    out = mfa.qk_norm_rope(q, k, qw, kw, cos, sin, pos)
    for a, b in zip(out, ref):
        assert a[4, :, :32].isnan().all() and torch.equal(a[4, :, 32:], b[4, :, 32:])
        keep = [i for i in range(9) if i != 4]
        assert torch.equal(a[keep], b[keep])
    empty = mfa.qk_norm_rope(q, k, qw, kw, cos[:0], sin[:0], pos)
    assert empty[0][..., :32].isnan().all() and torch.equal(empty[0][..., 32:], out[0][..., 32:])


def test_views_and_odd_alignment():
    Hq, Hkv, D = 6, 2, 64
    q, k, qw, kw, cos, sin, pos = inputs((2, 9), Hq, Hkv, D, D, torch.bfloat16)
    ref = mfa.qk_norm_rope(q, k, qw, kw, cos, sin, pos)
    same = lambda out: all(torch.equal(a, b) for a, b in zip(out, ref))  # noqa: E731
    packed = torch.randn(2, 9, Hq + 2 * Hkv, D, device=DEV, dtype=torch.bfloat16)
    packed[:, :, :Hq], packed[:, :, Hq:Hq + Hkv] = q, k
    assert same(mfa.qk_norm_rope(packed[:, :, :Hq], packed[:, :, Hq:Hq + Hkv], qw, kw, cos, sin, pos))
    swapped = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k)]
    assert same(mfa.qk_norm_rope(*swapped, qw, kw, cos, sin, pos))
    odd = []
    for t in (q, k):
        x = torch.empty(t.numel() + 1, device=DEV, dtype=t.dtype)[1:].view(t.shape)
        odd.append(x.copy_(t))
    for a, b in zip(mfa.qk_norm_rope(*odd, qw, kw, cos, sin, pos), ref):  # (single elements: sums in another order)
        assert bool(((a.float() - b.float()).abs() <= 2.0 ** -7 * b.float().abs()).all())
    wide = torch.empty(2, 9, Hq, 2 * D, device=DEV, dtype=torch.bfloat16)
    wide[..., ::2] = q
    assert same(mfa.qk_norm_rope(wide[..., ::2], k, qw, kw, cos, sin, pos))
    big = torch.stack((cos, cos + 1), 1).flatten(1)  # rows of a wider table
    assert same(mfa.qk_norm_rope(q, k, qw, kw, big[:, :D // 2], sin, pos))


def test_expanded_and_missing_gradients():
    q, k, qw, kw, cos, sin, pos = inputs((2, 5), 4, 2, 64, 64, torch.float32)
    leaves = [t.clone().requires_grad_() for t in (q, k, qw, kw)]
    oq, ok = mfa.qk_norm_rope(*leaves, cos, sin, pos)
    got = torch.autograd.grad(oq.sum(), leaves, allow_unused=True)
    check_grads(got, *leaves, cos, sin, pos, False, torch.ones_like(oq), torch.zeros_like(ok))
    # only the weight of k
    w = kw.clone().requires_grad_()
    oq, ok = mfa.qk_norm_rope(q, k, qw, w, cos, sin, pos)
    got = torch.autograd.grad((ok * 2).sum(), w)
    grads, mags = reference_grads(q, k, qw, kw, cos, sin, pos, False, torch.ones_like(oq), torch.full_like(ok, 2.0))
    assert bool(((got[0].double().cpu() - grads[1][1]).abs() <= U * grads[1][1].abs() + 256 * U * mags[1]).all())


def test_no_tokens():
    q, k, qw, kw, cos, sin, pos = inputs((0,), 4, 2, 64, 64, torch.bfloat16)
    leaves = [t.clone().requires_grad_() for t in (q, k, qw, kw)]
    oq, ok = mfa.qk_norm_rope(*leaves, cos, sin, pos)
    assert oq.shape == (0, 4, 64) and ok.shape == (0, 2, 64)
    got = torch.autograd.grad((oq, ok), leaves, (torch.zeros_like(oq), torch.zeros_like(ok)))
    assert not got[2].any() and not got[3].any()


def test_rows_of_zeros_and_large_values():
    q, k, qw, kw, cos, sin, pos = inputs((4,), 2, 2, 64, 64, torch.float32)
    q[0] = 0
    q[1] *= 1e15
    q[2] *= 1e-15
    oq, _ = mfa.qk_norm_rope(q, k, qw, kw, cos, sin, pos)
    check_rows(oq, formula(*d64(q, qw, cos, sin), pos.cpu().long(), 1e-6, False))
    q[3, 0, 5] = float("nan")
    out, _ = mfa.qk_norm_rope(q, k, qw, kw, cos, sin, pos)
    assert out[3, 0].isnan().all() and torch.equal(out[3, 1], oq[3, 1])


def test_captured_forward_and_backward():
    q, k, qw, kw, cos, sin, pos = inputs((2, 40), 4, 2, 64, 64, torch.bfloat16)
    leaves = [t.clone().requires_grad_() for t in (q, k, qw, kw)]
    ups = [torch.randn_like(q), torch.randn_like(k)]

    def step():
        outs = mfa.qk_norm_rope(*leaves, cos, sin, pos)
        return (*(o.detach() for o in outs), *torch.autograd.grad(outs, leaves, ups))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        with torch.no_grad():
            for t in leaves:
                t.normal_()
            pos.copy_((pos + 7) % 50)
            ups[0].normal_()
        graph.replay()
        torch.cuda.synchronize()
        ref = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, ref)), i


@pytest.mark.parametrize("D,rot", [(64, 64), (64, 16), (36, 18)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_tables_without_rows(D, rot, interleaved):
    """Every position is outside: the rotated elements are NaN, the others normalised."""
    q, k, qw, kw, cos, sin, pos = inputs((5,), 2, 1, D, rot, torch.float32)
    ref = mfa.qk_norm_rope(q, k, qw, kw, cos, sin, pos, interleaved=interleaved)
    got = mfa.qk_norm_rope(q, k, qw, kw, cos[:0], sin[:0], pos, interleaved=interleaved)
    for a, b in zip(got, ref):
        assert a[..., :rot].isnan().all() and torch.equal(a[..., rot:], b[..., rot:])


def test_heads_of_one_side_only_and_gradients_of_weights_only():
    q, k, qw, kw, cos, sin, pos = inputs((3, 50), 4, 2, 64, 64, torch.bfloat16)
    ref = mfa.qk_norm_rope(q, k, qw, kw, cos, sin, pos)
    no_k = mfa.qk_norm_rope(q, k[:, :, :0], qw, kw, cos, sin, pos)
    no_q = mfa.qk_norm_rope(q[:, :, :0], k, qw, kw, cos, sin, pos)
    assert torch.equal(no_k[0], ref[0]) and torch.equal(no_q[1], ref[1])
    assert no_k[1].shape == (3, 50, 0, 64) and no_q[0].shape == (3, 50, 0, 64)
    leaves = [t.clone().requires_grad_() for t in (q, k, qw, kw)]
    ups = [torch.randn_like(q), torch.randn_like(k)]
    full = torch.autograd.grad(mfa.qk_norm_rope(*leaves, cos, sin, pos), leaves, ups)
    some = torch.autograd.grad(mfa.qk_norm_rope(q, k, *leaves[2:], cos, sin, pos), leaves[2:], ups)
    assert all(torch.equal(a, b) for a, b in zip(some, full[2:]))
    some = torch.autograd.grad(mfa.qk_norm_rope(leaves[0], k, qw, kw, cos, sin, pos), leaves[:1], ups)
    assert torch.equal(some[0], full[0])
    one = mfa.qk_norm_rope(q, k[:, :, :0], leaves[2], leaves[3], cos, sin, pos)
    gw = torch.autograd.grad(one, leaves[2:], (ups[0], ups[1][:, :, :0]))
    assert torch.equal(gw[0], full[2]) and not gw[1].any()


def test_inputs_expanded_over_the_batch():
    """One sequence for three batches (batch stride 0): gradients are summed over them."""
    q, k, qw, kw, cos, sin, pos = inputs((1, 40), 4, 2, 64, 64, torch.float32)
    q0, k0 = q.clone().requires_grad_(), k.clone().requires_grad_()
    q3, k3 = q0.expand(3, -1, -1, -1), k0.expand(3, -1, -1, -1)
    p3 = torch.stack([pos[0], pos[0].flip(0), pos[0] // 2])
    outs = mfa.qk_norm_rope(q3, k3, qw, kw, cos, sin, p3)
    ups = [torch.randn_like(o) for o in outs]
    got = torch.autograd.grad(outs, (q0, k0), ups)
    qc, kc = (t.detach().repeat(3, 1, 1, 1).requires_grad_() for t in (q, k))
    ref = torch.autograd.grad(mfa.qk_norm_rope(qc, kc, qw, kw, cos, sin, p3), (qc, kc), ups)
    for a, b in zip(got, ref):
        assert torch.equal(a, b.sum(0, keepdim=True))


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradients_through_norm_rotation_and_attention(interleaved):
    """A training step's way from a packed projection: views, norm and rotation,
    causal grouped-query attention; gradients against float64 autograd on the CPU.

    fp32: the attention's gradients are within 2e-6 of their largest value, the
    norm's backward scales them and the reference by the same factors and adds 64 U,
    and its difference h - n mean(h n) at most doubles what is relative to h: below
    1e-5 of the largest value by a factor that leaves room for one row's.
    """
    B, L, Hq, Hkv, D = 2, 70, 4, 2, 64
    g = torch.Generator().manual_seed(3)
    packed = torch.randn(B, L, (Hq + 2 * Hkv) * D, generator=g).to(DEV).requires_grad_()
    _, _, qw, kw, cos, sin, _ = inputs((1,), 1, 1, D, D, torch.float32, top=L)
    qw, kw = qw.requires_grad_(), kw.requires_grad_()
    up = torch.randn(B, L, Hq, D, generator=g)

    def split(x):
        return [t.unflatten(-1, (-1, D)) for t in x.split([Hq * D, Hkv * D, Hkv * D], -1)]

    q, k, v = split(packed)
    q, k = mfa.qk_norm_rope(q, k, qw, kw, cos, sin, interleaved=interleaved)
    got = torch.autograd.grad(mfa.flash_attn_func(q, k, v, causal=True), (packed, qw, kw), up.to(DEV))

    leaves = [t.detach().cpu().double().requires_grad_() for t in (packed, qw, kw)]
    c, s, pos = cos.cpu().double(), sin.cpu().double(), torch.arange(L).expand(B, L)
    q, k, v = split(leaves[0])
    q, k = (formula(x, w, c, s, pos, 1e-6, interleaved) for x, w in ((q, leaves[1]), (k, leaves[2])))
    k, v = (x.repeat_interleave(Hq // Hkv, 2) for x in (k, v))
    w = torch.matmul(q.transpose(1, 2), k.permute(0, 2, 3, 1)) / D ** 0.5
    w = torch.softmax(w.masked_fill(~torch.ones(L, L, dtype=torch.bool).tril(), float("-inf")), -1)
    ref = torch.autograd.grad(torch.matmul(w, v.transpose(1, 2)).transpose(1, 2), leaves, up.double())
    for a, b in zip(got, ref):
        assert float((a.cpu().double() - b).abs().max()) <= 1e-5 * float(b.abs().max())
