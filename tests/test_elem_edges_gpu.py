"""embedding_scaled and group_norm_act at edges that ordinary values and sizes do not show."""
import pytest
import torch

import _elem_ref as R

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ['f32', 'bf16', 'f16']


def _randn(*shape, seed, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _norm_all(device, x, G, w, b, dy, act):
    """y, dx, dweight, dbias on the CPU."""
    from ag2video_amd import ops
    leaves = [t.to(device).requires_grad_(True) for t in (x, w, b)]
    y = ops.group_norm_act(leaves[0], G, *leaves[1:], act=act)
    return [t.detach().cpu() for t in (y,) + torch.autograd.grad(y, leaves, dy.to(device))]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("S", [20, 300, 6000])
@pytest.mark.parametrize("Cg", [1, 2, 3, 4, 5, 7, 8])
def test_parameters_that_are_not_finite_stay_in_their_group(Cg, S, dtype, device):
    """An infinite or NaN weight or bias of one channel reaches that channel's y and parameters' gradients and its group's dx; every other
    group keeps its bits.  Groups of fewer channels than a vector has elements, one a workgroup and several, and in parts."""
    G = 3
    C = G * Cg
    x, dy = _randn(2, S, C, seed=1, dtype=dtype), _randn(2, S, C, seed=2, dtype=dtype)
    w, b = 1 + 0.2 * _randn(C, seed=3), _randn(C, seed=4)
    c = Cg + Cg // 2                                          # a channel of the middle group
    for act in ('none', 'silu', 'lrelu'):
        want = _norm_all(device, x, G, w, b, dy, act)
        for which, value in ((0, float('inf')), (0, float('nan')), (1, float('-inf')), (1, float('nan'))):
            p = [w.clone(), b.clone()]
            p[which][c] = value
            got = _norm_all(device, x, G, *p, dy, act)
            others = torch.ones(C, dtype=torch.bool)
            others[Cg:2 * Cg] = False
            for name, q, r in zip(('y', 'dx', 'dweight', 'dbias'), got, want):
                assert torch.equal(q[..., others], r[..., others]), (name, act, which, value)
            own = torch.ones(C, dtype=torch.bool)             # y and the parameters' gradients: all but the channel itself
            own[c] = False
            for name, q, r in zip(('y', 'dweight', 'dbias'), (got[0], got[2], got[3]), (want[0], want[2], want[3])):
                assert torch.equal(q[..., own], r[..., own]), (name, act, which, value)


# Maps on which a group's mean is exact: sums of numbers of few bits, counts that are powers of two, values on both sides of the mean in pairs.  One
# launch and parts.
EXACT = [((2, 64, 16), 4), ((2, 64, 6), 3), ((2, 512, 8), 8), ((1, 16384, 16), 2), ((2, 8192, 64), 4)]


@pytest.mark.parametrize("shape,G", EXACT, ids=str)
def test_constant_groups_far_from_zero(shape, G, device):
    """x = mean exactly: h = 0, y = act(b), dweight = 0."""
    C = shape[-1]
    for value in (3.25, 1000.125, -31007.5):
        x = torch.full(shape, value)
        w, b, dy = 1 + 0.2 * _randn(C, seed=1), _randn(C, seed=2), _randn(*shape, seed=3)
        y, dx, dw, db = _norm_all(device, x, G, w, b, dy, 'silu')
        # fma(0, w, b) = b; the sigmoid from exp and a reciprocal: (4 + |z|) u relative, and the product
        want = b.double() * torch.sigmoid(b.double())
        assert ((y.double() - want).abs() <= (5 + b.double().abs()) * R.U * want.abs()).all()
        assert not dw.any()


@pytest.mark.parametrize("act", ['none', 'silu'])
@pytest.mark.parametrize("shape,G", EXACT, ids=str)
def test_gradients_far_from_zero(shape, G, act, device):
    """Values around 1000 whose mean is exact: the backward pass has h to a few roundings of h itself, not of |mean| / std.

    x - mean is exact, so h carries the relative error of 1 / std (the variance: at most DEPTH additions of positive terms; four more for the division, the
    root and the reciprocal) and of one product: e_h = |h| (DEPTH / 2 + 5) u.  In parts the statistics are joined in fp64, which adds less.  What
    follows from e_h is as in _elem_ref.group_norm."""
    N, S, C = shape
    Cg = C // G
    off = _randn(N, S, C, seed=1).mul(8).round().clamp(-40, 40) / 16
    if Cg == 1:                                               # symmetric: the mean of a group is 1000, exactly
        off[:, S // 2:] = -off[:, :S // 2]
    else:
        off[..., 1::2] = -off[..., ::2]
    x = 1000 + off
    w, b, dy = 1 + 0.2 * _randn(C, seed=3), _randn(C, seed=4), 1 + 0.1 * _randn(*shape, seed=5)
    y, dx, dw, db = _norm_all(device, x, G, w, b, dy, act)
    v = x.double().view(N, S, G, Cg)
    d = v - 1000.0
    rstd = ((d * d).mean((1, 3), keepdim=True) + 1e-5) ** -0.5
    r_rstd = (R.DEPTH / 2 + 4) * R.U
    h, e_h = d * rstd, (d * rstd).abs() * (r_rstd + R.U)
    wd, bd, g = w.double().view(1, 1, G, Cg), b.double().view(1, 1, G, Cg), dy.double().view(v.shape)
    z = h * wd + bd
    e_z = wd.abs() * e_h + 3 * R.U * ((wd * h).abs() + bd.abs())
    if act == 'silu':
        s = torch.sigmoid(z)
        dz, e_dz = g * s * (1 + z * (1 - s)), g.abs() * (0.5 * e_z + (8 + 2 * z.abs()) * R.U * (1 + z.abs()))
    else:
        dz, e_dz = g, torch.zeros_like(g)
    du = R.DEPTH * R.U
    total, err = (dz * h).sum((0, 1)).view(-1), (e_dz * h.abs() + dz.abs() * e_h + (2 * du + R.U) * (dz * h).abs()).sum((0, 1)).view(-1)
    R.check('dweight', dw, total, err + R.U * (total.abs() + err))
    t, e_t = wd * dz, wd.abs() * e_dz + R.U * (wd * dz).abs()
    dims = (1, 3)
    s1, s2 = t.mean(dims, keepdim=True), (t * h).mean(dims, keepdim=True)
    e_s1 = e_t.mean(dims, keepdim=True) + (du + 2 * R.U) * t.abs().mean(dims, keepdim=True)
    e_s2 = (e_t * h.abs() + t.abs() * e_h + R.U * (t * h).abs()).mean(dims, keepdim=True) + (du + 2 * R.U) * (t * h).abs().mean(dims, keepdim=True)
    ref = rstd * (t - s1 - h * s2)
    bound = rstd * (e_t + e_s1 + h.abs() * e_s2 + s2.abs() * e_h + 4 * R.U * (t.abs() + s1.abs() + (h * s2).abs())) + ref.abs() * (r_rstd + 2 * R.U)
    R.check('dx', dx.view(v.shape), ref, bound + R.U * (ref.abs() + bound))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize("shape,G", [((131, 64, 1024), 32), ((70, 64, 2048), 64), ((8199, 16, 16), 1), ((9001, 40, 16), 16), ((8201, 20, 12), 4), ((60, 200, 600), 200),
                                     ((2100, 10, 90), 6), ((3001, 9, 72), 9)], ids=str)
def test_batches_of_more_samples_than_workgroups(shape, G, dtype, device):
    """The one-launch backward pass walks several samples a workgroup where a batch has more of them than 2048 workgroups: several rounds, the last one
    not full, of one sample a workgroup and of four, of groups of whole vectors and of others."""
    from ag2video_amd import ops
    C = shape[-1]
    x, dy = _randn(*shape, seed=1, dtype=dtype), _randn(*shape, seed=2, dtype=dtype)
    w, b = 1 + 0.2 * _randn(C, seed=3), _randn(C, seed=4)
    ref = R.group_norm(x, G, w, b, 1e-5, 'silu', 0.2, dy)
    for name, got in zip(('y', 'dx', 'dweight', 'dbias'), _norm_all(device, x, G, w, b, dy, 'silu')):
        R.check(name, got, *ref[name])
    leaf = x.to(device).requires_grad_(True)
    (dx,) = torch.autograd.grad(ops.group_norm_act(leaf, G, w.to(device), b.to(device)), leaf, dy.to(device))
    for n in (0, shape[0] // 2, shape[0] - 1):
        one = x[n:n + 1].to(device).requires_grad_(True)
        (d1,) = torch.autograd.grad(ops.group_norm_act(one, G, w.to(device), b.to(device)), one, dy[n:n + 1].to(device))
        assert torch.equal(d1[0], dx[n])


@pytest.mark.parametrize("view", [lambda t: t, lambda t: t[..., 3:]], ids=['whole', 'slice'])
def test_group_norm_backward_past_32_bit_offsets(view, device):
    """x, dy and dx of more than 2^31 elements, all different: each sample as it is alone."""
    from ag2video_amd import ops
    N, S, C = 3, 1 << 20, 720
    x, dy = (torch.empty(N, S, C, device=device, dtype=torch.bfloat16) for _ in range(2))
    for n in range(N):
        x[n].normal_(generator=torch.Generator(device=device).manual_seed(n))
        dy[n].normal_(generator=torch.Generator(device=device).manual_seed(10 + n))
    x, dy = view(x), view(dy)
    C = x.shape[-1]
    G = 3
    w = [_randn(C, seed=1).to(device).requires_grad_(True), _randn(C, seed=2).to(device).requires_grad_(True)]
    leaf = x.detach().requires_grad_(True)
    dx, dw, db = torch.autograd.grad(ops.group_norm_act(leaf, G, *w), [leaf] + w, dy)
    sums, mags = torch.zeros(2, C, device=device, dtype=torch.float64), torch.zeros(2, C, device=device, dtype=torch.float64)
    for n in range(N):
        one = x.detach()[n:n + 1].clone().requires_grad_(True)
        d1, *p1 = torch.autograd.grad(ops.group_norm_act(one, G, *w), [one] + w, dy[n:n + 1].clone())
        assert torch.equal(d1[0], dx[n])
        p1 = torch.stack(p1).double()
        sums += p1
        mags += p1.abs()
    # one rounding of each sample's own, and one of the sum
    assert ((torch.stack((dw, db)).double() - sums).abs() <= R.U * (mags + sums.abs())).all()
    del x, dy, dx, leaf, one, d1
    torch.cuda.empty_cache()


# The ways of the gradient: one launch, tiles, ranks, a radix sort; rows far apart where there are few of them.
@pytest.mark.parametrize("n,V,D,apart", [(2000, 4, 64, 1 << 21), ((1 << 20) - 5, 27, 2100, 2100), (8000, 3000, 33, 1 << 19), ((1 << 25) + 77, 50, 72, 72),
                                         (300000, 3000, 40, 1 << 13)], ids=['one launch', 'tiles', 'ranks', 'radix, few words', 'radix'])
def test_embedding_gradient_rows_past_32_bit_offsets(n, V, D, apart, device):
    """A dense gradient of more than 2^31 elements, zero but for rows on both sides of that offset and the last ones.  Whole numbers."""
    from ag2video_amd import ops
    wide = torch.zeros(n, apart, device=device, dtype=torch.bfloat16)
    idx = (torch.arange(n, device=device) * 7 + 3) % V
    border = (1 << 31) // apart
    rows = torch.tensor(sorted({0, 1, border - 1, border, border + 1, border + n // 100, n - 2, n - 1}), device=device)
    assert border + n // 100 < n
    values = torch.randint(-8, 9, (rows.numel(), D), generator=torch.Generator().manual_seed(1)).to(device)
    wide[rows, :D] = values.bfloat16()
    table = torch.zeros(V, D, device=device, dtype=torch.bfloat16, requires_grad=True)
    (got,) = torch.autograd.grad(ops.embedding_scaled(idx, table, 2.0), table, wide[:, :D])
    want = torch.zeros(V, D, device=device, dtype=torch.float64).index_add_(0, idx[rows], values.double()) * 2
    assert want.any() and torch.equal(got.double(), want)
    del wide
    torch.cuda.empty_cache()


def test_embedding_tokens_past_32_bit_offsets(device):
    """Tokens 2^20 elements apart."""
    from ag2video_amd import ops
    n, V, D = 3000, 500, 12
    far = torch.zeros(n, 1 << 20, device=device, dtype=torch.int32)
    idx = torch.randint(V, (n,), generator=torch.Generator().manual_seed(1)).to(device)
    far[:, 5] = idx.int()
    table, dout = _randn(V, D, seed=2).to(device).requires_grad_(True), _randn(n, D, seed=3).to(device)
    a, b = ops.embedding_scaled(far[:, 5], table), ops.embedding_scaled(idx, table)
    assert torch.equal(a, b)
    assert torch.equal(torch.autograd.grad(a, table, dout)[0], torch.autograd.grad(b, table, dout)[0])
    del far
    torch.cuda.empty_cache()


@pytest.mark.parametrize("shape,G", [((3, 50, 24), 3), ((2, 6000, 36), 4), ((1, 4, 8192), 1)], ids=str)
def test_gradients_of_some_inputs_alone(shape, G, device):
    """x, weight and bias with a gradient or without, and absent: the same bits as all of them together."""
    from ag2video_amd import ops
    C = shape[-1]
    x, dy = _randn(*shape, seed=1).to(device), _randn(*shape, seed=2).to(device)
    w, b = (1 + 0.2 * _randn(C, seed=3)).to(device), _randn(C, seed=4).to(device)
    for have in ((True, True), (True, False), (False, True)):
        tensors = [x] + [t if h else None for t, h in zip((w, b), have)]
        leaves = [None if t is None else t.clone().requires_grad_(True) for t in tensors]
        y = ops.group_norm_act(leaves[0], G, *leaves[1:])
        full = dict(zip([k for k in range(3) if leaves[k] is not None], torch.autograd.grad(y, [t for t in leaves if t is not None], dy)))
        for mask in range(1, 8):
            want = [k for k in range(3) if mask >> k & 1 and tensors[k] is not None]
            if not want:
                continue
            some = [None if t is None else t.clone().requires_grad_(k in want) for k, t in enumerate(tensors)]
            y1 = ops.group_norm_act(some[0], G, *some[1:])
            assert torch.equal(y1, y)
            for k, g in zip(want, torch.autograd.grad(y1, [some[k] for k in want], dy)):
                assert torch.equal(g, full[k]), (have, want, k)
