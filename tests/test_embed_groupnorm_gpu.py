"""embedding_scaled and group_norm_act against 64-bit references with derived bounds (tests/_elem_ref.py)."""
import pytest
import torch

import _elem_ref as R

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ['f32', 'bf16', 'f16']


def _randn(*shape, seed, scale=1.0, shift=0.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype)


def _tokens(n, V, seed, kind='uniform'):
    g = torch.Generator().manual_seed(seed)
    if kind == 'uniform':
        return torch.randint(V, (n,), generator=g)
    if kind == 'one':                                      # every token the same: one long segment
        return torch.full((n,), V // 2)
    if kind == 'skewed':                                   # half of all tokens are one word, the rest follow 1 / rank
        t = (torch.exp(torch.rand(n, generator=g, dtype=torch.float64) * torch.log(torch.tensor(V + 1.0, dtype=torch.float64))) - 1).long().clamp(0, V - 1)
        return torch.where(torch.rand(n, generator=g) < 0.5, torch.full_like(t, V - 1), t)
    if kind == 'sorted':
        return torch.randint(V, (n,), generator=g).sort().values
    return torch.arange(n) % V                             # 'cyclic'


def _embed_case(device, idx, table, scale, pad, dout, name):
    from ag2video_amd import ops
    ref = R.embedding(idx, table, scale, pad, dout)
    t = table.to(device).requires_grad_(True)
    i = idx.to(device)
    out = ops.embedding_scaled(i, t, scale, pad)
    assert out.dtype == table.dtype and out.device == t.device
    R.check(name + '.out', out, ref[0], ref[1])
    (dt,) = torch.autograd.grad(out, t, dout.to(device))
    assert dt.dtype == table.dtype
    R.check(name + '.dtable', dt, ref[2], ref[3])
    with torch.no_grad():                                  # the path without a tape, and a second call: the same bits
        assert torch.equal(ops.embedding_scaled(i, t, scale, pad).nan_to_num(7.0), out.detach().nan_to_num(7.0))
    (again,) = torch.autograd.grad(ops.embedding_scaled(i, t, scale, pad), t, dout.to(device))
    assert torch.equal(dt, again)


EMBED = [
    # n, V, D, tokens
    (1, 1, 1, 'uniform'), (1, 5, 3, 'uniform'), (2, 1, 8, 'uniform'), (7, 3, 7, 'cyclic'), (10, 24, 128, 'uniform'),
    (63, 64, 16, 'cyclic'), (64, 64, 16, 'cyclic'), (65, 1000, 9, 'sorted'), (257, 2, 33, 'uniform'), (1280, 24, 128, 'uniform'),
    (1000, 7, 520, 'one'), (300, 40000, 12, 'uniform'), (4095, 511, 40, 'skewed'), (4096, 512, 24, 'sorted'), (4097, 513, 17, 'skewed'),
    (3, 70001, 2, 'uniform'), (2000, 100, 1027, 'skewed'),
    (8191, 33000, 31, 'skewed'), (8192, 300, 64, 'one'), (8193, 70000, 5, 'uniform'),
    (20000, 1025, 16, 'skewed'), (20001, 3, 48, 'uniform'), (33333, 60, 129, 'sorted'), (70000, 1, 4, 'one'), (66000, 262145, 4, 'uniform'),
    (120000, 5000, 1, 'skewed'),
]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("n,V,D,kind", EMBED, ids=lambda v: str(v))
def test_embedding_scaled(n, V, D, kind, dtype, device):
    idx = _tokens(n, V, n + V, kind)
    _embed_case(device, idx, _randn(V, D, seed=1, dtype=dtype), 0.37, None, _randn(n, D, seed=2, scale=0.1, dtype=dtype), 'embed')


# sizes at which the gradient changes its way: one launch, counted ranks, one radix pass, several, several rounds a workgroup
@pytest.mark.parametrize("n,V,D,kind", [(1024, 4, 300, 'skewed'), (1025, 4, 300, 'skewed'), (2048, 30, 128, 'one'), (2049, 30, 128, 'one'), (2048, 1100, 3, 'cyclic'),
                                        (6144, 511, 20, 'skewed'), (6145, 511, 20, 'skewed'), (6145, 512, 20, 'skewed'), (262144, 40, 8, 'skewed'),
                                        (262145, 700, 4, 'skewed'), (300001, 300000, 2, 'uniform')], ids=str)
def test_embedding_scaled_switching_sizes(n, V, D, kind, device):
    idx = _tokens(n, V, n, kind)
    for dtype in (torch.float32, torch.float16):
        _embed_case(device, idx, _randn(V, D, seed=1, dtype=dtype), 1.0, V // 3, _randn(n, D, seed=2, scale=0.1, dtype=dtype), 'embed')


@pytest.mark.parametrize("V", [255, 256, 257, 511, 512, 513], ids=str)
def test_embedding_scaled_large_tiles(V, device):
    """As many words as a tile of tokens has counters for, and one more; the last tile ends inside, and some tokens take no part."""
    n = 524288 + 77
    idx = _tokens(n, V, V, 'skewed')
    idx[::5] = V
    for dtype in (torch.float32, torch.float16):
        _embed_case(device, idx, _randn(V, 4, seed=1, dtype=dtype), 0.5, 3, _randn(n, 4, seed=2, scale=0.05, dtype=dtype), 'embed')


def test_embedding_scaled_past_the_caches(device):
    """Results and gradients large enough to go past the caches.  Whole numbers: every product and sum is exact."""
    from ag2video_amd import ops
    g = torch.Generator(device=device).manual_seed(0)
    for n, V, D in ((140001, 60000, 133), (80000, 70000, 130)):
        idx = torch.randint(V, (n,), device=device, generator=g)
        table = torch.randint(-50, 50, (V, D), device=device, generator=g).float().requires_grad_(True)
        dout = torch.randint(-50, 50, (n, D), device=device, generator=g).float()
        out = ops.embedding_scaled(idx, table, 2.0)
        assert torch.equal(out, table.detach()[idx] * 2)
        (grad,) = torch.autograd.grad(out, table, dout)
        assert torch.equal(grad, torch.zeros(V, D, device=device, dtype=torch.float64).index_add_(0, idx, dout.double()).float() * 2)


@pytest.mark.parametrize("pad", [None, 0, 11], ids=str)
@pytest.mark.parametrize("shape", [(), (5,), (3, 4), (2, 3, 50), (0,), (4, 0)], ids=str)
def test_embedding_scaled_shapes_and_padding(shape, pad, device):
    n = 1
    for s in shape:
        n *= s
    for itype in (torch.int32, torch.int64):
        idx = _tokens(n, 12, 5).view(shape).to(itype)
        _embed_case(device, idx, _randn(12, 20, seed=1), 4.5, pad, _randn(*shape, 20, seed=2), 'embed')


@pytest.mark.parametrize("n,V", [(40, 30), (3000, 30), (3000, 30000), (40000, 30)], ids=str)
def test_embedding_scaled_foreign_tokens(n, V, device):
    """Tokens outside the table: a row of NaN, no part in any gradient, nothing else disturbed."""
    idx = _tokens(n, V, 3)
    idx[::7] = V
    idx[1::11] = -1
    idx[2::13] = 2 ** 40
    idx[3::17] = -2 ** 62
    _embed_case(device, idx, _randn(V, 24, seed=1), 1.0, 2, _randn(n, 24, seed=2), 'foreign')
    idx = torch.full((n,), V)
    _embed_case(device, idx, _randn(V, 24, seed=1), 1.0, None, _randn(n, 24, seed=2), 'all foreign')


def test_embedding_scaled_strides(device):
    """Token and gradient views, a table inside a wider one and at an odd offset."""
    from ag2video_amd import ops
    base = _tokens(6 * 7 * 3, 9, 1).view(6, 7, 3)
    wide = _randn(9, 40, seed=2)
    for name, pick in (('slice', lambda t: t[:, :, 1]), ('transposed', lambda t: t.permute(2, 0, 1)), ('every other', lambda t: t[::2]),
                       ('expanded', lambda t: t[:1].expand(5, 7, 3)), ('reversed order', lambda t: t.transpose(0, 1))):
        idx = pick(base)
        table = wide[:, 3:24]
        dout = _randn(*idx.shape, 21, seed=3)
        out_ref, b_out, dt_ref, b_dt = R.embedding(idx, table, 1.5, None, dout)
        leaf = wide.to(device).requires_grad_(True)
        out = ops.embedding_scaled(pick(base.to(device)), leaf[:, 3:24], 1.5)
        R.check(name + '.out', out, out_ref, b_out)
        (g,) = torch.autograd.grad(out, leaf, dout.to(device))
        R.check(name + '.dtable', g[:, 3:24], dt_ref, b_dt)
        assert not g[:, :3].any() and not g[:, 24:].any()
    # broadcast gradients (sum().backward()) and gradients whose rows lie apart
    idx, table = base[..., 0].contiguous(), wide.to(device).requires_grad_(True)
    for name, d in (('ones', torch.ones(()).expand(6, 7, 40)), ('one row', _randn(40, seed=4).expand(6, 7, 40)),
                    ('row stride', _randn(6, 7, 50, seed=5)[..., 5:45]), ('transposed', _randn(40, 6, 7, seed=6).permute(1, 2, 0))):
        ref = R.embedding(idx, wide, 2.0, None, d)
        (g,) = torch.autograd.grad(ops.embedding_scaled(idx.to(device), table, 2.0), table, d.to(device))
        R.check(name, g, ref[2], ref[3])
    flat = _randn(9 * 13 + 1, seed=7, dtype=torch.bfloat16).to(device)         # rows at 2-byte offsets
    table = flat[1:].view(9, 13)
    ref = R.embedding(idx, table.cpu(), 1.0, None)
    R.check('offset', ops.embedding_scaled(idx.to(device), table), *ref)


def test_embedding_scaled_special_values(device):
    """Infinities and NaN stay in the rows and columns they are in."""
    V, D, n = 6, 10, 50
    table, dout, idx = _randn(V, D, seed=1), _randn(n, D, seed=2), _tokens(n, V, 3)
    table[2, 3], table[4, 0] = float('inf'), float('nan')
    from ag2video_amd import ops
    out = ops.embedding_scaled(idx.to(device), table.to(device), 2.0).cpu()
    assert torch.equal(out.nan_to_num(5.0, 6.0, 7.0), (table[idx] * 2.0).nan_to_num(5.0, 6.0, 7.0))
    i2, i3 = int((idx == 2).nonzero()[0]), int((idx == 3).nonzero()[0])
    dout[i2, 1], dout[i3, 2] = float('nan'), float('-inf')
    leaf = _randn(V, D, seed=1).to(device).requires_grad_(True)
    (g,) = torch.autograd.grad(ops.embedding_scaled(idx.to(device), leaf, 2.0, 5), leaf, dout.to(device))
    g = g.cpu()
    assert torch.isnan(g[2, 1]) and g[3, 2] == float('-inf') and int((~torch.isfinite(g)).sum()) == 2
    assert not g[5].any()


def test_embedding_scaled_long_offsets(device):
    """Offsets of the output beyond 2^31 elements and 2^32 bytes."""
    from ag2video_amd import ops
    n, D, V = (1 << 25) + 77, 72, 50                       # 2.4e9 elements
    idx = (torch.arange(n, device=device) * 7) % V
    table = _randn(V, D, seed=1, dtype=torch.bfloat16).to(device).requires_grad_(True)
    out = ops.embedding_scaled(idx, table, 2.0)
    for at in (0, 12345, (1 << 31) // D, (1 << 31) // D + 1, n - 1):
        assert torch.equal(out[at], table.detach()[at * 7 % V] * 2.0)
    dout = torch.zeros(1, device=device, dtype=torch.bfloat16).expand(n, D)
    (g,) = torch.autograd.grad(out, table, dout)
    assert not g.any()
    del dout
    # a gradient of ones counts the tokens; counts are sums of halves of 2^-1 exactly while they stay below 2^24 in fp32
    ones = torch.ones(n, 4, device=device).expand(n, 4)
    small = torch.zeros(V, 4, device=device, requires_grad=True)
    (g,) = torch.autograd.grad(ops.embedding_scaled(idx, small, 0.5), small, ones)
    assert torch.equal(g, 0.5 * torch.bincount(idx, minlength=V).float()[:, None].expand(V, 4))


NORM = [
    # shape, groups
    ((1, 1), 1), ((3, 4), 2), ((2, 1, 6), 6), ((1, 5, 7), 7), ((2, 9, 8), 1), ((3, 37, 90), 6), ((2, 16, 64), 4), ((1, 1000, 33), 3),
    ((4, 64, 64), 32), ((1, 63, 512), 32), ((2, 129, 40), 5), ((1, 17, 2050), 1), ((1, 3, 4104), 2), ((2, 2048, 16), 2), ((2, 7, 5, 3, 24), 3),
    ((200, 2, 24), 3), ((3000, 1, 8), 2), ((1, 1500, 6), 1), ((2, 700, 1030), 2), ((1, 1, 9000), 3), ((2, 40 * 40, 96), 32), ((1, 6000, 320), 32),
    ((2, 5000, 3), 3), ((1, 20, 512), 512),
]


def _norm_case(device, shape, groups, dtype, act, affine, ptype, seed=1, eps=1e-5, slope=0.2, shift=1.0):
    from ag2video_amd import ops
    C = shape[-1]
    x = (_randn(*shape, seed=seed) * torch.exp(0.3 * _randn(C, seed=seed + 1)) + shift * _randn(C, seed=seed + 2)).to(dtype)
    w = (1 + 0.3 * _randn(C, seed=seed + 3)).to(ptype) if affine else None
    b = _randn(C, seed=seed + 4, scale=0.3).to(ptype) if affine else None
    dy = _randn(*shape, seed=seed + 5).to(dtype)
    ref = R.group_norm(x, groups, w, b, eps, act, slope, dy)
    leaves = [t.to(device).requires_grad_(True) for t in (x, w, b) if t is not None]
    y = ops.group_norm_act(leaves[0], groups, *(leaves[1:] or (None, None)), eps=eps, act=act, slope=slope)
    assert y.dtype == dtype and y.is_contiguous()
    R.check('y', y, *ref['y'])
    grads = torch.autograd.grad(y, leaves, dy.to(device))
    for name, g, leaf in zip(('dx', 'dweight', 'dbias'), grads, leaves):
        assert g.dtype == leaf.dtype
        R.check(name, g, *ref[name])
    with torch.no_grad():
        y2 = ops.group_norm_act(leaves[0], groups, *(leaves[1:] or (None, None)), eps=eps, act=act, slope=slope)
    assert torch.equal(y2, y.detach())
    again = torch.autograd.grad(ops.group_norm_act(leaves[0], groups, *(leaves[1:] or (None, None)), eps=eps, act=act, slope=slope), leaves, dy.to(device))
    assert all(torch.equal(p, q) for p, q in zip(grads, again))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape,groups", NORM, ids=str)
def test_group_norm_act(shape, groups, dtype, device):
    _norm_case(device, shape, groups, dtype, 'silu', True, torch.float32)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("act", ['none', 'silu', 'lrelu'])
@pytest.mark.parametrize("affine", [False, True], ids=['plain', 'affine'])
def test_group_norm_act_forms(act, affine, dtype, device):
    for shape, groups in (((2, 50, 24), 3), ((2, 3000, 36), 4), ((2, 9, 10), 2)):
        _norm_case(device, shape, groups, dtype, act, affine, dtype, seed=7)
        _norm_case(device, shape, groups, dtype, act, affine, torch.float32, seed=9, eps=0.1, slope=0.0)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("S", [1024, 1025, 2047, 2049, 4096, 4097, 8193], ids=str)
def test_group_norm_act_switching_sizes(S, dtype, device):
    """Positions at which slabs get narrower or parts take over, in groups of whole vectors, of odd widths, and of all channels."""
    for C, G in ((64, 8), (44, 4), (15, 5), (24, 1)):
        _norm_case(device, (1, S, C), G, dtype, 'silu', True, torch.float32, seed=S)


@pytest.mark.parametrize("C,G", [(2312, 1), (2312, 2312), (1156, 4), (1200, 75)], ids=str)
def test_group_norm_act_wide(C, G, device):
    """Several tiles a row; groups of many tiles and many groups a tile."""
    for dtype in (torch.float32, torch.bfloat16):
        _norm_case(device, (2, 300, C), G, dtype, 'lrelu', True, torch.float32, seed=C)
        _norm_case(device, (1, 2600, C), G, dtype, 'silu', True, dtype, seed=G)


@pytest.mark.parametrize("N,S,C,G", [(2, 4, 8192, 1), (3, 5, 4100, 1), (1, 4096, 256, 2), (2, 1700, 530, 2), (1, 4100, 48, 1), (2, 9000, 96, 1)], ids=str)
def test_group_norm_act_wide_groups_in_parts(N, S, C, G, device):
    """Groups whose parts one workgroup joins, or several."""
    for dtype in (torch.float32, torch.float16):
        _norm_case(device, (N, S, C), G, dtype, 'silu', True, torch.float32)


@pytest.mark.parametrize("S,C,G", [(300, 6, 3), (93, 298, 149), (930, 298, 149), (480, 300, 100), (513, 48, 16), (400, 62, 31), (1025, 34, 17), (515, 66, 22)], ids=str)
def test_group_norm_act_narrow_groups(S, C, G, device):
    """Groups of a few channels: one of them, or as many as fill a vector, side by side in a workgroup."""
    for dtype in (torch.float32, torch.bfloat16):
        _norm_case(device, (2, S, C), G, dtype, 'lrelu', True, dtype)


@pytest.mark.parametrize("C", [64, 90, 112], ids=str)
def test_group_norm_act_batch_does_not_matter(C, device):
    """y and dx of a sample are the same bits alone and in a batch, also where only the batch is large enough to go past the caches."""
    from ag2video_amd import ops
    N, S = 3, 72000
    x = torch.randn(N, S, C, device=device, generator=torch.Generator(device=device).manual_seed(1))
    dy = torch.randn(N, S, C, device=device, generator=torch.Generator(device=device).manual_seed(2))
    w, b = _randn(C, seed=3).to(device), _randn(C, seed=4).to(device)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = ops.group_norm_act(leaves[0], 2, *leaves[1:])
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    sums, mags = torch.zeros(2, C, device=device, dtype=torch.float64), torch.zeros(2, C, device=device, dtype=torch.float64)
    for n in range(N):
        one = [t.clone().requires_grad_(True) for t in (x[n:n + 1], w, b)]
        y1 = ops.group_norm_act(one[0], 2, *one[1:])
        dx1, *dp = torch.autograd.grad(y1, one, dy[n:n + 1])
        assert torch.equal(y1[0], y[n]) and torch.equal(dx1[0], dx[n])
        dp = torch.stack(dp).double()
        sums += dp
        mags += dp.abs()
    # the parameters' gradients are the samples' own, joined by two fp32 additions of at most the magnitudes' sum each
    assert ((torch.stack((dw, db)).double() - sums).abs() <= 2 * R.U * mags).all()


def test_group_norm_act_far_mean(device):
    """A mean 300 deviations away, and one value 1e4 deviations away at the start of a group: the variance does not cancel."""
    from ag2video_amd import ops
    for shape, groups in (((2, 64, 16), 2), ((2, 6000, 16), 2)):
        x = _randn(*shape, seed=3) + 300.0
        x[0, 0, 0] += 1e4
        dy = _randn(*shape, seed=4)
        ref = R.group_norm(x, groups, None, None, 1e-5, 'none', 0.2, dy)
        leaf = x.to(device).requires_grad_(True)
        y = ops.group_norm_act(leaf, groups, act='none')
        R.check('y', y, *ref['y'])
        R.check('dx', torch.autograd.grad(y, leaf, dy.to(device))[0], *ref['dx'])


@pytest.mark.parametrize("S", [30, 5000])
def test_group_norm_act_one_parameter(S, device):
    """weight without bias, bias without weight; gradients of a part of the inputs."""
    from ag2video_amd import ops
    x, p, dy = _randn(2, S, 12, seed=1), _randn(12, seed=2), _randn(2, S, 12, seed=3)
    for w, b in ((p, None), (None, p)):
        ref = R.group_norm(x, 3, w, b, 1e-5, 'silu', 0.2, dy)
        gp = p.to(device).requires_grad_(True)
        gx = x.to(device).requires_grad_(True)
        args = (gp if w is not None else None, gp if b is not None else None)
        y = ops.group_norm_act(gx, 3, *args)
        R.check('y', y, *ref['y'])
        dx, dp = torch.autograd.grad(y, (gx, gp), dy.to(device))
        R.check('dx', dx, *ref['dx'])
        R.check('dp', dp, *ref['dweight' if w is not None else 'dbias'])
        only_p = torch.autograd.grad(ops.group_norm_act(gx.detach(), 3, *args), gp, dy.to(device))[0]
        assert torch.equal(only_p, dp)
        only_x = torch.autograd.grad(ops.group_norm_act(gx, 3, *(None if a is None else a.detach() for a in args)), gx, dy.to(device))[0]
        assert torch.equal(only_x, dx)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
def test_group_norm_act_strides(dtype, device):
    """Channel slices, channels-last NCHW tensors, samples apart, channels first (copied); gradients that are broadcast or lie apart."""
    from ag2video_amd import ops
    w, b = _randn(20, seed=8).to(device), _randn(20, seed=9).to(device)
    views = {
        'channel slice': (lambda t: t[..., 5:25], (3, 11, 13, 33)), 'one position apart': (lambda t: t[:, :, ::2], (3, 11, 14, 20)),
        'every other sample': (lambda t: t[::2], (5, 40, 20)), 'channels first': (lambda t: t.permute(0, 2, 3, 1), (2, 20, 9, 7)),
        'transposed positions': (lambda t: t.transpose(1, 2), (2, 9, 31, 20)), 'one sample repeated': (lambda t: t.expand(4, 30, 20), (1, 30, 20)),
        'odd offset': (lambda t: t.reshape(-1)[1:1 + 3 * 70 * 20].view(3, 70, 20), (3, 71, 20)),
        'long rows': (lambda t: t[..., 2:22], (2, 4500, 23)),
    }
    for name, (view, shape) in views.items():
        base = _randn(*shape, seed=1).to(dtype)
        x = view(base)
        dy = _randn(*x.shape, seed=2).to(dtype)
        ref = R.group_norm(x, 5, w.cpu(), b.cpu(), 1e-5, 'silu', 0.2, dy)
        leaf = base.to(device).requires_grad_(True)
        dx_at = view(leaf)
        dx_at.retain_grad()
        y = ops.group_norm_act(dx_at, 5, w, b)
        R.check(name + '.y', y, *ref['y'])
        y.backward(dy.to(device))
        R.check(name + '.dx', dx_at.grad, *ref['dx'])
    nchw = _randn(2, 20, 9, 7, seed=3).to(device).to(memory_format=torch.channels_last)
    ref = R.group_norm(nchw.cpu().permute(0, 2, 3, 1), 5, w.cpu(), b.cpu(), 1e-5, 'silu', 0.2)
    R.check('channels_last', ops.group_norm_act(nchw.permute(0, 2, 3, 1), 5, w, b), *ref['y'])
    x = _randn(2, 9, 7, 20, seed=4).to(dtype)
    for name, d in (('ones', torch.ones((), dtype=dtype).expand(2, 9, 7, 20)), ('one row', _randn(20, seed=5).to(dtype).expand(2, 9, 7, 20)),
                    ('slice', _randn(2, 9, 7, 30, seed=6).to(dtype)[..., 3:23]), ('channels first', _randn(2, 20, 9, 7, seed=7).to(dtype).permute(0, 2, 3, 1))):
        ref = R.group_norm(x, 5, w.cpu(), b.cpu(), 1e-5, 'silu', 0.2, d)
        leaf = x.to(device).requires_grad_(True)
        R.check(name, torch.autograd.grad(ops.group_norm_act(leaf, 5, w, b), leaf, d.to(device))[0], *ref['dx'])


@pytest.mark.parametrize("S", [20, 7000])
def test_group_norm_act_special_values(S, device):
    """An infinity or NaN reaches its own (sample, group) only; other groups keep their bits, forward and backward."""
    from ag2video_amd import ops
    x, dy, w, b = _randn(3, S, 16, seed=1), _randn(3, S, 16, seed=2), _randn(16, seed=3).to(device), _randn(16, seed=4).to(device)

    def run(x, dy):
        leaf = x.to(device).requires_grad_(True)
        y = ops.group_norm_act(leaf, 4, w, b)
        return y.detach().cpu(), torch.autograd.grad(y, leaf, dy.to(device))[0].cpu()

    y0, d0 = run(x, dy)
    x[1, S // 2, 5], x[2, 0, 15] = float('inf'), float('nan')
    y1, d1 = run(x, dy)
    bad = torch.zeros(3, S, 16, dtype=torch.bool)
    bad[1, :, 4:8] = bad[2, :, 12:16] = True
    for p, q in ((y0, y1), (d0, d1)):
        assert torch.isnan(q[bad]).all() and torch.equal(p[~bad], q[~bad])
    x[1, S // 2, 5], x[2, 0, 15] = 0.0, 0.0
    y2, d2 = run(x, dy)
    dy[0, 3, 1] = float('nan')
    y3, d3 = run(x, dy)
    bad = torch.zeros(3, S, 16, dtype=torch.bool)
    bad[0, :, :4] = True
    assert torch.equal(y2, y3) and torch.isnan(d3[bad]).all() and torch.equal(d2[~bad], d3[~bad])


def test_group_norm_act_constant_groups(device):
    """Variance zero: h = 0, y = act(bias), and a gradient that stays finite."""
    from ag2video_amd import ops
    x = torch.full((2, 40, 8), 3.25)
    x[1] = 0.0
    b = _randn(8, seed=1)
    dy = _randn(2, 40, 8, seed=2)
    ref = R.group_norm(x, 2, None, b, 1e-5, 'silu', 0.2, dy)
    leaf = x.to(device).requires_grad_(True)
    y = ops.group_norm_act(leaf, 2, None, b.to(device))
    R.check('y', y, *ref['y'])
    R.check('dx', torch.autograd.grad(y, leaf, dy.to(device))[0], *ref['dx'])


def test_empty(device):
    from ag2video_amd import ops
    w = torch.ones(8, device=device, requires_grad=True)
    for shape in ((0, 5, 8), (3, 0, 8), (2, 0, 4, 8)):
        x = torch.zeros(shape, device=device, requires_grad=True)
        y = ops.group_norm_act(x, 2, w)
        assert y.shape == x.shape
        dx, dw = torch.autograd.grad(y.sum(), (x, w))
        assert dx.shape == x.shape and not dw.any()
    table = torch.ones(4, 0, device=device, requires_grad=True)
    out = ops.embedding_scaled(torch.zeros(3, dtype=torch.long, device=device), table)
    assert out.shape == (3, 0) and torch.autograd.grad(out.sum(), table)[0].shape == (4, 0)


def test_group_norm_act_long_offsets(device):
    """A map of more than 2^31 elements."""
    from ag2video_amd import ops
    N, S, C = 3, 1 << 20, 720
    x = torch.empty(N, S, C, device=device, dtype=torch.bfloat16)
    for n in range(N):
        x[n].normal_(generator=torch.Generator(device=device).manual_seed(n))
    y = ops.group_norm_act(x, 8, act='none')
    for n in range(N):
        ref = ops.group_norm_act(x[n:n + 1].clone(), 8, act='none')
        assert torch.equal(ref[0, :1000], y[n, :1000]) and torch.equal(ref[0, -1000:], y[n, -1000:])
    m = y[2].float().view(S, 8, 90).mean((0, 2))
    assert m.abs().max() < 1e-3
    del y, ref
    leaf = x.requires_grad_(True)
    y = ops.group_norm_act(leaf, 8, act='none')
    (dx,) = torch.autograd.grad(y, leaf, x.detach())        # dy = x: what is left of it is rounding
    assert dx[2, -1000:].float().abs().max() < 0.05 and dx[0, :1000].float().abs().max() < 0.05


@pytest.mark.parametrize("S", [12, 6000])
def test_group_norm_act_against_differences(S, device):
    """The directional derivative by central differences of the operator itself: within the rounding of the two forward passes and the
    difference quotient's own error, which the 64-bit reference gives."""
    from ag2video_amd import ops
    N, C, G, e = 2, 12, 3, 2.0 ** -6
    x, w, b = _randn(N, S, C, seed=1), 1 + 0.2 * _randn(C, seed=2), _randn(C, seed=3)
    dy = _randn(N, S, C, seed=4)
    dirs = [_randn(*t.shape, seed=5 + i) for i, t in enumerate((x, w, b))]

    def at(k):
        return [t + k * e * d for t, d in zip((x, w, b), dirs)]

    vals, refs, slack = [], [], 0.0
    for k in (1, -1):
        px, pw, pb = at(k)
        y, bound = R.group_norm(px, G, pw, pb, 1e-5, 'silu', 0.2)['y']
        refs.append(float((y * dy.double()).sum()))
        slack += float((bound * dy.double().abs()).sum())
        got = ops.group_norm_act(px.to(device), G, pw.to(device), pb.to(device))
        vals.append(float((got.cpu().double() * dy.double()).sum()))
    by_op, by_ref = (vals[0] - vals[1]) / (2 * e), (refs[0] - refs[1]) / (2 * e)
    assert abs(by_op - by_ref) <= slack / (2 * e)
    leaves = [t.to(device).requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(ops.group_norm_act(leaves[0], G, *leaves[1:]), leaves, dy.to(device))
    ref = R.group_norm(x, G, w, b, 1e-5, 'silu', 0.2, dy)
    along = sum(float((g.cpu().double() * d.double()).sum()) for g, d in zip(grads, dirs))
    true = sum(float((ref[k][0] * d.double()).sum()) for k, d in zip(('dx', 'dweight', 'dbias'), dirs))
    rounding = sum(float((ref[k][1] * d.double().abs()).sum()) for k, d in zip(('dx', 'dweight', 'dbias'), dirs))
    assert abs(along - true) <= rounding
    assert abs(along - by_op) <= rounding + slack / (2 * e) + abs(true - by_ref)


def _chain(idx, table, w, b, groups=4):
    from ag2video_amd import ops
    rows = ops.embedding_scaled(idx, table, 3.0, 0)
    return ops.group_norm_act(rows, groups, w, b)


@pytest.mark.parametrize("shape", [(2, 6), (2, 9, 11), (3, 70, 64)], ids=str)
def test_run_together(shape, device):
    """A map of labels: its rows looked up, normalised over the map and activated, gradients back into the table."""
    n = 1
    for s in shape:
        n *= s
    V, D = 19, 32
    idx = _tokens(n, V, 1).view(shape)
    table, w, b = _randn(V, D, seed=2), 1 + 0.2 * _randn(D, seed=3), _randn(D, seed=4)
    dy = _randn(*shape, D, seed=5)
    leaves = [t.to(device).requires_grad_(True) for t in (table, w, b)]
    y = _chain(idx.to(device), *leaves)
    # the intermediate rows, as the operator rounds them, are the reference's input; the table's gradient takes the reference's dx with
    # its bound through the sum
    rows = (table.double()[idx] * 3.0).float()
    ref = R.group_norm(rows, 4, w, b, 1e-5, 'silu', 0.2, dy)
    R.check('y', y, *ref['y'])
    dt, dw, db = torch.autograd.grad(y, leaves, dy.to(device))
    R.check('dweight', dw, *ref['dweight'])
    R.check('dbias', db, *ref['dbias'])
    dx, e_dx = ref['dx']
    at = idx.reshape(-1)
    total = torch.zeros(V, D, dtype=torch.float64).index_add_(0, at, dx.reshape(-1, D)) * 3.0
    off = torch.zeros(V, D, dtype=torch.float64).index_add_(0, at, (e_dx + R.DEPTH * R.U * dx.abs()).reshape(-1, D)) * 3.0
    total[0], off[0] = 0.0, 0.0
    R.check('dtable', dt, total, off * (1 + R.U) + 4 * R.U * total.abs())


@pytest.mark.parametrize("V,D,shape", [(20, 16, (2, 30)), (300, 48, (4, 900)), (20, 48, (2, 9000)), (70000, 20, (3, 7000))], ids=str)
def test_other_stream_and_replay(V, D, shape, device):
    """Forward and backward on a side stream, then captured into a graph and replayed on new values between eager calls: the same bits."""
    torch.manual_seed(0)
    idx = torch.randint(V, shape, device=device)
    fresh = [torch.randn(V, D, device=device), torch.randn(D, device=device), torch.randn(D, device=device)]
    dys = [torch.randn(*shape, D, device=device) for _ in range(4)]

    def step(idx, table, w, b, dy):
        leaves = [t.detach().requires_grad_(True) for t in (table, w, b)]
        y = _chain(idx, *leaves)
        return (y.detach(),) + torch.autograd.grad(y, leaves, dy)

    eager = step(idx, *fresh, dys[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = step(idx, *fresh, dys[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(eager, there))

    s_idx, s_in, s_dy = idx.clone(), [t.clone() for t in fresh], dys[0].clone()
    with torch.cuda.stream(side):
        step(s_idx, *s_in, s_dy)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):                                     # two graphs, one memory pool
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            out = step(s_idx, *s_in, s_dy)
        graphs.append(graph)
        outs.append(out)
    for k in range(4):
        s_idx.copy_(torch.randint(V, shape, device=device, generator=torch.Generator(device=device).manual_seed(k)))
        for t in s_in:
            t.add_(0.25)
        s_dy.copy_(dys[k])
        for graph, out in zip(graphs, outs):
            graph.replay()
            got = [t.clone() for t in out]
            torch.cuda.synchronize()
            want = step(s_idx, *s_in, s_dy)
            assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_calls_on_two_streams_at_once(device):
    torch.manual_seed(1)
    idx = torch.randint(5000, (30000,), device=device)
    table, x = torch.randn(5000, 40, device=device), torch.randn(4, 5000, 64, device=device)
    dout, dy = torch.randn(30000, 40, device=device), torch.randn(4, 5000, 64, device=device)
    from ag2video_amd import ops

    def embed():
        t = table.detach().requires_grad_(True)
        return torch.autograd.grad(ops.embedding_scaled(idx, t, 1.5), t, dout)[0]

    def norm():
        t = x.detach().requires_grad_(True)
        return torch.autograd.grad(ops.group_norm_act(t, 8), t, dy)[0]

    want = embed(), norm()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for _ in range(3):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((k % 2, (embed, norm)[k % 2]()))
    torch.cuda.synchronize()
    assert all(torch.equal(t, want[k]) for k, t in got)


def test_calls_of_two_threads(device):
    """Each thread on a stream of its own, forward and backward."""
    import threading
    from ag2video_amd import ops
    x, dy = torch.randn(3, 700, 64, device=device), torch.randn(3, 700, 64, device=device)
    idx, table, dout = torch.randint(900, (9000,), device=device), torch.randn(900, 24, device=device), torch.randn(9000, 24, device=device)

    def norm():
        t = x.detach().requires_grad_(True)
        return torch.autograd.grad(ops.group_norm_act(t, 8), t, dy)[0]

    def embed():
        t = table.detach().requires_grad_(True)
        return torch.autograd.grad(ops.embedding_scaled(idx, t, 0.5), t, dout)[0]

    want, got = (norm(), embed()), []
    torch.cuda.synchronize()

    def work(k):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            mine = [(norm, embed)[k]() for _ in range(20)]
            stream.synchronize()
        got.extend((k, t) for t in mine)

    threads = [threading.Thread(target=work, args=(k % 2,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 80 and all(torch.equal(t, want[k]) for k, t in got)


def test_parameters_inside_flat_buffers(device):
    """Tables and norm parameters that are views of a flat buffer at any element offset (as the fused optimizer keeps them)."""
    from ag2video_amd import ops
    flat = _randn(2000, seed=1).to(device)
    for off in (1, 2, 3, 5):
        w, b, table = flat[off:off + 52], flat[100 + off:152 + off], flat[200 + off:200 + off + 19 * 52].view(19, 52)
        idx = _tokens(300, 19, off)
        ref = R.embedding(idx, table.cpu(), 2.0, None)
        rows = ops.embedding_scaled(idx.to(device), table, 2.0)
        R.check('rows', rows, *ref)
        x = rows.view(3, 100, 52)
        for S in (100, 50):
            want = R.group_norm(x[:, :S].cpu(), 13, w.cpu(), b.cpu(), 1e-5, 'silu', 0.2)
            R.check('y', ops.group_norm_act(x[:, :S], 13, w, b), *want['y'])


def test_modules(device):
    """layers.Embedding with a scale and layers.GroupNormAct: the operators with nn.Embedding's and nn.GroupNorm's parameters."""
    from ag2video_amd import ops
    from ag2video_amd.models.layers import Embedding, GroupNormAct
    emb = Embedding(11, 24, padding_idx=3, scale=2.0).to(device)
    norm = GroupNormAct(4, 24, act='lrelu', slope=0.1).to(device)
    assert set(norm.state_dict()) == {'weight', 'bias'} and set(emb.state_dict()) == {'weight'}
    idx = _tokens(40, 11, 1).view(2, 20).to(device)
    y = norm(emb(idx))
    want = ops.group_norm_act(ops.embedding_scaled(idx, emb.weight, 2.0, 3), 4, norm.weight, norm.bias, act='lrelu', slope=0.1)
    assert torch.equal(y, want)
    y.square().sum().backward()
    assert not emb.weight.grad[3].any() and emb.weight.grad[4].any() and norm.weight.grad.any()
    plain = Embedding(11, 24).to(device)
    assert torch.equal(plain(idx), ops.embedding(idx, plain.weight))
    half = Embedding(11, 24).to(device).to(torch.bfloat16)
    assert half(idx).dtype == torch.bfloat16


def test_module_takes_tokens_of_any_integer_type(device):
    """A padding_idx changes the operator behind layers.Embedding, not the tokens it takes."""
    from ag2video_amd.models.layers import Embedding
    idx = _tokens(40, 11, 1).to(device)
    emb = Embedding(11, 24, padding_idx=3).to(device)
    for itype in (torch.uint8, torch.int16, torch.int32):
        assert torch.equal(emb(idx.to(itype)), emb.weight[idx])


def test_no_second_derivative(device):
    """Differentiating a gradient is an error and not a wrong number: the backward pass is refused where its graph is asked for."""
    from ag2video_amd import ops
    x = torch.randn(2, 5, 8, device=device, requires_grad=True)
    table = torch.randn(6, 8, device=device, requires_grad=True)
    for leaf, y in ((x, ops.group_norm_act(x, 2)), (table, ops.embedding_scaled(torch.arange(4, device=device), table))):
        with pytest.raises(RuntimeError, match='second derivative'):
            torch.autograd.grad(y.square().sum(), leaf, create_graph=True)


def test_refusals(device):
    """What the operators refuse of tensors on the device."""
    from ag2video_amd import ops
    idx, table = torch.zeros(3, dtype=torch.long, device=device), torch.zeros(4, 8, device=device)
    x = torch.zeros(2, 3, 8, device=device)
    for call in (lambda: ops.embedding_scaled(idx.cpu(), table), lambda: ops.embedding_scaled(idx.float(), table), lambda: ops.embedding_scaled(idx.short(), table),
                 lambda: ops.embedding_scaled(idx, table.double()), lambda: ops.embedding_scaled(idx, table[0]), lambda: ops.embedding_scaled(idx, table[:0]),
                 lambda: ops.embedding_scaled(idx, table, 1.0, 4), lambda: ops.embedding_scaled(idx, table, 1.0, -1), lambda: ops.embedding_scaled(idx, table.long()),
                 lambda: ops.group_norm_act(x, 3), lambda: ops.group_norm_act(x, 0), lambda: ops.group_norm_act(x, -2), lambda: ops.group_norm_act(x[0, 0], 2),
                 lambda: ops.group_norm_act(x.double(), 2), lambda: ops.group_norm_act(x, 2, act='tanh'), lambda: ops.group_norm_act(x, 2, eps=-1.0),
                 lambda: ops.group_norm_act(x, 2, eps=float('nan')), lambda: ops.group_norm_act(x, 2, slope=float('nan')),
                 lambda: ops.group_norm_act(x, 2, torch.ones(7, device=device)), lambda: ops.group_norm_act(x, 2, torch.ones(8)),
                 lambda: ops.group_norm_act(x, 2, None, torch.ones(8, 1, device=device)), lambda: ops.group_norm_act(x, 2, torch.ones(8, device=device).half()),
                 lambda: ops.group_norm_act(x.half(), 2, torch.ones(8, device=device), torch.ones(8, device=device).half()),
                 lambda: ops.group_norm_act(x[..., :0], 1), lambda: ops.group_norm_act(torch.zeros(1, device=device).expand(1 << 22, 1, 8), 8)):
        with pytest.raises(RuntimeError):
            call()
