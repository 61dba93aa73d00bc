"""embedding_scaled and group_norm_act at the sizes that their documentation ends with: batches of more workgroups than one launch takes, rows of 2^29
channels and 2^23 columns."""
import pytest
import torch

import _elem_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _give_memory_back():
    yield
    torch.cuda.empty_cache()


def _normal(device, seed, *shape, dtype=torch.bfloat16):
    g = torch.Generator(device=device).manual_seed(seed)
    t = torch.empty(*shape, device=device, dtype=dtype)
    for part in t.flatten().split(1 << 30):
        part.normal_(generator=g)
    return t


# One launch for a sample: 2^23 workgroups of 2 samples do not fit one grid.  Parts: 17 a sample, over 2^24 in all; 10 columns of 4 samples' parts.
@pytest.mark.parametrize("N,S", [((1 << 23) + 5, 130), ((1 << 20) + 3, 8704)], ids=['one launch', 'parts'])
def test_samples_of_large_batches(N, S, device):
    """y and dx of a sample are the same bits in a batch of any size, on both sides of every border between launches."""
    from ag2video_amd import ops
    x, dy = _normal(device, 1, N, S, 1), _normal(device, 2, N, S, 1)
    p = [torch.full((1,), v, device=device, requires_grad=True) for v in (1.25, 0.5)]
    x.requires_grad_(True)
    y = ops.group_norm_act(x, 1, *p)
    dx, _, _ = torch.autograd.grad(y, [x] + p, dy)
    y = y.detach()
    first = N // 2
    for at in [0, N - 9] + [k for b in range(1, 4) for k in (b * ((1 << 23) - 1) // 17 - 4, b * ((1 << 22) - 1) * 2 - 4) if 0 <= k < N - 9]:
        few = x.detach()[at:at + 9].clone().requires_grad_(True)
        y1 = ops.group_norm_act(few, 1, *p)
        dx1 = torch.autograd.grad(y1, few, dy[at:at + 9])[0]
        assert torch.equal(y1, y[at:at + 9]) and torch.equal(dx1, dx[at:at + 9]), at
    for at, n in ((0, first), (first, N - first)):              # and all of it against two calls of half the batch
        half = x.detach()[at:at + n].requires_grad_(True)
        y1 = ops.group_norm_act(half, 1, *p)
        assert torch.equal(y1, y[at:at + n])
        assert torch.equal(torch.autograd.grad(y1, half, dy[at:at + n])[0], dx[at:at + n])


def test_very_many_channels(device):
    """2^29 + 8 channels of one position: the parameters' gradients are single products."""
    from ag2video_amd import ops
    C, G = (1 << 29) + 8, 8
    x, dy = _normal(device, 1, 1, 1, C, dtype=torch.float16), _normal(device, 2, 1, 1, C, dtype=torch.float16)
    w, b = torch.ones(C, device=device, dtype=torch.float16), torch.zeros(C, device=device, dtype=torch.float16)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = ops.group_norm_act(x, G, w, b, act='none')
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    assert torch.equal(db, dy.view(C))
    ut = R.half_step(torch.float16)
    for g in range(G):
        at = slice(g * (C // G), (g + 1) * (C // G))
        v, d = x.detach().view(C)[at].double(), dy.view(C)[at].double()
        mean = v.mean()
        h = (v - mean) * (((v - mean) ** 2).mean() + 1e-5) ** -0.5
        # the statistics' sums: no thread adds more than DEPTH terms in fp32, what joins them is in fp64
        e_h = 2 * R.DEPTH * R.U * (1 + h.abs())
        assert ((y.detach().view(C)[at].double() - h).abs() <= ut * h.abs() + 2 * e_h + R.tiny(torch.float16)).all()
        assert ((dw[at].double() - d * h).abs() <= ut * (d * h).abs() + 2 * e_h * d.abs() + R.tiny(torch.float16)).all()
    assert torch.isfinite(dx).all()


@pytest.mark.parametrize("n,V,D,dtype", [(100, 128, 1 << 23, torch.float32), (3, 2, (1 << 30) - 1, torch.bfloat16)], ids=['2^23', '2^30 - 1'])
def test_very_wide_rows(n, V, D, dtype, device):
    """Whole numbers: every product and sum is exact."""
    from ag2video_amd import ops
    idx = (torch.arange(n, device=device) * 5) % V
    table = _normal(device, 1, V, D, dtype=dtype).mul_(4).round_().requires_grad_(True)
    dout = _normal(device, 2, n, D, dtype=dtype).mul_(4).round_()
    out = ops.embedding_scaled(idx, table, 2.0)
    for i in range(n):
        assert torch.equal(out[i], table.detach()[idx[i]] * 2)
    (got,) = torch.autograd.grad(out, table, dout)
    del out
    for v in range(V):
        rows = dout[idx == v]
        assert torch.equal(got[v], rows.sum(0, dtype=torch.float32).mul(2).to(dtype) if rows.shape[0] else torch.zeros_like(got[v]))


# One launch, whose workgroups walk many samples each, and parts, whose samples are added up at the end.
@pytest.mark.parametrize("N,S,C", [(1 << 23, 16, 1), (1 << 18, 1100, 1), (1 << 20, 16, 12), (70000, 1500, 3)], ids=str)
def test_parameter_gradients_of_very_many_samples(N, S, C, device):
    """dbias where every term is the same number, whose last bits a long fp32 sum would drop one by one, and dweight.

    No fp32 sum is deeper than a walker's 256 samples of at most two rows each and, before and behind it, the joins of a workgroup (14 levels)."""
    from ag2video_amd import ops
    c = (13107 + 63 / 128) / 2 ** 17                            # 21 bits
    x = _normal(device, 1, N, S, C, dtype=torch.float32)
    dy = torch.full((), c, device=device).expand(N, S, C)
    p = [torch.full((C,), v, device=device, requires_grad=True) for v in (1.0, 0.0)]
    dw, db = torch.autograd.grad(ops.group_norm_act(x, C, *p, act='none'), p, dy)
    total = float(N) * S * c
    depth = 256 + 2 + 14 + 1
    assert ((db.double() - total).abs() <= depth * R.U * total).all(), ((db.double() - total) / total / R.U).tolist()
    # dweight = c * sum of h, which is 0 but for rounding: that of the mean (DEPTH additions) in each h, and of the sums
    mags = torch.zeros(C, device=device, dtype=torch.float64)
    for part in x.split(1 << 18):
        d = part.double()
        d -= d.mean(1, keepdim=True)
        mags += (d.abs() * ((d * d).mean(1, keepdim=True) + 1e-5) ** -0.5).sum((0, 1))
    assert (dw.double().abs() <= c * (depth + 3 * R.DEPTH) * R.U * mags).all()
