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
