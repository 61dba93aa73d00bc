"""What embedding_scaled and group_norm_act refuse, at the Python and at the C boundary, and the reference's own gradients."""
import ctypes

import pytest
import torch

import _elem_ref as R


def _refused(fn, *args, **kwargs):
    with pytest.raises(RuntimeError):
        fn(*args, **kwargs)


def test_cpu_tensors_are_refused():
    from ag2video_amd import ops
    _refused(ops.embedding_scaled, torch.zeros(3, dtype=torch.long), torch.zeros(4, 8))
    _refused(ops.group_norm_act, torch.zeros(2, 3, 8), 2)


def _entry():
    from ag2video_amd import _lib
    return _lib.load(), ctypes.c_void_p(4096)           # a non-null pointer that no refused call follows


def test_embed_entry_points_refuse():
    """Arguments the kernels cannot take come back as AG2V_EINVAL before anything is launched."""
    lib, p = _entry()
    fwd = dict(dtype=0, idx=p, ib=8, istride=1, table=p, tstride=8, out=p, n=4, V=5, D=8, scale=1.0, stream=None)
    for change in (dict(dtype=3), dict(dtype=-1), dict(idx=None), dict(table=None), dict(out=None), dict(ib=2), dict(n=0), dict(n=-1), dict(n=1 << 31),
                   dict(V=0), dict(V=1 << 31), dict(D=0), dict(D=1 << 30), dict(tstride=7)):
        assert lib.ag2v_embed_fwd(*{**fwd, **change}.values()) == -1, change
    need = lib.ag2v_embed_bwd_workspace_floats(0, 5000, 5, 8)
    bwd = dict(dtype=0, idx=p, ib=8, istride=1, dout=p, dstride=8, dtable=p, n=5000, V=5, D=8, scale=1.0, pad=-1, ws=p, nws=need, stream=None)
    for change in (dict(dtype=7), dict(idx=None), dict(dout=None), dict(dtable=None), dict(ib=1), dict(n=0), dict(V=0), dict(D=-3), dict(n=1 << 32)):
        assert lib.ag2v_embed_bwd(*{**bwd, **change}.values()) == -1, change
    for n, V, D in ((100000, 50000, 8), (9000, 9000, 700)):
        need = lib.ag2v_embed_bwd_workspace_floats(1, n, V, D)
        big = {**bwd, 'dtype': 1, 'n': n, 'V': V, 'D': D}
        assert need > 0
        assert lib.ag2v_embed_bwd(*{**big, 'nws': need - 1}.values()) == -1
        assert lib.ag2v_embed_bwd(*{**big, 'ws': None, 'nws': need}.values()) == -1
        assert lib.ag2v_embed_bwd(*{**big, 'ws': ctypes.c_void_p(4100), 'nws': need}.values()) == -1
    assert lib.ag2v_embed_bwd_workspace_floats(0, 0, 5, 8) == 0 and lib.ag2v_embed_bwd_workspace_floats(9, 10, 5, 8) == 0


def test_group_norm_entry_points_refuse():
    lib, p = _entry()
    fwd = dict(dtype=0, x=p, xs=24, xr=8, w=p, b=p, pt=0, y=p, mean=p, rstd=p, N=2, S=3, C=8, G=2, eps=1e-5, act=1, slope=0.2, ws=p, nws=1 << 20, stream=None)
    for change in (dict(dtype=3), dict(pt=5), dict(x=None), dict(y=None), dict(mean=None), dict(rstd=None), dict(N=0), dict(S=0), dict(S=-4), dict(S=1 << 30), dict(C=0), dict(N=1 << 23), dict(pt=1),
                   dict(G=0), dict(G=3), dict(eps=-1.0), dict(eps=float('nan')), dict(act=3), dict(act=-1)):
        assert lib.ag2v_group_norm_fwd(*{**fwd, **change}.values()) == -1, change
    bwd = dict(dtype=0, dy=p, ds=24, dr=8, x=p, xs=24, xr=8, w=p, b=p, pt=0, mean=p, rstd=p, dx=p, dw=p, db=p, N=2, S=3, C=8, G=2, act=1, slope=0.2,
               ws=p, nws=1 << 20, stream=None)
    for change in (dict(dtype=-1), dict(dy=None), dict(x=None), dict(mean=None), dict(rstd=None), dict(N=-1), dict(C=7), dict(G=16), dict(act=9)):
        assert lib.ag2v_group_norm_bwd(*{**bwd, **change}.values()) == -1, change
    for backward, entry, base in ((0, lib.ag2v_group_norm_fwd, fwd), (1, lib.ag2v_group_norm_bwd, bwd)):
        big = {**base, 'N': 4, 'S': 100000, 'C': 64, 'G': 4}
        need = lib.ag2v_group_norm_workspace_floats(0, 4, 100000, 64, 4, backward)
        assert need > 0
        assert entry(*{**big, 'nws': need - 1}.values()) == -1
        assert entry(*{**big, 'ws': None, 'nws': need}.values()) == -1
        assert entry(*{**big, 'ws': ctypes.c_void_p(4100), 'nws': need}.values()) == -1


def test_reference_gradients_against_differences():
    """The 64-bit formulas the GPU tests compare with: gradients against central differences (error ~ step^2 and rounding / step)."""
    torch.manual_seed(0)
    x, w, b = torch.randn(2, 9, 12), 1 + 0.2 * torch.randn(12), torch.randn(12)
    dy, e = torch.randn(2, 9, 12), 2.0 ** -10
    for act in ('none', 'silu', 'lrelu'):
        ref = R.group_norm(x.double(), 3, w.double(), b.double(), 1e-5, act, 0.2, dy.double())
        for k, name in enumerate(('dx', 'dweight', 'dbias')):
            d = torch.randn((x, w, b)[k].shape, dtype=torch.float64)
            f = []
            for s in (1, -1):
                p = [x.double(), w.double(), b.double()]
                p[k] = p[k] + s * e * d
                f.append(float((R.group_norm(p[0], 3, p[1], p[2], 1e-5, act, 0.2)['y'][0] * dy.double()).sum()))
            along = float((ref[name][0] * d).sum())
            # a third derivative of order 10^2 at most here, times e^2; a leaky kink inside the step adds its width times the slope's jump
            slack = 1e-3 if act != 'lrelu' else 0.2
            assert abs((f[0] - f[1]) / (2 * e) - along) <= slack * max(1.0, abs(along)), (act, name)
    idx = torch.tensor([3, 1, 3, 0, 5, -1, 3])
    table, dout = torch.randn(5, 4), torch.randn(7, 4)
    out, _, dt, _ = R.embedding(idx, table, 2.0, 0, dout)
    assert torch.isnan(out[4:6]).all() and torch.equal(out[0], 2.0 * table[3].double())
    assert torch.equal(dt[3], 2.0 * (dout[0].double() + dout[2].double() + dout[6].double())) and not dt[0].any() and not dt[4].any()


@pytest.mark.parametrize("shape,view,expect", [
    ((2, 3, 4, 8), lambda t: t, (96, 8)), ((2, 3, 4, 8), lambda t: t[..., 2:6], (96, 8)), ((2, 3, 4, 8), lambda t: t[:, :, ::2], (96, 16)),
    ((2, 3, 4, 8), lambda t: t[:, 1:2], (96, 8)), ((2, 8, 3, 4), lambda t: t.permute(0, 2, 3, 1), None), ((2, 3, 4, 8), lambda t: t.transpose(1, 2), None),
    ((1, 5, 8), lambda t: t.expand(3, 5, 8), (0, 8)), ((5, 8), lambda t: t, (8, 8)), ((5, 8), lambda t: t[::2], (16, 4)), ((5, 1, 8), lambda t: t, (8, 8)),
    ((2, 6, 1), lambda t: t[:, ::3], (6, 3)),
], ids=range(11))
def test_channel_rows(shape, view, expect):
    """Which views are read in place: (sample stride, row stride), None where the operator copies."""
    from ag2video_amd import _lib
    n = 1
    for s in shape:
        n *= s
    x = view(torch.arange(float(n)).view(shape))
    t, xs, xr = _lib.elem_ops().channel_rows(x)
    if expect is None:
        assert t.data_ptr() != x.data_ptr() and t.is_contiguous()
    else:
        assert t.data_ptr() == x.data_ptr()
        if x.dim() > 2:
            assert (xs, xr) == expect
        else:
            assert xs == expect[0]
    C, rows = x.shape[-1], x[0].numel() // x.shape[-1]
    flat = torch.as_strided(t, (x.shape[0], rows, C), (xs, xr, 1), t.storage_offset())
    assert torch.equal(flat, x.reshape(x.shape[0], rows, C))


@pytest.mark.parametrize("view,stride", [(lambda t: t, 1), (lambda t: t[:, :, 1], 3), (lambda t: t[::2], None), (lambda t: t[1], 1), (lambda t: t[:, 0, 0], 12),
                                         (lambda t: t.permute(2, 0, 1), None), (lambda t: t[0, 0, 0], 1), (lambda t: t[:1].expand(4, 4, 3), None)], ids=range(8))
def test_token_rows(view, stride):
    from ag2video_amd import _lib
    idx = view(torch.arange(5 * 4 * 3).view(5, 4, 3))
    t, st = _lib.elem_ops().token_rows(idx)
    if stride is not None:
        assert st == stride and t.data_ptr() == idx.data_ptr()
    assert torch.equal(torch.as_strided(t, (idx.numel(),), (st,), t.storage_offset()), idx.reshape(-1))
