"""embedding_scaled and group_norm_act in 64 bits, each with a bound on how far a correct fp32 computation of it may be off.

u = 2^-24 is half a step of fp32, ut half a step of the tensors' type.  No sum of the kernels is deeper than DEPTH additions at the sizes
tested (a thread's own rows, the workgroup's tree, the join of the parts), so a sum is off by at most DEPTH u times the sum of its terms'
magnitudes.  The bounds follow the formulas step by step; nothing in them is measured.
"""
import torch

U = 2.0 ** -24
DEPTH = 256


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half a step of the type's subnormal numbers."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def embedding(idx, table, scale, pad, dout=None):
    """out, bound [, dtable, bound].  idx, table, dout: CPU tensors of the types the operator takes."""
    V, D = table.shape
    ut, tn = half_step(table.dtype), tiny(table.dtype)
    flat = idx.reshape(-1).long()
    inside = (flat >= 0) & (flat < V)
    rows = table.double()[flat.clamp(0, V - 1)] * scale
    rows[~inside] = float('nan')
    out = rows.view(*idx.shape, D)
    # scale to fp32, the product, the store
    bound = (ut + 2 * U) * (1 + ut) * out.abs() + tn
    if dout is None:
        return out, bound
    take = inside if pad is None else inside & (flat != pad)
    d = dout.double().reshape(-1, D)[take]
    at = flat[take]
    total = torch.zeros(V, D, dtype=torch.float64).index_add_(0, at, d)
    mags = torch.zeros(V, D, dtype=torch.float64).index_add_(0, at, d.abs())
    count = torch.zeros(V, dtype=torch.float64).index_add_(0, at, torch.ones(at.numel(), dtype=torch.float64))
    depth = torch.clamp(count, max=DEPTH)[:, None]
    err = abs(scale) * mags * (depth + 2) * U
    dt = total * scale
    return out, bound, dt, err + ut * (dt.abs() + err) + tn


def _act(z, act, slope):
    if act == 'silu':
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if act == 'lrelu':
        return torch.where(z > 0, z, z * slope), torch.where(z > 0, torch.ones_like(z), torch.full_like(z, slope))
    return z, torch.ones_like(z)


def group_norm(x, groups, weight, bias, eps, act, slope, dy=None):
    """{'y': (value, bound) [, 'dx', 'dweight', 'dbias']} for x [N, ..., C]."""
    shape, C = x.shape, x.shape[-1]
    N = shape[0]
    ut, tn = half_step(x.dtype), tiny(x.dtype)
    v = x.double().reshape(N, -1, groups, C // groups)
    S, M = v.shape[1], v.shape[1] * (C // groups)
    w = (torch.ones(C) if weight is None else weight).double().view(1, 1, groups, -1)
    b = (torch.zeros(C) if bias is None else bias).double().view(1, 1, groups, -1)
    dims = (1, 3)
    mean = v.mean(dims, keepdim=True)
    d = v - mean
    var = (d * d).mean(dims, keepdim=True)
    rstd = (var + eps) ** -0.5
    h = d * rstd
    z = h * w + b
    y, slope_z = _act(z, act, slope)
    du = DEPTH * U
    e_mean = du * v.abs().mean(dims, keepdim=True) + U * mean.abs()
    # the variance from deviations around a value of the group's own range: a thread's sum of squares is at most its count (<= DEPTH)
    # times its sum of squares about the mean, hence the second DEPTH term on the variance, and the mean's error enters squared and once
    # more through the deviations
    e_var = 2 * du * var + e_mean * e_mean + 2 * e_mean * d.abs().mean(dims, keepdim=True) + 4 * U * (v * v).mean(dims, keepdim=True).sqrt() * var.sqrt()
    r_rstd = 0.5 * e_var / (var + eps) + 4 * U
    e_h = (e_mean + U * (v.abs() + mean.abs())) * rstd + h.abs() * (r_rstd + 3 * U)
    e_z = w.abs() * e_h + 3 * U * ((w * h).abs() + b.abs())
    # silu' <= 1.1; the sigmoid from exp and a reciprocal: (4 + |z|) u relative
    if act == 'silu':
        e_y = 1.1 * e_z + (4 + z.abs()) * U * y.abs()
    elif act == 'lrelu':
        e_y = max(1.0, abs(slope)) * e_z + U * y.abs()
    else:
        e_y = e_z
    out = {'y': (y.reshape(shape), (e_y + ut * (y.abs() + e_y) + tn).reshape(shape))}
    if dy is None:
        return out
    g = dy.double().reshape(v.shape)
    dz = g * slope_z
    if act == 'silu':           # |silu''| <= 0.5
        e_dz = g.abs() * (0.5 * e_z + (8 + 2 * z.abs()) * U * (1 + z.abs()))
    elif act == 'lrelu':        # within e_z of the kink either slope is right
        e_dz = torch.where(z.abs() <= e_z, g.abs() * abs(1 - slope), U * dz.abs())
    else:
        e_dz = torch.zeros_like(dz)
    t, e_t = w * dz, w.abs() * e_dz + U * (w * dz).abs()
    s1, s2 = t.mean(dims, keepdim=True), (t * h).mean(dims, keepdim=True)
    e_s1 = e_t.mean(dims, keepdim=True) + (du + 2 * U) * t.abs().mean(dims, keepdim=True)
    e_th = e_t * h.abs() + t.abs() * e_h + U * (t * h).abs()
    e_s2 = e_th.mean(dims, keepdim=True) + (du + 2 * U) * (t * h).abs().mean(dims, keepdim=True)
    dx = rstd * (t - s1 - h * s2)
    e_dx = rstd * (e_t + e_s1 + h.abs() * e_s2 + s2.abs() * e_h + 4 * U * (t.abs() + s1.abs() + (h * s2).abs())) + dx.abs() * (r_rstd + 2 * U)
    out['dx'] = (dx.reshape(shape), (e_dx + ut * (dx.abs() + e_dx) + tn).reshape(shape))
    up = ut if weight is None else half_step(weight.dtype)
    e_p = {'dweight': ((dz * h), e_dz * h.abs() + dz.abs() * e_h + U * (dz * h).abs()), 'dbias': (dz, e_dz)}
    for name, (terms, err) in e_p.items():
        s = terms.sum((0, 1)).reshape(-1)
        e = (err + 2 * du * terms.abs()).sum((0, 1)).reshape(-1)
        out[name] = (s, e + up * (s.abs() + e) + (tiny(x.dtype) if weight is None else tiny(weight.dtype)))
    return out


def check(name, got, ref, bound):
    """Element by element within the bound; NaN exactly where the reference has one."""
    got = got.detach().cpu().double()
    assert got.shape == ref.shape, "%s: shape %s, expected %s" % (name, tuple(got.shape), tuple(ref.shape))
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(got), nan), "%s: NaN in other places" % name
    off = (got - ref).abs()[~nan]
    lim = bound.expand(ref.shape)[~nan]
    if off.numel():
        k = int((off - lim).argmax())
        assert off[k] <= lim[k], "%s: off by %.3e where %.3e is allowed (value %.3e)" % (name, off[k], lim[k], ref[~nan][k])
