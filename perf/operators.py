"""The cases on which the embedding and group-norm operators are measured.

``ops.embedding_scaled``: rows of a table looked up by token and multiplied by a constant; its gradient sums the rows of the output's
gradient by token.  ``ops.group_norm_act``: group norm with an activation on channels-last maps, forward and backward.  The plain forms
below are the same operators in elementary torch operations; ``exact`` has them once more in 64 bits.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
_BYTES = {'f32': 4, 'bf16': 2, 'f16': 2}


# ------------------------------------------------------------------------------------------------ cases
def _embed(name, train, n, V, D, dtype, tokens, scale, pad=-1, index='i64'):
    return {'name': name, 'op': 'embed', 'train': train, 'n': n, 'V': V, 'D': D, 'dtype': dtype, 'tokens': tokens, 'scale': scale,
            'pad': pad, 'index': index}


def _norm(name, train, N, S, C, G, dtype, act, affine=True, params='f32'):
    return {'name': name, 'op': 'norm', 'train': train, 'N': N, 'S': S, 'C': C, 'G': G, 'dtype': dtype, 'act': act, 'affine': affine,
            'params': params}


def listed():
    return [
        # the object attributes of one clip at inference: 10 objects, a table of two dozen words (latency)
        _embed('embed_objects', False, 10, 24, 128, 'f32', 'uniform', 1.0),
        # a label map for 8 frames of 256 x 256, each label's row at its pixel (the output is all the work)
        _embed('embed_label_map', False, 8 * 256 * 256, 27, 128, 'bf16', 'runs', math.sqrt(128.0), index='i32'),
        # the actions of a training step: batch 8, 16 frames, 10 edges
        _embed('embed_train_actions', True, 8 * 16 * 10, 24, 128, 'f32', 'uniform', 1.0, pad=0),
        # captions of a training step: words of a large vocabulary by their frequency
        _embed('embed_train_captions', True, 8192, 32000, 1024, 'bf16', 'frequency', 32.0, pad=0),
        # a long ragged batch, an odd width: rows that no vector load is aligned to
        _embed('embed_train_long', True, 131071, 50001, 389, 'f16', 'frequency', math.sqrt(389.0)),
        # a label map in training: 8 maps of 128 x 128 whose gradient meets in 27 rows
        _embed('embed_train_label_map', True, 8 * 128 * 128, 27, 128, 'f32', 'runs', 1.0),
        # the decoder's head of one clip at inference: an 8 x 8 map (latency)
        _norm('norm_head', False, 1, 64, 1024, 32, 'bf16', 'silu'),
        # frames at the output resolution at inference, the largest map
        _norm('norm_full', False, 16, 256 * 256, 64, 32, 'bf16', 'silu'),
        # the decoder's head in training
        _norm('norm_train_head', True, 8, 64, 1024, 32, 'f32', 'silu'),
        # a middle level in training, parameters in the maps' type
        _norm('norm_train_mid', True, 8, 64 * 64, 256, 32, 'f16', 'silu', params='same'),
        # odd maps: 37 x 53, 15 channels a group, a leaky slope
        _norm('norm_train_odd', True, 3, 37 * 53, 90, 6, 'f32', 'lrelu'),
        # clips whose statistics span 16 frames of 64 x 64, the largest training case
        _norm('norm_train_clip', True, 4, 16 * 64 * 64, 256, 32, 'bf16', 'silu'),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


_TENSOR_BYTES = 1 << 27     # no drawn tensor is larger than the largest listed one


def draw(rng):
    dtype = rng.choice(['f32', 'bf16', 'f16'])
    most = _TENSOR_BYTES // _BYTES[dtype]
    train = rng.random() < 0.65
    case = _draw_embed(rng, dtype, most, train) if rng.random() < 0.5 else _draw_norm(rng, dtype, most, train)
    del case['name']
    return case


def _draw_embed(rng, dtype, most, train):
    D = _log(rng, 1, 2048)
    n = _log(rng, 1, max(1, min(1 << 19, most // D)))
    V = _log(rng, 1, max(1, min(1 << 17, most // D)))
    return _embed('', train, n, V, D, dtype, rng.choice(['uniform', 'frequency', 'runs']), rng.choice([1.0, math.sqrt(D), 0.37]),
                  pad=rng.choice([-1, rng.randrange(V)]), index=rng.choice(['i64', 'i32']))


def _draw_norm(rng, dtype, most, train):
    Cg = rng.choice([1, 2, 3, 4, 5, 8, 8, 15, 16, 16, 32, 64])
    G = _log(rng, 1, max(1, 2048 // Cg))
    C = Cg * G
    N = _log(rng, 1, 32)
    # at least 16 values a group: with two, what is left of the gradient is rounding, in 32 bits as in 16
    S = _log(rng, -(-16 // Cg), max(16, min(1 << 17, most // (N * C))))
    return _norm('', train, N, S, C, G, dtype, rng.choice(['none', 'silu', 'lrelu']), affine=rng.random() < 0.8,
                 params=rng.choice(['f32', 'same']))


# ------------------------------------------------------------------------------------------------ inputs
def _tokens(case, gen, dev):
    n, V = case['n'], case['V']
    if case['tokens'] == 'frequency':           # word r with probability ~ 1 / (r + 1)
        u = torch.rand(n, generator=gen, device=dev, dtype=torch.float64)
        t = (torch.exp(u * math.log(V + 1.0)) - 1.0).floor().long().clamp_(0, V - 1)
    elif case['tokens'] == 'runs':              # regions of a label map: runs of 16 equal labels
        t = torch.randint(V, (n // 16 + 1,), generator=gen, device=dev).repeat_interleave(16)[:n]
    else:
        t = torch.randint(V, (n,), generator=gen, device=dev)
    if case['pad'] >= 0:                        # a padded batch: a tenth of the slots
        t = torch.where(torch.rand(n, generator=gen, device=dev) < 0.1, torch.full_like(t, case['pad']), t)
    return t.to(torch.int32 if case['index'] == 'i32' else torch.int64)


def prepare(case, seed):
    dev = torch.device('cuda')
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    dtype = _TYPES[case['dtype']]
    if case['op'] == 'embed':
        n, V, D = case['n'], case['V'], case['D']
        state = {'idx': _tokens(case, gen, dev), 'table': (normal(V, D) * 0.05).to(dtype).requires_grad_(case['train'])}
        if case['train']:
            state['dout'] = (normal(n, D) * 0.05).to(dtype)
    else:
        N, S, C = case['N'], case['S'], case['C']
        ptype = torch.float32 if case['params'] == 'f32' else dtype
        # channels of a convolution's output: means and widths of their own
        x = normal(N, S, C).mul_(torch.exp(0.3 * normal(C))).add_(normal(C)).to(dtype).requires_grad_(case['train'])
        state = {'x': x, 'weight': None, 'bias': None}
        if case['affine']:
            state['weight'] = (1.0 + 0.2 * normal(C)).to(ptype).requires_grad_(case['train'])
            state['bias'] = (0.2 * normal(C)).to(ptype).requires_grad_(case['train'])
        if case['train']:
            state['dy'] = normal(N, S, C).to(dtype)
    state['case'] = case
    return state


# ------------------------------------------------------------------------------------------------ one pass
def _plain_embed(case, idx, table, dout):
    idx = idx.long()
    result = {'out': (table[idx].float() * case['scale']).to(table.dtype)}
    if dout is not None:
        # rows that very many tokens share are long sums: those in 64 bits
        wide = torch.float64 if case['n'] > 64 * case['V'] else torch.float32
        d = torch.zeros(table.shape, dtype=wide, device=table.device).index_add_(0, idx, dout.to(wide)) * case['scale']
        if case['pad'] >= 0:
            d[case['pad']] = 0
        result['dtable'] = d.to(table.dtype)
    return result


_EPS, _SLOPE = 1e-5, 0.2


def _plain_norm(case, x, weight, bias, dy):
    N, S, C, G = case['N'], case['S'], case['C'], case['G']
    v = x.float().view(N, S, G, C // G)
    mean = v.mean(dim=(1, 3), keepdim=True)
    d = v - mean
    rstd = ((d * d).mean(dim=(1, 3), keepdim=True) + _EPS).rsqrt()
    xhat = (d * rstd).view(N, S, C)
    z = xhat if weight is None else xhat * weight.float() + bias.float()
    if case['act'] == 'silu':
        gate = 1.0 / (1.0 + torch.exp(-z))
        y = z * gate
    else:
        y = torch.where(z > 0, z, z * _SLOPE) if case['act'] == 'lrelu' else z
    result = {'y': y.to(x.dtype)}
    if dy is None:
        return result
    dz = dy.float()
    if case['act'] == 'silu':
        dz = dz * gate * (1.0 + z * (1.0 - gate))
    elif case['act'] == 'lrelu':
        dz = torch.where(z > 0, dz, dz * _SLOPE)
    dxhat = dz if weight is None else dz * weight.float()
    h, e = xhat.view(N, S, G, C // G), dxhat.view(N, S, G, C // G)
    dx = rstd * (e - e.mean(dim=(1, 3), keepdim=True) - h * (e * h).mean(dim=(1, 3), keepdim=True))
    result['dx'] = dx.view(N, S, C).to(x.dtype)
    if weight is not None:
        result['dweight'] = (dz * xhat).sum(dim=(0, 1)).to(weight.dtype)
        result['dbias'] = dz.sum(dim=(0, 1)).to(bias.dtype)
    return result


def run(state):
    case = state['case']
    if case['op'] == 'embed':
        idx, table, dout = state['idx'], state['table'], state.get('dout')
        if not own:
            return _plain_embed(case, idx, table.detach(), dout)
        from ag2video_amd import ops
        out = ops.embedding_scaled(idx, table, scale=case['scale'], padding_idx=case['pad'] if case['pad'] >= 0 else None)
        if dout is None:
            return {'out': out}
        return {'out': out, 'dtable': torch.autograd.grad(out, table, dout)[0]}
    x, weight, bias, dy = state['x'], state['weight'], state['bias'], state.get('dy')
    if not own:
        plain = [None if t is None else t.detach() for t in (x, weight, bias)]
        return _plain_norm(case, *plain, dy)
    from ag2video_amd import ops
    y = ops.group_norm_act(x, case['G'], weight, bias, eps=_EPS, act=case['act'], slope=_SLOPE)
    if dy is None:
        return {'y': y}
    if weight is None:
        return {'y': y, 'dx': torch.autograd.grad(y, x, dy)[0]}
    dx, dw, db = torch.autograd.grad(y, (x, weight, bias), dy)
    return {'y': y, 'dx': dx, 'dweight': dw, 'dbias': db}


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def _distinct(case):
    """Expected number of table rows that the tokens name."""
    n, V = case['n'], case['V']
    if case['tokens'] == 'frequency':
        r = np.arange(V, dtype=np.float64)
        p = np.log((r + 2.0) / (r + 1.0)) / math.log(V + 1.0)
    else:
        p = np.full(V, 1.0 / V)
    draws = n / 16.0 if case['tokens'] == 'runs' else float(n)
    return float(np.minimum(1.0 - np.power(1.0 - np.minimum(p, 1.0), draws), 1.0).sum())


def work(case):
    e = _BYTES[case['dtype']]
    if case['op'] == 'embed':
        n, V, D = case['n'], case['V'], case['D']
        ib = 4 if case['index'] == 'i32' else 8
        bytes_, flops = n * ib + max(1.0, _distinct(case)) * D * e + n * D * e, n * D
        if case['train']:
            bytes_, flops = bytes_ + n * D * e + V * D * e, 2 * n * D + V * D
        return {'bytes': bytes_, 'flops': flops}
    elems = case['N'] * case['S'] * case['C']
    p = (4 if case['params'] == 'f32' else e) * (2 * case['C'] if case['affine'] else 0)
    per = {'none': 6, 'lrelu': 8, 'silu': 10}[case['act']]
    if case['train']:       # the backward pass reads x and dy and writes dx; the forward pass has read x already, once is the floor
        return {'bytes': 4 * elems * e + 2 * p, 'flops': 3 * per * elems}
    return {'bytes': 2 * elems * e + p, 'flops': per * elems}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case['op'] == 'embed':
        table, idx = state['table'].detach().double(), state['idx'].long()
        result = {'out': torch.index_select(table, 0, idx) * case['scale']}
        if case['train']:
            order = torch.argsort(idx, stable=True)
            rows = state['dout'].double()
            g = torch.zeros_like(table)
            g.index_put_((idx[order],), rows[order], accumulate=True)
            keep = torch.arange(case['V'], device=g.device) != case['pad']
            result['dtable'] = g * keep[:, None] * case['scale']
        return result
    N, S, C, G = case['N'], case['S'], case['C'], case['G']
    leaves = [None if state[k] is None else state[k].detach().double().requires_grad_(case['train']) for k in ('x', 'weight', 'bias')]
    x, weight, bias = leaves
    rows = x.reshape(N, S, G, C // G).permute(0, 2, 1, 3).reshape(N * G, -1)
    centred = rows - rows.sum(1, keepdim=True) / rows.shape[1]
    variance = centred.pow(2).sum(1, keepdim=True) / rows.shape[1]
    z = (centred / (variance + _EPS).sqrt()).reshape(N, G, S, C // G).permute(0, 2, 1, 3).reshape(N, S, C)
    if weight is not None:
        z = z * weight + bias
    if case['act'] == 'silu':
        y = z * torch.sigmoid(z)
    elif case['act'] == 'lrelu':
        y = torch.clamp(z, min=0) + _SLOPE * torch.clamp(z, max=0)
    else:
        y = z
    result = {'y': y.detach()}
    if case['train']:
        grads = torch.autograd.grad(y, [t for t in leaves if t is not None], state['dy'].double())
        for name, g in zip(('dx', 'dweight', 'dbias'), grads):
            result[name] = g
    return result
