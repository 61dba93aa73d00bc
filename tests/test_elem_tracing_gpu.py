"""embedding_scaled and group_norm_act under what watches a program at torch's dispatcher: traces, dispatch modes, vmap, forward-mode duals."""
import types
import warnings

import pytest
import torch

pytestmark = pytest.mark.gpu


def _randn(*shape, seed, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to('cuda')


def _embed(idx, table):
    from ag2video_amd import ops
    return ops.embedding_scaled(idx, table, 2.0, 3)


def _norm(x, w, b):
    from ag2video_amd import ops
    return ops.group_norm_act(x, 4, w, b, act='lrelu', slope=0.1)


def _no_weight(x, b):
    from ag2video_amd import ops
    return ops.group_norm_act(x, 2, None, b)


def _module(idx, table):
    from ag2video_amd.models.layers import Embedding
    return Embedding.forward(types.SimpleNamespace(scale=None, padding_idx=3, weight=table), idx)


def _inputs(fn, seed, grad=False):
    """Inputs of `fn`; other shapes of the same rank for another seed."""
    n = 5 + seed
    if fn in (_embed, _module):
        idx = torch.randint(11, (3, n), generator=torch.Generator().manual_seed(seed)).cuda()
        return (idx, _randn(11, 24, seed=seed).requires_grad_(grad))
    x = _randn(2, 7 * n, 24, seed=seed, dtype=torch.bfloat16).requires_grad_(grad)
    p = (_randn(24, seed=seed + 1).requires_grad_(grad), _randn(24, seed=seed + 2).requires_grad_(grad))
    return (x,) + (p if fn is _norm else p[:1])


CALLS = [_embed, _norm, _no_weight, _module]


def _grads(y, inputs, seed=9):
    leaves = [t for t in inputs if t.requires_grad]
    return torch.autograd.grad(y, leaves, _randn(*y.shape, seed=seed, dtype=y.dtype))


@pytest.mark.parametrize("grad", [False, True], ids=['values', 'tape'])
@pytest.mark.parametrize("fn", CALLS)
def test_traced_functions(fn, grad, device):
    """torch.jit.trace records the operator: new inputs of another size give what the function gives, forward and backward."""
    with warnings.catch_warnings():
        warnings.simplefilter('ignore')
        traced = torch.jit.trace(fn, _inputs(fn, 0, grad))
    for seed in (0, 1, 2):
        a, b = _inputs(fn, seed, grad), _inputs(fn, seed, grad)
        junk = [torch.full_like(t, 7) for t in a]              # (what an empty result may find in memory)
        del junk
        want, got = fn(*a), traced(*b)
        assert torch.equal(want, got)
        if grad:
            assert all(torch.equal(p, q) for p, q in zip(_grads(want, a), _grads(got, b)))


@pytest.mark.parametrize("fn", CALLS)
def test_graphs_of_dispatch_modes(fn, device):
    """make_fx records the operators of the forward and of the backward pass."""
    from torch.fx.experimental.proxy_tensor import make_fx

    def both(dy, *inputs):
        y = fn(*inputs)
        return (y,) + torch.autograd.grad(y, [t for t in inputs if t.requires_grad], dy)

    first = _inputs(fn, 0, True)
    y = fn(*first)
    graph = make_fx(both)(_randn(*y.shape, seed=7, dtype=y.dtype), *first)
    names = [str(node.target) for node in graph.graph.nodes]
    assert any(n.startswith('ag2v.') and n.endswith('_backward.default') for n in names), names
    other = [t if t.dtype == torch.long else (t.detach() * 0.5 + 1).requires_grad_(True) for t in first]
    dy = _randn(*y.shape, seed=8, dtype=y.dtype)
    for p, q in zip(both(dy, *other), graph(dy, *other)):
        assert torch.equal(p, q)


@pytest.mark.parametrize("fn", CALLS)
def test_shapes_alone(fn, device):
    """Fake tensors: the results' shapes, types and device, forward and backward, and nothing runs."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    real = _inputs(fn, 1, True)
    want = fn(*real)
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        fake = [mode.from_tensor(t) for t in real]
        y = fn(*fake)
        assert (y.shape, y.dtype, y.device) == (want.shape, want.dtype, want.device)
        leaves = [t for t in fake if t.requires_grad]
        for g, t in zip(torch.autograd.grad(y, leaves, torch.ones_like(y)), leaves):
            assert g.shape == t.shape and g.dtype == t.dtype


@pytest.mark.parametrize("backend", ['eager', 'aot_eager'])
@pytest.mark.parametrize("fn", [_embed, _norm, _no_weight])
def test_compiled_functions(fn, backend, device):
    compiled = torch.compile(fn, backend=backend)
    for seed in (0, 1):
        a, b = _inputs(fn, seed, True), _inputs(fn, seed, True)
        want, got = fn(*a), compiled(*b)
        assert torch.equal(want, got)
        assert all(torch.equal(p, q) for p, q in zip(_grads(want, a), _grads(got, b)))


@pytest.mark.parametrize("fn", CALLS)
def test_forward_mode_is_refused(fn, device):
    """A dual input has no tangent here: an error, with a tape and without, and not a result without a tangent."""
    import torch.autograd.forward_ad as fwad
    for grad in (False, True):
        inputs = _inputs(fn, 0, grad)
        for k, t in enumerate(inputs):
            if not t.is_floating_point():
                continue
            with fwad.dual_level():
                dual = list(inputs)
                dual[k] = fwad.make_dual(t, torch.ones_like(t))
                with pytest.raises(RuntimeError):
                    fn(*dual)
                with torch.no_grad(), pytest.raises(RuntimeError):
                    fn(*dual)
            assert fn(*inputs).shape                           # and outside nothing is refused
    inputs = _inputs(fn, 0)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: fn(*inputs[:-1], t), (inputs[-1],), (torch.ones_like(inputs[-1]),))


@pytest.mark.parametrize("fn", [_embed, _norm, _no_weight])
def test_function_transforms(fn, device):
    """vmap and func.grad: the right result or an error, never a wrong one."""
    sets = [_inputs(fn, 0), [t if t.dtype == torch.long else t * 0.5 for t in _inputs(fn, 0)]]
    batch = [torch.stack(ts) for ts in zip(*sets)]
    try:
        with warnings.catch_warnings():
            warnings.simplefilter('ignore')
            got = torch.vmap(fn)(*batch)
    except RuntimeError:
        got = None
    assert got is None or torch.equal(got, torch.stack([fn(*s) for s in sets]))
    last = len(batch) - 1
    try:
        got = torch.func.grad(lambda *a: fn(*a).float().sum(), last)(*sets[0])
    except RuntimeError:
        got = None
    leaf = [t.detach().clone() for t in sets[0]]
    leaf[last].requires_grad_(True)
    want = torch.autograd.grad(fn(*leaf).float().sum(), leaf[last])[0]
    assert got is None or torch.equal(got, want)
    # several output gradients at once
    y = fn(*leaf)
    many = torch.stack([torch.ones_like(y), 2 * torch.ones_like(y)])
    one = [torch.autograd.grad(y, leaf[last], m, retain_graph=True)[0] for m in many]
    try:
        with warnings.catch_warnings():
            warnings.simplefilter('ignore')
            got = torch.autograd.grad(y, leaf[last], many, is_grads_batched=True)[0]
    except RuntimeError:
        got = None
    assert got is None or torch.equal(got, torch.stack(one))


def test_recorded_operators_refuse_what_the_functions_refuse(device):
    """A trace may be called with other tensors than it was made with: the operators themselves check them."""
    from ag2video_amd import _lib
    _lib.elem_ops()
    op = torch.ops.ag2v
    idx, table = torch.zeros(3, 2, dtype=torch.long, device=device), torch.zeros(4, 8, device=device)
    dout, x = torch.zeros(3, 2, 8, device=device), torch.zeros(2, 3, 8, device=device)
    w, stats = torch.ones(8, device=device), torch.ones(2, 2, 2, device=device)
    every = [True, True, True]
    ok = [(op.embedding_scaled, (idx, table, 1.0, -1)), (op.embedding_scaled_backward, (dout, idx, 4, 1.0, -1)), (op.group_norm_act, (x, 2, w, None, 1e-5, 1, 0.2)),
          (op.group_norm_act_backward, (x, x, w, None, stats, 1, 0.2, every))]
    for fn, args in ok:
        fn(*args)
    bad = [
        (op.embedding_scaled, [(idx.float(), table, 1.0, -1), (idx.cpu(), table, 1.0, -1), (idx, table.cpu(), 1.0, -1), (idx, table.double(), 1.0, -1),
                               (idx, table[0], 1.0, -1), (idx, table[:0], 1.0, -1), (idx, table, 1.0, 4), (idx, table, 1.0, -2)]),
        (op.embedding_scaled_backward, [(dout[:2], idx, 4, 1.0, -1), (dout, idx, 0, 1.0, -1), (dout, idx.int().short(), 4, 1.0, -1), (dout.cpu(), idx, 4, 1.0, -1),
                                        (dout.double(), idx, 4, 1.0, -1), (dout, idx, 4, 1.0, 4), (dout[0], idx, 4, 1.0, -1), (dout, idx, 1 << 31, 1.0, -1)]),
        (op.group_norm_act, [(x.double(), 2, w, None, 1e-5, 1, 0.2), (x, 3, w, None, 1e-5, 1, 0.2), (x, 2, w[:7], None, 1e-5, 1, 0.2), (x, 2, w, None, 1e-5, 3, 0.2),
                             (x, 2, w, None, -1.0, 1, 0.2), (x, 2, w.cpu(), None, 1e-5, 1, 0.2), (x, 0, w, None, 1e-5, 1, 0.2), (x.cpu(), 2, None, None, 1e-5, 1, 0.2)]),
        (op.group_norm_act_backward, [(x[:1], x, w, None, stats, 1, 0.2, every), (x.half(), x, w, None, stats, 1, 0.2, every), (x, x, w, None, stats[:1], 1, 0.2, every),
                                      (x, x, w, None, stats.double(), 1, 0.2, every), (x, x, w, None, stats[:, :1], 1, 0.2, every),
                                      (x, x, w, None, stats.transpose(0, 2), 1, 0.2, every), (x, x, w, None, stats, 5, 0.2, every),
                                      (x.cpu(), x, w, None, stats, 1, 0.2, every), (x, x, w[:4], None, stats, 1, 0.2, every)]),
    ]
    for fn, calls in bad:
        for k, args in enumerate(calls):
            with pytest.raises((RuntimeError, NotImplementedError)):
                fn(*args)
                pytest.fail('%s %d was not refused' % (fn, k))


@pytest.mark.parametrize("fn", CALLS)
def test_modes_of_torch(fn, device):
    """inference_mode, autocast, checkpoints of either kind, and a saved trace: the plain call's bits."""
    import io
    from torch.utils.checkpoint import checkpoint
    plain = _inputs(fn, 1, True)
    want = fn(*plain)
    grads = _grads(want, plain)
    with torch.inference_mode():
        assert torch.equal(fn(*_inputs(fn, 1)), want)
    with torch.autocast('cuda', torch.bfloat16):
        assert torch.equal(fn(*_inputs(fn, 1)), want)
    for reentrant in (False, True):
        again = _inputs(fn, 1, True)
        y = checkpoint(fn, *again, use_reentrant=reentrant)
        assert torch.equal(y, want)
        leaves = [t for t in again if t.requires_grad]
        y.backward(_randn(*y.shape, seed=9, dtype=y.dtype))
        assert all(torch.equal(t.grad, g) for t, g in zip(leaves, grads))
    with warnings.catch_warnings():
        warnings.simplefilter('ignore')
        buffer = io.BytesIO()
        torch.jit.save(torch.jit.trace(fn, _inputs(fn, 0)), buffer)
        buffer.seek(0)
        assert torch.equal(torch.jit.load(buffer)(*_inputs(fn, 1)), want)
