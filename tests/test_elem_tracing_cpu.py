"""The operators of embedding_scaled and group_norm_act as torch's dispatcher sees them, without a device."""
import pytest
import torch


def _fake():
    from torch._subclasses.fake_tensor import FakeTensorMode
    return FakeTensorMode(allow_non_fake_inputs=True)


def test_shapes_alone():
    from ag2video_amd import ops
    with _fake():
        idx = torch.zeros(3, 5, dtype=torch.int32, device='cuda')
        table = torch.zeros(7, 8, device='cuda', dtype=torch.float16)
        y = ops.embedding_scaled(idx, table, 2.0, 1)
        assert y.shape == (3, 5, 8) and y.dtype == torch.float16 and y.device.type == 'cuda' and not y.requires_grad
        assert ops.embedding_scaled(idx, table.requires_grad_(True)).requires_grad
        x = torch.zeros(2, 12, 9, 4, device='cuda').permute(0, 2, 3, 1)
        y = ops.group_norm_act(x, 3, torch.ones(12, device='cuda'))
        assert y.shape == x.shape and y.is_contiguous()
        for call in (lambda: ops.embedding_scaled(idx.float(), table), lambda: ops.embedding_scaled(idx, table, 1.0, 7), lambda: ops.embedding_scaled(idx, table, 1.0, -1),
                     lambda: ops.group_norm_act(x, 5), lambda: ops.group_norm_act(x, 3, torch.ones(4, device='cuda')), lambda: ops.group_norm_act(x, 3, act='relu')):
            with pytest.raises(RuntimeError):
                call()


def test_a_graph_holds_the_operators():
    from torch.fx.experimental.proxy_tensor import make_fx
    from ag2video_amd import ops
    with _fake():
        idx, table = torch.zeros(9, dtype=torch.long, device='cuda'), torch.zeros(7, 8, device='cuda')
        graph = make_fx(lambda i, t: ops.group_norm_act(ops.embedding_scaled(i, t, 2.0, 1).view(1, 9, 8), 2))(idx, table)
    names = [str(node.target) for node in graph.graph.nodes]
    assert 'ag2v.embedding_scaled.default' in names and 'ag2v.group_norm_act.default' in names, names


def test_a_dual_is_refused():
    import torch.autograd.forward_ad as fwad
    from ag2video_amd import ops
    with _fake(), fwad.dual_level():
        idx, table = torch.zeros(9, dtype=torch.long, device='cuda'), torch.zeros(7, 8, device='cuda')
        x, w = torch.zeros(2, 9, 8, device='cuda'), torch.ones(8, device='cuda')
        dual = [fwad.make_dual(t, torch.ones_like(t)) for t in (table, x, w)]
        for call in (lambda: ops.embedding_scaled(idx, dual[0]), lambda: ops.group_norm_act(dual[1], 2), lambda: ops.group_norm_act(x, 2, dual[2]),
                     lambda: ops.group_norm_act(x, 2, None, dual[2])):
            with pytest.raises(RuntimeError, match='forward-mode'):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match='forward-mode'):
                call()
