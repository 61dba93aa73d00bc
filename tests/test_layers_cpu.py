"""Modules of models/layers.py without a device."""
import pickle

import torch


def test_an_embedding_pickled_without_a_scale(monkeypatch):
    """A module pickled whole before layers.Embedding had a scale looks up as it did."""
    from ag2video_amd import ops
    from ag2video_amd.models.layers import Embedding
    emb = Embedding(5, 4)
    emb.__dict__.pop('scale')
    emb = pickle.loads(pickle.dumps(emb))
    assert 'scale' not in emb.__dict__
    monkeypatch.setattr(ops, 'embedding', lambda idx, table: table[idx])
    idx = torch.tensor([3, 0])
    assert torch.equal(emb(idx), emb.weight[idx])
    again = pickle.loads(pickle.dumps(Embedding(5, 4, scale=2.0)))
    assert again.scale == 2.0
