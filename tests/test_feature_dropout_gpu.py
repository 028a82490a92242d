"""`feature_dropout` of the epoch drivers: the gathered rows with the mask of the batch's own key."""
import numpy as np
import pytest
import torch

import ops_formulas as f
from helpers import rmat_csr

pytestmark = pytest.mark.gpu

STREAM = 0x66656174 << 32


@pytest.fixture(scope="module")
def graph():
    import aethergraph_b200 as ag

    n, off, dst, _ = rmat_csr(11, 8, seed=17)
    return ag.Graph.from_csr(off, dst), np.random.default_rng(5).standard_normal((n, 21)).astype(np.float32)


@pytest.mark.parametrize("kw", [dict(), dict(num_workers=2, group=1), dict(disjoint=True)])
def test_rows_of_a_batch(graph, kw):
    from aethergraph_b200 import _lib
    from aethergraph_b200.pytorch import NeighborLoader
    from aethergraph_b200.pytorch.loader import epoch_sampling_seed

    g, feats = graph
    make = lambda **more: NeighborLoader(g, [5, 3], input_nodes=np.arange(300), batch_size=70, shuffle=False, seed=7,  # noqa: E731
                                         features=feats, **kw, **more)
    plain, dropped, again = make(), make(feature_dropout=0.3), make(feature_dropout=0.3)
    seeds = np.random.SeedSequence(7)
    first = []
    for epoch in range(2):
        key = epoch_sampling_seed(seeds)
        for b, (p, d, e) in enumerate(zip(plain, dropped, again)):
            assert torch.equal(p.n_id, d.n_id) and torch.equal(d.x, e.x)
            x = feats[p.n_id.cpu().numpy()]
            assert np.array_equal(p.x.cpu().numpy(), x)
            m = f.mask(*x.shape, 0.3, _lib.lib().ag_batch_seed(key, b), STREAM)
            # scale and product are rounded once each
            off = (d.x.cpu().double() - torch.from_numpy(x).double() * m).abs()
            assert bool((off <= 2 * 2.0 ** -24 * torch.from_numpy(x).double().abs() * m).all())
            first.append(d.x.cpu())
    half = len(first) // 2
    assert all(a.shape != b.shape or not torch.equal(a == 0, b == 0) for a, b in zip(first[:half], first[half:]))


def test_unseeded_epochs_differ_and_refusals(graph):
    from aethergraph_b200.pytorch import NeighborLoader

    g, feats = graph
    make = lambda **kw: NeighborLoader(g, [4], input_nodes=np.arange(100), batch_size=100, shuffle=False, features=feats, **kw)  # noqa: E731
    loader = make(feature_dropout=0.5)
    (a,), (b,) = list(loader), list(loader)
    k = min(len(a.x), len(b.x), 100)
    assert not torch.equal(a.x[:k] == 0, b.x[:k] == 0)
    for kw in (dict(feature_dropout=1.0), dict(feature_dropout=-0.1), dict(feature_dropout=0.1, neighbor_sampler=lambda g, s: s)):
        with pytest.raises(ValueError, match="feature_dropout"):
            make(**kw)
    with pytest.raises(ValueError, match="feature_dropout"):
        NeighborLoader(g, [4], feature_dropout=0.1)


def test_typed_graph():
    import aethergraph_b200 as ag
    from aethergraph_b200 import _lib
    from aethergraph_b200.pytorch import HeteroNeighborLoader
    from aethergraph_b200.pytorch.loader import epoch_sampling_seed

    rng = np.random.default_rng(3)
    e = lambda n, a, b: (rng.integers(0, a, n).astype(np.uint32), rng.integers(0, b, n).astype(np.uint32))  # noqa: E731
    h = ag.HeteroCsrGraph.from_edge_arrays({"a": 300, "b": 200}, [("a", "to", "b", *e(3000, 300, 200)), ("b", "to", "a", *e(3000, 200, 300))])
    feats = {"a": rng.standard_normal((300, 16)).astype(np.float32), "b": rng.standard_normal((200, 9)).astype(np.float32)}
    make = lambda **kw: HeteroNeighborLoader(h, {("a", "to", "b"): [4, 3], ("b", "to", "a"): [4, 3]}, ("b", np.arange(90)),  # noqa: E731
                                             batch_size=40, shuffle=False, seed=5, features=feats, **kw)
    key = epoch_sampling_seed(np.random.SeedSequence(5))
    for b, (p, d) in enumerate(zip(make(), make(feature_dropout=0.4))):
        for t, nt in enumerate(h.node_types()):
            assert torch.equal(p[nt].n_id, d[nt].n_id)
            m = f.mask(*p[nt].x.shape, 0.4, _lib.lib().ag_batch_seed(key, b), STREAM + t)
            want = p[nt].x.cpu().double() * m
            assert bool(((d[nt].x.cpu().double() - want).abs() <= 2 * 2.0 ** -24 * want.abs()).all())
    with pytest.raises(ValueError, match="feature_dropout"):
        HeteroNeighborLoader(h, {("a", "to", "b"): [4]}, ("b", None), feature_dropout=0.2)
