"""The type vectors' modules on the device under activation checkpointing."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

import type_vector_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mg():
    import libmolgrid_amd
    return libmolgrid_amd


@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpointed_grids_of_learned_types(mg, reentrant):
    """A checkpointed layer with an encoder and a dropout behind it gives the bits of the same layer that keeps
    everything, under the same numbers."""
    g = torch.Generator().manual_seed(5)
    coords = (torch.rand((2, 30, 3), generator=g) * 6 - 3).cuda()
    types = torch.randint(0, 6, (2, 30), generator=g).float().cuda()
    radii = (torch.rand((2, 30), generator=g) + 1.0).cuda()
    encoder, drop = mg.TypeEncoder(6, 8, p=0.3).cuda(), mg.TypeDropout(0.5)
    layer = mg.Coords2Grid(mg.GridMaker(0.5, 5.5), (0, 0, 0), encoder)
    w = torch.randn((2, 8, 12, 12, 12), generator=g).cuda().requires_grad_()
    coords.requires_grad_()
    leaves = [coords, w] + list(encoder.parameters())

    def stretch(coords):
        return drop(layer(coords, types, radii)) * w

    results = []
    for run in (lambda c: checkpoint(stretch, c, use_reentrant=reentrant), stretch):
        for leaf in leaves:
            leaf.grad = None
        torch.manual_seed(8)
        y = run(coords)
        y.sum().backward()
        results.append([y.detach()] + [leaf.grad for leaf in leaves])
    for got, expected in zip(*results):
        assert torch.equal(got, expected)
    assert 0.3 < float((results[0][0] == 0).float().mean())


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_counted_call_says_which_it_is(mg, reentrant):
    g = torch.Generator().manual_seed(6)
    x, w = (torch.randn(3001, generator=g).cuda().requires_grad_() for _ in range(2))
    drop = mg.TypeDropout(0.5, seed=4)
    with pytest.raises(RuntimeError, match="offset"):
        checkpoint(lambda t: drop(t) * w, x, use_reentrant=reentrant).sum().backward()
    w.grad = x.grad = None
    checkpoint(lambda t: drop(t, offset=7) * w, x, use_reentrant=reentrant).sum().backward()
    keep = torch.from_numpy(ref.kept(3001, 0.5, 4, 7)[0] * 2.0).float().cuda()
    assert torch.equal(w.grad, keep * x.detach()) and torch.equal(x.grad, keep * w.detach())


def test_modules_that_share_a_state_in_one_graph(mg):
    """Two modules and a second call of one of them, captured together: masks of their own in every replay, those
    of the plain form for seed and offset with the state added."""
    x = torch.ones(4099).cuda()
    state = torch.tensor([0, 0]).cuda()
    first, second = mg.TypeDropout(0.5, seed=2 ** 64 - 5, state=state), mg.TypeDropout(0.25, seed=2, state=state)
    calls = ((first, None, 2 ** 64 - 5, 0.5), (second, None, 2, 0.25), (first, 6, 2 ** 64 - 5, 0.5))
    for module, offset, _, _ in calls:      # (loads the kernels before the capture)
        module(x, offset=offset)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outputs = [module(x, offset=offset) for module, offset, _, _ in calls]
    for replay in range(4):
        state.copy_(torch.tensor([100 * replay + 11, -replay]).cuda())
        graph.replay()
        torch.cuda.synchronize()
        for out, (module, offset, seed, p) in zip(outputs, calls):
            keep, factor = ref.kept(4099, p, (seed + 100 * replay + 11) % 2 ** 64, ((offset or 0) - replay) % 2 ** 64)
            assert torch.equal(out.cpu(), torch.from_numpy(keep * factor).float()), replay
            assert torch.equal(out, module(x, offset=offset)), replay
