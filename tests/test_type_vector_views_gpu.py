"""Grid views and managed grids stand for their tensors in the type vectors' calls, whichever argument they are."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mg():
    import libmolgrid_amd
    return libmolgrid_amd


def same(got, expected):
    got, expected = ([r] if isinstance(r, torch.Tensor) else list(r) for r in (got, expected))
    assert len(got) == len(expected)
    for a, b in zip(got, expected):
        assert (a is None and b is None) or (a.is_cuda and torch.equal(a, b))


@pytest.mark.parametrize("managed", [False, True])
def test_views_behind_a_device_tensor(mg, managed):
    g = torch.Generator().manual_seed(3)

    def random(*shape):
        return torch.randn(shape, generator=g).cuda()

    def view(t):
        if not managed:
            return (mg.Grid1fCUDA if t.dim() == 1 else mg.Grid2fCUDA)(t)
        m = (mg.MGrid1f if t.dim() == 1 else mg.MGrid2f)(*t.shape)
        m.copyFrom(t)
        m.gpu()
        return m

    index = torch.tensor([0.0, 2.0, 1.0, -1.0, 2.0]).cuda()
    table, x, grad, scales = random(3, 6), random(5, 6), random(5, 6), random(5)
    weight, bias = random(6), random(6)
    same(mg.embed_types(index, view(table), view(scales)), mg.embed_types(index, table, scales))
    same(mg.embed_types(index, table, scale=view(scales)), mg.embed_types(index, table, scales))
    same(mg.embed_types_backward(grad, view(index), view(table), view(scales)),
         mg.embed_types_backward(grad, index, table, scales))
    same(mg.layer_norm(x, view(weight), view(bias)), mg.layer_norm(x, weight, bias))
    _, mean, rstd = mg.layer_norm(x)
    same(mg.layer_norm_backward(grad, view(x), view(mean), view(rstd), view(weight)),
         mg.layer_norm_backward(grad, x, mean, rstd, weight))
    numbers = dict(scale=1.5, p=0.25, seed=3)
    same(mg.encode_types(index, table, view(weight), bias=view(bias), **numbers),
         mg.encode_types(index, table, weight, bias, **numbers))
    same(mg.encode_types_backward(grad, view(index), view(table), view(weight), **numbers),
         mg.encode_types_backward(grad, index, table, weight, **numbers))
    same(mg.dropout(view(x), 0.25, 3), mg.dropout(x, 0.25, 3))
    refused = [lambda: mg.layer_norm(x, view(random(7))), lambda: mg.layer_norm_backward(grad, x, view(random(4)), rstd),
               lambda: mg.embed_types(index, table, view(random(4))), lambda: mg.encode_types(index, table, scale=view(scales)),
               lambda: mg.dropout(x, 0.25, state=view(random(2)))]
    for i, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
            pytest.fail("call %d was not refused" % i)
