"""The random numbers that the type vectors' modules take, call by call: which calls have to agree
(a call that activation checkpointing runs again, a module saved and loaded) and which have to
differ.  The host layer alone: the mask comes from the plain form, so no device is needed."""
import copy
import io

import numpy as np
import pytest
import torch
from torch.utils.checkpoint import checkpoint

import type_vector_reference as ref


@pytest.fixture
def mg(monkeypatch):
    import libmolgrid_amd
    from libmolgrid_amd import type_vectors

    def dropout(x, p, seed=0, offset=0, state=None):
        if state is not None:
            seed, offset = ((int(n) + m) % 2 ** 64 for n, m in zip(state, (seed, offset)))
        keep, factor = ref.kept(x.numel(), p, seed, offset)
        mask = torch.from_numpy(keep.reshape(tuple(x.shape)))
        return torch.where(mask, x * factor, torch.zeros((), dtype=x.dtype))

    def encode_types(type_index, table, weight, bias, scale, eps, p, seed, offset, state=None):
        return dropout(scale * table[type_index.long()], p, seed, offset, state)

    def encode_types_backward(grad, type_index, table, weight, scale, eps, p, seed, offset, state,
                              table_gradient, param_gradients):
        g = dropout(grad, p, seed, offset, state) * scale
        return torch.zeros_like(table).index_add_(0, type_index.long(), g), torch.zeros_like(weight), \
            torch.zeros_like(weight)

    monkeypatch.setattr(type_vectors, "dropout", dropout)
    monkeypatch.setattr(type_vectors, "encode_types", encode_types)
    monkeypatch.setattr(type_vectors, "encode_types_backward", encode_types_backward)
    return libmolgrid_amd


def _inputs(n=64):
    g = torch.Generator().manual_seed(3)
    x, w = (torch.randn(n, generator=g).requires_grad_() for _ in range(2))
    return x, w


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_repeated_call_drops_the_same_elements(mg, reentrant):
    """Two checkpointed stretches with two calls each: gradients of everything behind the dropped
    elements are those of the output's own masks (elements are kept or not, so a gradient of another
    mask is off by whole elements)."""
    x, w = _inputs()
    drops = [mg.TypeDropout(0.5), mg.TypeDropout(0.5)]
    seen = []

    def stretch(t):
        for drop in drops:
            t = drop(t)
            seen.append(t.detach() != 0)
            t = t * w
        return t

    y = checkpoint(stretch, x, use_reentrant=reentrant)
    y = checkpoint(stretch, y, use_reentrant=reentrant)
    masks = list(seen)
    assert len(masks) == 4
    y.sum().backward()
    assert len(seen) == 8
    # every call dropped as its repetition did (the stretches are repeated last to first)
    for first, again in zip(masks, seen[6:] + seen[4:6]):
        assert torch.equal(first, again)
    keep = torch.ones(x.shape, dtype=torch.bool)
    for m in masks:
        keep &= m
    kept, xd, wd = keep.double() * 2 ** 4, x.detach().double(), w.detach().double()
    # y = 16 kept x w^4
    for got, expected in ((x.grad, kept * wd ** 4), (w.grad, 4 * kept * xd * wd ** 3)):
        assert torch.allclose(got.double(), expected, rtol=16 * 2.0 ** -24, atol=0)


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_repeated_encoder_drops_the_same_elements(mg, reentrant):
    encoder = mg.TypeEncoder(5, 16, p=0.5)
    index, w = torch.arange(12) % 5, torch.randn(12, 16).requires_grad_()
    seen = []

    def stretch(w):
        y = encoder(index)
        seen.append(y.detach() != 0)
        return y * w

    checkpoint(stretch, w, use_reentrant=reentrant).sum().backward()
    assert torch.equal(seen[0], seen[1])
    vectors = 2.0 * seen[0] * encoder.weight.detach()[index]
    assert torch.equal(w.grad, vectors)
    expected = torch.zeros_like(encoder.weight).index_add_(0, index, 2.0 * seen[0] * w.detach())
    assert torch.equal(encoder.weight.grad, expected)


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_counted_call_is_not_repeated_under_another_number(mg, reentrant):
    """With a seed the offset is a count, which a repetition would move on: it is refused, and the
    caller says which call it is."""
    x, w = _inputs()
    drop = mg.TypeDropout(0.5, seed=4)
    y = checkpoint(lambda t: drop(t) * w, x, use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match="offset"):
        y.sum().backward()
    w.grad = x.grad = None
    y = checkpoint(lambda t: drop(t, offset=7) * w, x, use_reentrant=reentrant)
    y.sum().backward()
    keep, _ = ref.kept(x.numel(), 0.5, 4, 7)
    assert np.array_equal(y.detach().numpy() != 0, keep)
    assert torch.equal(w.grad, torch.from_numpy(2.0 * keep).float() * x.detach())
    assert torch.equal(x.grad, torch.from_numpy(2.0 * keep).float() * w.detach())


def test_calls_differ_and_a_seed_counts(mg):
    x, _ = _inputs(4096)
    drop = mg.TypeDropout(0.5)
    torch.manual_seed(1)
    a, b = drop(x), drop(x)
    torch.manual_seed(1)
    assert not torch.equal(a, b) and torch.equal(drop(x), a) and torch.equal(drop(x), b)
    drop = mg.TypeDropout(0.5, seed=9)
    assert drop.offset == 0
    for call in range(3):
        assert np.array_equal(drop(x).detach().numpy() != 0, ref.kept(4096, 0.5, 9, call)[0])
    before = torch.get_rng_state()
    drop(x), drop(x, offset=5), mg.TypeDropout(0.0)(x), mg.TypeDropout(0.5).eval()(x)
    assert torch.equal(before, torch.get_rng_state())           # nothing drawn that is not needed
    assert drop.offset == 4


@pytest.mark.parametrize("seed", [None, 6])
def test_replicas_move_the_module_on(mg, seed):
    """Replicas are made anew for every step (as DataParallel makes them): their calls count."""
    x, _ = _inputs(4096)
    drop = mg.TypeDropout(0.5, seed=seed)
    steps = [drop._replicate_for_data_parallel()(x) for _ in range(3)]
    for i in range(3):
        for j in range(i):
            assert not torch.equal(steps[i], steps[j])


def test_copies_count_for_themselves(mg):
    x, _ = _inputs(4096)
    drop = mg.TypeDropout(0.5, seed=6)
    drop(x)
    copied = copy.deepcopy(drop)
    assert torch.equal(copied(x), drop(x))
    copied(x)
    assert (copied.offset, drop.offset) == (3, 2)


@pytest.mark.parametrize("seed", [0, 5, 2 ** 63, 2 ** 64 - 1])
def test_a_loaded_module_goes_on_where_the_saved_one_was(mg, seed):
    x, _ = _inputs(4096)
    drop = mg.TypeDropout(0.5, seed=seed)
    drop(x), drop(x)
    file = io.BytesIO()
    torch.save(torch.nn.Sequential(drop).state_dict(), file)
    file.seek(0)
    resumed = mg.TypeDropout(0.5, seed=1)
    torch.nn.Sequential(resumed).load_state_dict(torch.load(file, weights_only=True))
    assert (resumed.seed, resumed.offset) == (seed, 2)
    assert torch.equal(resumed(x), drop(x))
    for bad in (-1, 2 ** 64):
        with pytest.raises(ValueError):
            mg.TypeDropout(0.5, seed=bad)


def test_a_state_dict_without_numbers_is_loaded(mg):
    encoder = mg.TypeEncoder(5, 8, p=0.5, seed=3)
    saved = {k: v for k, v in encoder.state_dict().items() if not k.endswith("_extra_state")}
    assert len(saved) == 3
    other = mg.TypeEncoder(5, 8, p=0.5, seed=4)
    other.load_state_dict(saved)
    assert other.seed == 4 and torch.equal(other.weight, encoder.weight)
    with pytest.raises(RuntimeError):
        other.load_state_dict({k: v for k, v in saved.items() if k != "norm_bias"})


def test_modules_that_share_a_state_drop_other_elements(mg):
    """A state is added to the module's own numbers, whether the seed was given or drawn, and to the offset
    that a call is given."""
    x, _ = _inputs(4096)
    state = torch.tensor([100, -1])
    drops = [mg.TypeDropout(0.5, seed=3, state=state), mg.TypeDropout(0.5, seed=4, state=state),
             mg.TypeDropout(0.5, state=state), mg.TypeDropout(0.5, state=state)]
    masks = [drop(x).detach() != 0 for drop in drops] + [drops[0](x, offset=1).detach() != 0]
    for i, mask in enumerate(masks):
        assert all(not torch.equal(mask, other) for other in masks[:i])
    assert np.array_equal(masks[0].numpy(), ref.kept(4096, 0.5, 103, 2 ** 64 - 1)[0])
    assert np.array_equal(masks[4].numpy(), ref.kept(4096, 0.5, 103, 0)[0])
    for drop, mask in zip(drops, masks):                        # the same numbers: the same elements
        assert torch.equal(drop(x).detach() != 0, mask)
