"""Learned type vectors (libmolgrid_amd/type_vectors.py) on the device against plain 64-bit forms."""
import math

import numpy as np
import pytest
import torch

import type_vector_reference as ref
from type_vector_reference import check, f64

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def mg():
    import libmolgrid_amd
    return libmolgrid_amd


def on_device(t, shifted=False):
    """t on the device; shifted: a contiguous view that starts one element into its memory."""
    if not shifted:
        return t.cuda()
    room = torch.zeros(t.numel() + 1, dtype=t.dtype).cuda()
    room[1:].copy_(t.reshape(-1))
    return room[1:].view(t.shape)


def values(rng, shape, dtype, scale=1.0, shift=0.0):
    return torch.tensor(rng.standard_normal(shape) * scale + shift, dtype=torch.float32).to(dtype)


def indices(rng, shape, rows, kind, frac_ignored=0.1):
    t = rng.integers(0, max(rows, 1), shape)
    off = rng.random(shape) < frac_ignored
    t = np.where(off, rng.choice([-1, rows, rows + 5, -7], shape), t)
    if kind == F32:
        t = t + np.where(rng.random(shape) < 0.3, 0.5, 0.0)       # the whole number below counts
    return torch.tensor(t).to(kind)


# ------------------------------------------------------------------------------------------------
# embedding
# ------------------------------------------------------------------------------------------------
EMBED = [
    # shape of the indices, rows, channels, type, kind of index, a scale per token
    ((1,), 28, 32, F32, F32, False), ((1,), 1, 1, BF16, torch.int64, True),
    ((0,), 5, 8, F32, torch.int32, True), ((7,), 0, 8, F16, torch.int64, False),
    ((64,), 28, 28, F32, F32, True), ((3, 41), 28, 28, F32, F32, False),
    ((130,), 2, 7, F16, torch.int32, True), ((257,), 300, 33, BF16, torch.int64, False),
    ((65,), 1000, 64, BF16, F32, True), ((31,), 77, 1001, F16, torch.int64, False),
    ((40,), 9, 2056, BF16, torch.int32, True), ((9,), 4, 4099, F32, torch.int64, False),
    ((700,), 3, 16, F32, F32, True), ((700,), 513, 5, F16, torch.int32, False),
    ((2500,), 40, 12, BF16, torch.int64, True), ((2100,), 3000, 24, F32, torch.int64, False),
    ((500,), 28, 300, F32, torch.int64, True), ((400,), 20, 1024, BF16, F32, False), ((3000,), 32, 24, F32, F32, True),
]


@pytest.mark.parametrize("shape,rows,channels,dtype,kind,per_token", EMBED)
@pytest.mark.parametrize("shifted", [False, True])
def test_embedding(mg, shape, rows, channels, dtype, kind, per_token, shifted):
    rng = np.random.default_rng(rows + 7 * channels)
    index = indices(rng, shape, rows, kind)
    table = values(rng, (rows, channels), dtype)
    grad = values(rng, shape + (channels,), dtype)
    scale = torch.tensor(rng.uniform(0.5, 1.5, shape), dtype=F32) if per_token else 5.65
    d_scale = on_device(scale, shifted) if per_token else scale
    d_index, d_table, d_grad = (on_device(t, shifted) for t in (index, table, grad))
    at = ref.rows_of(index, rows)
    s = f64(scale).reshape(-1) if per_token else float(np.float32(scale))
    y, d_y = ref.embed(at, f64(table), s)
    got = mg.embed_types(d_index, d_table, d_scale)
    check(got.view(-1, channels), y, d_y, dtype, "vectors")
    assert got.shape == shape + (channels,)
    (dw, d_dw), (ds, d_ds) = ref.embed_backward(at, f64(grad).reshape(-1, channels), f64(table), s)
    to_table, to_scale = mg.embed_types_backward(d_grad, d_index, d_table, d_scale)
    check(to_table, dw, d_dw, dtype, "gradient of the table")
    if per_token:
        check(to_scale.view(-1), ds, d_ds, F32, "gradient of the scale")
    else:
        assert to_scale is None
    again, none = mg.embed_types_backward(d_grad, d_index, d_table, d_scale, scale_gradient=False)
    assert none is None and torch.equal(again, to_table)          # the same bits
    none, only = mg.embed_types_backward(d_grad, d_index, d_table, d_scale, table_gradient=False)
    assert none is None and (only is None or torch.equal(only, to_scale))


@pytest.mark.parametrize("case", ["one row", "nothing", "two rows far apart", "sorted", "reversed"])
@pytest.mark.parametrize("tokens", [5, 64, 1000, 5000])
def test_gradient_of_the_table_for_unusual_orders(mg, case, tokens):
    """Every token on one row, no token on any, only the first and the last row, rising and falling
    indices: the sums of the rows and zeros elsewhere."""
    rows, channels = 1300, 20
    rng = np.random.default_rng(tokens)
    index = {"one row": np.full(tokens, 77), "nothing": np.full(tokens, -1),
             "two rows far apart": np.where(np.arange(tokens) % 3 == 0, 0, rows - 1),
             "sorted": np.sort(rng.integers(0, rows, tokens)),
             "reversed": np.sort(rng.integers(0, rows, tokens))[::-1].copy()}[case]
    grad = values(rng, (tokens, channels), F32)
    index = torch.tensor(index)
    table = torch.zeros((rows, channels))
    (dw, d_dw), _ = ref.embed_backward(index.numpy(), f64(grad), f64(table), 2.0)
    got, _ = mg.embed_types_backward(grad.cuda(), index.cuda(), table.cuda(), 2.0)
    check(got, dw, d_dw, F32, case)


@pytest.mark.parametrize("case", ["one row", "nothing", "even", "uneven", "sorted"])
@pytest.mark.parametrize("tokens,rows", [(32768, 700), (32769, 33), (33000, 511), (40960, 512), (50001, 5000),
                                         (36000, 300000)])
def test_gradient_of_the_table_for_many_tokens(mg, case, tokens, rows):
    """On either side of where the tokens are sorted by digits: one, two and three digits, whole and
    broken tiles, tokens without a row."""
    channels = 3
    rng = np.random.default_rng(tokens)
    index = {"one row": np.full(tokens, rows - 1), "nothing": np.full(tokens, -1),
             "even": rng.integers(0, rows, tokens),
             "uneven": np.minimum(rng.integers(0, rows, tokens), rng.integers(0, rows, tokens) // 50),
             "sorted": np.sort(rng.integers(0, rows, tokens))}[case]
    index[rng.random(tokens) < 0.1] = rows                        # names no row
    grad = values(rng, (tokens, channels), F32)
    (dw, d_dw), _ = ref.embed_backward(np.where(index < rows, index, -1), f64(grad), np.zeros((rows, channels)), 1.0)
    index, table = torch.tensor(index).cuda(), torch.zeros((rows, channels)).cuda()
    got, _ = mg.embed_types_backward(grad.cuda(), index, table)
    check(got, dw, d_dw, F32, case)
    weight = torch.ones(channels).cuda()
    to = mg.encode_types_backward(grad.cuda(), index, table + 1, weight, p=0.5, seed=3)
    at = np.where(index.cpu().numpy() < rows, index.cpu().numpy(), -1)
    for g, expected in zip(to, ref.encode_backward(at, f64(grad), np.ones((rows, channels)), 1.0, np.ones(channels),
                                                   1e-5, 0.5, 3, 0)):
        check(g, *expected, F32, case)


def test_indices_that_name_no_row(mg):
    """Not-a-number, infinities, numbers beyond 32 bits and between the rows; infinities and
    not-a-number in the gradients of tokens without a row stay out of the sums."""
    table = torch.arange(1., 13.).view(4, 3).cuda()
    inf, nan = math.inf, math.nan
    t = torch.tensor([nan, inf, -inf, -0.5, -0.0, 0.99, 3.99, 4.0, 2.0 ** 31, 1e30, 1e-45])
    expected = torch.tensor([-1, -1, -1, -1, 0, 0, 3, -1, -1, -1, 0])
    got = mg.embed_types(t.cuda(), table).cpu()
    for i, row in enumerate(expected.tolist()):
        assert torch.equal(got[i], table[row].cpu() if row >= 0 else torch.zeros(3)), i
    big = torch.tensor([2 ** 31, 2 ** 32 + 1, -2 ** 33, 2 ** 62, 3], dtype=torch.int64)
    got = mg.embed_types(big.cuda(), table).cpu()
    assert torch.equal(got[:4], torch.zeros(4, 3)) and torch.equal(got[4], table[3].cpu())
    grad = torch.ones(11, 3)
    grad[expected < 0] = nan
    dw, ds = mg.embed_types_backward(grad.cuda(), t.cuda(), table, torch.full((11,), 2.0).cuda())
    assert dw.cpu().tolist() == [[6.] * 3, [0.] * 3, [0.] * 3, [2.] * 3]
    assert ds.cpu()[expected < 0].tolist() == [0.] * 7      # (zero times what stands there is not looked at)


# ------------------------------------------------------------------------------------------------
# layer norm
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows", [1, 5, 67, 520])
@pytest.mark.parametrize("channels", [1, 3, 8, 28, 32, 64, 100, 255, 256, 1000, 1001, 2048])
@pytest.mark.parametrize("dtype,param", [(F32, F32), (F16, F32), (BF16, BF16)])
def test_layer_norm(mg, rows, channels, dtype, param):
    _layer_norm(mg, rows, channels, dtype, param, False)


@pytest.mark.parametrize("rows,channels", [(1, 4096), (3, 5000), (2, 8200), (2, 20000), (1, 66000), (2, 16388)])
@pytest.mark.parametrize("dtype,param", [(F32, F32), (F16, F16), (BF16, F32)])
def test_layer_norm_of_wide_rows(mg, rows, channels, dtype, param):
    _layer_norm(mg, rows, channels, dtype, param, False)


@pytest.mark.parametrize("rows,channels", [(5, 7), (9, 64), (4, 2048), (3, 9000)])
@pytest.mark.parametrize("dtype,param", [(F32, F32), (F16, F16), (BF16, F32)])
def test_layer_norm_off_alignment(mg, rows, channels, dtype, param):
    _layer_norm(mg, rows, channels, dtype, param, True)


@pytest.mark.parametrize("rows,channels", [(40000, 4), (9001, 30), (4099, 100)])
def test_layer_norm_of_many_rows(mg, rows, channels):
    _layer_norm(mg, rows, channels, F32, F32, False)


def _layer_norm(mg, rows, channels, dtype, param, shifted):
    rng = np.random.default_rng(rows * 31 + channels)
    x = (values(rng, (rows, channels), F32) * torch.tensor(np.exp(rng.standard_normal(channels)), dtype=F32)
         + torch.tensor(rng.standard_normal(channels), dtype=F32)).to(dtype)
    grad = values(rng, (rows, channels), dtype)
    weight, bias = values(rng, channels, param, 0.2, 1.0), values(rng, channels, param, 0.1)
    d = [on_device(t, shifted) for t in (x, grad, weight, bias)]
    norm = ref.Norm(f64(x), 1e-5)
    got, mean, rstd = mg.layer_norm(d[0], d[2], d[3], 1e-5)
    check(got, *norm.forward(f64(weight), f64(bias)), dtype, "result")
    check(mean, norm.mean[:, 0], norm.d_mean[:, 0], F32, "mean")
    check(rstd, norm.rstd[:, 0], norm.d_rstd[:, 0], F32, "rstd")
    dx, dw, db = norm.backward(f64(grad), f64(weight))
    to_x, to_weight, to_bias = mg.layer_norm_backward(d[1], d[0], mean, rstd, d[2])
    check(to_x, *dx, dtype, "gradient of the input")
    check(to_weight, *dw, param, "gradient of the weight")
    check(to_bias, *db, param, "gradient of the bias")
    only = mg.layer_norm_backward(d[1], d[0], mean, rstd, d[2], param_gradients=False)
    assert torch.equal(only[0], to_x) and only[1:] == (None, None)
    only = mg.layer_norm_backward(d[1], d[0], mean, rstd, d[2], input_gradient=False)
    assert only[0] is None and torch.equal(only[1], to_weight) and torch.equal(only[2], to_bias)
    plain, _, _ = mg.layer_norm(d[0])                             # without parameters
    check(plain, *norm.forward(1.0, 0.0), dtype, "without parameters")
    dx, dw, db = norm.backward(f64(grad), np.ones(channels))
    to_x, to_weight, _ = mg.layer_norm_backward(d[1], d[0], mean, rstd)
    check(to_x, *dx, dtype, "gradient without parameters")
    check(to_weight, *dw, F32, "gradient of absent weights")


def test_layer_norm_of_rows_with_a_large_mean(mg):
    """A mean of 1000 beside a spread of 1: the variance comes from the differences."""
    rng = np.random.default_rng(4)
    x = values(rng, (6, 500), F32, 1.0, 1000.0)
    norm = ref.Norm(f64(x), 1e-5)
    got, _, _ = mg.layer_norm(x.cuda())
    y, d = norm.forward(1.0, 0.0)
    assert d.max() < 0.05                                         # (squares of x would lose all of it)
    check(got, y, d, F32)


def test_layer_norm_of_rows_without_spread(mg):
    """Equal elements: zero, whatever the mean, and a gradient whose mean is taken out."""
    x = torch.full((3, 40), 2.5)
    got, mean, rstd = mg.layer_norm(x.cuda(), eps=1e-5)
    assert not got.any() and torch.all(mean == 2.5)
    check(rstd, np.full(3, 1 / math.sqrt(float(np.float32(1e-5)))), np.full(3, 1e-4), F32)


@pytest.mark.parametrize("channels", [28, 300, 3000])
def test_layer_norm_keeps_what_is_not_finite_in_its_row(mg, channels):
    rng = np.random.default_rng(5)
    x = values(rng, (9, channels), F32)
    clean, _, _ = mg.layer_norm(x.cuda())
    x[2, 5], x[6, 0] = math.inf, math.nan
    got, mean, rstd = mg.layer_norm(x.cuda())
    assert torch.isnan(got[2]).any() and torch.isnan(got[6]).all()
    rest = [0, 1, 3, 4, 5, 7, 8]
    assert torch.equal(got[rest], clean[rest])
    dx, _, _ = mg.layer_norm_backward(torch.ones_like(got), x.cuda(), mean, rstd)
    assert torch.isfinite(dx[rest]).all() and torch.isnan(dx[6]).all()


def test_layer_norm_of_nothing(mg):
    for shape in ((0, 8), (4, 0), (0, 0), (2, 0, 8)):
        x = torch.zeros(shape).cuda()
        y, mean, rstd = mg.layer_norm(x)
        assert y.shape == shape and mean.shape == shape[:-1]
        dx, dw, db = mg.layer_norm_backward(y, x, mean, rstd)
        assert dx.shape == shape and not dw.any() and not db.any() and dw.shape == shape[-1:]


# ------------------------------------------------------------------------------------------------
# dropout
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n", [1, 7, 8, 9, 63, 513, 4100, 70001])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shifted", [False, True])
def test_dropout(mg, n, p, dtype, shifted):
    rng = np.random.default_rng(n)
    x = values(rng, n, dtype)
    seed, offset = 0xFEDCBA9876543210, 2 ** 63 + n
    y, d = ref.dropout(f64(x), p, seed, offset)
    got = mg.dropout(on_device(x, shifted), p, seed, offset)
    check(got, y, d, dtype)
    keep, _ = ref.kept(n, p, seed, offset)
    if n > 4000 and 0 < p < 1:                                    # six standard deviations
        assert abs(keep.mean() - (1 - p)) < 6 * math.sqrt(p * (1 - p) / n)
    nothing = mg.dropout(on_device(x, shifted), p, seed, offset + 1)
    assert p in (0.0, 1.0) or n < 64 or not torch.equal(nothing, got)


def test_dropout_hides_what_it_drops(mg):
    x = torch.full((4096,), math.nan)
    x[::2] = math.inf
    keep, factor = ref.kept(4096, 0.3, 3, 4)
    got = mg.dropout(x.cuda(), 0.3, 3, 4).cpu()
    assert not got[~torch.tensor(keep)].any()
    kept = torch.tensor(keep)
    assert torch.isnan(got[1::2][kept[1::2]]).all() and torch.isinf(got[::2][kept[::2]]).all()
    assert not mg.dropout(x.cuda(), 1.0, 3, 4).any()
    assert mg.dropout(x.cuda(), 2.0 ** -18, 3, 4).isnan().sum() == 2048    # below half of a step of p


def test_dropout_takes_its_numbers_from_a_state(mg):
    x = torch.randn(1003, generator=torch.Generator().manual_seed(1)).cuda()
    for seed, offset in ((5, 9), (2 ** 63 - 1, 0), (-1, -2)):     # int64 bits stand for 64-bit numbers
        state = torch.tensor([seed, offset]).cuda()
        assert torch.equal(mg.dropout(x, 0.25, state=state), mg.dropout(x, 0.25, seed % 2 ** 64, offset % 2 ** 64))


# ------------------------------------------------------------------------------------------------
# the three in one
# ------------------------------------------------------------------------------------------------
ENCODE = [
    ((1,), 28, 32, F32, F32, F32, 0.0), ((6, 50), 28, 32, F32, F32, F32, 0.1),
    ((64,), 28, 28, F32, F32, torch.int32, 0.5), ((300,), 5, 7, F16, F32, torch.int64, 0.1),
    ((33,), 500, 130, BF16, BF16, torch.int64, 0.3), ((20,), 40, 1001, F16, F16, F32, 0.1),
    ((12,), 30, 2048, BF16, F32, torch.int64, 0.1), ((5,), 3, 9001, F32, F32, torch.int32, 0.2),
    ((0,), 4, 8, F32, F32, F32, 0.1), ((5,), 0, 8, F32, F32, F32, 0.1), ((4000,), 28, 8, F32, F32, F32, 0.1),
    ((3000,), 700, 24, BF16, F32, torch.int64, 0.1), ((9,), 2, 1, F32, F32, F32, 1.0),
    ((500,), 28, 300, F32, F32, torch.int64, 0.3), ((400,), 20, 1024, BF16, F32, F32, 0.1),
    ((60,), 20, 8200, F16, F32, torch.int32, 0.1),
]


@pytest.mark.parametrize("shape,rows,channels,dtype,param,kind,p", ENCODE)
@pytest.mark.parametrize("shifted", [False, True])
def test_encoding(mg, shape, rows, channels, dtype, param, kind, p, shifted):
    rng = np.random.default_rng(rows + 7 * channels)
    index = indices(rng, shape, rows, kind)
    table, grad = values(rng, (rows, channels), dtype), values(rng, shape + (channels,), dtype)
    weight, bias = values(rng, channels, param, 0.2, 1.0), values(rng, channels, param, 0.1)
    numbers = dict(scale=1.7, eps=1e-5, p=p, seed=12345678901234567890, offset=77)
    d_index, d_table, d_grad, d_weight, d_bias = (on_device(t, shifted) for t in
                                                  (index, table, grad, weight, bias))
    at = ref.rows_of(index, rows)
    args = (1.7, f64(weight), 1e-5, p, numbers["seed"], 77)
    got = mg.encode_types(d_index, d_table, d_weight, d_bias, **numbers)
    y, d = ref.encode(at, f64(table), 1.7, f64(weight), f64(bias), 1e-5, p, numbers["seed"], 77)
    check(got.view(-1, channels), y, d, dtype, "vectors")
    dt, dw, db = ref.encode_backward(at, f64(grad).reshape(-1, channels), f64(table), *args)
    to = mg.encode_types_backward(d_grad, d_index, d_table, d_weight, **numbers)
    check(to[0], *dt, dtype, "gradient of the table")
    check(to[1], *dw, param, "gradient of the weight")
    check(to[2], *db, param, "gradient of the bias")
    again = mg.encode_types_backward(d_grad, d_index, d_table, d_weight, **numbers)
    assert all(torch.equal(a, b) for a, b in zip(again, to))
    only = mg.encode_types_backward(d_grad, d_index, d_table, d_weight, **numbers, table_gradient=False)
    assert only[0] is None and torch.equal(only[1], to[1]) and torch.equal(only[2], to[2])
    only = mg.encode_types_backward(d_grad, d_index, d_table, d_weight, **numbers, param_gradients=False)
    assert only[1:] == (None, None) and torch.equal(only[0], to[0])
    state = torch.tensor([numbers["seed"] - 2 ** 64, 77]).cuda()
    numbers.update(seed=0, offset=0)
    assert torch.equal(mg.encode_types(d_index, d_table, d_weight, d_bias, **numbers, state=state), got)
    assert torch.equal(mg.encode_types_backward(d_grad, d_index, d_table, d_weight, **numbers, state=state)[0], to[0])


@pytest.mark.parametrize("rows,channels", [(6, 8), (6, 300), (6, 9001), (60, 8), (60, 300), (40, 9001)])
@pytest.mark.parametrize("tokens", [0, 3, 500])
def test_rows_without_tokens_have_no_part(mg, rows, channels, tokens):
    """Infinities, not-a-number and rows without spread (eps 0) in rows that no token names: zeros in
    their own gradient, nothing in the others'."""
    rng = np.random.default_rng(rows + channels)
    index = torch.tensor(rng.integers(0, 3, tokens))
    table, grad = values(rng, (rows, channels), F32), values(rng, (tokens, channels), F32)
    weight = values(rng, channels, F32, 0.2, 1.0)
    args = (1.5, f64(weight), 0.0, 0.25, 7, 8)
    expected = ref.encode_backward(index.numpy(), f64(grad), f64(table[:3]), *args)
    table[3], table[4], table[5:] = math.nan, math.inf, 0.5
    got = mg.encode_types_backward(grad.cuda(), index.cuda(), table.cuda(), weight.cuda(), scale=1.5, eps=0.0,
                                   p=0.25, seed=7, offset=8)
    assert not got[0][3:].any()
    for g, (value, bound) in zip((got[0][:3], got[1], got[2]), expected):
        check(g, value, bound, F32)
    y = mg.encode_types(index.cuda(), table.cuda(), weight.cuda(), scale=1.5, eps=0.0)
    assert torch.isfinite(y).all()


def test_encoding_is_its_parts_one_after_the_other(mg):
    """float32, where the parts round nothing away: within the bounds of the one pass, twice."""
    rng = np.random.default_rng(8)
    index, table = indices(rng, (50, 30), 28, F32), values(rng, (28, 32), F32)
    weight, bias = values(rng, 32, F32, 0.2, 1.0), values(rng, 32, F32, 0.1)
    d_index, d_table, d_weight, d_bias = (t.cuda() for t in (index, table, weight, bias))
    one = mg.encode_types(d_index, d_table, d_weight, d_bias, scale=1.7, p=0.2, seed=5, offset=6)
    x = mg.embed_types(d_index, d_table, 1.7)
    named = torch.tensor(ref.rows_of(index, 28) >= 0).view(50, 30, 1)
    parts = mg.dropout(mg.layer_norm(x, d_weight, d_bias)[0], 0.2, 5, 6).cpu() * named
    at = ref.rows_of(index, 28)
    _, d = ref.encode(at, f64(table), 1.7, f64(weight), f64(bias), 1e-5, 0.2, 5, 6)
    assert np.all(np.abs(f64(one) - f64(parts)).reshape(-1, 32) <= 2.1 * d)


# ------------------------------------------------------------------------------------------------
# autograd, modules and the grids behind them
# ------------------------------------------------------------------------------------------------
def test_modules_give_the_functions_gradients(mg):
    rng = np.random.default_rng(9)
    index = indices(rng, (4, 21), 28, F32).cuda()
    embedding, norm = mg.TypeEmbedding(28, 24, scale=2.0).cuda(), mg.TypeNorm(24).cuda()
    drop = mg.TypeDropout(0.25, seed=11)
    scale = torch.tensor(rng.uniform(0.5, 1.5, (4, 21)), dtype=F32).cuda().requires_grad_()
    up = values(rng, (24, 4, 21), F32).cuda().permute(1, 2, 0)    # a gradient that is not contiguous
    x = embedding(index, scale)
    z = drop(norm(x))
    z.backward(up)
    up = up.contiguous()
    y, mean, rstd = mg.layer_norm(x.detach(), norm.weight.detach(), norm.bias.detach())
    assert torch.equal(z.detach(), mg.dropout(y, 0.25, 11, 0))
    g = mg.dropout(up, 0.25, 11, 0)
    dx, dw, db = mg.layer_norm_backward(g, x.detach(), mean, rstd, norm.weight.detach())
    dt, ds = mg.embed_types_backward(dx, index, embedding.weight.detach(), scale.detach())
    for got, expected in ((norm.weight.grad, dw), (norm.bias.grad, db), (embedding.weight.grad, dt),
                          (scale.grad, ds)):
        assert torch.equal(got, expected)
    assert torch.equal(embedding(index).detach(), mg.embed_types(index, embedding.weight.detach(), 2.0))
    assert not torch.equal(drop(x.detach()), mg.dropout(x.detach(), 0.25, 11, 0))    # the next offset
    drop.eval()
    assert drop(x) is x


def test_encoder_module(mg):
    rng = np.random.default_rng(10)
    index = indices(rng, (70,), 28, torch.int64).cuda()
    encoder = mg.TypeEncoder(28, 16, scale=4.0, p=0.2, seed=3).cuda()
    up = values(rng, (70, 16), F32).cuda()
    for call in range(2):
        encoder.zero_grad()
        y = encoder(index)
        y.backward(up)
        table, w, b = (t.detach() for t in (encoder.weight, encoder.norm_weight, encoder.norm_bias))
        numbers = dict(scale=4.0, p=0.2, seed=3, offset=call)
        assert torch.equal(y.detach(), mg.encode_types(index, table, w, b, **numbers))
        for got, expected in zip((encoder.weight, encoder.norm_weight, encoder.norm_bias),
                                 mg.encode_types_backward(up, index, table, w, **numbers)):
            assert torch.equal(got.grad, expected)
    encoder.eval()
    assert torch.equal(encoder(index).detach(), mg.encode_types(index, table, w, b, scale=4.0))
    y = encoder(index).sum()
    (g,) = torch.autograd.grad(y, encoder.norm_bias, create_graph=True)
    with pytest.raises(RuntimeError):                             # no second derivative, said so
        g.sum().backward()
    mg.set_random_seed(5)
    first = mg.TypeDropout(0.5).seed
    mg.set_random_seed(5)
    assert first == mg.TypeDropout(0.5).seed != mg.TypeDropout(0.5).seed


def _atoms(rng, shape, ntypes):
    coords = torch.tensor(rng.uniform(-3, 3, shape + (3,)), dtype=F32).cuda()
    types = torch.tensor(rng.integers(0, ntypes, shape), dtype=F32).cuda()
    radii = torch.tensor(rng.uniform(1.2, 2.0, shape), dtype=F32).cuda()
    return coords, types, radii


@pytest.mark.parametrize("batched", [False, True])
def test_grids_of_learned_types(mg, batched):
    """Coords2Grid with a type encoder is Coords2Grid on the encoder's vectors, gradients included;
    a table of one-hot rows gives the grids of the index types."""
    rng = np.random.default_rng(12)
    gmaker = mg.GridMaker(0.5, 5.5)
    coords, types, radii = _atoms(rng, (3, 14) if batched else (14,), 6)
    if batched:
        types[1, 9:], radii[1, 9:] = 0, 0                         # padding as the datasets' collate makes it
    encoder = mg.TypeEncoder(6, 8, p=0.1, seed=4).cuda()
    layer = mg.Coords2Grid(gmaker, (0, 0, 0), type_encoder=encoder)
    assert dict(layer.named_parameters()).keys() == {"type_encoder.weight", "type_encoder.norm_weight",
                                                     "type_encoder.norm_bias"}
    coords.requires_grad_()
    grid = layer(coords, types, radii)
    up = torch.tensor(rng.standard_normal(tuple(grid.shape)), dtype=F32).cuda()
    grid.backward(up)
    c2 = coords.detach().clone().requires_grad_()
    w, nw, nb = (t.detach() for t in (encoder.weight, encoder.norm_weight, encoder.norm_bias))
    vectors = mg.encode_types(types, w, nw, nb, p=0.1, seed=4, offset=0).requires_grad_()
    plain = mg.Coords2Grid(gmaker, (0, 0, 0))(c2, vectors, radii)
    plain.backward(up)
    assert torch.equal(grid, plain) and torch.equal(coords.grad, c2.grad)
    expected = mg.encode_types_backward(vectors.grad, types, w, nw, p=0.1, seed=4, offset=0)
    for got, e in zip((encoder.weight, encoder.norm_weight, encoder.norm_bias), expected):
        assert torch.equal(got.grad, e)
    one_hot = mg.TypeEmbedding(6, 6).cuda()
    with torch.no_grad():
        one_hot.weight.copy_(torch.eye(6))
        grid = mg.Coords2Grid(gmaker, (0, 0, 0), one_hot)(coords, types, radii)
        vectors = torch.nn.functional.one_hot(types.long().cpu(), 6).float().cuda()
        assert torch.equal(grid, mg.Coords2Grid(gmaker, (0, 0, 0))(coords, vectors, radii))


def test_bfloat16_encoder_feeds_the_grids(mg):
    rng = np.random.default_rng(13)
    coords, types, radii = _atoms(rng, (20,), 28)
    encoder = mg.TypeEncoder(28, 16, dtype=BF16, norm_dtype=F32).cuda()
    grid = mg.Coords2Grid(mg.GridMaker(0.5, 5.5), (0, 0, 0), encoder)(coords, types, radii)
    grid.sum().backward()
    assert grid.dtype == F32 and encoder.weight.grad.dtype == BF16
    assert torch.isfinite(encoder.weight.grad).all() and encoder.norm_weight.grad.dtype == F32


def test_gradients_against_differences(mg):
    """The layer's gradients against central differences of its own grids (float32 grids, a step of
    2^-6: rounding of the sum over the grid and the third derivative stay below a hundredth)."""
    rng = np.random.default_rng(14)
    gmaker = mg.GridMaker(1.0, 5.0)
    coords, types, radii = _atoms(rng, (9,), 4)
    encoder = mg.TypeEncoder(4, 5).cuda()
    with torch.no_grad():
        encoder.weight.copy_(torch.tensor(rng.standard_normal((4, 5)), dtype=F32))
    layer = mg.Coords2Grid(gmaker, (0, 0, 0), encoder)
    up = torch.tensor(rng.standard_normal((5, 6, 6, 6))).cuda()

    def loss():
        return float((layer(coords, types, radii).double() * up).sum())

    layer(coords, types, radii).backward(up.float())
    for parameter in (encoder.weight, encoder.norm_weight, encoder.norm_bias):
        flat, step = parameter.data.view(-1), 2.0 ** -6
        size = float(parameter.grad.abs().max())
        for i in range(0, flat.numel(), 3):
            keep = float(flat[i])
            flat[i] = keep + step
            high = loss()
            flat[i] = keep - step
            low = loss()
            flat[i] = keep
            assert abs((high - low) / (2 * step) - float(parameter.grad.view(-1)[i])) < 1e-2 * size


def test_host_arrays_are_staged(mg):
    rng = np.random.default_rng(15)
    index, table = indices(rng, (12,), 9, F32), values(rng, (9, 6), F32)
    x = values(rng, (12, 6), F32)
    got = mg.embed_types(index, table, 3.0)
    assert not got.is_cuda and torch.equal(got, mg.embed_types(index.cuda(), table.cuda(), 3.0).cpu())
    assert torch.equal(mg.embed_types(index.numpy(), table.numpy(), 3.0), got)
    assert torch.equal(mg.layer_norm(x)[0], mg.layer_norm(x.cuda())[0].cpu())
    encoder = mg.TypeEncoder(9, 6)
    encoder(index).sum().backward()
    assert encoder.weight.grad is not None and not encoder.weight.grad.is_cuda
    managed = mg.MGrid1f(12)
    managed.copyFrom(index.numpy())
    assert torch.equal(mg.embed_types(managed, table, 3.0), got)


def test_refusals(mg):
    t, w = torch.zeros(4).cuda(), torch.zeros((5, 6)).cuda()
    x = torch.zeros((4, 6)).cuda()
    m = torch.zeros(4).cuda()
    bad = [
        lambda: mg.embed_types(t.double(), w), lambda: mg.embed_types(t, w.double()),
        lambda: mg.embed_types(t, w[0]), lambda: mg.embed_types(t, w.t()), lambda: mg.embed_types(t, w.cpu()),
        lambda: mg.embed_types(t, w, torch.ones(3).cuda()), lambda: mg.embed_types(t, w, torch.ones(4).double().cuda()),
        lambda: mg.embed_types(t, w, torch.tensor(2.0).cuda()), lambda: mg.embed_types(t, w, torch.ones((4, 1)).cuda()),
        lambda: mg.encode_types(t, w, scale=torch.ones(4).cuda()),
        lambda: mg.encode_types_backward(x, t, w, scale=torch.tensor(1.0).cuda()),
        lambda: mg.embed_types_backward(x.half(), t, w), lambda: mg.embed_types_backward(x[:3], t, w),
        lambda: mg.embed_types_backward(x[:, ::2], t, w),
        lambda: mg.layer_norm(x, m), lambda: mg.layer_norm(x, w[0].half()), lambda: mg.layer_norm(x.double()),
        lambda: mg.layer_norm(x[:, ::2]), lambda: mg.layer_norm(x, eps=-1.0), lambda: mg.layer_norm(x, eps=math.nan),
        lambda: mg.layer_norm(x.half(), w[0], w[0].half()), lambda: mg.layer_norm(torch.tensor(1.0).cuda()),
        lambda: mg.layer_norm_backward(x, x, m[:3], m), lambda: mg.layer_norm_backward(x, x, m, m.double()),
        lambda: mg.layer_norm_backward(x.half(), x, m, m),
        lambda: mg.dropout(x, -0.1), lambda: mg.dropout(x, 1.1), lambda: mg.dropout(x, math.nan),
        lambda: mg.dropout(x, 0.1, -1), lambda: mg.dropout(x, 0.1, 2 ** 64), lambda: mg.dropout(x, 0.1, 0, 2 ** 64),
        lambda: mg.dropout(x.t(), 0.1), lambda: mg.dropout(x, 0.1, state=m), lambda: mg.dropout(x.double(), 0.1),
        lambda: mg.dropout(x, 0.1, state=torch.zeros(2, dtype=torch.int64)),
        lambda: mg.encode_types(t, w, m), lambda: mg.encode_types(t, w, p=2.0), lambda: mg.encode_types(t, w, eps=-1.0),
        lambda: mg.encode_types_backward(x.half(), t, w), lambda: mg.TypeDropout(1.5), lambda: mg.TypeEncoder(4, 4, p=-1),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail("call %d was not refused" % i)


# ------------------------------------------------------------------------------------------------
# streams and graphs
# ------------------------------------------------------------------------------------------------
def test_two_streams_at_once(mg):
    """Calls that overlap on two streams have nothing in common."""
    rng = np.random.default_rng(16)
    index, table = indices(rng, (3000,), 500, torch.int64).cuda(), values(rng, (500, 64), F32).cuda()
    grads = [values(rng, (3000, 64), F32).cuda() for _ in range(2)]
    weight = torch.ones(64).cuda()
    expected = [mg.encode_types_backward(g, index, table, weight, p=0.1, seed=1) for g in grads]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(4):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(mg.encode_types_backward(grads[k], index, table, weight, p=0.1, seed=1))
    torch.cuda.synchronize()
    for k in range(2):
        for r in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(r, expected[k]))


def test_captured_step(mg):
    """A training step of the encoder and the grids behind it, captured and replayed with other
    random numbers and inputs, against the same step run eagerly; eager work in between."""
    rng = np.random.default_rng(17)
    gmaker = mg.GridMaker(0.5, 5.5)
    coords, types, radii = _atoms(rng, (2, 40), 28)
    state = torch.tensor([7, 0]).cuda()
    encoder = mg.TypeEncoder(28, 8, p=0.2, seed=1, state=state).cuda()
    layer = mg.Coords2Grid(gmaker, (0, 0, 0), encoder)
    up = torch.tensor(rng.standard_normal((2, 8, 12, 12, 12)), dtype=F32).cuda()
    parameters = list(encoder.parameters())

    def step():
        return torch.autograd.grad(layer(coords, types, radii), parameters, up)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for replay in range(4):
        types.copy_(torch.tensor(rng.integers(0, 28, (2, 40)), dtype=F32).cuda())
        state[1] = replay
        graph.replay()
        got = [g.clone() for g in captured]
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b), replay
    encoder.state = None
    with pytest.raises(RuntimeError):                             # a mask that would repeat itself
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            encoder(types)
    torch.cuda.synchronize()


def test_state_changed_before_the_backward_pass_is_noticed(mg):
    state = torch.tensor([7, 0]).cuda()
    encoder = mg.TypeEncoder(28, 8, p=0.2, state=state).cuda()
    y = encoder(torch.zeros(5).cuda())
    state[1] += 1
    with pytest.raises(RuntimeError):
        y.sum().backward()
