"""TEST INFRASTRUCTURE: the kernels of learned type vectors on the emulated device, through the C ABI
on arrays that end at an inaccessible page, against the plain 64-bit forms of
tests/type_vector_reference.py; sizes, types and kinds of indices are drawn.
    python tests/emu/type_vectors.py [rounds] [seed]"""
import os
import sys

import numpy as np
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)
sys.path.insert(0, os.path.dirname(HERE))

import emu_capi as e  # noqa: E402
import type_vector_reference as ref  # noqa: E402
from type_vector_reference import check, f64  # noqa: E402

TYPES = [torch.float32, torch.float16, torch.bfloat16]
KINDS = [torch.float32, torch.int32, torch.int64]
STORED = {torch.float32: np.float32, torch.float16: np.uint16, torch.bfloat16: np.uint16,
          torch.int32: np.int32, torch.int64: np.int64}
SHIFT = 0                        # elements that arrays start behind their block's first one


def stored(t):
    return t.contiguous().view(torch.int16).numpy().view(np.uint16) if t.element_size() == 2 else t.numpy()


def place(shape, dtype, fill=None):
    """Array of `dtype` in guarded memory that ends where its block ends, or SHIFT elements before."""
    n = int(np.prod(shape))
    a = e.array((n + SHIFT,), STORED[dtype])
    a = (a[SHIFT:] if SHIFT else a).reshape(shape)
    if fill is not None:
        a[...] = fill
    return a


def put(t):
    return place(tuple(t.shape), t.dtype, stored(t))


def back(a, dtype):
    t = torch.from_numpy(np.array(a).view(np.int16) if a.dtype == np.uint16 else np.array(a))
    return t.view(dtype) if t.dtype != dtype else t


def ok(code):
    assert code == 0, code


def workspace(size):
    """Bytes that hold something else than zeros, aligned to 256, with a guard behind them."""
    if not size:
        return None, 0
    w = e.array(((size + 255) // 256 * 256,), np.uint8, fill=0xA5, tight=False)
    return w.ctypes.data, size


def values(rng, shape, dtype, scale=1.0, shift=0.0):
    return torch.tensor(rng.standard_normal(shape) * scale + shift, dtype=torch.float32).to(dtype)


def drawn_size(rng, most):
    return int(round(np.exp(rng.uniform(0, np.log(most)))))


def tokens_case(rng):
    tokens, rows = drawn_size(rng, 3000), drawn_size(rng, 1500)
    channels = drawn_size(rng, max(2, min(1500, 150000 // max(tokens, rows))))
    if rng.random() < 0.5:
        channels = max(8, channels // 8 * 8)
    if rng.random() < 0.08:                                        # sorted by digits
        tokens, rows, channels = int(rng.integers(32769, 45000)), drawn_size(rng, 3000) + 32, int(rng.integers(1, 5))
    dtype, kind = TYPES[rng.integers(3)], KINDS[rng.integers(3)]
    t = rng.integers(0, rows, tokens)
    how = rng.integers(4)
    if how == 0:                                                   # most tokens on few rows
        t = np.minimum(t, rng.integers(0, rows, tokens) // max(1, rows // 3))
    elif how == 1:
        t = np.sort(t)
    t = np.where(rng.random(tokens) < 0.1, rng.choice([-1, rows, rows + 3], tokens), t)
    return tokens, rows, channels, dtype, kind, torch.tensor(t).to(kind)


def embed(rng):
    tokens, rows, channels, dtype, kind, index = tokens_case(rng)
    table, grad = values(rng, (rows, channels), dtype), values(rng, (tokens, channels), dtype)
    per_token = rng.random() < 0.5
    scale = torch.tensor(rng.uniform(0.5, 1.5, tokens), dtype=torch.float32) if per_token else None
    number = 1.75
    a_index, a_table, a_grad = put(index), put(table), put(grad)
    a_scale = put(scale) if per_token else None
    head = (tokens, rows, channels, TYPES.index(dtype), KINDS.index(kind), e.ptr(a_index))
    out = place((tokens, channels), dtype)
    ok(e.lib.mg_embed_types(*head, e.ptr(a_table), number, e.ptr(a_scale), e.ptr(out), None))
    at = ref.rows_of(index, rows)
    s = f64(scale) if per_token else number
    check(back(out, dtype), *ref.embed(at, f64(table), s), dtype, "vectors")
    to_table = place((rows, channels), dtype)
    to_scale = place((tokens,), torch.float32) if per_token else None
    w, size = workspace(e.lib.mg_embed_types_backward_workspace_size(tokens, rows, channels))
    ok(e.lib.mg_embed_types_backward(*head, e.ptr(a_grad), e.ptr(a_table), number, e.ptr(a_scale),
                                     e.ptr(to_table), e.ptr(to_scale), w, size, None))
    dw, ds = ref.embed_backward(at, f64(grad), f64(table), s)
    check(back(to_table, dtype), *dw, dtype, "gradient of the table")
    if per_token:
        check(back(to_scale, torch.float32), *ds, torch.float32, "gradient of the scale")
    return "embed %s %s %d tokens %d rows %d channels" % (dtype, kind, tokens, rows, channels)


def norm(rng):
    rows = drawn_size(rng, 1500)
    channels = drawn_size(rng, max(2, min(9000, 150000 // rows)))
    if rng.random() < 0.5:
        channels = max(8, channels // 8 * 8)
    dtype = TYPES[rng.integers(3)]
    param = dtype if rng.random() < 0.5 else torch.float32
    x, grad = values(rng, (rows, channels), dtype, 2.0, 0.5), values(rng, (rows, channels), dtype)
    weight, bias = values(rng, channels, param, 0.2, 1.0), values(rng, channels, param, 0.1)
    a_x, a_grad, a_weight, a_bias = put(x), put(grad), put(weight), put(bias)
    if rng.random() < 0.2:
        a_weight, weight = None, torch.ones(channels, dtype=param)
    head = (rows, channels, TYPES.index(dtype), TYPES.index(param))
    out = place((rows, channels), dtype)
    mean, rstd = (place((rows,), torch.float32) for _ in range(2))
    ok(e.lib.mg_layer_norm(*head, e.ptr(a_x), e.ptr(a_weight), e.ptr(a_bias), 1e-5, e.ptr(out),
                           e.ptr(mean), e.ptr(rstd), None))
    n = ref.Norm(f64(x), 1e-5)
    check(back(out, dtype), *n.forward(f64(weight), f64(bias)), dtype, "normed")
    check(back(mean, torch.float32), n.mean[:, 0], n.d_mean[:, 0], torch.float32, "mean")
    check(back(rstd, torch.float32), n.rstd[:, 0], n.d_rstd[:, 0], torch.float32, "rstd")
    over = put(x)                                                  # in place
    ok(e.lib.mg_layer_norm(*head, e.ptr(over), e.ptr(a_weight), e.ptr(a_bias), 1e-5, e.ptr(over), None, None, None))
    assert np.array_equal(over, out)
    to_x = place((rows, channels), dtype)
    to_weight, to_bias = (place((channels,), param) for _ in range(2))
    w, size = workspace(e.lib.mg_layer_norm_backward_workspace_size(rows, channels))
    ok(e.lib.mg_layer_norm_backward(*head, e.ptr(a_grad), e.ptr(a_x), e.ptr(mean), e.ptr(rstd),
                                    e.ptr(a_weight), e.ptr(to_x), e.ptr(to_weight), e.ptr(to_bias), w,
                                    size, None))
    dx, dw, db = n.backward(f64(grad), f64(weight))
    check(back(to_x, dtype), *dx, dtype, "gradient of the input")
    check(back(to_weight, param), *dw, param, "gradient of the weight")
    check(back(to_bias, param), *db, param, "gradient of the bias")
    return "norm %s %s %d rows %d channels" % (dtype, param, rows, channels)


def dropout(rng):
    n, dtype = drawn_size(rng, 30000), TYPES[rng.integers(3)]
    p, seed, offset = float(rng.random()), int(rng.integers(2 ** 62)) * 4 + 3, int(rng.integers(2 ** 62))
    x = values(rng, n, dtype)
    a, out = put(x), place((n,), dtype)
    ok(e.lib.mg_dropout(n, TYPES.index(dtype), e.ptr(a), p, seed, offset, None, e.ptr(out), None))
    check(back(out, dtype), *ref.dropout(f64(x), p, seed, offset), dtype, "dropped")
    ok(e.lib.mg_dropout(n, TYPES.index(dtype), e.ptr(a), p, seed, offset, None, e.ptr(a), None))
    assert np.array_equal(a, out)                                  # in place
    return "dropout %s %d" % (dtype, n)


def encode(rng):
    tokens, rows, channels, dtype, kind, index = tokens_case(rng)
    param = dtype if rng.random() < 0.5 else torch.float32
    table, grad = values(rng, (rows, channels), dtype), values(rng, (tokens, channels), dtype)
    weight, bias = values(rng, channels, param, 0.2, 1.0), values(rng, channels, param, 0.1)
    p, seed, offset = float(rng.choice([0.0, 0.1, 0.6])), int(rng.integers(2 ** 62)), int(rng.integers(100))
    a_index, a_table, a_grad, a_weight, a_bias = (put(t) for t in (index, table, grad, weight, bias))
    head = (tokens, rows, channels, TYPES.index(dtype), TYPES.index(param), KINDS.index(kind), e.ptr(a_index))
    out = place((tokens, channels), dtype)
    ok(e.lib.mg_encode_types(*head, e.ptr(a_table), 1.5, e.ptr(a_weight), e.ptr(a_bias), 1e-5, p, seed,
                             offset, None, e.ptr(out), None))
    at = ref.rows_of(index, rows)
    check(back(out, dtype), *ref.encode(at, f64(table), 1.5, f64(weight), f64(bias), 1e-5, p, seed, offset),
          dtype, "vectors")
    to_table = place((rows, channels), dtype)
    to_weight, to_bias = (place((channels,), param) for _ in range(2))
    w, size = workspace(e.lib.mg_encode_types_backward_workspace_size(tokens, rows, channels))
    ok(e.lib.mg_encode_types_backward(*head, e.ptr(a_grad), e.ptr(a_table), 1.5, e.ptr(a_weight), 1e-5, p,
                                      seed, offset, None, e.ptr(to_table), e.ptr(to_weight), e.ptr(to_bias),
                                      w, size, None))
    dt, dw, db = ref.encode_backward(at, f64(grad), f64(table), 1.5, f64(weight), 1e-5, p, seed, offset)
    check(back(to_table, dtype), *dt, dtype, "gradient of the table")
    check(back(to_weight, param), *dw, param, "gradient of the weight")
    check(back(to_bias, param), *db, param, "gradient of the bias")
    return "encode %s %s %d tokens %d rows %d channels" % (dtype, kind, tokens, rows, channels)


def main(rounds, seed):
    global SHIFT
    rng = np.random.default_rng(seed)
    for r in range(rounds):
        for fn in (embed, norm, dropout, encode):
            SHIFT = int(rng.choice([0, 0, 1, 2, 3, 4]))
            state = rng.bit_generator.state["state"]["state"]
            try:
                said = fn(rng)
            except AssertionError as problem:
                print("round %d, %s, shift %d, state %d: %s" % (r, fn.__name__, SHIFT, state, problem))
                return 1
            if "-v" in sys.argv:
                print(said, "shift", SHIFT, flush=True)
            e.release_all()
    print("%d rounds passed" % rounds)
    return 0


if __name__ == "__main__":
    numbers = [int(a) for a in sys.argv[1:] if a.lstrip("-").isdigit()]
    sys.exit(main(numbers[0] if numbers else 20, numbers[1] if len(numbers) > 1 else 1))
