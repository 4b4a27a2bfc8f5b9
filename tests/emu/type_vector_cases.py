"""TEST INFRASTRUCTURE: fixed cases of the type vectors' kernels on the emulated device, by name, with the
helpers of type_vectors.py.
    python tests/emu/type_vector_cases.py name ..."""
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

import type_vectors as tv  # noqa: E402
from type_vectors import KINDS, TYPES, back, check, e, f64, ok, place, put, ref, values, workspace  # noqa: E402


def numbers_beside_a_state():
    """seed and offset are added to a state's, modulo 2^64."""
    rng = np.random.default_rng(2)
    n, rows, channels = 515, 40, 9
    x, index = values(rng, n * channels, torch.float32), torch.arange(n) % rows
    table, weight = values(rng, (rows, channels), torch.float32), torch.ones(channels)
    grad = values(rng, (n, channels), torch.float32)
    for seed, offset, state in ((3, 4, (5, 9)), (2 ** 64 - 2, 2 ** 63, (7, 2 ** 63 + 1)), (0, 0, (8, 1))):
        a_state = e.array((2,), np.uint64)
        a_state[...] = state
        both = [(a + b) % 2 ** 64 for a, b in zip((seed, offset), state)]
        a, out = put(x), place((n * channels,), torch.float32)
        ok(e.lib.mg_dropout(n * channels, 0, e.ptr(a), 0.4, seed, offset, e.ptr(a_state), e.ptr(out), None))
        check(back(out, torch.float32), *ref.dropout(f64(x), 0.4, *both), torch.float32, "dropped")
        a_index, a_table, a_weight, a_grad = (put(t) for t in (index, table, weight, grad))
        head = (n, rows, channels, 0, 0, KINDS.index(torch.int64), e.ptr(a_index))
        out = place((n, channels), torch.float32)
        ok(e.lib.mg_encode_types(*head, e.ptr(a_table), 1.5, None, None, 1e-5, 0.4, seed, offset, e.ptr(a_state),
                                 e.ptr(out), None))
        ones, zeros = np.ones(channels), np.zeros(channels)
        check(back(out, torch.float32), *ref.encode(f64(index).astype(int), f64(table), 1.5, ones, zeros, 1e-5, 0.4, *both),
              torch.float32, "vectors")
        to_table = place((rows, channels), torch.float32)
        w, size = workspace(e.lib.mg_encode_types_backward_workspace_size(n, rows, channels))
        ok(e.lib.mg_encode_types_backward(*head, e.ptr(a_grad), e.ptr(a_table), 1.5, None, 1e-5, 0.4, seed, offset,
                                          e.ptr(a_state), e.ptr(to_table), None, None, w, size, None))
        dt, _, _ = ref.encode_backward(f64(index).astype(int), f64(grad), f64(table), 1.5, ones, 1e-5, 0.4, *both)
        check(back(to_table, torch.float32), *dt, torch.float32, "gradient of the table")


def many_tiles():
    """Tokens of more tiles than the digit sort reads the counts of one by one, the last one ragged, two passes of
    digits: whole numbers, so the sums are exact in any order."""
    rng = np.random.default_rng(4)
    tokens, rows = 129 * 4096 + 77, 600
    at = rng.integers(-1, rows + 1, tokens)
    at[:40000] = 3                                                # (a row that fills tiles)
    grad = rng.integers(-8, 9, (tokens, 1)).astype(np.float32)
    index, a_grad = put(torch.tensor(at, dtype=torch.int32)), e.put(grad)
    to_table = place((rows, 1), torch.float32)
    w, size = workspace(e.lib.mg_embed_types_backward_workspace_size(tokens, rows, 1))
    ok(e.lib.mg_embed_types_backward(tokens, rows, 1, 0, KINDS.index(torch.int32), e.ptr(index), e.ptr(a_grad), None, 1.0,
                                     None, e.ptr(to_table), None, w, size, None))
    named = (at >= 0) & (at < rows)
    expected = np.bincount(at[named], grad[named, 0].astype(np.float64), rows)
    assert np.array_equal(to_table[:, 0], expected)


def digest():
    """Prints digests of the gradients that both sources compute with products and sums: layer norm's of its input (whose
    forward pass has no product that could be fused), and an encoder's of its table by sorted tokens."""
    import hashlib
    rng = np.random.default_rng(3)
    rows, channels = 60, 96
    a_x, a_grad = (put(values(rng, (rows, channels), torch.float32, 2.0, 0.7)) for _ in range(2))
    a_weight, index = put(values(rng, channels, torch.float32)), put(torch.arange(rows))
    a_mean, a_rstd = put(values(rng, rows, torch.float32)), put(values(rng, rows, torch.float32, 0.1, 1.0))
    to_x, to_table = (place((rows, channels), torch.float32) for _ in range(2))
    ok(e.lib.mg_layer_norm_backward(rows, channels, 0, 0, e.ptr(a_grad), e.ptr(a_x), e.ptr(a_mean), e.ptr(a_rstd),
                                    e.ptr(a_weight), e.ptr(to_x), None, None, None, 0, None))
    w, size = workspace(e.lib.mg_encode_types_backward_workspace_size(rows, rows, channels))
    ok(e.lib.mg_encode_types_backward(rows, rows, channels, 0, 0, KINDS.index(torch.int64), e.ptr(index), e.ptr(a_grad),
                                      e.ptr(a_x), 1.3, e.ptr(a_weight), 1e-5, 0.0, 0, 0, None, e.ptr(to_table), None,
                                      None, w, size, None))
    for what, a in (("layer_norm", to_x), ("embed", to_table)):
        print(what, hashlib.sha256(np.ascontiguousarray(a).tobytes()).hexdigest())


if __name__ == "__main__":
    for name in sys.argv[1:]:
        globals()[name]()
        e.release_all()
        print(name, "passed", flush=True)
