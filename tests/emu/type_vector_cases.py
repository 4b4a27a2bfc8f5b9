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


if __name__ == "__main__":
    for name in sys.argv[1:]:
        globals()[name]()
        e.release_all()
        print(name, "passed", flush=True)
