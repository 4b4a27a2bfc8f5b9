"""Calls whose workgroups go round: more tokens or rows than the launches have workgroups for, so that a team takes a
second one; and the encoder of a small table either side of the number of tokens that norms it once a workgroup."""
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


def inputs(tokens, rows, channels, dtype):
    rng = np.random.default_rng(tokens + channels)
    at = rng.integers(-1, rows + 1, tokens)
    table, grad = (torch.tensor(rng.standard_normal((n, channels)), dtype=F32).to(dtype) for n in (rows, tokens))
    weight, bias = (torch.tensor(rng.uniform(0.5, 1.5, channels), dtype=F32) for _ in range(2))
    return torch.tensor(at), table, grad, weight, bias


@pytest.mark.parametrize("tokens,rows,channels,dtype", [
    (9000, 50, 130, BF16),        # embed: a wave a token, more tokens than waves
    (40000, 3, 5, F16),           # several tokens a team
])
def test_embed(mg, tokens, rows, channels, dtype):
    index, table, grad, _, _ = inputs(tokens, rows, channels, dtype)
    at = ref.rows_of(index, rows)
    check(mg.embed_types(index.cuda(), table.cuda(), 1.5), *ref.embed(at, f64(table), 1.5), dtype, "vectors")
    to_table, _ = mg.embed_types_backward(grad.cuda(), index.cuda(), table.cuda(), 1.5)
    check(to_table, *ref.embed_backward(at, f64(grad), f64(table), 1.5)[0], dtype, "gradient of the table")


@pytest.mark.parametrize("tokens,rows,channels,dtype", [
    # a small table normed once a workgroup, more elements than the launch has lanes for (a position is then carried
    # from channels to tokens), and either side of the rule
    (80000, 28, 28, F32), (20000, 2, 130, BF16), (20000, 28, 7, BF16), (19999, 28, 7, BF16), (50000, 32, 8, F16),
    (49999, 32, 8, F16), (50000, 33, 4, F32), (29999, 33, 3, F32), (30000, 33, 3, F32), (50000, 1, 72, BF16),
    (300, 1, 8192, F32), (300, 2, 4096, BF16), (300, 2, 1001, F16), (300, 1, 8191, F32),
    (2600, 2500, 1001, F16),      # more rows than teams of four waves
])
def test_encode(mg, tokens, rows, channels, dtype):
    index, table, _, weight, bias = inputs(tokens, rows, channels, dtype)
    at = ref.rows_of(index, rows)
    got = mg.encode_types(index.cuda(), table.cuda(), weight.cuda(), bias.cuda(), 1.5, p=0.25, seed=9, offset=4)
    check(got, *ref.encode(at, f64(table), 1.5, f64(weight), f64(bias), 1e-5, 0.25, 9, 4), dtype, "vectors")


@pytest.mark.parametrize("tokens,rows,channels,dtype", [
    (300, 1100, 2048, BF16), (300, 1100, 1500, F32),    # more rows than workgroups of four waves
])
def test_encode_backward(mg, tokens, rows, channels, dtype):
    index, table, grad, weight, _ = inputs(tokens, rows, channels, dtype)
    at = ref.rows_of(index, rows)
    got = mg.encode_types_backward(grad.cuda(), index.cuda(), table.cuda(), weight.cuda(), 1.5, p=0.25, seed=9, offset=4)
    expected = ref.encode_backward(at, f64(grad), f64(table), 1.5, f64(weight), 1e-5, 0.25, 9, 4)
    for g, (value, bound), t, what in zip(got, expected, (dtype, F32, F32), ("table", "weight", "bias")):
        check(g, value, bound, t, "gradient of the " + what)


def test_time_of_a_few_wide_rows(mg):
    """The encoder is not beyond three times its parts called one after the other (a third of them on the card that this
    was written on; beyond five times them where eight lanes norm the row in every workgroup)."""
    index, table = torch.zeros(300, dtype=torch.int32).cuda(), torch.randn(1, 8192).cuda()
    weight, bias = torch.ones(8192).cuda(), torch.zeros(8192).cuda()

    def best(call):
        call()
        times = []
        for _ in range(8):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            for _ in range(10):
                call()
            end.record()
            torch.cuda.synchronize()
            times.append(start.elapsed_time(end))
        return min(times)

    one = best(lambda: mg.encode_types(index, table, weight, bias, p=0.1, seed=1))
    parts = best(lambda: mg.dropout(mg.layer_norm(mg.embed_types(index, table), weight, bias)[0], 0.1, 1))
    assert one <= 3 * parts
