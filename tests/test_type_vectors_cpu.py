"""Learned type vectors without a GPU: the plain 64-bit forms against differences and published
numbers, refusals of the C ABI, and the kernels on the emulated device."""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest

import type_vector_reference as ref

HERE = os.path.dirname(os.path.abspath(__file__))


def emulated(args, env=None):
    return subprocess.run([sys.executable, os.path.join(HERE, "emu", args[0])] + args[1:],
                          env=dict(os.environ, **(env or {})), stdout=subprocess.PIPE,
                          stderr=subprocess.STDOUT, text=True, timeout=1500)


@pytest.fixture(scope="module")
def emulated_library():
    sys.path.insert(0, os.path.join(HERE, "emu"))
    import build_emu
    return build_emu.build()


# ------------------------------------------------------------------------------------------------
# the plain forms themselves
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("counter,key,words", [
    # the generator's published known answers: counters and keys of zeros, of ones, and digits of pi
    (0, 0, (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
    (2 ** 128 - 1, 2 ** 64 - 1, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
    (0x0370734413198a2e85a308d3243f6a88, 0x299f31d0a4093822, (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1)),
])
def test_generator_known_answers(counter, key, words):
    got = ref.philox(np.array([counter & (2 ** 64 - 1)], np.uint64), counter >> 64, key)[0]
    assert tuple(int(w) for w in got) == words


def _differences(f, x, up, step=1e-6):
    out = np.zeros_like(x)
    for i in np.ndindex(*x.shape):
        high, low = x.copy(), x.copy()
        high[i] += step
        low[i] -= step
        out[i] = ((f(high) - f(low)) * up).sum() / (2 * step)
    return out


def test_plain_gradients_against_differences():
    rng = np.random.default_rng(1)
    rows = np.array([0, 2, 2, -1, 1, 2, 0])
    table, weight, bias = rng.standard_normal((4, 5)), rng.standard_normal(5), rng.standard_normal(5)
    up, scale = rng.standard_normal((7, 5)), rng.uniform(0.5, 1.5, 7)
    (dw, _), (ds, _) = ref.embed_backward(rows, up, table, scale)
    assert np.allclose(dw, _differences(lambda t: ref.embed(rows, t, scale)[0], table, up), atol=1e-8)
    assert np.allclose(ds, _differences(lambda s: ref.embed(rows, table, s)[0], scale, up), atol=1e-8)
    x = rng.standard_normal((7, 5))
    (dx, _), (dn, _), (db, _) = ref.Norm(x, 1e-5).backward(up, weight)
    assert np.allclose(dx, _differences(lambda v: ref.Norm(v, 1e-5).forward(weight, bias)[0], x, up), atol=1e-7)
    assert np.allclose(dn, _differences(lambda v: ref.Norm(x, 1e-5).forward(v, bias)[0], weight, up), atol=1e-7)
    assert np.allclose(db, _differences(lambda v: ref.Norm(x, 1e-5).forward(weight, v)[0], bias, up), atol=1e-7)
    numbers = (1e-5, 0.3, 5, 6)
    dt, dn, db = (g for g, _ in ref.encode_backward(rows, up, table, 1.5, weight, *numbers))
    for got, at, f in ((dt, table, lambda v: ref.encode(rows, v, 1.5, weight, bias, *numbers)[0]),
                       (dn, weight, lambda v: ref.encode(rows, table, 1.5, v, bias, *numbers)[0]),
                       (db, bias, lambda v: ref.encode(rows, table, 1.5, weight, v, *numbers)[0])):
        assert np.allclose(got, _differences(f, at, up), atol=1e-7)


def test_bounds_notice_a_planted_mistake():
    """A gradient that leaves out one token, a variance over channels - 1, a mask shifted by one
    element: all of them beyond the bounds the device is held to."""
    import torch
    rng = np.random.default_rng(2)
    rows, up = rng.integers(0, 4, 60), rng.standard_normal((60, 24))
    (dw, d), _ = ref.embed_backward(rows, up, np.zeros((4, 24)), 1.0)
    for wrong, bound, right in (
            (ref.embed_backward(rows[:-1], up[:-1], np.zeros((4, 24)), 1.0)[0][0], d, dw),
            (ref.Norm(up, 1e-5).forward(1.0, 0.0)[0] * np.sqrt(23 / 24), ref.Norm(up, 1e-5).forward(1.0, 0.0)[1],
             ref.Norm(up, 1e-5).forward(1.0, 0.0)[0]),
            (np.roll(ref.dropout(up, 0.5, 1, 2)[0].reshape(-1), 1).reshape(60, 24), ref.dropout(up, 0.5, 1, 2)[1],
             ref.dropout(up, 0.5, 1, 2)[0])):
        ref.check(torch.tensor(right, dtype=torch.float32), right, bound, torch.float32)
        with pytest.raises(AssertionError):
            ref.check(torch.tensor(wrong, dtype=torch.float32), right, bound, torch.float32)


# ------------------------------------------------------------------------------------------------
# refusals: nothing is launched, so the built library answers without a GPU
# ------------------------------------------------------------------------------------------------
def test_entry_points_refuse_before_they_launch():
    from libmolgrid_amd import _capi
    lib, inv, null = _capi.lib, _capi.MG_ERR_INVALID_ARGUMENT, _capi.MG_ERR_NULL_POINTER
    a, odd = 0x10000, 0x10001                     # addresses that nothing reads

    def embed(n=3, v=4, c=5, dtype=0, kind=0, index=a, table=a, scales=None, out=a):
        return lib.mg_embed_types(n, v, c, dtype, kind, index, table, 1.0, scales, out, None)
    for bad in (dict(n=-1), dict(v=-1), dict(c=-1), dict(dtype=3), dict(dtype=-1), dict(kind=3),
                dict(kind=-1), dict(index=odd), dict(table=odd), dict(out=odd), dict(scales=odd)):
        assert embed(**bad) == inv, bad
    for bad in (dict(index=None), dict(table=None), dict(out=None)):
        assert embed(**bad) == null, bad
    assert embed(n=0, index=None, out=None) == 0 and embed(c=0, table=None) == 0
    for bad in (dict(n=1 << 28), dict(v=1 << 28), dict(c=(1 << 20) + 1)):
        assert embed(**bad) == _capi.MG_ERR_UNSUPPORTED, bad

    def embed_back(n=3, v=4, c=5, dtype=0, kind=0, index=a, grad=a, table=a, scales=None, to_table=a,
                   to_scales=None, workspace=a, size=1 << 30):
        return lib.mg_embed_types_backward(n, v, c, dtype, kind, index, grad, table, 1.0, scales, to_table,
                                           to_scales, workspace, size, None)
    for bad in (dict(n=-1), dict(dtype=5), dict(grad=odd), dict(to_table=odd), dict(to_scales=odd)):
        assert embed_back(**bad) == inv, bad
    for bad in (dict(index=None), dict(grad=None), dict(table=None, to_scales=a, to_table=None)):
        assert embed_back(**bad) == null, bad
    need = lib.mg_embed_types_backward_workspace_size(5000, 4000, 8)
    if need:
        big = dict(n=5000, v=4000, c=8)
        assert embed_back(size=need - 1, **big) == inv and embed_back(workspace=a + 16, **big) == inv
        assert embed_back(workspace=None, **big) == null

    def norm(n=3, c=5, dtype=0, param=0, x=a, weight=a, bias=a, eps=1e-5, out=a, mean=a, rstd=a):
        return lib.mg_layer_norm(n, c, dtype, param, x, weight, bias, eps, out, mean, rstd, None)
    for bad in (dict(n=-1), dict(c=-2), dict(dtype=3), dict(param=1), dict(dtype=1, param=2), dict(eps=-1.0),
                dict(eps=float("nan")), dict(x=odd), dict(weight=odd), dict(bias=odd), dict(out=odd),
                dict(mean=odd), dict(rstd=odd)):
        assert norm(**bad) == inv, bad
    for bad in (dict(x=None), dict(out=None), dict(mean=None), dict(rstd=None)):
        assert norm(**bad) == null, bad
    assert norm(n=0, x=None) == 0

    def norm_back(n=3, c=5, dtype=0, param=0, grad=a, x=a + 64, mean=a, rstd=a, weight=a, to_x=a + 128,
                  to_weight=a, to_bias=a, workspace=a, size=1 << 30):
        return lib.mg_layer_norm_backward(n, c, dtype, param, grad, x, mean, rstd, weight, to_x, to_weight,
                                          to_bias, workspace, size, None)
    for bad in (dict(n=-1), dict(param=2), dict(grad=odd), dict(to_x=a), dict(to_x=a + 64), dict(workspace=a + 8),
                dict(size=lib.mg_layer_norm_backward_workspace_size(3, 5) - 1)):
        assert norm_back(**bad) == inv, bad
    for bad in (dict(grad=None), dict(x=None), dict(mean=None), dict(rstd=None), dict(workspace=None)):
        assert norm_back(**bad) == null, bad
    assert norm_back(c=0) == 0 and norm_back(to_x=None, to_weight=None, to_bias=None) == 0

    def drop(n=5, dtype=0, x=a, p=0.5, state=None, out=a):
        return lib.mg_dropout(n, dtype, x, p, 1, 2, state, out, None)
    for bad in (dict(dtype=3), dict(p=-0.1), dict(p=1.5), dict(p=float("nan")), dict(x=odd), dict(out=odd),
                dict(state=a + 4)):
        assert drop(**bad) == inv, bad
    assert drop(x=None) == null and drop(out=None) == null and drop(n=0, x=None) == 0
    assert drop(n=1 << 50) == _capi.MG_ERR_OUT_OF_RANGE

    def encode(n=3, v=4, c=5, dtype=0, param=0, kind=0, index=a, table=a, weight=a, bias=a, eps=1e-5, p=0.1,
               out=a):
        return lib.mg_encode_types(n, v, c, dtype, param, kind, index, table, 1.0, weight, bias, eps, p, 1, 2,
                                   None, out, None)
    for bad in (dict(v=-1), dict(param=1), dict(kind=4), dict(eps=-1.0), dict(p=2.0), dict(out=odd), dict(bias=odd)):
        assert encode(**bad) == inv, bad
    assert encode(index=None) == null and encode(table=None) == null and encode(n=0, out=None) == 0

    def encode_back(n=3, v=4, c=5, grad=a, table=a, p=0.1, to_table=a, workspace=a, size=1 << 30):
        return lib.mg_encode_types_backward(n, v, c, 0, 0, 0, a, grad, table, 1.0, a, 1e-5, p, 1, 2, None,
                                            to_table, a, a, workspace, size, None)
    for bad in (dict(n=-1), dict(p=2.0), dict(grad=odd), dict(to_table=odd), dict(workspace=a + 4),
                dict(size=lib.mg_encode_types_backward_workspace_size(3, 4, 5) - 1)):
        assert encode_back(**bad) == inv, bad
    for bad in (dict(grad=None), dict(table=None), dict(workspace=None)):
        assert encode_back(**bad) == null, bad


def test_host_layer_needs_a_device_or_says_so():
    import torch
    import libmolgrid_amd as mg
    if torch.cuda.is_available():
        pytest.skip("a device is there")
    with pytest.raises(RuntimeError):
        mg.embed_types(torch.zeros(3), torch.zeros((4, 5)))
    with pytest.raises(ValueError):
        mg.TypeDropout(2.0)
    with pytest.raises(ValueError):
        mg.TypeNorm(4, eps=-1.0)


# ------------------------------------------------------------------------------------------------
# the kernels on the emulated device
# ------------------------------------------------------------------------------------------------
def test_drawn_cases(emulated_library):
    p = emulated(["type_vectors.py", "25", "7"])
    assert p.returncode == 0 and "25 rounds passed" in p.stdout, p.stdout[-3000:]


@pytest.mark.parametrize("env", [{"EMU_ORDER": "reverse"}, {"EMU_APPROX": "hash"}, {"EMU_CONTRACT": "1"},
                                 {"EMU_SANITIZE": "1"},
                                 {"EMU_SANITIZE": "address", "ASAN_OPTIONS": "verify_asan_link_order=0:detect_leaks=0"}])
def test_drawn_cases_in_other_modes(emulated_library, env):
    """Threads and workgroups last to first; approximate instructions one unit off; fused
    multiply-adds; clang's run-time checks of undefined behaviour and of addresses."""
    p = emulated(["type_vectors.py", "8", "8"], env)
    assert p.returncode == 0 and "8 rounds passed" in p.stdout, p.stdout[-3000:]


def test_device_tests_on_the_emulated_device(emulated_library):
    """Some of the GPU test file's cases of the functions (what needs autograd on device tensors, streams or
    graphs is left to the device; all of the others pass here as well, in five minutes)."""
    p = emulated(["gpu_tests_on_fake_device.py", os.path.join(HERE, "test_type_vectors_gpu.py"), "-m", "gpu", "-q",
                  "-x", "-k", "(unusual or name_no_row or no_part or hides or off_alignment or large_mean or "
                  "without_spread or of_nothing or parts_one_after) and not 9001"])
    assert p.returncode == 0 and "passed" in p.stdout, p.stdout[-3000:]
