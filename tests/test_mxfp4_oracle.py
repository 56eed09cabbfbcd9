"""CPU: the MXFP4 oracle against the format's definition, and what the operators refuse before anything is launched."""
import ctypes

import numpy as np
import pytest
import torch

import oracle


def test_levels_borders_and_scales():
    x = np.zeros((1, 64))
    x[0, :14] = [4, 0.25, 0.26, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 5.01, 7.9, -0.75, -7.9, 0.74]
    x[0, 32:35] = [3.999, -1.0, 2.0 ** -20]
    codes, scales = oracle.mxfp4_quant_rows(x)
    assert scales.tolist() == [[127, 126]]
    got = oracle.mxfp4_values(codes, scales)[0]
    assert got[:14].tolist() == [4, 0, 0.5, 1, 1, 2, 2, 4, 4, 6, 6, -1, -6, 0.5]
    assert got[32:35].tolist() == [3.0, -1.0, 0.0]  # 7.998 units of 1/2 become 6


def test_scale_limits():
    x = np.zeros((5, 32))
    x[1, 3] = np.inf
    x[2, 3] = np.nan
    x[3, 3] = 2.0 ** -140
    x[4, 3] = 2.0 ** 127
    codes, scales = oracle.mxfp4_quant_rows(x)
    assert scales[:, 0].tolist() == [127, 255, 255, 0, 252]
    assert not codes[1].any() and not codes[2].any() and np.isnan(oracle.mxfp4_values(codes, scales)[1:3]).all()


def test_every_level_comes_back():
    values = np.concatenate([oracle.mxfp4_oracle.LEVELS, -oracle.mxfp4_oracle.LEVELS])
    x = np.tile(values, (1, 2))
    for shift in (-100, -3, 0, 90):
        assert (oracle.mxfp4_held(x * 2.0 ** shift) == x * 2.0 ** shift).all()


def test_doubt_covers_both_sides_of_a_border():
    x = np.zeros((1, 32))
    x[0, 0], x[0, 1] = 4.0 + 1e-9, 0.75 - 1e-9  # the scale is 1, and 1/2 if the first were below 4
    d = oracle.mxfp4_doubt(x, np.full((1, 32), 1e-8))
    assert d[0, 1] >= 0.25 and d[0, 0] >= 1.0 - 1e-6 and d[0, 2] == 0
    assert oracle.mxfp4_doubt(x * 1.5, np.full((1, 32), 1e-8)).max() == 0


def test_layer_of_one_expert_is_the_dense_formula():
    rng = np.random.default_rng(3)
    x = torch.from_numpy(rng.standard_normal((3, 64)))
    w1, w2 = rng.standard_normal((1, 128, 64)), rng.standard_normal((1, 64, 64))
    q1, q2 = oracle.mxfp4_quant_rows(w1[0]), oracle.mxfp4_quant_rows(w2[0])
    out, doubt = oracle.fused_moe_mxfp4(x, q1[0][None], q1[1][None], q2[0][None], q2[1][None], torch.zeros(3, 1), 1)
    h = oracle.mxfp4_held(x) @ oracle.mxfp4_held(w1[0]).T
    act = h[:, :64] / (1 + np.exp(-h[:, :64])) * h[:, 64:]
    assert np.allclose(out, oracle.mxfp4_held(act) @ oracle.mxfp4_held(w2[0]).T, rtol=1e-12, atol=1e-12)
    assert (doubt >= 0).all()


# ---- refusals: nothing below may reach a launch ----------------------------------------------------------------

P = ctypes.c_void_p(1 << 20)  # never dereferenced


def _refused(native, code, call, *args):
    assert getattr(native, call)(*args) == code, (call, args)
    assert native.fr_last_error_string()


def test_c_entry_points_refuse(native):
    from fast_route_amd import _native as N
    odd = ctypes.c_void_p((1 << 20) + 4)
    q = "fr_quant_mxfp4_rows"
    _refused(native, -2, q, P, N.FR_BF16, -1, 64, 64, P, P, None)
    _refused(native, -2, q, P, N.FR_BF16, 4, 48, 48, P, P, None)
    _refused(native, -2, q, P, N.FR_BF16, 4, 0, 0, P, P, None)
    _refused(native, -2, q, P, N.FR_BF16, 1 << 40, 64, 64, P, P, None)
    _refused(native, -3, q, P, N.FR_F32, 4, 64, 64, P, P, None)
    _refused(native, -1, q, None, N.FR_BF16, 4, 64, 64, P, P, None)
    _refused(native, -4, q, P, N.FR_BF16, 4, 64, 60, P, P, None)
    _refused(native, -4, q, P, N.FR_BF16, 4, 64, 68, P, P, None)
    _refused(native, -4, q, odd, N.FR_BF16, 4, 64, 64, P, P, None)
    assert native.fr_quant_mxfp4_rows(None, N.FR_BF16, 0, 64, 64, None, None, None) == 0
    d = "fr_dequant_mxfp4_rows"
    _refused(native, -2, d, P, P, 4, 40, N.FR_BF16, P, None)
    _refused(native, -3, d, P, P, 4, 64, N.FR_I32, P, None)
    _refused(native, -1, d, P, None, 4, 64, N.FR_BF16, P, None)
    _refused(native, -4, d, odd, P, 4, 64, N.FR_BF16, P, None)
    t = "fr_mxfp4_tile_weights"
    _refused(native, -2, t, P, P, 0, 64, 64, 0, P, None)
    _refused(native, -2, t, P, P, 1, 96, 64, 1, P, None)  # 48 gate rows
    _refused(native, -2, t, P, P, 1, 64, 33, 0, P, None)
    _refused(native, -2, t, P, P, 1 << 20, 1 << 20, 64, 0, P, None)
    _refused(native, -1, t, P, P, 1, 64, 64, 0, None, None)
    assert native.fr_mxfp4_tiled_bytes(1, 64, 64) == 2 * 4352 and native.fr_mxfp4_tiled_bytes(3, 33, 257) == 3 * 4 * 4352
    assert native.fr_mxfp4_tiled_bytes(1 << 20, 1 << 30, 64) == -1 and native.fr_mxfp4_tiled_bytes(-1, 1, 32) == -1
    m = "fr_linear_mxfp4"
    big = 1 << 40
    _refused(native, -2, m, P, N.FR_BF16, -1, 64, 64, P, 8, P, P, big, None)
    _refused(native, -2, m, P, N.FR_BF16, 4, 40, 40, P, 8, P, P, big, None)
    _refused(native, -2, m, P, N.FR_BF16, 4, 64, 64, P, 0, P, P, big, None)
    _refused(native, -3, m, P, N.FR_F32, 4, 64, 64, P, 8, P, P, big, None)
    _refused(native, -1, m, P, N.FR_BF16, 4, 64, 64, None, 8, P, P, big, None)
    _refused(native, -4, m, P, N.FR_BF16, 4, 64, 32, P, 8, P, P, big, None)
    _refused(native, -5, m, P, N.FR_BF16, 40, 64, 64, P, 8, P, P, 128, None)
    _refused(native, -5, m, P, N.FR_BF16, 20, 64, 64, P, 8, P, None, big, None)
    assert native.fr_linear_mxfp4(None, N.FR_BF16, 0, 64, 64, None, 8, None, None, 0, None) == 0
    assert native.fr_linear_mxfp4_workspace_bytes(4, 0, 64) == -1
    f = "fr_fused_moe_mxfp4"

    def layer(rc, x=P, dt=N.FR_BF16, w1=P, w2=P, lg=P, ldt=N.FR_F32, M=4, H=64, F=64, E=8, k=2, out=P, ws=P, size=big):
        _refused(native, rc, f, x, dt, w1, w2, lg, ldt, M, H, F, E, k, 1, out, ws, size, None)
    layer(-2, M=-1)
    layer(-2, M=(1 << 24) + 1)
    layer(-2, M=1 << 23, k=4)
    layer(-2, H=48)
    layer(-2, F=0)
    layer(-2, E=257, k=1)
    layer(-2, k=9)
    layer(-2, k=0)
    layer(-3, dt=N.FR_F32)
    layer(-3, ldt=N.FR_I32)
    layer(-1, lg=None)
    layer(-4, x=odd)
    layer(-5, ws=None)
    layer(-5, size=1024)
    layer(-4, ws=ctypes.c_void_p((1 << 20) + 128))
    assert native.fr_moe_mxfp4_workspace_bytes(4, 64, 64, 8, 9) == -1
    for M in (0, 1, 32, 33, 300, 1 << 20):
        for H, F, E, k in ((64, 64, 8, 2), (32, 32, 1, 1), (4096, 14336, 8, 2), (2048, 1408, 64, 6), (1056, 1120, 256, 9)):
            assert native.fr_moe_mxfp4_workspace_bytes(M, H, F, E, k) >= 0


def test_python_entry_points_refuse_cpu_tensors():
    import fast_route_amd as fr
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    codes, scales = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    for call in (lambda: fr.quantize_rows_mxfp4(x), lambda: fr.dequantize_rows_mxfp4(codes, scales),
                 lambda: fr.prepare_linear_mxfp4(codes, scales), lambda: fr.linear_mxfp4(x, fr.MXFP4Weight(codes, 4, 64)),
                 lambda: fr.prepare_weights_mxfp4(codes[None], scales[None], codes[None], scales[None]),
                 lambda: fr.fused_moe_mxfp4(x, fr.MXFP4Experts(codes, codes, 1, 64, 64), torch.zeros(4, 1), 1)):
        with pytest.raises(AssertionError):
            call()


def test_prepared_weights_of_other_sizes_are_refused(native):
    """A handle whose data are not what its sizes say would be read beyond its end: the check that every product makes first, on
    the CPU; the sizes are those that the layout's own entry point states."""
    from fast_route_amd.layers.mxfp4 import _check_tiled
    cpu = torch.device("cpu")
    for matrices, rows, K in ((1, 1, 32), (1, 33, 256), (3, 64, 288), (8, 1120, 1056)):
        nbytes = native.fr_mxfp4_tiled_bytes(matrices, rows, K)
        data = torch.empty(nbytes, dtype=torch.uint8)
        _check_tiled(data, matrices, rows, K, cpu, "w")
        bad = [(data[:-1], rows, K, cpu), (data, rows + 32, K, cpu), (data, rows, K + 256, cpu), (data[::2], rows, K, cpu),
               (torch.empty(nbytes, dtype=torch.int8), rows, K, cpu), (data, rows, K, torch.device("meta"))]
        for d, r, k, dev in bad:
            with pytest.raises(AssertionError):
                _check_tiled(d, matrices, r, k, dev, "w")
