"""CPU checks of the 8-bit activation form: the 64-bit restatement the GPU tests use agrees with PyTorch's e4m3 conversion
and with the properties the header states, and the entry points refuse a null context."""
import ctypes

import numpy as np
import pytest

import act8_ref as r8


def test_restatement_agrees_with_the_e4m3_conversion_of_torch():
    import torch
    assert np.array_equal(r8.E4M3[:0x7F], torch.arange(0x7F, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy())
    rng = np.random.default_rng(0)
    x = r8.activations(rng, 200, 904, 3.0)
    q, scale = r8.pack(x)
    k = scale.astype(np.int64) - 127
    t = torch.from_numpy(r8.blocks(x) * np.exp2(-k.astype(np.float64))[..., None]).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(q, t.reshape(200, -1)[:, :904])


def test_value_is_within_half_a_step_and_exact_in_bf16():
    rng = np.random.default_rng(1)
    x = r8.bf16(rng.standard_normal((64, 256)) * np.exp2(rng.integers(-140, 118, (64, 256)).astype(np.float64)))
    q, scale = r8.pack(x)
    v = r8.widen(q, scale)
    k = (scale.astype(np.float64) - 127).repeat(32, axis=1)
    assert (np.abs(v - x) <= np.maximum(2.0 ** -4 * np.abs(x), np.exp2(k - 10))).all()
    assert np.array_equal(r8.bf16(v), v)


def test_borders_of_the_scale():
    top = np.zeros((4, 32))
    top[0, 3], top[1, 3], top[2, 3], top[3, 3] = 448.0, 449.0, 3.3e38, 0.0
    q, scale = r8.pack(top)
    assert list(scale[:, 0]) == [127, 128, 246, 10]
    assert r8.E4M3[q[2, 3]] == 448.0
    bad = np.full((1, 32), 1.5)
    bad[0, 7], bad[0, 9] = np.inf, np.nan
    q, scale = r8.pack(bad)
    v = r8.widen(q, scale)[0]
    assert np.isnan(v[7]) and np.isnan(v[9]) and (np.delete(v, [7, 9]) == 1.5).all()


@pytest.mark.parametrize("name", ["ta_q8_store", "ta_q8_load", "ta_add_rms_norm_q8_fwd", "ta_rms_norm_q8_bwd", "ta_silu_mul_q8_fwd",
                                  "ta_silu_mul_q8_bwd", "ta_gemm_tokens_q8_f32"])
def test_null_context_is_refused(name):
    import tensor_adapt_b200 as ta
    fn = getattr(ta.lib, name)
    args = [a(1) if a is ctypes.c_float else (0 if a in (ctypes.c_int, ctypes.c_long) else None) for a in fn.argtypes]
    assert fn(*args) == -1
