"""The decode-step operators at the ends of their ranges, against float64 restatements: gate, beta and conv values where
e^x overflows.

Tolerances, derived before the first run, beside each test; the bars of outputs and states are those of
tests/test_gpu_decode.py."""

import numpy as np
import pytest
import torch

from oracle import kda as ok
from test_gpu_decode import D, kda_check, kda_dev, kda_make, kda_run, recurrence64

pytestmark = pytest.mark.gpu

# ---- KDA: arguments of the exponentials beyond where e^x is finite in 32 bits (|x| > 88.7) ---------------------------


@pytest.mark.parametrize("a_log", [0.0, float(np.log(16.0))])
def test_kda_decay_over_the_whole_range_of_gates(cuda, a_log):
    """The decay alone, read in fp32: with beta = -inf nothing is written to the state, so a state of ones becomes
    a_c = exp(lower_bound sigmoid(z_c)), z = exp(A_log) (g + dt_bias) from -200 to 200 in steps of 0.1, and +-inf.
    Bar: sigmoid within 2^-21 (an exponential of 2^-22 and a quotient of 2 ulp) moves the exponent by at most
    5 x 2^-21, the fp32 product z by 5 x 0.25 |z| sigmoid(1 - sigmoid) x 2^-22 or less, the outer exponential adds
    2^-22: together below 16 x 2^-22 of a."""
    rng = np.random.default_rng(41)
    H = 32
    d = kda_make(rng, 2, H, 2)
    rate = float(np.exp(np.float64(np.float32(a_log))))
    z = np.linspace(-200.0, 200.0, H * D)
    d["a_log"] = np.full(H, a_log, np.float32)
    d["dtb"] = (z / rate).astype(np.float32)
    d["g"] = np.zeros((2, H * D), np.float32)
    d["g"][1, 0::2], d["g"][1, 1::2] = -np.inf, np.inf
    d["beta"] = np.full((2, H), -np.inf, np.float32)
    d["rst"] = np.ones((2, H, D, D), np.float32)
    seqs = [(0, 1, 0, 1), (1, 2, 1, 1)]
    with np.errstate(over="ignore"):
        want = np.exp(ok.gate(d["g"], d["a_log"], d["dtb"], -5.0, H, D))           # [2, H, D]
    out, _, rst, status = kda_run(cuda, d, seqs, H)
    assert status == 0 and np.isfinite(out).all()
    for r in range(2):
        assert (rst[r] == rst[r][:, :1, :]).all()                                  # every value row alike
        err = np.abs(rst[r][:, 0, :] - want[r]) / want[r]
        assert err.max() < 16 * 2.0 ** -22, (r, float(err.max()))


def test_kda_trained_gates(cuda):
    """A in 1 .. 16 and dt_bias = softplus^-1 of steps of 1e-3 .. 0.1 (-6.9 .. -2.3), as trained layers have them:
    arguments down to -130; five tokens a request, the state kept from token to token."""
    rng = np.random.default_rng(43)
    H, R, n = 8, 6, 5
    d = kda_make(rng, R * n, H, R)
    d["a_log"] = np.log(rng.uniform(1.0, 16.0, H)).astype(np.float32)
    dt = np.exp(rng.uniform(np.log(1e-3), np.log(0.1), H * D))
    d["dtb"] = np.log(np.expm1(dt)).astype(np.float32)
    seqs = [(r * n, (r + 1) * n, r, 1) for r in range(R)]
    z = np.exp(d["a_log"].astype(np.float64))[:, None] * (d["g"].reshape(-1, H, D) + d["dtb"].reshape(H, D))
    assert (z < -88.8).mean() > 0.01
    with np.errstate(over="ignore"):
        want = recurrence64(d, seqs, H)
    out, cst, rst, status = kda_run(cuda, d, seqs, H)
    assert status == 0
    kda_check(out, cst, rst, want, seqs, tol_state=2e-5)


@pytest.mark.parametrize("what", ["beta", "conv"])
def test_kda_beta_and_conv_values_from_minus_200_to_200(cuda, what):
    """Every bf16 value on a grid of 0.25 (0.5 above 64, 1 above 128) as a beta, +-inf too, and as a conv output."""
    rng = np.random.default_rng(47)
    H = 8
    if what == "beta":
        v = np.concatenate([np.arange(-200.0, 200.0, 0.25), [np.inf, -np.inf]])
        v = np.pad(v, (0, -len(v) % H), constant_values=90.5)
        R = len(v) // H
        d = kda_make(rng, R, H, R)
        d["beta"] = torch.from_numpy(v.reshape(R, H)).to(torch.bfloat16).double().numpy()
    else:
        R = 40
        d = kda_make(rng, R, H, R)
        x = rng.uniform(-200.0, 200.0, (R, 3 * H * D))
        # whole rows of v beyond the range (q and k keep their large values, so that the products stay of order one)
        x[0, 2 * H * D:], x[1, 2 * H * D:] = rng.uniform(-200, -85, H * D), rng.uniform(-95, -88, H * D)
        d["x"] = torch.from_numpy(x).to(torch.bfloat16).double().numpy()
        d["w"] = np.zeros((3 * H * D, 4), np.float32)
        d["w"][:, 3] = 1.0                                   # the conv output is the token's own value
    seqs = [(r, r + 1, r, 1) for r in range(R)]
    with np.errstate(over="ignore"):
        want = recurrence64(d, seqs, H)
    assert all(np.isfinite(w).all() for w in want)
    out, cst, rst, status = kda_run(cuda, d, seqs, H)
    assert status == 0
    kda_check(out, cst, rst, want, seqs)


@pytest.mark.parametrize("name", ["g", "beta", "x"])
def test_kda_nan_inputs_stay_nan(cuda, name):
    """A NaN gate, beta or value makes its own head NaN (a gate: its state column and the head's outputs), not another."""
    rng = np.random.default_rng(53)
    H = 3
    d = kda_make(rng, 2, H, 2)
    col = {"g": D + 5, "beta": 1, "x": 2 * H * D + D + 5}[name]           # all of head 1
    d[name] = np.array(d[name])
    d[name][0, col] = np.nan
    out, _, rst, _ = kda_run(cuda, d, [(0, 1, 0, 1), (1, 2, 1, 1)], H)
    bad = out[0].reshape(H, D)
    assert np.isnan(bad[1, 5]) and (name == "x" or np.isnan(bad[1]).all())
    assert np.isfinite(bad[[0, 2]]).all() and np.isfinite(out[1]).all()
    assert np.isnan(rst[0, 1]).any() and np.isfinite(rst[0, [0, 2]]).all() and np.isfinite(rst[1]).all()
