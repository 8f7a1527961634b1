"""-m gpu: the pointwise operators where their results are small, masked, shared between streams or made by another kernel; against
float64 (oracle/pointwise.py).  U and half_step as in test_gpu_pointwise."""
import pytest
import torch

from oracle import pointwise as O
from test_gpu_pointwise import APPROX, TYPES, U, check, half_step, rnd, run_linear

pytestmark = pytest.mark.gpu


# the stored slopes of saturated units, which are negative: an error relative to the slope and an absolute one below its normal numbers.
# fp32: as computed; bf16: 9 bits of mantissa down to 2^-60; fp16: 10 bits down to 2^-33, half a step of its subnormal numbers 2^-44
STORED = {"f32": (0.0, 0.0), "bf16": (2.0 ** -10, 2.0 ** -60), "f16": (2.0 ** -11, 2.0 ** -44)}
SATURATED = [("f32", "silu", -14, -6), ("f32", "gelu", -4.5, -3), ("f16", "silu", -14, -6), ("f16", "gelu", -4.5, -3),
             ("f16", "silu", -20, -16), ("f16", "gelu", -6.25, -5.5), ("bf16", "silu", -20, -17), ("bf16", "gelu", -6, -5.5),
             ("bf16", "silu", -36, -30), ("bf16", "gelu", -8.25, -7.75)]


@pytest.mark.parametrize("p", [0.0, 0.25])
@pytest.mark.parametrize("N,K,M", [(3, 8, 5), (300, 35, 7), (300, 64, 40)])
@pytest.mark.parametrize("dtype,activation,low,high", SATURATED)
def test_gradients_of_saturated_units(gpu, dtype, activation, low, high, N, K, M, p):
    """pre-activations where the slope is far below 1: every gradient within a bound relative to the slopes themselves.  dy is large (a scaled
    loss), so that dz = dy slope is not lost among fp16's subnormal numbers"""
    t = TYPES[dtype]
    g = torch.Generator().manual_seed(5)
    x, w = rnd(1, N, K).to(t), (rnd(2, K, M) * 0.1 * K ** -0.5).to(t)
    b = (low + (high - low) * torch.rand(M, generator=g, dtype=torch.float64)).to(t)
    dy = (4096 * rnd(3, N, M)).to(t)
    rng = torch.tensor([3, 4], dtype=torch.int64, device=gpu)
    keep = O.keep(3, 4, N, M, p) if p else None
    got = run_linear(gpu, x, w, b, None, activation, 1, p, rng, dy)
    X, W, B, DY = (v.double() for v in (x, w, b, dy))
    o = O.linear(X, W, B, None, activation, 1, keep, p, DY)
    h, (relative, absolute) = half_step(t), STORED[dtype]
    tiny = torch.finfo(t).smallest_normal * h  # half the smallest subnormal number
    ez = (K + 4) * U * (X.abs() @ W.abs() + B.abs())
    # |act'' / act'| <= 9 over these ranges (GELU: (2 - z^2) phi over z phi + Phi, at most |z| (1 + 1 / z^2); SiLU: 1 at most); act' itself:
    # exponents of up to 52, rounded three times
    f = o["f"].abs()
    ef = f * (9 * ez + 2 * APPROX[t] + 160 * U + relative) + (absolute / (1 - p) if p == 0 else absolute / (1 - p) * keep.double())
    edz = DY.abs() * ef + (h + 4 * U) * o["dz"].abs() + tiny / (1 - p)
    check(got[1], o["dx"], 1.01 * ((edz + (M + 4) * U * o["dz"].abs()) @ W.abs().t() + h * o["dx"].abs() + tiny), "dx")
    rounds = (N + 4) * U * o["dz"].abs()
    check(got[2], o["dw"], 1.01 * (X.abs().t() @ (edz + rounds) + h * o["dw"].abs() + tiny), "dweight")
    check(got[3], o["db"], 1.01 * ((edz + rounds).sum(0) + h * o["db"].abs() + tiny), "dbias")
