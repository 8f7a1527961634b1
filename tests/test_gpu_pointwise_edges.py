"""-m gpu: the pointwise operators where their results are small, masked, shared between streams or made by another kernel; against
float64 (oracle/pointwise.py).  U and half_step as in test_gpu_pointwise."""
import pytest
import torch

from oracle import pointwise as O
from test_gpu_pointwise import APPROX, TYPES, U, batch_tensor, check, check_group_norm, half_step, rnd, run_group_norm, run_linear

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
    # dz itself: two operands of the type, the second a rounding of at most h of it, rounded in turn
    edz = DY.abs() * ef + (2 * h * h + 4 * U) * o["dz"].abs() + tiny / (1 - p)
    check(got[1], o["dx"], 1.01 * ((edz + (2 * M + 4) * U * o["dz"].abs()) @ W.abs().t() + h * o["dx"].abs() + tiny), "dx")
    rounds = (2 * N + 4) * U * o["dz"].abs()
    check(got[2], o["dw"], 1.01 * (X.abs().t() @ (edz + rounds) + h * o["dw"].abs() + tiny), "dweight")
    check(got[3], o["db"], 1.01 * ((edz + rounds).sum(0) + h * o["db"].abs() + tiny), "dbias")


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("N,K,M", [(300, 64, 1), (1, 64, 300), (700, 130, 1), (9, 20, 3)])
@pytest.mark.parametrize("activation,leak", [("silu", 1), ("gelu", 1), ("leaky_relu", 0.333)])
def test_gradients_lose_one_rounding(gpu, dtype, N, K, M, activation, leak):
    """sums of one or a few terms: the operand's rounding would show beside the result's"""
    t = TYPES[dtype]
    x, w, b, dy = rnd(11, N, K).to(t), (rnd(12, K, M) * K ** -0.5).to(t), (0.1 * rnd(13, M)).to(t), rnd(14, N, M).to(t)
    got = run_linear(gpu, x, w, b, None, activation, leak, 0.0, None, dy)
    X, W, B, DY = (v.double() for v in (x, w, b, dy))
    o = O.linear(X, W, B, None, activation, leak, None, 0.0, DY)
    h = half_step(t)
    tiny = torch.finfo(t).smallest_normal * h
    ez = (K + 4) * U * (X.abs() @ W.abs() + B.abs())
    if activation == "leaky_relu":
        assert (o["z"].abs() > ez).all()  # (on one side of the kink; the slope is the caller's fp32 number)
        ef = U * o["f"].abs()
    else:  # stored slopes: fp16 2^-13 of positive ones, 2^-11 of negative ones, 2^-19 where they are below 2^-6
        relative, absolute = (2.0 ** -10, 0.0) if dtype == "bf16" else (2.0 ** -11, 2.0 ** -19)
        ef = 0.8 * ez + (8 * U + APPROX[t]) * (1 + o["z"].abs()) + relative * o["f"].abs() + absolute
        if dtype == "f16":
            ef = torch.where(o["f"] > 2.0 ** -5, ef - (2.0 ** -11 - 2.0 ** -13) * o["f"] - absolute, ef)
    edz = DY.abs() * ef + (2 * h * h + 4 * U) * o["dz"].abs() + tiny
    check(got[1], o["dx"], 1.01 * ((edz + (2 * M + 4) * U * o["dz"].abs()) @ W.abs().t() + h * o["dx"].abs() + tiny), "dx")
    rounds = (2 * N + 4) * U * o["dz"].abs()
    check(got[2], o["dw"], 1.01 * (X.abs().t() @ (edz + rounds) + h * o["dw"].abs() + tiny), "dweight")
    check(got[3], o["db"], 1.01 * ((edz + rounds).sum(0) + h * o["db"].abs() + tiny), "dbias")


def test_gradients_next_to_the_largest_number(gpu):
    """fp16: dy 60,000 times a slope above 1 leaves the type, the products with small weights and rows do not"""
    N, K, M = 40, 16, 8
    x, w = (rnd(1, N, K) * 2.0 ** -8).half(), (rnd(2, K, M) * 2.0 ** -6).half()
    b = torch.full((M,), 1.4).half()
    dy = torch.full((N, M), 60000.0).half()
    got = run_linear(gpu, x, w, b, None, "gelu", 1, 0.0, None, dy)
    o = O.linear(x.double(), w.double(), b.double(), None, "gelu", 1, None, 0.0, dy.double())
    assert (o["dz"] > 65504).all() and float(o["dx"].abs().max()) < 65504 and float(o["dw"].abs().max()) < 65504
    e = (2.0 ** -13 + 2 * APPROX[torch.float16] + 64 * U) * o["dz"]  # stored slope, its computation; dz's second operand is exact
    check(got[1], o["dx"], 1.01 * (e @ w.double().abs().t() + 2.0 ** -11 * o["dx"].abs() + 2.0 ** -25), "dx")
    check(got[2], o["dw"], 1.01 * (x.double().abs().t() @ e + 2.0 ** -11 * o["dw"].abs() + 2.0 ** -25), "dweight")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("activation,leak", [("silu", 1), ("gelu", 1), ("leaky_relu", 1), ("leaky_relu", 0.25), ("leaky_relu", 0)])
@pytest.mark.parametrize("N,K,M", [(3, 5, 4), (200, 70, 33), (300, 130, 72)])
def test_bad_gradients_of_dropped_elements_stay_there(gpu, dtype, activation, leak, N, K, M):
    """as a dropout layer's do: the gradients are those of zeros in their places, bit for bit.  A bad one that is kept reaches its row of dx
    and its column of dW and db"""
    t = TYPES[dtype]
    x, w, b, dy = rnd(21, N, K).to(t), (rnd(22, K, M) * K ** -0.5).to(t), (0.1 * rnd(23, M)).to(t), rnd(24, N, M).to(t)
    rng = torch.tensor([6, 7], dtype=torch.int64, device=gpu)
    keep = O.keep(6, 7, N, M, 0.5)
    clean = torch.where(keep, dy, torch.zeros_like(dy))
    bad = torch.full_like(dy, float("inf"))
    bad[::2] = float("nan")
    bad[:, ::3] = -float("inf")
    want = run_linear(gpu, x, w, b, None, activation, leak, 0.5, rng, clean)
    got = run_linear(gpu, x, w, b, None, activation, leak, 0.5, rng, torch.where(keep, dy, bad))
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    if activation == "leaky_relu" and leak == 0:
        return  # (a ReLU's slope may be 0 where nothing was dropped)
    r, c = [int(i) for i in keep.nonzero()[len(keep.nonzero()) // 2]]
    clean[r, c] = float("nan")
    got = run_linear(gpu, x, w, b, None, activation, leak, 0.5, rng, clean)
    rows, columns = torch.arange(N) != r, torch.arange(M) != c
    assert got[1][r].isnan().all() and torch.equal(got[1][rows], want[1][rows])
    assert got[2][:, c].isnan().all() and torch.equal(got[2][:, columns], want[2][:, columns])
    assert got[3][c].isnan() and torch.equal(got[3][columns], want[3][columns])


def test_sample_offsets_on_several_streams(gpu):
    """the stream that asks first makes them behind its own work; another, ordered behind the batch's build alone, waits for them and leaves
    the memory to itself until it is through"""
    import occuseg_amd.sparseconvnet as scn
    lengths = [900, 0, 333, 1]
    x = rnd(31, sum(lengths), 16).float().to(gpu)
    module = scn.GroupNormSiLU(16, 4).to(gpu)
    with torch.no_grad():
        want = module(batch_tensor(gpu, scn, x, lengths)).features.clone()
        for turn in range(3):
            inp = batch_tensor(gpu, scn, x, lengths)
            first, second = torch.cuda.Stream(), torch.cuda.Stream()
            torch.cuda.synchronize()
            with torch.cuda.stream(first):
                torch.cuda._sleep(100000000)  # (some 40 ms: the second stream's call is queued before the offsets are made)
                a = module(inp).features
            with torch.cuda.stream(second):
                b = module(inp).features
            inp.metadata._sample_offsets.clear()
            torch.cuda.synchronize()
            assert torch.equal(a, want) and torch.equal(b, want), turn


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lengths,C,groups", [([2048, 0, 0, 0], 128, 128), ([2049], 128, 128), ([1024, 0, 3000, 72], 32, 32), ([8192], 4, 4), ([8193], 4, 4),
                                              ([300] * 3, 1024, 1024)], ids=lambda v: str(v) if isinstance(v, int) else "%dx%d" % (len(v), sum(v)))
def test_group_norm_where_one_launch_ends(gpu, lengths, C, groups, dtype):
    t, N = TYPES[dtype], sum(lengths)
    x = (rnd(41, N, C) * torch.exp(0.5 * rnd(42, C)) + rnd(43, C)).to(t)
    dy, w, b = rnd(44, N, C).to(t), (1 + 0.2 * rnd(45, C)).float(), (0.2 * rnd(46, C)).float()
    args = (x, lengths, groups, w, b, 1e-4, "silu", 1, dy)
    check_group_norm(run_group_norm(gpu, *args), *args, "one launch or three")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("K,M", [(7, 3), (100, 130), (448, 448)])
def test_linear_of_few_rows_and_of_more(gpu, K, M, dtype):
    """up to four rows are another kernel's, with an order of summation of its own: the bits of a row depend on which of the two it was, and
    on nothing else; both are within the roundings of K products and of what follows them"""
    from occuseg_amd import SCN
    t = TYPES[dtype]
    x, w, b, res = rnd(51, 300, K).to(t), (rnd(52, K, M) * K ** -0.5).to(t), (0.1 * rnd(53, M)).to(t), rnd(54, 300, M).to(t)
    on = [v.to(gpu) for v in (x, w, b, res)]
    o = O.linear(x.double(), w.double(), b.double(), res.double(), "gelu", 1, None, 0.0)
    ez = (K + 4) * U * (x.double().abs() @ w.double().abs() + b.double().abs())
    bound = 1.13 * ez + (8 * U + APPROX[t]) * (o["z"].abs() + 1) + 4 * U * (o["value"].abs() + o["y"].abs()) + half_step(t) * o["y"].abs()

    def run(n):
        y, factor = on[0].new_empty(0), torch.empty(0, dtype=SCN.factor_dtype(on[0]), device=gpu)
        SCN.FusedNetworkInNetwork_updateOutput(on[0][:n], y, on[1], on[2], on[3][:n], "gelu", 1, 0.0, None, factor)
        check(y, o["y"][:n], 1.01 * bound[:n], "%d rows" % n)
        return y, factor

    for sizes in ((4, 1, 2, 3), (300, 5, 17, 33, 100)):
        whole = run(sizes[0])
        for n in sizes[1:]:
            assert all(torch.equal(a[:n], c) for a, c in zip(whole, run(n))), n


def test_a_random_state_that_moved_on_is_not_taken_for_the_one_that_was_drawn_from(gpu):
    """a layer's own state handed to another as its `rng`: backward needs it as it was"""
    import occuseg_amd.sparseconvnet as scn
    a, b = scn.Dropout(0.5).to(gpu), scn.Dropout(0.5).to(gpu)
    x = torch.ones(64, 64, device=gpu, requires_grad=True)
    y = a(scn.SparseConvNetTensor(x), rng=b.rng_state).features
    b(scn.SparseConvNetTensor(x.detach()))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y = a(scn.SparseConvNetTensor(x), rng=b.rng_state.clone()).features
    b(scn.SparseConvNetTensor(x.detach()))
    y.sum().backward()
    assert torch.equal(x.grad, y.detach())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("N,K,M", [(3, 5, 4), (200, 70, 33), (300, 64, 128)])
def test_slopes_that_are_nan_reach_the_gradients(gpu, dtype, activation, N, K, M):
    """a row of NaN, of either sign: its row of dx, and all of dW and db; the other rows of dx are as without it"""
    t = TYPES[dtype]
    x, w, b, dy = rnd(61, N, K).to(t), (rnd(62, K, M) * K ** -0.5).to(t), (0.1 * rnd(63, M)).to(t), rnd(64, N, M).to(t)
    want = run_linear(gpu, x, w, b, None, activation, 1, 0.0, None, dy)[1]
    for bad in (float("nan"), -float("nan")):
        x[N // 2] = bad
        y, dx, dw, db = run_nan(gpu, x, w, b, activation, dy)
        rows = torch.arange(N) != N // 2
        assert y[N // 2].isnan().all() and dx[N // 2].isnan().all() and dw.isnan().all() and db.isnan().all()
        assert torch.equal(dx[rows], want[rows])


def run_nan(gpu, x, w, b, activation, dy):
    import occuseg_amd.sparseconvnet as scn
    m = scn.FusedNetworkInNetwork(w.size(0), w.size(1), True, activation).to(gpu).to(x.dtype)
    with torch.no_grad():
        m.weight.copy_(w)
        m.bias.copy_(b)
    xg = x.to(gpu).requires_grad_(True)
    y = m(scn.SparseConvNetTensor(xg)).features
    return [y] + list(torch.autograd.grad(y, [xg, m.weight, m.bias], dy.to(gpu)))
