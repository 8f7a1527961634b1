"""-m gpu: group norm over ragged samples, dropout and the 1x1 convolution with its epilogue against float64 (oracle/pointwise.py).

Tolerances count roundings.  U = 2^-24 (fp32), h = half a step of the type, relative.  A value made by n fp32 operations on terms of
total magnitude M is within n U M of the formula's; what is stored is within h |value| on top.  GELU is made of a polynomial whose
error relative to the value is below 2^-20 (fp32), 2^-18 (fp16), 2^-14 (bf16): APPROX.
"""
import numpy as np
import pytest
import torch

from oracle import pointwise as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


APPROX = {torch.float32: 2.0 ** -20, torch.float16: 2.0 ** -18, torch.bfloat16: 2.0 ** -14}


def half_step(t):
    return torch.finfo(t).eps / 2


def check(got, want, bound, what):
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if want.numel() == 0:
        return
    bad = (got - want).abs() / bound.clamp(min=1e-300)
    assert torch.isfinite(got).all(), what
    assert float(bad.max()) <= 1, "%s: %.3g times the bound at %s" % (what, float(bad.max()), np.unravel_index(int(bad.argmax()), bad.shape))


def rnd(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


# ---------------------------------------------------------------------------------------------------------- group norm ---
def run_group_norm(gpu, x, lengths, groups, weight, bias, eps, activation, leakiness, dy):
    from occuseg_amd import SCN
    from occuseg_amd.sparseconvnet.norm import _GroupNormFunction
    offsets = torch.tensor([0] + list(np.cumsum(lengths)), dtype=torch.int64, device=gpu)
    xg = x.to(gpu).requires_grad_(True)
    none = torch.Tensor()
    w = weight.float().to(gpu).requires_grad_(True) if weight is not None else none
    b = bias.float().to(gpu).requires_grad_(True) if bias is not None else none
    y = _GroupNormFunction.apply(xg, w, b, offsets, eps, groups, activation, leakiness)
    leaves = [xg] + ([w, b] if weight is not None else [])
    return [y] + list(torch.autograd.grad(y, leaves, dy.to(gpu)))


def check_group_norm(got, x, lengths, groups, weight, bias, eps, activation, leakiness, dy, what):
    t = x.dtype
    o = O.group_norm(x.double(), lengths, groups, weight, bias, eps, activation, leakiness, dy.double())
    w = (torch.ones(x.size(1)) if weight is None else weight).double().abs()
    b = (torch.zeros(x.size(1)) if bias is None else bias).double().abs()
    h, approx = half_step(t), APPROX[t]
    # statistics: at most 64 additions in a thread's chain, 64 in the joins, of deviations from a value of the plane; the mean is
    # stored in fp32
    n_stat = 128
    far = o["rstd"] * (x.double().abs() + o["mean"].abs())  # magnitudes that cancel in x - mean
    spread = 1 + o["xh"].abs()
    ez = U * (n_stat * spread + far) * w + 4 * U * (o["z"].abs() + b)
    # |act'| <= 1.13, |act''| <= 0.8; the functions themselves: 8 operations
    bound = 1.13 * ez + (8 * U + approx) * (o["z"].abs() + 1) * (activation != "leaky_relu") + h * o["y"].abs()
    check(got[0], o["y"], bound * 1.01, what + " y")
    dz = dy.double() * o["slope"]
    slope_error = lambda approx: 0.8 * ez * (activation != "leaky_relu") + (8 * U + approx) * (1 + o["z"].abs()) + U  # noqa: E731
    # (the sums, which are stored in fp32, are made of fp32's slopes whatever the features are)
    e_dx_dz, e_dz = dy.double().abs() * slope_error(approx), dy.double().abs() * slope_error(APPROX[torch.float32])
    e_xh = U * (n_stat * spread + far)
    # sums over a sample: relative to the absolute terms, plus the terms' own errors
    e_dx = torch.zeros_like(dz)
    r, C = 0, x.size(1)
    e_dw, e_db = torch.zeros(C, dtype=torch.float64), torch.zeros(C, dtype=torch.float64)
    for n in lengths:
        rows, r = slice(r, r + n), r + n
        if not n:
            continue
        ax, adz = o["xh"][rows].abs(), dz[rows].abs()
        e_db += (e_dz[rows] + n_stat * U * adz).sum(0)
        e_dw += (e_dz[rows] * ax + adz * e_xh[rows] + n_stat * U * adz * ax).sum(0)
        mean = lambda v: v.view(n, groups, -1).mean((0, 2), keepdim=True).expand(n, groups, C // groups).reshape(n, C)  # noqa: E731
        e1 = mean((e_dz[rows] + n_stat * U * adz) * w)
        e2 = mean((e_dz[rows] * ax + adz * e_xh[rows] + n_stat * U * adz * ax) * w)
        terms = dz[rows].abs() * w + o["m1"][rows].abs() + (o["xh"][rows] * o["m2"][rows]).abs()
        e_dx[rows] = o["rstd"][rows] * (e_dx_dz[rows] * w + e1 + ax * e2 + e_xh[rows] * o["m2"][rows].abs() + n_stat * U * terms)
    check(got[1], o["dx"], 1.01 * (e_dx + h * o["dx"].abs()), what + " dx")
    if weight is not None:
        check(got[2], o["dw"], 1.01 * (e_dw + U * o["dw"].abs()) + 1e-30, what + " dweight")
        check(got[3], o["db"], 1.01 * (e_db + U * o["db"].abs()) + 1e-30, what + " dbias")


GN_CASES = [
    # lengths, planes, groups
    ([1], 1, 1),
    ([1], 8, 8),               # one value a group: variance 0
    ([3, 0, 1, 2], 4, 2),
    ([0, 0, 5, 0], 20, 5),
    ([37, 1, 0, 211], 21, 7),   # odd planes
    ([300, 5], 35, 5),
    ([129, 64], 64, 8),
    ([1000], 448, 32),
    ([70, 71], 257, 1),         # odd and above 256
    ([33], 385, 77),
    ([40, 3], 1536, 16),        # more vectors a row than threads
    ([12], 4096, 1024),
    ([20001, 0, 9999], 32, 32),
    ([5] * 130, 12, 3),         # more samples than a wave
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lengths,C,groups", GN_CASES, ids=lambda v: str(v) if isinstance(v, int) else "%dx%d" % (len(v), sum(v)))
def test_group_norm(gpu, lengths, C, groups, dtype):
    t, N = TYPES[dtype], sum(lengths)
    x = (rnd(1, N, C) * torch.exp(0.5 * rnd(2, C)) + rnd(3, C)).to(t)
    dy, w, b = rnd(4, N, C).to(t), (1 + 0.2 * rnd(5, C)).float(), (0.2 * rnd(6, C)).float()
    for activation in ("silu", "gelu"):
        got = run_group_norm(gpu, x, lengths, groups, w, b, 1e-4, activation, 1, dy)
        check_group_norm(got, x, lengths, groups, w, b, 1e-4, activation, 1, dy, activation)
    got = run_group_norm(gpu, x, lengths, groups, None, None, 1e-4, "leaky_relu", 1, dy)
    check_group_norm(got, x, lengths, groups, None, None, 1e-4, "leaky_relu", 1, dy, "bare")


def test_group_norm_leaky_slope(gpu):
    """values of +-1 in equal numbers: the pre-activations are +-w + b, far from the kink"""
    x = torch.tensor([1.0, -1.0]).repeat(64).view(32, 4)
    dy, w, b = rnd(1, 32, 4).float(), torch.ones(4), torch.full((4,), 0.25)
    got = run_group_norm(gpu, x, [32], 2, w, b, 1e-4, "leaky_relu", 0.333, dy)
    check_group_norm(got, x, [32], 2, w, b, 1e-4, "leaky_relu", 0.333, dy, "leaky")


def test_group_norm_far_from_zero(gpu):
    """mean 1000 times the spread: sums of squares in fp32 would lose the variance"""
    x = (1000 + rnd(1, 5000, 16)).float()
    dy, w, b = rnd(2, 5000, 16).float(), torch.ones(16), torch.zeros(16)
    got = run_group_norm(gpu, x, [3000, 2000], 4, w, b, 1e-4, "silu", 1, dy)
    check_group_norm(got, x, [3000, 2000], 4, w, b, 1e-4, "silu", 1, dy, "far")


def test_group_norm_rows_outside_the_samples_are_left(gpu):
    from occuseg_amd import SCN
    x = rnd(1, 50, 8).float().to(gpu)
    offsets = torch.tensor([7, 20, 20, 41], dtype=torch.int64, device=gpu)
    out = torch.full((50, 8), 123.0, device=gpu)
    stats = torch.empty(0, device=gpu)
    SCN.GroupNormalization_updateOutput(x, out, stats, offsets, None, None, 1e-4, 2, "leaky_relu", 1)
    assert (out[:7] == 123).all() and (out[41:] == 123).all()
    want = O.group_norm(x.double().cpu()[7:41], [13, 0, 21], 2, None, None, 1e-4, "leaky_relu", 1)
    check(out[7:41], want["y"], 256 * U * (1 + want["y"].abs()), "inside")
    assert stats.shape == (3, 2, 2) and (stats[1] == 0).all()
    dx = torch.full((50, 8), 5.0, device=gpu)
    dw, db = torch.empty(8, device=gpu), torch.empty(8, device=gpu)
    SCN.GroupNormalization_backward(x, dx, torch.ones_like(x), stats, offsets, None, None, dw, db, 2, "leaky_relu", 1)
    assert (dx[:7] == 5).all() and (dx[41:] == 5).all() and torch.equal(db, torch.full_like(db, 34))


@pytest.mark.parametrize("samples", [300, 5000])
def test_group_norm_many_samples(gpu, samples):
    lengths = [(7 * s) % 5 % 4 for s in range(samples)]  # 0 to 3 sites each
    lengths[samples // 2] = 1500
    n = sum(lengths)
    x, dy, w, b = rnd(31, n, 24).float(), rnd(32, n, 24).float(), rnd(33, 24).float().double(), rnd(34, 24).float().double()
    args = (x, lengths, 2, w, b, 1e-2, "silu", 1.0, dy)
    check_group_norm(run_group_norm(gpu, *args), *args, "%d samples" % samples)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_group_norm_bad_values_stay_in_their_group(gpu, bad):
    x = rnd(1, 60, 8).float()
    clean = run_group_norm(gpu, x, [30, 30], 2, None, None, 1e-4, "silu", 1, torch.ones(60, 8))[0]
    x[4, 1] = bad
    got = run_group_norm(gpu, x, [30, 30], 2, None, None, 1e-4, "silu", 1, torch.ones(60, 8))[0]
    assert got[:30, :4].isnan().all()
    assert torch.equal(got[30:], clean[30:]) and torch.equal(got[:30, 4:], clean[:30, 4:])


def batch_tensor(gpu, scn, features, lengths):
    """the features over a batch whose sample s has lengths[s] distinct voxels"""
    parts = []
    for s, n in enumerate(lengths):
        i = torch.arange(n)
        parts.append(torch.stack([i % 16, i // 16 % 16, i // 256, torch.full_like(i, s)], 1))
    meta, size = scn.Metadata(3), torch.tensor([512] * 3)
    meta.inputLayer(size, torch.cat(parts).to(gpu), len(lengths), 4, gpu)
    return scn.SparseConvNetTensor(features, meta, size)


@pytest.mark.parametrize("occ", [True, False])
def test_group_norm_module_takes_the_samples_from_the_batch(gpu, occ, monkeypatch):
    import occuseg_amd.sparseconvnet as scn
    from occuseg_amd import SCN
    monkeypatch.setattr(SCN, "OCC_BUILD", occ)
    lengths = [300, 0, 17, 1]
    x = rnd(1, 318, 16).float()
    for module, act, leak in ((scn.GroupNormReLU(16, 4), "leaky_relu", 0), (scn.GroupNormLeakyReLU(16, 4, leakiness=0.1), "leaky_relu", 0.1),
                              (scn.GroupNormSiLU(16, 2), "silu", 1), (scn.GroupNormalization(16, 8, affine=False), "leaky_relu", 1)):
        module = module.to(gpu)
        inp = batch_tensor(gpu, scn, x.to(gpu), lengths)
        assert inp.metadata.sampleOffsets(inp.spatial_size).tolist() == [0, 300, 300, 317, 318]
        out = module(inp)
        want = O.group_norm(x.double(), lengths, module.nGroups, None, None, 1e-4, act, leak)
        check(out.features, want["y"], 256 * U * (1 + want["z"].abs()), repr(module))
        module.eval()
        assert torch.equal(module(inp).features, out.features)
    with pytest.raises(RuntimeError, match="rows of features"):
        scn.GroupNormalization(16, 4).to(gpu)(scn.SparseConvNetTensor(x[:10].to(gpu), inp.metadata, inp.spatial_size))
    # the parameters in the features' type
    half = scn.GroupNormSiLU(16, 2).to(gpu).to(torch.bfloat16)
    out = half(scn.SparseConvNetTensor(x.to(gpu, torch.bfloat16).requires_grad_(True), inp.metadata, inp.spatial_size))
    out.features.float().sum().backward()
    assert out.features.dtype == torch.bfloat16 and half.weight.grad.dtype == torch.bfloat16


def test_group_norm_coarser_scale(gpu):
    """the samples of a scale that a strided convolution made"""
    import occuseg_amd.sparseconvnet as scn
    inp = batch_tensor(gpu, scn, rnd(1, 410, 8).float().to(gpu), [400, 10])
    coarse = scn.Convolution(3, 8, 8, 2, 2, False).to(gpu)(inp)
    loc = coarse.get_spatial_locations()
    lengths = [int((loc[:, 3] == s).sum()) for s in range(2)]
    out = scn.GroupNormSiLU(8, 4).to(gpu)(coarse)
    want = O.group_norm(coarse.features.detach().double().cpu(), lengths, 4, None, None, 1e-4, "silu", 1)
    check(out.features, want["y"], 256 * U * (1 + want["z"].abs()), "coarse")


# ------------------------------------------------------------------------------------------------------------- dropout ---
def masked(x, keep, p):
    """the kernel's arithmetic: one fp32 product, one rounding to the type"""
    v = (x.float() * np.float32(1.0 / (1.0 - p))).to(x.dtype)
    return torch.where(keep, v, torch.zeros_like(v))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N,C", [(1, 1), (3, 2), (7, 3), (1, 448), (100, 35), (65, 64), (9, 1023), (5000, 20), (4097, 128)])
def test_dropout(gpu, N, C, dtype):
    import occuseg_amd.sparseconvnet as scn
    for seed, offset, p in ((12345, 0, 0.5), (-1, 2 ** 40 + 3, 0.1), (2 ** 62, -1, 0.99)):
        rng = torch.tensor([seed, offset], dtype=torch.int64, device=gpu)
        x, dy = rnd(1, N, C).to(TYPES[dtype]), rnd(2, N, C).to(TYPES[dtype])
        xg = x.to(gpu).requires_grad_(True)
        y = scn.Dropout(p).to(gpu)(scn.SparseConvNetTensor(xg), rng=rng).features
        (dx,) = torch.autograd.grad(y, [xg], dy.to(gpu))
        keep = O.keep(seed, offset, N, C, p)
        assert torch.equal(y.cpu(), masked(x, keep, p)) and torch.equal(dx.cpu(), masked(dy, keep, p))


def test_dropout_slices_bad_values_and_empty(gpu):
    import occuseg_amd.sparseconvnet as scn
    rng = torch.tensor([5, 6], dtype=torch.int64, device=gpu)
    drop = scn.Dropout(0.5).to(gpu)
    wide = rnd(1, 200, 24).float().to(gpu)
    keep = O.keep(5, 6, 200, 9, 0.5)
    for x in (wide[:, 3:12], wide[:, ::2][:, :9], wide.t().contiguous().t()[:, :9], wide[::2][:, 5:14]):
        y = drop(scn.SparseConvNetTensor(x), rng=rng).features
        assert torch.equal(y.cpu(), masked(x.cpu(), keep[:x.size(0)], 0.5))
    x = torch.full((8, 8), float("nan"))
    x[::2] = float("inf")
    y = drop(scn.SparseConvNetTensor(x.to(gpu)), rng=rng).features.cpu()
    keep = O.keep(5, 6, 8, 8, 0.5)
    assert (y[~keep] == 0).all() and not y[keep].isfinite().any()
    assert drop(scn.SparseConvNetTensor(torch.zeros(0, 8, device=gpu)), rng=rng).features.shape == (0, 8)


def test_dropout_state_moves_on(gpu):
    import occuseg_amd.sparseconvnet as scn
    drop = scn.Dropout(0.5).to(gpu)
    drop.reseed(77, 0)
    x = torch.ones(64, 64, device=gpu)
    a, b = (drop(scn.SparseConvNetTensor(x)).features for _ in range(2))
    assert drop.rng_state.tolist() == [77, 2] and not torch.equal(a, b)
    assert torch.equal((a > 0).cpu(), O.keep(77, 0, 64, 64, 0.5)) and torch.equal((b > 0).cpu(), O.keep(77, 1, 64, 64, 0.5))
    # an rng of the caller's leaves the state alone
    c = drop(scn.SparseConvNetTensor(x), rng=torch.tensor([77, 1], device=gpu)).features
    assert torch.equal(b, c) and drop.rng_state.tolist() == [77, 2]


# -------------------------------------------------------------------------------------------------------------- linear ---
def run_linear(gpu, x, w, b, res, activation, leakiness, p, rng, dy):
    import occuseg_amd.sparseconvnet as scn
    m = scn.FusedNetworkInNetwork(w.size(0), w.size(1), b is not None, activation, leakiness, p).to(gpu).to(x.dtype)
    with torch.no_grad():
        m.weight.copy_(w)
        if b is not None:
            m.bias.copy_(b)
    xg = x.to(gpu).requires_grad_(True)
    rg = res.to(gpu).requires_grad_(True) if res is not None else None
    y = m(scn.SparseConvNetTensor(xg), residual=rg, rng=rng).features
    leaves = [xg, m.weight] + ([m.bias] if b is not None else []) + ([rg] if res is not None else [])
    got = [y] + list(torch.autograd.grad(y, leaves, dy.to(gpu)))
    with torch.no_grad():  # the serving call: the same numbers
        assert torch.equal(m(scn.SparseConvNetTensor(xg), residual=rg, rng=rng).features, y)
    return got


def check_linear(got, x, w, b, res, activation, leakiness, keep, p, dy, what):
    t = x.dtype
    d = [None if v is None else v.double() for v in (x, w, b, res, dy)]
    x, w, b, res, dy = d
    o = O.linear(x, w, b, res, activation, leakiness, keep, p, dy)
    K, M, N = w.size(0), w.size(1), x.size(0)
    h, approx = half_step(t), APPROX[t]
    ez = (K + 4) * U * (x.abs() @ w.abs() + (0 if b is None else b.abs()))
    up = (1 if keep is None else 1 / (1 - p))
    smooth = activation != "leaky_relu"
    ev = up * (1.13 * ez + (8 * U + approx) * (o["z"].abs() + 1) * smooth) + 4 * U * o["value"].abs()
    check(got[0], o["y"], 1.01 * (ev + 2 * U * (o["value"].abs() + o["y"].abs()) + h * o["y"].abs()) + 1e-30, what + " y")
    # dz: the stored slope (bf16: in fp16, within h; fp16: in steps of 2^-14) and the operand are rounded (fp32: two roundings of U);
    # nothing is, without a factor
    ef = up * (0.8 * ez + (8 * U + approx) * (1 + o["z"].abs()) + (2.0 ** -15 if t == torch.float16 else 0)) * smooth
    tiny = torch.finfo(t).smallest_normal * h  # below the normal numbers a rounding is half the smallest subnormal
    bare = activation == "leaky_relu" and leakiness == 1 and keep is None
    edz = torch.zeros_like(dy) if bare else dy.abs() * (ef + h * o["f"].abs() + 2 * tiny) + (h + 2 * U) * o["dz"].abs() + 2 * tiny
    check(got[1], o["dx"], 1.01 * ((edz + (M + 4) * U * o["dz"].abs()) @ w.abs().t() + h * o["dx"].abs() + tiny) + 1e-30, what + " dx")
    terms = x.abs().t() @ (edz + min(N + 4, 4096) * U * o["dz"].abs())
    check(got[2], o["dw"], 1.01 * (terms + h * o["dw"].abs() + tiny) + 1e-30, what + " dweight")
    i = 3
    if b is not None:
        check(got[i], o["db"], 1.01 * ((edz + min(N + 4, 4096) * U * o["dz"].abs()).sum(0) + h * o["db"].abs() + tiny) + 1e-30, what + " dbias")
        i += 1
    if res is not None:
        assert torch.equal(got[i].double().cpu(), dy)


LIN_CASES = [
    # sites, planes in, out
    (1, 1, 1), (1, 448, 448), (2, 3, 5), (5, 16, 16), (17, 35, 77), (33, 64, 20), (127, 20, 33), (128, 64, 64), (129, 65, 129),
    (1000, 128, 512), (300, 512, 128), (2049, 7, 200), (64, 1000, 40), (700, 449, 31), (20011, 32, 64),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N,K,M", LIN_CASES)
def test_linear(gpu, N, K, M, dtype):
    t = TYPES[dtype]
    x, w, b = rnd(1, N, K).to(t), (rnd(2, K, M) * (2.0 / K) ** 0.5).to(t), (0.1 * rnd(3, M)).to(t)
    res, dy = rnd(4, N, M).to(t), rnd(5, N, M).to(t)
    rng = torch.tensor([99, 2 ** 33], dtype=torch.int64, device=gpu)
    for activation, leak, p, bias, residual in (("leaky_relu", 1, 0.0, None, None), ("silu", 1, 0.0, b, res), ("gelu", 1, 0.3, b, res),
                                                ("silu", 1, 0.9, None, None), ("leaky_relu", 1, 0.5, b, None)):
        keep = O.keep(99, 2 ** 33, N, M, p) if p else None
        got = run_linear(gpu, x, w, bias, residual, activation, leak, p, rng, dy)
        check_linear(got, x, w, bias, residual, activation, leak, keep, p, dy, "%s p %s" % (activation, p))


@pytest.mark.parametrize("leak", [0, 0.333])
def test_linear_leaky_slope(gpu, leak):
    """small integers: the pre-activations are exact, zeros among them"""
    g = torch.Generator().manual_seed(1)
    ints = lambda *s: torch.randint(-3, 4, s, generator=g).float()  # noqa: E731
    x, w, b, dy = ints(300, 24), ints(24, 40), ints(40), rnd(2, 300, 40).float()
    assert ((x @ w + b) == 0).any()
    got = run_linear(gpu, x, w, b, None, "leaky_relu", leak, 0.0, None, dy)
    check_linear(got, x, w, b, None, "leaky_relu", leak, None, 0.0, dy, "leaky")


def test_linear_slices_and_empty(gpu):
    """column slices of wider tensors are read in place; a transposed gradient is not; no sites"""
    import occuseg_amd.sparseconvnet as scn
    m = scn.FusedNetworkInNetwork(9, 6, True, "silu").to(gpu)
    wide = rnd(1, 70, 33).float().to(gpu)
    x, res = wide[:, 5:14], wide[:, 20:26]
    y = m(scn.SparseConvNetTensor(x), residual=res).features
    assert torch.equal(y, m(scn.SparseConvNetTensor(x.clone()), residual=res.clone()).features)
    xg = x.clone().requires_grad_(True)
    y = m(scn.SparseConvNetTensor(xg)).features
    dy = rnd(2, 70, 6).float().to(gpu)
    slice_of = torch.zeros(70, 20, device=gpu)
    slice_of[:, 7:13] = dy
    want = torch.autograd.grad(y, [xg, m.weight, m.bias], dy, retain_graph=True)
    for other in (slice_of[:, 7:13], dy.t().contiguous().t()):
        assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(y, [xg, m.weight, m.bias], other, retain_graph=True)))
    e = torch.zeros(0, 9, device=gpu, requires_grad=True)
    y = m(scn.SparseConvNetTensor(e)).features
    grads = torch.autograd.grad(y, [e, m.weight, m.bias], torch.zeros(0, 6, device=gpu))
    assert y.shape == (0, 6) and grads[0].shape == (0, 9) and (grads[1] == 0).all() and (grads[2] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_linear_many_outputs_are_those_of_few(gpu, dtype):
    """a product's order of summation is that of its planes whatever the number of sites: large calls (other column blocks, weights laid
    out anew) give the bits of small ones, which test_linear compares with float64.  (33.75 million outputs.)"""
    from occuseg_amd import SCN
    t, N, K, M, few = TYPES[dtype], 67500, 100, 500, 300
    g = torch.Generator(device=gpu).manual_seed(6)
    x, w, b, res, dy = (torch.randn(*shape, device=gpu, generator=g).to(t) for shape in ((N, K), (K, M), (M,), (N, M), (N, M)))
    rng = torch.tensor([8, 9], device=gpu)

    def run(rows, p):
        y, factor, dx = x.new_empty(0), torch.empty(0, dtype=SCN.factor_dtype(x), device=gpu), x.new_empty(0)
        SCN.FusedNetworkInNetwork_updateOutput(x[rows], y, w, b, res[rows], "gelu", 1, p, rng, factor)
        SCN.FusedNetworkInNetwork_backward(x[rows], dx, dy[rows], w, None, None, "gelu", 1, p, factor)
        return y, factor, dx

    for p, parts in ((0.0, (slice(0, few), slice(N - few, N))), (0.4, (slice(0, few),))):
        whole = run(slice(0, N), p)
        for rows in parts:
            assert all(torch.equal(a[rows], c) for a, c in zip(whole, run(rows, p))), (p, rows)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("K,M", [(352, 64), (353, 64), (704, 64), (705, 64), (128, 416), (128, 417), (64, 353), (64, 705)])
def test_linear_weights_that_just_fit(gpu, K, M, dtype):
    """both sides of where the weights of a column block stop staying on a CU: the bits of small calls, as above"""
    from occuseg_amd import SCN
    t, N, few = TYPES[dtype], 33000, 200
    g = torch.Generator(device=gpu).manual_seed(7)
    x, w, b, dy = (torch.randn(*shape, device=gpu, generator=g).to(t) for shape in ((N, K), (K, M), (M,), (N, M)))

    def run(rows):
        y, factor, dx = x.new_empty(0), torch.empty(0, dtype=SCN.factor_dtype(x), device=gpu), x.new_empty(0)
        SCN.FusedNetworkInNetwork_updateOutput(x[rows], y, w, b, None, "silu", 1, 0.0, None, factor)
        SCN.FusedNetworkInNetwork_backward(x[rows], dx, dy[rows], w, None, None, "silu", 1, 0.0, factor)
        return y, factor, dx

    whole = run(slice(0, N))
    for rows in (slice(0, few), slice(N - few, N)):
        assert all(torch.equal(a[rows], c) for a, c in zip(whole, run(rows))), rows


def test_rows_do_not_mix(gpu):
    """a row of NaN or infinity reaches its own output and the weight's gradient only"""
    import occuseg_amd.sparseconvnet as scn
    for t, k in ((torch.float32, 35), (torch.bfloat16, 35), (torch.float16, 64)):
        m = scn.FusedNetworkInNetwork(k, 50, True, "gelu").to(gpu).to(t)
        x = rnd(1, 200, k).to(gpu, t)
        clean = m(scn.SparseConvNetTensor(x)).features
        x[77], x[199] = float("nan"), float("inf")
        y = m(scn.SparseConvNetTensor(x)).features
        rest = [i for i in range(200) if i not in (77, 199)]
        assert torch.equal(y[rest], clean[rest]) and y[77].isnan().all()


# ------------------------------------------------------------------------------------------------------------ together ---
def block(scn, gpu, p, dtype=torch.float32):
    torch.manual_seed(0)
    return torch.nn.ModuleList([scn.GroupNormSiLU(16, 4), scn.FusedNetworkInNetwork(16, 48, True, "gelu", dropout=p),
                                scn.FusedNetworkInNetwork(48, 16, True, dropout=p), scn.Dropout(p)]).to(gpu).to(dtype)


def run_block(scn, mods, inp):
    h = mods[1](mods[0](inp))
    return mods[3](mods[2](h, residual=inp)).features


def test_block_against_float64(gpu):
    """group norm -> hidden layer with dropout -> output layer with the block's input as residual -> dropout; every gradient"""
    import occuseg_amd.sparseconvnet as scn
    mods = block(scn, gpu, 0.25)
    lengths = [211, 0, 40]
    x = rnd(1, 251, 16).float()
    xg = x.to(gpu).requires_grad_(True)
    for i, m in enumerate(mods[1:]):
        m.reseed(100 + i)
    y = run_block(scn, mods, batch_tensor(gpu, scn, xg, lengths))
    dy = rnd(2, 251, 16).float()
    params = [p for m in mods for p in m.parameters()]
    got = [y] + list(torch.autograd.grad(y, [xg] + params, dy.to(gpu)))
    # float64
    P = [p.detach().double().cpu().requires_grad_(True) for p in params]
    X = x.double().requires_grad_(True)
    k = [O.keep(100 + i, 0, 251, c, 0.25) / 0.75 for i, c in enumerate((48, 16, 16))]
    n = torch.cat([((g - g.mean((0, 2), keepdim=True)) * (g.var((0, 2), keepdim=True, unbiased=False) + 1e-4).rsqrt()).reshape(-1, 16)
                   for g in X.view(-1, 4, 4).split([211, 40])])
    h = torch.nn.functional.silu(n * P[0] + P[1])
    h = torch.nn.functional.gelu(h @ P[2] + P[3]) * k[0]
    out = (X + (h @ P[4] + P[5]) * k[1]) * k[2]
    want = [out] + list(torch.autograd.grad(out, [X] + P, dy.double()))
    for i, (a, b) in enumerate(zip(got, want)):
        # five products in a row, each relative to sums of at most 251 terms: 2^-24 x (4 x 64 + 251) of the largest value
        check(a, b.detach(), torch.full_like(b, 512 * U * max(1.0, float(b.detach().abs().max()))), "output %d" % i)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_block_is_reproducible_and_replays_in_a_graph(gpu, dtype):
    """the same numbers bit for bit: twice in a row, on another stream, and from a captured pass replayed between eager work"""
    import occuseg_amd.sparseconvnet as scn
    mods = block(scn, gpu, 0.25, dtype)
    params = [p for m in mods for p in m.parameters()]
    inp = batch_tensor(gpu, scn, rnd(1, 700, 16).to(gpu, dtype).requires_grad_(True), [300, 400])
    dy = rnd(2, 700, 16).to(gpu, dtype)

    def step():
        # (detached: a backward pass must not be captured while an eager graph of the same leaves lives -- the leaves' accumulation
        #  nodes belong to that graph's stream, and torch ends the capture with a crash)
        y = run_block(scn, mods, inp)
        return [y.detach()] + list(torch.autograd.grad(y, [inp.features] + params, dy))

    def seeded(offset):
        for m in mods[1:]:
            m.reseed(5, offset)

    want = []
    for offset in range(4):
        seeded(offset)
        want.append([t.clone() for t in step()])
    seeded(0)
    assert all(torch.equal(a, b) for a, b in zip(step(), want[0]))
    seeded(0)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    seeded(0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    seeded(0)
    for offset in range(4):
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(static, want[offset])), "replay %d" % offset
        junk = torch.randn(1 << 20, device=gpu).sum()  # other work and memory between the replays
        torch.cuda.synchronize()
        del junk


def test_gradients_against_differences(gpu):
    """fp32 block along random directions: (f(x + h v) - f(x - h v)) / 2 h.  The sums of f are made in float64; an output's fp32 error
    is some 2^-21, of 3200 outputs' signs at random 2^-15, over 2 h = 2^-7: 2^-8; the third derivative's term h^2 / 6 f''' is of
    that size too"""
    import occuseg_amd.sparseconvnet as scn
    mods = block(scn, gpu, 0.25)
    x, dy = rnd(1, 200, 16).float().to(gpu), rnd(2, 200, 16).float().to(gpu)

    def f(x):
        for m in mods[1:]:
            m.reseed(5)
        return run_block(scn, mods, batch_tensor(gpu, scn, x, [150, 50]))

    xg = x.clone().requires_grad_(True)
    (grad,) = torch.autograd.grad(f(xg), [xg], dy)
    h = 2.0 ** -8
    for seed in range(3):
        v = rnd(10 + seed, 200, 16).float().to(gpu)
        with torch.no_grad():
            diff = float(((f(x + h * v).double() - f(x - h * v).double()) * dy.double()).sum()) / (2 * h)
        want = float((grad.double() * v.double()).sum())
        # the directional derivative is itself a sum of 3200 terms of size 1
        assert abs(diff - want) < 2.0 ** -6 * 3200 ** 0.5, (diff, want)


def test_trains_inside_a_network(gpu):
    """beside the convolutions, under the flat gradient buffer of data-parallel training"""
    import occuseg_amd.sparseconvnet as scn
    from occuseg_amd import dp
    torch.manual_seed(0)
    net = scn.Sequential().add(scn.SubmanifoldConvolution(3, 3, 16, 3, False)).add(scn.GroupNormSiLU(16, 4)) \
        .add(scn.SubmanifoldConvolution(3, 16, 16, 3, False)).add(scn.Dropout(0.2)).add(scn.FusedNetworkInNetwork(16, 5, True))
    net = net.to(gpu)
    bucket = dp.FlatGradBucket(net.parameters())
    inp = batch_tensor(gpu, scn, rnd(1, 320, 3).float().to(gpu), [300, 20])
    bucket.zero()
    net(inp).features.sum().backward()
    assert all(p.grad is not None and p.grad.isfinite().all() and p.grad.abs().max() > 0 for p in net.parameters())
    assert bucket.flat.abs().max() > 0


def test_refusals(gpu):
    import occuseg_amd.sparseconvnet as scn
    from occuseg_amd import SCN
    x = torch.zeros(4, 8, device=gpu)
    t = scn.SparseConvNetTensor
    for call in (lambda: scn.Dropout(0.5).to(gpu)(t(x.double())),
                 lambda: scn.Dropout(0.5).to(gpu)(t(x), rng=torch.zeros(2, dtype=torch.int64)),
                 lambda: scn.Dropout(0.5).to(gpu)(t(x), rng=torch.zeros(3, dtype=torch.int64, device=gpu)),
                 lambda: scn.Dropout(0.5)(t(x)),  # (state on the CPU)
                 lambda: scn.FusedNetworkInNetwork(8, 4).to(gpu)(t(x.half())),
                 lambda: scn.FusedNetworkInNetwork(7, 4).to(gpu)(t(x)),
                 lambda: scn.FusedNetworkInNetwork(8, 4).to(gpu)(t(x), residual=x),
                 lambda: scn.FusedNetworkInNetwork(8, 8).to(gpu)(t(x), residual=x.bfloat16()),
                 lambda: scn.FusedNetworkInNetwork(8, 8).to(gpu)(t(x), residual=x.cpu()),
                 lambda: scn.GroupNormalization(16, 4).to(gpu)(t(x)),
                 lambda: SCN.GroupNormalization_updateOutput(x, x.new_empty(0), x.new_empty(0), torch.zeros(2, device=gpu), None, None,
                                                             1e-4, 2, "silu", 1),
                 lambda: SCN.GroupNormalization_updateOutput(torch.zeros(4, 8192, device=gpu), x.new_empty(0), x.new_empty(0),
                                                             torch.tensor([0, 4], device=gpu), None, None, 1e-4, 2, "silu", 1),
                 lambda: SCN.FusedNetworkInNetwork_backward(x, None, x, torch.zeros(8, 4, device=gpu), None, None, "silu", 1, 0.0)):
        with pytest.raises(RuntimeError):
            call()
    xg = x.clone().requires_grad_(True)
    y = scn.FusedNetworkInNetwork(8, 4, True, "silu").to(gpu)(t(xg)).features
    (g,) = torch.autograd.grad(y.sum(), [xg], create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()  # no second derivatives


def test_outputs_of_another_type_or_device_are_refused(gpu):
    """an output that is smaller than what the kernel writes"""
    from occuseg_amd import SCN
    x, w, rng = torch.zeros(6, 8, device=gpu), torch.zeros(8, 4, device=gpu), torch.zeros(2, dtype=torch.int64, device=gpu)
    offsets = torch.tensor([0, 6], device=gpu)
    e, half, host = x.new_empty(0), x.new_empty(0).half(), torch.empty(0)
    stats = torch.zeros(1, 2, 2, device=gpu)
    for bad in (half, host):
        for call in (lambda: SCN.Dropout_updateOutput(x, bad, 0.5, rng),
                     lambda: SCN.GroupNormalization_updateOutput(x, bad, e, offsets, None, None, 1e-4, 2, "silu", 1),
                     lambda: SCN.GroupNormalization_updateOutput(x, e, bad, offsets, None, None, 1e-4, 2, "silu", 1),
                     lambda: SCN.GroupNormalization_backward(x, bad, x, stats, offsets, None, None, None, None, 2, "silu", 1),
                     lambda: SCN.GroupNormalization_backward(x, e, x, stats.to(bad), offsets, None, None, None, None, 2, "silu", 1),
                     lambda: SCN.GroupNormalization_backward(x, e, x, stats, offsets, None, None, torch.zeros(8).to(bad), None, 2, "silu", 1),
                     lambda: SCN.GroupNormalization_backward(x, e, x, stats, offsets, None, None, None, torch.zeros(8).to(bad), 2, "silu", 1),
                     lambda: SCN.FusedNetworkInNetwork_updateOutput(x, bad, w, None, None, "silu", 1, 0.0, None),
                     lambda: SCN.FusedNetworkInNetwork_updateOutput(x, e, w, None, None, "silu", 1, 0.0, None, bad),
                     lambda: SCN.FusedNetworkInNetwork_backward(x, bad, x[:, :4], w, None, None, "leaky_relu", 1, 0.0),
                     lambda: SCN.FusedNetworkInNetwork_backward(x, None, x[:, :4], w, bad, None, "leaky_relu", 1, 0.0),
                     lambda: SCN.FusedNetworkInNetwork_backward(x, None, x[:, :4], w, x.new_empty(0), bad, "leaky_relu", 1, 0.0)):
            with pytest.raises(RuntimeError, match="output on"):
                call()
