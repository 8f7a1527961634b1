"""not gpu: the oracle of the pointwise operators against published vectors and differences; what the operators refuse."""
import numpy as np
import pytest
import torch

from oracle import pointwise as O


def test_philox_known_answers():
    """the three vectors the generator is published with (counter and key of zeros, of ones, of pi's digits)"""
    ones = 0xFFFFFFFF
    for ctr, key, want in (
            ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
            ((ones,) * 4, (ones,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
            ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
             (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        assert tuple(int(w) for w in O.philox(np.array(ctr), key)) == want


def _difference(f, x, direction, h=1e-6):
    return float((f(x + h * direction) - f(x - h * direction)) / (2 * h))


@pytest.mark.parametrize("activation", ["leaky_relu", "silu", "gelu"])
def test_oracle_gradients_against_differences(activation):
    g = torch.Generator().manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    lengths, C, groups = [5, 0, 1, 9], 6, 3
    x, w, b, dy = rnd(15, C), rnd(C), rnd(C), rnd(15, C)
    out = O.group_norm(x, lengths, groups, w, b, 1e-3, activation, 0.3, dy)
    loss = lambda x=x, w=w, b=b: (O.group_norm(x, lengths, groups, w, b, 1e-3, activation, 0.3)["y"] * dy).sum()  # noqa: E731
    for name, leaf, grad in (("x", x, out["dx"]), ("w", w, out["dw"]), ("b", b, out["db"])):
        d = rnd(*leaf.shape)
        assert abs(_difference(lambda t: loss(**{name: t}), leaf, d) - float((grad * d).sum())) < 1e-6, name
    x, w, b, res, dy = rnd(7, 4), rnd(4, 5), rnd(5), rnd(7, 5), rnd(7, 5)
    mask = O.keep(11, 3, 7, 5, 0.4)
    out = O.linear(x, w, b, res, activation, 0.3, mask, 0.4, dy)
    loss = lambda x=x, w=w, b=b: (O.linear(x, w, b, res, activation, 0.3, mask, 0.4)["y"] * dy).sum()  # noqa: E731
    for name, leaf, grad in (("x", x, out["dx"]), ("w", w, out["dw"]), ("b", b, out["db"])):
        d = rnd(*leaf.shape)
        assert abs(_difference(lambda t: loss(**{name: t}), leaf, d) - float((grad * d).sum())) < 1e-6, name


def test_mask_frequency():
    """4 x 10^5 words: the share kept is within five standard deviations of 1 - p, per lane of the counter too"""
    k = O.keep(-5, 2 ** 40 + 1, 2000, 200, 0.3).numpy()
    assert abs(k.mean() - 0.7) < 5 * np.sqrt(0.21 / k.size)
    for lane in range(4):
        part = k[:, lane::4]
        assert abs(part.mean() - 0.7) < 5 * np.sqrt(0.21 / part.size)


def test_modules_refuse():
    import occuseg_amd.sparseconvnet as scn
    for make in (lambda: scn.GroupNormalization(8, 3), lambda: scn.GroupNormalization(8, 0), lambda: scn.GroupNormalization(0, 1),
                 lambda: scn.GroupNormalization(8, 2, activation="tanh"), lambda: scn.Dropout(1.0), lambda: scn.Dropout(-0.1),
                 lambda: scn.Dropout(float("nan")), lambda: scn.FusedNetworkInNetwork(4, 4, activation="relu6"),
                 lambda: scn.FusedNetworkInNetwork(4, 4, dropout=1.5)):
        with pytest.raises(ValueError):
            make()
    x = scn.SparseConvNetTensor(torch.zeros(3, 4))
    for module in (scn.Dropout(0.5), scn.FusedNetworkInNetwork(4, 2)):
        with pytest.raises(RuntimeError, match="GPU"):
            module(x)
    # evaluation, and p = 0, hand the input on
    assert scn.Dropout(0.5).eval()(x) is x and scn.Dropout(0.0)(x) is x
    with pytest.raises(RuntimeError, match=r"\[sites, planes\]"):
        scn.FusedNetworkInNetwork(4, 2)(scn.SparseConvNetTensor(torch.zeros(3)))


def test_boundary_refuses_on_the_host():
    from occuseg_amd import SCN, _lib
    lib = _lib.load()
    e = torch.empty(0)
    with pytest.raises(RuntimeError, match="GPU"):
        SCN.GroupNormalization_updateOutput(torch.zeros(2, 4), e, e, torch.zeros(2, dtype=torch.int64), None, None, 1e-4, 2, "silu", 1)
    # the C entries look at their arguments before they launch anything
    assert lib.scn_group_norm_temp_bytes(100, 8, 3, 1, 0, 0) == 0 and lib.scn_group_norm_temp_bytes(100, 8, 2, 1, 0, 1) > 0
    assert lib.scn_group_norm_forward(None, None, None, None, None, None, 1e-4, 0, 1.0, 10, 8, 2, 1, 0, None, 0, None) == 2
    assert lib.scn_group_norm_forward(None, None, None, None, None, None, 1e-4, 7, 1.0, 10, 8, 2, 1, 0, None, 0, None) == 2
    assert lib.scn_group_norm_temp_bytes(100, 8, 2, 1, 0, 0) == 0 and lib.scn_group_norm_temp_bytes(10000, 8, 2, 1, 0, 0) > 0
    assert lib.scn_group_norm_backward(None, None, None, None, None, None, None, None, None, 0, 1.0, 10, 8, 2, 1, 3, None, 0, None) == 2
    assert lib.scn_dropout(None, 8, None, 10, 8, 0, 0.5, None, None) == 2
    assert lib.scn_dropout(None, 8, None, 10, 8, 0, 1.0, None, None) == 2
    assert lib.scn_dropout(None, 8, None, 0, 8, 0, 0.5, None, None) == 0
    assert lib.scn_linear_forward(None, 8, None, None, None, 0, None, None, 10, 8, 4, 0, 1.0, 0.0, None, 0, None, 0, None) == 2
    assert lib.scn_linear_forward(None, 8, None, None, None, 0, None, None, 10, 0, 4, 0, 1.0, 0.0, None, 0, None, 0, None) == 2
    assert lib.scn_linear_dinput(None, 4, None, None, None, 10, 8, 4, 0, 1.0, 0.0, 5, None) == 2
    assert lib.scn_linear_dweight(None, 8, None, 4, None, None, None, 10, 8, 4, 0, 1.0, 0.0, 0, None, 0, None) == 2
    assert lib.scn_rng_take(None, None, None) == 2
    assert lib.scn_sample_offsets(None, 0, 0, None, None) == 2
    assert lib.scn_linear_dweight_temp_bytes(1000, 8, 4) >= 4 * (8 * 4 + 4)


def test_dropout_state():
    import occuseg_amd.sparseconvnet as scn
    torch.manual_seed(4)
    a = scn.Dropout(0.5)
    torch.manual_seed(4)
    b = scn.FusedNetworkInNetwork(1, 1, dropout=0.5)
    assert a.rng_state.dtype == torch.int64 and int(a.rng_state[1]) == 0 and "rng_state" in a.state_dict()
    b.reseed(7, 9)
    assert b.rng_state.tolist() == [7, 9]
    assert a.to(torch.bfloat16).rng_state.dtype == torch.int64


def test_boundary_refuses_sizes_beyond_a_launch():
    """the pointers are not looked at: sizes and strides are refused first, on the host"""
    from occuseg_amd import _lib
    lib = _lib.load()
    p = torch.zeros(4).data_ptr()
    # strides whose multiples leave 32 bits, weights of more than 2^32 threads, sites beyond 2^31
    assert lib.scn_linear_forward(p, 1 << 27, p, None, None, 0, p, None, 40, 8, 4, 0, 1.0, 0.0, None, 0, None, 0, None) == 2
    assert lib.scn_linear_forward(p, 8, p, None, p, 1 << 27, p, None, 40, 8, 4, 0, 1.0, 0.0, None, 0, None, 0, None) == 2
    assert lib.scn_linear_dinput(p, 1 << 27, None, p, p, 40, 8, 4, 0, 1.0, 0.0, 0, None) == 2
    for ldx, ld_dy in ((1 << 27, 4), (8, 1 << 27)):
        assert lib.scn_linear_dweight(p, ldx, p, ld_dy, None, p, None, 40, 8, 4, 0, 1.0, 0.0, 0, p, 1 << 40, None) == 2
    assert lib.scn_linear_dweight(p, 1 << 15, p, 1 << 15, None, p, None, 40, 1 << 15, 1 << 15, 0, 1.0, 0.0, 0, p, 1 << 40, None) == 2
    assert lib.scn_linear_forward(p, 8, p, None, None, 0, p, None, 1 << 31, 8, 4, 0, 1.0, 0.0, None, 0, p, 1 << 40, None) == 2
    assert lib.scn_dropout(p, 8, p, 1 << 31, 8, 0, 0.5, p, None) == 2
    assert lib.scn_dropout(p, 7, p, 40, 8, 0, 0.5, p, None) == 2
    assert lib.scn_group_norm_temp_bytes(1 << 31, 8, 2, 1, 0, 0) == 0 and lib.scn_group_norm_temp_bytes(10, 8, 2, 1 << 16, 0, 0) == 0


def test_fused_layer_takes_the_parameters_of_a_plain_one():
    import occuseg_amd.sparseconvnet as scn
    plain, fused = scn.NetworkInNetwork(5, 3, True), scn.FusedNetworkInNetwork(5, 3, True, "silu", dropout=0.1)
    fused.reseed(3, 4)
    torch.nn.Sequential(fused).load_state_dict(torch.nn.Sequential(plain).state_dict())
    assert torch.equal(fused.weight, plain.weight) and fused.rng_state.tolist() == [3, 4]
    other = scn.FusedNetworkInNetwork(5, 3, True, "silu", dropout=0.1)
    other.load_state_dict(fused.state_dict())
    assert other.rng_state.tolist() == [3, 4] and torch.equal(other.weight, fused.weight)


def test_group_norm_of_few_sites_needs_no_workspace():
    """one launch where that is few workgroups with few values each, three and their workspace where not"""
    from occuseg_amd import _lib
    temp = lambda N, C, G, S: _lib.load().scn_group_norm_temp_bytes(N, C, G, S, 0, 0)  # noqa: E731
    for few in ((1, 1, 1, 1), (402, 448, 32, 4), (402, 448, 32, 1), (1024, 128, 128, 4), (4096, 32, 32, 4), (1024, 1024, 32, 4), (8192, 4, 4, 1), (0, 64, 8, 1)):
        assert temp(*few) == 0, few
    for many in ((32768, 1024, 1024, 1), (1024, 448, 32, 1), (256, 1024, 512, 4), (32768, 32, 32, 4), (16384, 64, 32, 4), (100, 8, 2, 512)):
        assert temp(*many) > 0, many


def test_plain_layer_takes_the_parameters_of_a_fused_one_without_dropout():
    import occuseg_amd.sparseconvnet as scn
    plain, fused = scn.NetworkInNetwork(5, 3, True), scn.FusedNetworkInNetwork(5, 3, True, "silu")
    torch.nn.Sequential(plain).load_state_dict(torch.nn.Sequential(fused).state_dict())
    assert torch.equal(plain.weight, fused.weight)
    # and one that was saved with its state
    old = dict(fused.state_dict(), rng_state=torch.tensor([8, 9]))
    other = scn.FusedNetworkInNetwork(5, 3, True, "silu")
    other.load_state_dict(old)
    assert torch.equal(other.weight, fused.weight) and other.rng_state.tolist() == [8, 9]
