"""Group norm, dropout and the 1x1 convolution with its epilogue, over the active sites of a batch: the cases they are
measured on, their plain forms, their calls, and their values in 64 bits.

    group norm   per sample s and group g of C/G planes, over the sample's sites:  y = act((x - mean) / sqrt(var + eps) * w + b)
    dropout      y = x / (1 - p) where the site's random word is >= p 2^32, else 0; the words are Philox4x32-10 of
                 key = seed, counter = (plane / 4, row, offset)
    1x1 conv     y = residual + dropout(act(x W + b))

Features are [sites, planes]; a training pass returns the gradients beside the outputs.  Leaky ReLU is measured forwards only:
its slope jumps at zero, so two correct roundings of one pre-activation may differ in a gradient by a whole term.
"""
import math

import torch

own = False

EPS = 1e-4
LEAK = 0.333
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
MASK32 = 0xFFFFFFFF


# ------------------------------------------------------------------------------------------------------------- cases ---
def listed():
    return [
        # the coarsest level of the m64 network in a serving pass: a few hundred sites, a sample without any, one with one
        dict(name="gn_f32_coarse", op="gn", type="f32", lengths="211,190,0,1", planes=448, groups=32, act="leaky", train=False),
        # four scenes at the input level of a train step
        dict(name="gn_f32_scenes_train", op="gn", type="f32", lengths="150211,149870,151003,150590", planes=64, groups=8,
             act="silu", train=True),
        # the next level in half the bytes; one scene was dropped by the loader
        dict(name="gn_bf16_level1_train", op="gn", type="bf16", lengths="44250,44251,0,88500", planes=128, groups=32,
             act="silu", train=True),
        # planes of a head with seven classes of three numbers each: rows that no wide load fits
        dict(name="gn_f16_odd", op="gn", type="f16", lengths="30011,1,7", planes=21, groups=7, act="leaky", train=False),
        # dropout behind the coarsest level
        dict(name="drop_f32_coarse", op="drop", type="f32", rows=402, planes=448, p=0.5, train=False),
        # ... behind the input level of four scenes
        dict(name="drop_bf16_scenes_train", op="drop", type="bf16", rows=601674, planes=128, p=0.1, train=True),
        # ... in front of an odd head
        dict(name="drop_f16_odd_train", op="drop", type="f16", rows=50001, planes=35, p=0.3, train=True),
        # one site through a hidden layer: the smallest call of a serving loop
        dict(name="nin_f32_one_site", op="nin", type="f32", rows=1, n_in=448, n_out=448, act="silu", residual=True, p=0.0,
             train=False),
        # the classifier: 64 planes to 20 classes for every voxel of four scenes
        dict(name="nin_f32_classifier", op="nin", type="f32", rows=601674, n_in=64, n_out=20, act="none", residual=False, p=0.0,
             train=False),
        # first layer of a residual channel block at level 1
        dict(name="nin_f32_level1_train", op="nin", type="f32", rows=177001, n_in=64, n_out=128, act="gelu", residual=True, p=0.1,
             train=True),
        # the wide layer of such a block
        dict(name="nin_bf16_wide_train", op="nin", type="bf16", rows=177001, n_in=128, n_out=512, act="gelu", residual=False, p=0.1,
             train=True),
        # planes that no wide load or whole tile fits
        dict(name="nin_f16_odd_train", op="nin", type="f16", rows=50001, n_in=35, n_out=77, act="silu", residual=True, p=0.2,
             train=True),
    ]


def _log_size(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["gn", "drop", "nin"])
    case = dict(op=op, type=rng.choice(["f32", "bf16", "f16"]), train=rng.random() < 0.6)
    rows = _log_size(rng, 1, 600000)
    if op == "gn":
        per_group = rng.choice([1, 2, 3, 4, 7, 8, 14, 16])
        case["groups"] = _log_size(rng, 1, 32)
        case["planes"] = per_group * case["groups"]
        rows = min(rows, 77000000 // case["planes"])
        cuts = sorted(rng.randint(0, rows) for _ in range(rng.randint(0, 7)))
        case["lengths"] = ",".join(str(b - a) for a, b in zip([0] + cuts, cuts + [rows]))
        case["act"] = rng.choice(["none", "silu", "gelu"] if case["train"] else ["none", "leaky", "silu", "gelu"])
    elif op == "drop":
        case["planes"] = _log_size(rng, 1, 512)
        case["rows"] = min(rows, 77000000 // case["planes"])
        case["p"] = round(rng.uniform(0.05, 0.9), 3)
    else:
        case["n_in"], case["n_out"] = _log_size(rng, 1, 512), _log_size(rng, 1, 512)
        case["rows"] = min(rows, 11000000000 // (case["n_in"] * case["n_out"]), 110000000 // (case["n_in"] + 2 * case["n_out"]))
        case["act"] = rng.choice(["none", "silu", "gelu"] if case["train"] else ["none", "leaky", "silu", "gelu"])
        case["residual"] = rng.random() < 0.5
        case["p"] = rng.choice([0.0, 0.1, 0.5])
    return case


def _lengths(case):
    return [int(n) for n in case["lengths"].split(",")]


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "nin":
        rows, n_in, n_out = case["rows"], case["n_in"], case["n_out"]
        tensors = n_in + n_out + (n_out if case["residual"] else 0) + ((n_in + n_out) if case["train"] else 0)
        weights = (n_in + 1) * n_out * (2 if case["train"] else 1)
        return {"bytes": size * (rows * tensors + weights), "flops": 2 * rows * n_in * n_out * (3 if case["train"] else 1)}
    elements = (sum(_lengths(case)) if case["op"] == "gn" else case["rows"]) * case["planes"]
    passes = 4 if case["train"] else 2
    per_element = 8 if case["op"] == "gn" else 1
    return {"bytes": size * elements * passes, "flops": per_element * elements * (2 if case["train"] else 1)}


# ------------------------------------------------------------------------------------------------------------ inputs ---
def _sites(lengths, device):
    """distinct voxels [sites, 4] = (x, y, z, sample), one sample behind the other"""
    parts = []
    for sample, n in enumerate(lengths):
        i = torch.arange(n, device=device)
        parts.append(torch.stack([i % 128, i // 128 % 128, i // 16384, torch.full_like(i, sample)], 1))
    return torch.cat(parts)


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    dtype = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=device)

    state = {"case": case, "rng": torch.randint(-2**63, 2**63 - 1, (2,), generator=gen, device=device)}
    if case["op"] == "nin":
        rows, n_in, n_out = case["rows"], case["n_in"], case["n_out"]
        state["x"] = normal(rows, n_in).to(dtype)
        state["weight"] = (normal(n_in, n_out) * math.sqrt(2.0 / n_in)).to(dtype)
        state["bias"] = (0.1 * normal(n_out)).to(dtype)
        state["residual"] = normal(rows, n_out).to(dtype) if case["residual"] else None
        state["dy"] = normal(rows, n_out).to(dtype) if case["train"] else None
    else:
        planes = case["planes"]
        rows = sum(_lengths(case)) if case["op"] == "gn" else case["rows"]
        # (a convolution's output: planes of different scale and level)
        state["x"] = (normal(rows, planes) * torch.exp(0.5 * normal(planes)) + normal(planes)).to(dtype)
        state["dy"] = normal(rows, planes).to(dtype) if case["train"] else None
        if case["op"] == "gn":
            state["weight"], state["bias"] = 1 + 0.1 * normal(planes), 0.1 * normal(planes)
    if own:
        _prepare_own(case, state)
    return state


def _prepare_own(case, state):
    """what a program that uses the framework keeps: the module with its parameters, and the tensor over its batch's sites"""
    import occuseg_amd.sparseconvnet as scn
    leak = LEAK if case.get("act") == "leaky" else 1
    act = case.get("act") if case.get("act") in ("silu", "gelu") else "leaky_relu"
    metadata, size = None, None
    if case["op"] == "gn":
        module = scn.GroupNormalization(case["planes"], case["groups"], eps=EPS, activation=act, leakiness=leak)
        metadata, size = scn.Metadata(3), torch.tensor([4096] * 3)
        lengths = _lengths(case)
        metadata.inputLayer(size, _sites(lengths, state["x"].device), len(lengths), 3, state["x"].device)
    elif case["op"] == "drop":
        module = scn.Dropout(case["p"])
    else:
        module = scn.FusedNetworkInNetwork(case["n_in"], case["n_out"], True, activation=act, leakiness=leak, dropout=case["p"])
        module.to(state["x"].dtype)
    module.to(state["x"].device)
    if "weight" in state:
        with torch.no_grad():
            module.weight.copy_(state["weight"])
            module.bias.copy_(state["bias"])
    state["module"] = module.train(case["train"] or case.get("p", 0) > 0)
    state["x"].requires_grad_(case["train"])
    if state.get("residual") is not None:
        state["residual"].requires_grad_(case["train"])
    state["input"] = scn.SparseConvNetTensor(state["x"], metadata, size)


def _run_own(state):
    case, module, dy = state["case"], state["module"], state["dy"]
    extra = {}
    if case.get("p", 0) > 0:
        extra["rng"] = state["rng"]
    if state.get("residual") is not None:
        extra["residual"] = state["residual"]
    if not case["train"]:
        with torch.no_grad():
            return module(state["input"], **extra).features
    out = module(state["input"], **extra).features
    leaves = [state["x"]] + ([module.weight, module.bias] if "weight" in state else [])
    if "residual" in extra:
        leaves.append(state["residual"])
    return [out] + list(torch.autograd.grad(out, leaves, dy))


# ------------------------------------------------------------------------------------------------------- plain forms ---
def _act(z, act):
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "leaky":
        return torch.where(z > 0, z, z * LEAK)
    return z


def _act_slope(z, act):
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * math.sqrt(0.5 / math.pi)
    if act == "leaky":
        return torch.where(z > 0, torch.ones_like(z), torch.full_like(z, LEAK))
    return torch.ones_like(z)


def _threshold(p):
    return int(p * 4294967296.0)


def _keep(rng, rows, planes, p):
    """truth values [rows, planes]: the random word of an element is at least p 2^32.  Products of two 32-bit words wrap in
    int64, but all their 64 bits are there."""
    quads = (planes + 3) // 4
    device = rng.device
    k0, k1 = rng[0] & MASK32, (rng[0] >> 32) & MASK32
    c0 = torch.arange(quads, device=device).expand(rows, quads)
    c1 = torch.arange(rows, device=device).view(rows, 1).expand(rows, quads)
    c2, c3 = (rng[1] & MASK32).expand(rows, quads), ((rng[1] >> 32) & MASK32).expand(rows, quads)
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & MASK32) ^ c1 ^ k0, b & MASK32, ((a >> 32) & MASK32) ^ c3 ^ k1, a & MASK32
        k0, k1 = (k0 + 0x9E3779B9) & MASK32, (k1 + 0xBB67AE85) & MASK32
    words = torch.stack([c0, c1, c2, c3], 2).view(rows, quads * 4)
    return words[:, :planes] >= _threshold(p)


def _run_gn(state):
    case = state["case"]
    groups, act, dtype = case["groups"], case["act"], state["x"].dtype
    planes = case["planes"]
    weight, bias = state["weight"], state["bias"]
    outs, dxs = [], []
    dweight, dbias = torch.zeros_like(weight), torch.zeros_like(bias)
    lengths = _lengths(case)
    for n, x, dy in zip(lengths, state["x"].split(lengths), state["dy"].split(lengths) if case["train"] else [None] * len(lengths)):
        if n == 0:
            continue
        x = x.float().view(n, groups, planes // groups)
        x = x - x.mean((0, 2), keepdim=True)
        scale = 1 / torch.sqrt((x * x).mean((0, 2), keepdim=True) + EPS)
        normed = x * scale
        w = weight.view(1, groups, -1)
        z = normed * w + bias.view(1, groups, -1)
        outs.append(_act(z, act).view(n, planes))
        if case["train"]:
            dz = dy.float().view(n, groups, -1) * _act_slope(z, act)
            dweight += (dz * normed).sum(0).view(-1)
            dbias += dz.sum(0).view(-1)
            dn = dz * w
            dxs.append((scale * (dn - dn.mean((0, 2), keepdim=True) - normed * (dn * normed).mean((0, 2), keepdim=True))).view(n, planes))
    if not outs:
        outs, dxs = [state["x"].float()], [state["x"].float()]
    out = torch.cat(outs).to(dtype)
    return [out, torch.cat(dxs).to(dtype), dweight, dbias] if case["train"] else out


def _drop(values, keep, p):
    return torch.where(keep, values * (1 / (1 - p)), torch.zeros_like(values))


def _run_drop(state):
    case, x = state["case"], state["x"]
    keep = _keep(state["rng"], case["rows"], case["planes"], case["p"])
    out = _drop(x.float(), keep, case["p"]).to(x.dtype)
    return [out, _drop(state["dy"].float(), keep, case["p"]).to(x.dtype)] if case["train"] else out


def _run_nin(state):
    case, dtype, p = state["case"], state["x"].dtype, state["case"]["p"]
    x, weight = state["x"].float(), state["weight"].float()
    z = x @ weight + state["bias"].float()
    out = _act(z, case["act"])
    keep = _keep(state["rng"], case["rows"], case["n_out"], p) if p > 0 else None
    if keep is not None:
        out = _drop(out, keep, p)
    if state["residual"] is not None:
        out = out + state["residual"].float()
    if not case["train"]:
        return out.to(dtype)
    dz = state["dy"].float()
    if keep is not None:
        dz = _drop(dz, keep, p)
    dz = dz * _act_slope(z, case["act"])
    grads = [(dz @ weight.t()).to(dtype), (x.t() @ dz).to(dtype), dz.sum(0).to(dtype)]
    return [out.to(dtype)] + grads + ([state["dy"]] if state["residual"] is not None else [])


def run(state):
    if own:
        return _run_own(state)
    return {"gn": _run_gn, "drop": _run_drop, "nin": _run_nin}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------- values in 64 bits ---
def _mulhilo(c, m):
    """high and low word of the product of 32-bit words, in 16-bit limbs that stay below 2^63"""
    c_hi, c_lo = c // 65536, c % 65536
    low = c_lo * m
    mid = c_hi * m + low // 65536
    return mid // 65536, mid % 65536 * 65536 + low % 65536


def _exact_keep(rng, rows, planes, p):
    seed, offset = (int(v) % 2**64 for v in rng.tolist())
    key = [seed % 2**32, seed // 2**32]
    plane, row = torch.arange((planes + 3) // 4, device=rng.device), torch.arange(rows, device=rng.device)
    zero = torch.zeros(rows, plane.numel(), dtype=torch.int64, device=rng.device)
    ctr = [zero + plane, zero + row[:, None], zero + offset % 2**32, zero + offset // 2**32]
    for _ in range(10):
        hi0, lo0 = _mulhilo(ctr[0], 0xD2511F53)
        hi1, lo1 = _mulhilo(ctr[2], 0xCD9E8D57)
        ctr = [hi1.bitwise_xor(ctr[1]).bitwise_xor(torch.full_like(hi1, key[0])), lo1,
               hi0.bitwise_xor(ctr[3]).bitwise_xor(torch.full_like(hi0, key[1])), lo0]
        key = [(key[0] + 0x9E3779B9) % 2**32, (key[1] + 0xBB67AE85) % 2**32]
    words = torch.empty(rows, plane.numel(), 4, dtype=torch.int64, device=rng.device)
    for lane in range(4):
        words[:, :, lane] = ctr[lane]
    return words.flatten(1)[:, :planes] >= math.floor(p * 2.0**32)


def _exact_act(z, act):
    """the activation and its slope"""
    if act == "silu":
        s = torch.special.expit(z)
        return z * s, s + z * s * (1 - s)
    if act == "gelu":
        cdf = torch.special.ndtr(z)
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    slope = torch.where(z > 0, 1.0, LEAK if act == "leaky" else 1.0).double()
    return z * slope, slope


def exact(case, seed):
    state = prepare(case, seed)
    x = state["x"].detach().double()
    dy = state["dy"].double() if case["train"] else None
    if case["op"] == "drop":
        factor = _exact_keep(state["rng"], case["rows"], case["planes"], case["p"]).double() / (1 - case["p"])
        return [x * factor, dy * factor] if case["train"] else x * factor
    weight, bias = state["weight"].detach().double(), state["bias"].detach().double()
    if case["op"] == "nin":
        z = torch.addmm(bias, x, weight)
        value, slope = _exact_act(z, case["act"])
        factor = torch.ones_like(z)
        if case["p"] > 0:
            factor = _exact_keep(state["rng"], case["rows"], case["n_out"], case["p"]).double() / (1 - case["p"])
        residual = state["residual"]
        out = value * factor + (residual.detach().double() if residual is not None else 0)
        if not case["train"]:
            return out
        dz = dy * factor * slope
        return [out, torch.mm(dz, weight.t().contiguous()), torch.mm(x.t().contiguous(), dz), dz.sum(0)] + \
            ([dy] if residual is not None else [])
    # group norm: sums by sample and group
    lengths = _lengths(case)
    rows, planes, groups = x.size(0), case["planes"], case["groups"]
    sample = torch.repeat_interleave(torch.arange(len(lengths), device=x.device), torch.tensor(lengths, device=x.device))
    count = torch.tensor(lengths, device=x.device, dtype=torch.float64).clamp(min=1)[:, None] * (planes // groups)

    def means(values):
        sums = torch.zeros(len(lengths), planes, dtype=torch.float64, device=x.device).index_add_(0, sample, values)
        sums = sums.view(len(lengths), groups, -1).sum(2) / count
        return sums.repeat_interleave(planes // groups, 1)[sample]

    centred = x - means(x)
    rstd = (means(centred * centred) + EPS).rsqrt()
    normed = centred * rstd
    value, slope = _exact_act(normed * weight + bias, case["act"])
    if not case["train"]:
        return value
    dz = dy * slope
    dn = dz * weight
    dx = rstd * (dn - means(dn) - normed * means(dn * normed))
    return [value, dx, (dz * normed).sum(0), dz.sum(0)]
