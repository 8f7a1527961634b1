"""Dropout, and the 1x1 convolution with its epilogue.

Dropout makes its mask from a counter, forwards and backwards, and stores none; FusedNetworkInNetwork is NetworkInNetwork
(sparseconvnet/networkInNetwork.py:14-88: same `weight` [nIn, nOut], same initialisation) with what usually follows it inside
its kernel.
"""
import torch
from torch.autograd import Function
from torch.nn import Module, Parameter

from .. import SCN
from . import counters
from .tensor import SparseConvNetTensor, apply_function, first_order, optionalTensor


def _new(like, *shape):
    return torch.empty(shape, dtype=like.dtype, device=like.device)


def _like(input, features):
    return SparseConvNetTensor(features, input.metadata, input.spatial_size)


class _DropoutFunction(Function):
    @staticmethod
    def forward(ctx, features, p, rng):
        out = _new(features, *features.shape)
        SCN.Dropout_updateOutput(features, out, p, rng)
        ctx.p = p
        ctx.save_for_backward(rng)
        return out

    @staticmethod
    @first_order
    def backward(ctx, grad_output):
        (rng,) = ctx.saved_tensors
        grad_input = _new(grad_output, *grad_output.shape)
        SCN.Dropout_updateGradInput(grad_input, grad_output, ctx.p, rng)
        return grad_input, None, None


class _Random(Module):
    """a module that draws: the buffer `rng_state` = (seed, offset), int64 [2].  The seed comes from torch's CPU generator when the
    module is made; every training forward pass uses one offset.  The counting happens on the device, so a pass captured into a
    graph draws a new mask at every replay.  Ranks of a data-parallel job that are seeded alike draw alike: `reseed` them.  A forward
    pass that is run again for its gradients (activation checkpointing) draws again: hand it `rng`.  A copy of a module draws what
    its original draws until it is reseeded.  A state_dict without the buffer (of a NetworkInNetwork) leaves it as it is; that of a
    module that never draws (probability 0) is without it, and a NetworkInNetwork loads it."""

    def _save_to_state_dict(self, destination, prefix, keep_vars):
        Module._save_to_state_dict(self, destination, prefix, keep_vars)
        if not self.p:
            destination.pop(prefix + "rng_state", None)

    def _load_from_state_dict(self, state_dict, prefix, *args):
        state_dict.setdefault(prefix + "rng_state", self.rng_state)
        Module._load_from_state_dict(self, state_dict, prefix, *args)

    def _init_rng(self):
        self.register_buffer("rng_state", torch.stack([torch.randint(-2 ** 63, 2 ** 63 - 1, ()), torch.zeros((), dtype=torch.int64)]))

    def reseed(self, seed, offset=0):
        self.rng_state.copy_(torch.tensor([seed, offset], dtype=torch.int64))

    def _draw(self, rng):
        return SCN.rng_take(self.rng_state) if rng is None else rng


class Dropout(_Random):
    """features / (1 - p) for the elements kept, 0 for the others, in training; the input itself in evaluation.  No mask is stored:
    backward makes it again.  ``forward(input, rng)`` with an int64 tensor (seed, offset) on the features' device uses that instead
    of the module's own state and leaves the state alone -- the same ``rng``, the same mask."""

    def __init__(self, p=0.5):
        Module.__init__(self)
        self.p = SCN._drop_p("Dropout", p)
        self._init_rng()

    def forward(self, input, rng=None):
        if not self.training or self.p == 0:
            return input
        return _like(input, apply_function(_DropoutFunction, input.features, self.p, self._draw(rng)))

    def input_spatial_size(self, out_size):
        return out_size

    def __repr__(self):
        return "Dropout(p=%s)" % self.p


class _FusedNiNFunction(Function):
    @staticmethod
    def forward(ctx, features, weight, bias, residual, activation, leakiness, p, rng):
        shape = features.size(0), weight.size(1)
        out = _new(features, *shape)
        # what the backward pass needs of activation and mask: their common derivative, one value per output
        wanted = any(ctx.needs_input_grad[:3]) and (p > 0 or activation != "leaky_relu" or leakiness != 1)
        factor = torch.empty(shape, dtype=SCN.factor_dtype(features), device=features.device) if wanted else None
        macs = SCN.FusedNetworkInNetwork_updateOutput(features, out, weight, bias, residual, activation, leakiness, p, rng, factor)
        counters.add(macs, out.nelement())
        ctx.has_bias, ctx.args = bias.numel() > 0, (activation, leakiness, p)
        ctx.save_for_backward(features, weight, factor)
        return out

    @staticmethod
    @first_order
    def backward(ctx, grad_output):
        features, weight, factor = ctx.saved_tensors
        need_x, need_w, need_b, need_res = ctx.needs_input_grad[:4]
        need_b = need_b and ctx.has_bias
        grad_input = _new(features, *features.shape) if need_x else None
        grad_weight = _new(weight, *weight.shape) if need_w or need_b else None
        grad_bias = _new(weight, weight.size(1)) if need_b else None
        if need_x or need_w or need_b:
            SCN.FusedNetworkInNetwork_backward(features, grad_input, grad_output, weight, grad_weight, grad_bias, *ctx.args, factor)
        return (grad_input, grad_weight if need_w else None, grad_bias, grad_output if need_res else None) + (None,) * 4


class FusedNetworkInNetwork(_Random):
    """(not in the reference) ``residual + dropout(act(features @ weight + bias))`` in one kernel: ``activation`` "leaky_relu" with
    ``leakiness`` (0 = ReLU, 1 = none), "silu" or "gelu"; ``dropout`` = probability, in training.  ``forward(input, residual, rng)``:
    residual = a SparseConvNetTensor or a tensor [sites, nOut] (None: none), rng as Dropout's.  float32, bfloat16 or float16; the
    parameters must be of the features' type."""

    def __init__(self, nIn, nOut, bias=True, activation="leaky_relu", leakiness=1, dropout=0.0):
        Module.__init__(self)
        SCN._activation("FusedNetworkInNetwork", activation)
        self.nIn, self.nOut = nIn, nOut
        self.activation, self.leakiness = activation, leakiness
        self.p = SCN._drop_p("FusedNetworkInNetwork", dropout)
        self.weight = Parameter(torch.empty(nIn, nOut).normal_(0, (2.0 / nIn) ** 0.5))
        if bias:
            self.bias = Parameter(torch.zeros(nOut))
        self._init_rng()

    def forward(self, input, residual=None, rng=None):
        p = self.p if self.training else 0.0
        if isinstance(residual, SparseConvNetTensor):
            residual = residual.features
        return _like(input, apply_function(_FusedNiNFunction, input.features, self.weight, optionalTensor(self, "bias"), residual,
                                           self.activation, self.leakiness, p, self._draw(rng) if p > 0 else None))

    def input_spatial_size(self, out_size):
        return out_size

    def __repr__(self):
        s = "FusedNetworkInNetwork(%d->%d" % (self.nIn, self.nOut)
        if self.activation != "leaky_relu" or self.leakiness != 1:
            s += ",%s" % self.activation + (",leakiness=%s" % self.leakiness if self.activation == "leaky_relu" else "")
        return s + (",dropout=%s)" % self.p if self.p else ")")
