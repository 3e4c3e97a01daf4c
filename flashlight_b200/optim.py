"""fl::SGDOptimizer (flashlight/fl/optim/SGDOptimizer.{h,cpp}) over the fused step kernel, and AdamW over all
parameters at once."""
from __future__ import annotations

from typing import List

import torch

from . import _lib as L
from . import functions as F
from .autograd import Variable
from .extension import ptr, stream_handle


class SGDOptimizer:
    """Same constructor arguments and update rule as fl::SGDOptimizer(parameters, learningRate,
    momentum, weightDecay, useNesterov).  `step(grad_scale, zero_grad)` applies one update per
    parameter in a single pass (flb200_sgd_step); grad_scale is the 1/world-size of a
    data-parallel average when the all-reduce summed, zero_grad clears the gradients in the
    same pass instead of a separate zeroGrad()."""

    def __init__(self, parameters: List[Variable], learning_rate: float, momentum: float = 0.0,
                 weight_decay: float = 0.0, use_nesterov: bool = False):
        self.parameters = list(parameters)
        self.lr, self.mu, self.wd, self.nesterov = learning_rate, momentum, weight_decay, use_nesterov
        self.velocities = [torch.zeros_like(p.tensor) if momentum != 0 else None
                           for p in self.parameters]

    def step(self, grad_scale: float = 1.0, zero_grad: bool = False) -> None:
        for p, v in zip(self.parameters, self.velocities):
            if p.grad is None:  # isGradAvailable() false: skipped like the reference
                continue
            g = p.grad if p.grad.is_contiguous() else p.grad.contiguous()
            if not p.tensor.is_contiguous():
                raise ValueError("SGDOptimizer: parameters must be contiguous")
            L.check(L.lib.flb200_sgd_step(ptr(p.tensor), ptr(g), ptr(v), p.tensor.numel(), self.lr,
                                          self.mu, self.wd, 1 if self.nesterov else 0, grad_scale,
                                          1 if zero_grad else 0, L.F32, stream_handle()))

    def zeroGrad(self) -> None:
        for p in self.parameters:
            p.zeroGrad()


class AdamWOptimizer:
    """The moments of fl::AdamOptimizer (flashlight/fl/optim/AdamOptimizer.{h,cpp}) with the weight decay beside
    the step: p -= lr * (m^ / (sqrt(v^) + epsilon) + weight_decay * p).  One launch for all parameters
    (functions.adamw_step).  state_bits=8 keeps m and sqrt(v) as e4m3 bytes with a scale per 256 elements:
    2 bytes per element instead of 8.  Parameters without a gradient are passed over; the step's number counts
    all calls that made a step.  The states of all parameters lie one after another in `first` and `second`.  The
    step's number, the rate and the addresses are arguments of the launch: a step captured in a CUDA graph repeats one
    number's corrections of the moments and one rate with every replay, so capture the model's step without it, or
    capture it again."""

    def __init__(self, parameters: List[Variable], learning_rate: float, beta1: float = 0.9,
                 beta2: float = 0.999, epsilon: float = 1e-8, weight_decay: float = 0.0, state_bits: int = 32):
        if state_bits not in (32, 8):
            raise ValueError("AdamWOptimizer: states have 32 or 8 bits")
        self.parameters = list(parameters)
        self.lr, self.beta1, self.beta2 = learning_rate, beta1, beta2
        self.eps, self.wd, self.state_bits, self.steps = epsilon, weight_decay, state_bits, 0
        tensors = [p.tensor for p in self.parameters]
        if not all(t.is_contiguous() for t in tensors):
            raise ValueError("AdamWOptimizer: parameters must be contiguous")
        blocks = [(t.numel() + L.ADAMW_BLOCK - 1) // L.ADAMW_BLOCK for t in tensors]
        self.first, self.firsts = self._states(tensors, blocks)
        self.second, self.seconds = self._states(tensors, blocks)
        self.first_scale = self.second_scale = self.first_scales = self.second_scales = None
        if state_bits == 8:
            device = self.first.device
            self.first_scale, self.second_scale = (torch.zeros(sum(blocks), device=device) for _ in range(2))
            self.first_scales, self.second_scales = self.first_scale.split(blocks), self.second_scale.split(blocks)

    def _states(self, tensors, blocks):
        """Zeros for all parameters in one buffer, each parameter on blocks of its own, and its part of them."""
        device = tensors[0].device if tensors else "cuda"
        eight = self.state_bits == 8
        buffer = torch.zeros(sum(blocks) * L.ADAMW_BLOCK, dtype=torch.uint8 if eight else torch.float32,
                             device=device)
        if eight:
            buffer = buffer.view(torch.float8_e4m3fn)
        parts = buffer.split([n * L.ADAMW_BLOCK for n in blocks])
        return buffer, [part[:t.numel()] for part, t in zip(parts, tensors)]

    def step(self, grad_scale: float = 1.0) -> None:
        grads = [p.grad for p in self.parameters]
        F.adamw_step([p.tensor for p in self.parameters],
                     [g if g is None or g.is_contiguous() else g.contiguous() for g in grads], self.firsts,
                     self.seconds, step=self.steps + 1, lr=self.lr, beta1=self.beta1, beta2=self.beta2, eps=self.eps,
                     weight_decay=self.wd, grad_scale=grad_scale, first_scales=self.first_scales,
                     second_scales=self.second_scales)
        self.steps += 1  # (a step that was refused has changed nothing and does not count)

    def zeroGrad(self) -> None:
        for p in self.parameters:
            p.zeroGrad()
