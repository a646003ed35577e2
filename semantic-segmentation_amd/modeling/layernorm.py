"""Layer normalisation of every position over its channels, for (N, C, H, W) maps: the counterpart of SwitchNorm2d and
HipBatchNorm2d for blocks whose normalisation must not depend on other positions or images (batch of one, tiled
inference).  The maps are NHWC in memory, so the C values of a position are one contiguous row: forward is one pass over
the input, backward one pass over input and gradient that also reduces the parameter gradients.
There is no CPU path: a CPU tensor raises.
"""
import torch
import torch.nn as nn

from snws import ops


class LayerNorm2d(nn.Module):
    """y = (x - mean) / sqrt(var + eps) * weight + bias, mean and (biased) variance over the channels of each position.
    weight, bias: (num_features,), ones and zeros at the start; affine=False leaves them out."""

    def __init__(self, num_features, eps=1e-5, affine=True):
        super(LayerNorm2d, self).__init__()
        self.num_features, self.eps = num_features, eps
        if affine:
            self.weight = nn.Parameter(torch.ones(num_features))
            self.bias = nn.Parameter(torch.zeros(num_features))
        else:
            self.register_parameter('weight', None)
            self.register_parameter('bias', None)

    def extra_repr(self):
        return '{}, eps={}, affine={}'.format(self.num_features, self.eps, self.weight is not None)

    def forward(self, x):
        if x.dim() != 4:
            raise ValueError('expected 4D input (got {}D input)'.format(x.dim()))
        if x.shape[1] != self.num_features:
            raise ValueError('expected {} channels (got {})'.format(self.num_features, x.shape[1]))
        ops.require_gpu(x, "LayerNorm2d")
        return ops.layer_norm(x.permute(0, 2, 3, 1), self.weight, self.bias, self.eps).permute(0, 3, 1, 2)
