"""MI355X-native implementation of the PyramidConvBlock hot path: channels-last large-kernel
depthwise conv2d with the adaptive average pooling, gate and bilinear upsampling that
``ConvBlock`` composes around it, forward and backward, on hand-written gfx950 kernels; and what goes around and
beside such a block in a model: channel norms, gated residuals, a gated linear recurrence along an axis, and with matrices for states the
gated delta rule, with the norms and rotated positions of its queries and keys."""
from .avgpool import AdaptiveAvgPool2dFunction, OptimizedAdaptiveAvgPool2d
from .conv_block import ConvBlock, GateFunction, SimpleGate
from .delta import GatedDelta, GatedDeltaFunction, gated_delta, gated_delta_step
from .dwconv import DepthwiseConv2DFunction, OptimizedDepthwiseConv2d
from .norm import (ChannelNorm, ChannelNormFunction, GatedResidual, GatedResidualFunction, ResidualConvStack, channel_norm,
                   gated_residual)
from .rotary import HeadRotary, HeadRotaryFunction, head_rotary
from .scan import GatedScan, GatedScanFunction, gated_scan, gated_scan_step
from .up import BilinearInterp2dFunction, OptimizedBilinearInterp2d

__all__ = [
    "ConvBlock", "SimpleGate", "GateFunction",
    "OptimizedDepthwiseConv2d", "DepthwiseConv2DFunction",
    "OptimizedAdaptiveAvgPool2d", "AdaptiveAvgPool2dFunction",
    "OptimizedBilinearInterp2d", "BilinearInterp2dFunction",
    "ChannelNorm", "ChannelNormFunction", "channel_norm",
    "GatedResidual", "GatedResidualFunction", "gated_residual", "ResidualConvStack",
    "GatedScan", "GatedScanFunction", "gated_scan", "gated_scan_step",
    "HeadRotary", "HeadRotaryFunction", "head_rotary",
    "GatedDelta", "GatedDeltaFunction", "gated_delta", "gated_delta_step",
]
