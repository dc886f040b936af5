"""B200-native (sm_100a) wavelet filter-bank transforms with the API of ``fdwt``.

* :func:`dwt`, :func:`idwt`, :func:`wavedec`, :func:`waverec`, :class:`DWT1D`,
  :class:`IDWT1D` -- Mallat fast wavelet transform, PyWavelets-compatible.
* :func:`cwt`, :class:`CWT1D` -- Morlet continuous wavelet transform with the O(N)-per-scale
  octave pyramid (``method="fast"``).
* :class:`MorletTokenMixer`, :class:`WaveletTokenMixer`, :class:`MorletAttention`,
  :class:`MorletChannelMixAttention` -- attention replacements.
* :func:`layer_norm`, :func:`linear_attention`, :func:`linear_attention_step` and the layers
  :class:`LayerNorm`, :class:`DecayTokenMixer` -- a causal token mixer for training, prompts and
  single tokens.
* :func:`rms_norm`, :func:`rms_norm_quantized` (:class:`RMSNorm`), :func:`causal_conv1d` and
  :func:`selective_scan` with their single-token forms :func:`causal_conv1d_step` and
  :func:`selective_scan_step` -- the norm with the residual's addition, the short convolution and
  the selective state space scan of a causal mixer, :class:`SelectiveTokenMixer`, and of stacks of
  them, :class:`SelectiveTokenStack`.

Every transform runs in hand-written CUDA kernels for sm_100a behind the C ABI of
``include/fdwt_b200.h`` (``libfdwt_b200.so``); inputs must be CUDA tensors.
"""

from . import config
from .causal_conv import causal_conv1d, causal_conv1d_step
from .cwt import CWT1D, MorletPlan, cwt, freqs_to_scales, scales_to_freqs
from .dwt import DWT1D, IDWT1D, dwt, dwt_max_level, idwt, wavedec, waverec
from .layers import (DecayTokenMixer, MorletAttention, MorletChannelMixAttention,
                     MorletTokenMixer, SelectiveTokenMixer, SelectiveTokenStack,
                     WaveletTokenMixer)
from .linear_attention import linear_attention, linear_attention_step
from .norm import LayerNorm, RMSNorm, layer_norm, rms_norm, rms_norm_quantized
from .selective_scan import selective_scan, selective_scan_step
from .wavelets import FilterBank, get_filter_bank

__version__ = "0.1.0"

__all__ = [
    "config", "CWT1D", "MorletPlan", "cwt", "freqs_to_scales", "scales_to_freqs",
    "DWT1D", "IDWT1D", "dwt", "dwt_max_level", "idwt", "wavedec", "waverec",
    "MorletAttention", "MorletChannelMixAttention", "MorletTokenMixer", "WaveletTokenMixer",
    "DecayTokenMixer", "LayerNorm", "layer_norm", "linear_attention", "linear_attention_step",
    "RMSNorm", "rms_norm", "rms_norm_quantized", "causal_conv1d", "causal_conv1d_step",
    "selective_scan", "selective_scan_step", "SelectiveTokenMixer", "SelectiveTokenStack",
    "FilterBank", "get_filter_bank",
]
