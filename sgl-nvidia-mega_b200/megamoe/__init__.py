"""megamoe: B200-native (sm_100a) routed-MoE chain behind the reference's step API.

``RoutedMoE`` binds one MoE layer's MXFP4 weights; the stateless ops
(``router_gemv``, ``gate_topk``, ``route``, ``finalize``) mirror the reference's
individual kernels; ``rms_norm``, ``quantize_int8``, ``int8_linear`` and
``int8_ffn`` are the dense 8-bit operators beside it (the norm that makes the
layer's input, dense layers, an int8 shared expert). All compute runs in libmegamoe.so (hand-written CUDA for
sm_100a); there is no CPU path.
"""

from .moe import (  # noqa: F401
    RoutedMoE,
    finalize,
    finalize_partial,
    gate_topk,
    route,
    route_words,
    router_gemv,
)
from .dense import NormOutput, int8_check, int8_ffn, int8_linear, int8_set_wait_budget, quantize_int8, rms_norm  # noqa: F401
from .comm import PeerAllReduce  # noqa: F401
from .stack import MoEStack  # noqa: F401

__all__ = ["MoEStack", "NormOutput", "PeerAllReduce", "RoutedMoE", "finalize", "finalize_partial", "gate_topk", "int8_check",
           "int8_ffn", "int8_linear", "int8_set_wait_budget", "quantize_int8", "rms_norm", "route", "route_words", "router_gemv"]
