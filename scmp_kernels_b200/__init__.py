"""B200-native (sm_100a) stochastic-computing matmul.

Drop-in for the ``sc_matmul`` path of scmp_kernels: the same Python API
(:func:`sc_matmul`, :func:`clear_rng_cache`, the ``quant`` package) over a
C-ABI library of hand-written CUDA kernels (``libscmp_b200.so``).

Next to it, the exact layers a model runs and trains around an SC product:
:func:`layer_norm`, :func:`linear` and 8-bit activation checkpoints
(:class:`Act8`), each with its backward pass.
"""
from .act8 import Act8, pack_act8, unpack_act8
from .dense import linear, linear_backward, linear_forward
from .norm import layer_norm, layer_norm_backward, layer_norm_forward
from .sc import clear_rng_cache, det_kernel_tuning, prepare_weight, sc_matmul, sc_matmul_levels, sc_matmul_prepared

__all__ = ["sc_matmul", "clear_rng_cache", "det_kernel_tuning", "prepare_weight", "sc_matmul_prepared",
           "sc_matmul_levels", "layer_norm", "layer_norm_forward", "layer_norm_backward", "linear", "linear_forward",
           "linear_backward", "Act8", "pack_act8", "unpack_act8"]
