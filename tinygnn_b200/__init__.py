"""tinygnn_b200 -- a B200-native GNN inference engine with TinyGNN's API.

The compute path is libtinygnn_b200.so (hand-written sm_100a CUDA kernels
behind the C ABI in include/tinygnn_b200.h).  This package is its Python
host side: ctypes bindings (``_lib``), torch-tensor front ends of every
entry point (``ops``; training operators: ``training``), seeded synthetic inputs (``synth``) and the
row-partitioned multi-GPU driver (``dist``).  Importing it without the
built library raises: there is no CPU fallback.
"""
from . import _lib
from ._lib import InvalidArgument, OutOfRange, TinyGNNError, launches
from .ops import (CSR, add_bias_, add_self_loops, csr_validate, degree_order, edge_list_to_csr,
                  edge_softmax, elu_, gat_layer, gcn_layer, gcn_norm, gelu_, leaky_relu_, log_softmax_,
                  matmul, relu_, sage_aggregate, sage_layer, sage_max_aggregate, sigmoid_, softmax_,
                  spmm, tanh_)
# The training operators' names, imported on their first use: their module is
# built against one torch, and the rest of the package needs none of it.
_TRAINING = ("Saved8", "activation_backward", "activation_save8", "check_row_offsets", "layer_norm",
             "layer_norm_backward", "save8", "typed_linear", "typed_linear_backward", "typed_linear_grad_input",
             "typed_linear_grad_weight")

__version__ = "0.1.0"


def version() -> str:
    return _lib.lib.tg_version().decode()


def device_count() -> int:
    return int(_lib.lib.tg_device_count())


def __getattr__(name: str):
    if name != "training" and name not in _TRAINING:
        raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
    import importlib
    module = importlib.import_module(".training", __name__)
    globals().update({n: getattr(module, n) for n in _TRAINING})
    return module if name == "training" else globals()[name]


def __dir__():
    return sorted({*globals(), "training", *_TRAINING})


__all__ = [n for n in __dir__() if not n.startswith("_")]
