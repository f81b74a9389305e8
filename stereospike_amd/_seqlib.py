"""Loader of the sequence operators' library: lib/ss_seq_torch.so (csrc/ss_seq_torch.cpp), the PyTorch side of libss_sequence.so (include/ss_sequence.h).

As with the neuron library there is no fallback: a missing library, a CPU tensor or an operand of another type raises SSNeuronError.
"""
import importlib.machinery
import importlib.util
import os

import torch  # noqa: F401  (before the library, so that one HIP runtime is shared)

from ._lib import SSNeuronError

_PKG = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_PKG, 'lib', 'libss_sequence.so')
OPS_PATH = os.path.join(_PKG, 'lib', 'ss_seq_torch.so')
ABI_VERSION = 1
MAX_HEAD_DIM = 256
MAX_NORM_WIDTH = 16384
MAX_INT8_K = 131071
MAX_STATES = 65535
MAX_STEPS, MAX_SIDE, MAX_TILES = 1 << 30, 1 << 27, 1 << 24

_ops = None


def ops():
    """Load (once) and return the library.  Raises loudly when it has not been built."""
    global _ops
    if _ops is not None:
        return _ops
    for path in (LIB_PATH, OPS_PATH):
        if not os.path.exists(path):
            raise SSNeuronError(f'{path} not found: the HIP extension is not built.  Run `python -c "import __graft_entry__ as g; g.build()"` or '
                                f'`make -C stereospike_amd/csrc` (hipcc --offload-arch=gfx950).  There is no CPU fallback.')
    spec = importlib.util.spec_from_file_location('ss_seq_torch', OPS_PATH, loader=importlib.machinery.ExtensionFileLoader('ss_seq_torch', OPS_PATH))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    if m.abi_version() != ABI_VERSION:
        raise SSNeuronError(f'libss_sequence.so ABI {m.abi_version()} != expected {ABI_VERSION}; rebuild')
    m.set_error(SSNeuronError)
    _ops = m
    return _ops
