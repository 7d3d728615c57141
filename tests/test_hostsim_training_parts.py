"""Parts of the gradients and sums over rows of the training operators, on the kernels' host build: the
GPU tests' bodies (see test_hostsim_parity)."""

import tests.test_training_ops_parts_gpu as _parts
from tests.test_hostsim_parity import _twin

for _mod in (_parts,):
    for _attr, _fn in list(vars(_mod).items()):
        if _attr.startswith("test_") and callable(_fn):
            globals()[f"test_host__{_attr[5:]}"] = _twin(_mod, _fn)
