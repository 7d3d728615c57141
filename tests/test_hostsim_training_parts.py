"""Parts of the gradients and sums over rows of the training operators, on the kernels' host build: the
GPU tests' bodies (see test_hostsim_parity)."""

import tests.test_training_ops_parts_gpu as _parts
import tests.test_training_ops_row_sums_gpu as _sums
from tests.test_hostsim_parity import _twin

# minutes of CPU time
SKIP = {"test_weight_gradients_hold_every_row_large"}

for _mod in (_parts, _sums):
    for _attr, _fn in list(vars(_mod).items()):
        if _attr.startswith("test_") and callable(_fn) and _attr not in SKIP:
            globals()[f"test_host__{_attr[5:]}"] = _twin(_mod, _fn)
