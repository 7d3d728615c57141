"""The training operators' GPU tests on the kernels' host build (see test_hostsim_parity)."""

import tests.test_training_ops_gpu as _mod
from tests.test_hostsim_parity import _twin

# needs streams and graphs of a device
SKIP = {"test_training_ops_streams_and_graphs"}

for _attr, _fn in list(vars(_mod).items()):
    if _attr.startswith("test_") and callable(_fn) and _attr not in SKIP:
        globals()[f"test_host_training__{_attr[5:]}"] = _twin(_mod, _fn)
