"""The limits of tests/test_zy_host_model_limits_gpu.py on the kernels' host build, where nothing differs."""

import tests.test_zy_host_model_limits_gpu as _mod
from tests.test_hostsim_parity import _twin


def test_host_every_case_within_its_limit():
    _twin(_mod, _mod.test_every_case_within_its_limit)()


def test_host_diffusion_attention_within_its_rows_limits():
    _twin(_mod, _mod.test_diffusion_attention_within_its_rows_limits)()
