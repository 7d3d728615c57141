"""The GPU's results against the host build's vectors (see test_zy_host_model_vectors_gpu) with a limit of its
own for each case: 16 units of a value's bf16 spacing, as few roundings apart as all cases but one are, and for
the diffusion attention a limit per row that follows from the share of values that differ.

That case's output is a product with 768 terms per value behind a chain of bf16 roundings (adaptive norm, q, k, v,
attention), so the two sides' values before the last rounding differ everywhere, a row's by about as much in all of its
768 channels: by many small terms of either sign, normally distributed with a deviation sigma of the row.  Such a
difference d changes the rounded value with probability |d| / step, if it is below the step; with a step of 2^-7 / m of the
value (mantissa m in [1, 2), 1.44 * 2^-8 on average), E|value| = 0.8 RMS and E|d| = 0.8 sigma the share f of a row's values
that differ tells sigma = 1.44 * 2^-8 f RMS.  No value of 61440 is expected beyond five sigma, and the rounding itself adds
one step.  The share is counted from 768 values: n found stand for at most n + 3 sqrt(n) + 3 expected."""

import pytest
import torch

from tests.golden.make_host_model_vectors import cases
from tests.test_zy_host_model_vectors_gpu import VECTORS, compare
from tests.util import ulp_bf16

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
DIFFUSION = "apb_diffusion_bf16"
MAX_UNITS = 16


def diffusion_limit(ref, got):
    """Largest difference of each value by the rule above; ref, got: [..., rows, 768] in fp32."""
    n = (ref != got).float().sum(-1, keepdim=True)
    share = (n + 3 * n.sqrt() + 3) / ref.shape[-1]
    sigma = 1.44 * 2.0 ** -8 * share * ref.square().mean(-1, keepdim=True).sqrt()
    return 5 * sigma + ulp_bf16(torch.maximum(ref.abs(), got.abs()))


def test_every_case_within_its_limit():
    for name, (share, worst) in compare(DEV).items():
        print(f"case {name}: {worst:.2f} units", flush=True)
        assert name.endswith("_f32") or name == DIFFUSION or worst <= MAX_UNITS, (name, share, worst)


def test_diffusion_attention_within_its_rows_limits():
    print(f"case {DIFFUSION}", flush=True)
    build, inputs, call = cases()[DIFFUSION]
    ref = torch.load(VECTORS, weights_only=True)[DIFFUSION].float()
    with torch.no_grad():
        got = call(build().to(DEV), {k: v.to(DEV) for k, v in inputs.items()}).detach().cpu().float()
    ratio = (got - ref).abs() / diffusion_limit(ref, got)
    print(f"  largest difference / limit {ratio.max().item():.3f}", flush=True)
    assert (ratio <= 1).all(), ratio.max().item()
    # a mistake in one of 16 heads (48 of 768 terms gone from the last product) is far beyond it
    wrong = ref + (48 / 768) ** 0.5 * ref.square().mean(-1, keepdim=True).sqrt() * torch.randn(
        ref.shape, generator=torch.Generator().manual_seed(0))
    wrong = wrong.bfloat16().float()
    assert ((wrong - ref).abs() > diffusion_limit(ref, wrong)).any(-1).all()
