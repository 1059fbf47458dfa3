"""4-bit decode products: scales and activations that are not finite, and every number of warps."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import vkblas_b200 as vk  # noqa: E402
from fused_util import TYPES, rand, rounded, within  # noqa: E402


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("K,group", [(33, 32), (65, 32), (129, 64), (257, 128)])
def test_infinite_scale_of_the_last_group(cuda, kind, K, group):
    """The last group has one weight: an infinite scale makes it an infinity of its sign, or NaN where it
    is 0, whatever the rest of its step is padded with."""
    gen = torch.Generator(device="cuda").manual_seed(K)
    t, M, N = TYPES[kind], 3, 40
    ng = -(-K // group)
    q = torch.randint(0, 256, (N, (K + 1) // 2), generator=gen, device="cuda", dtype=torch.uint8)
    n = torch.stack((q & 15, q >> 4), -1).reshape(N, -1)[:, :K].double() - 8
    s = torch.rand(N, ng, generator=gen, device="cuda").to(t) + 0.5
    s[::2, -1] = float("inf")
    x = rand(gen, t, M, K)
    y = vk.gemv_q4_tensors(x, vk.q4_pack_tensors(q, s, None, K, group))
    want = x[:, -1:].double() * n[None, ::2, -1] * float("inf")
    assert torch.equal(torch.isnan(y[:, ::2]), torch.isnan(want)) and bool((~torch.isnan(want)).any())
    assert torch.equal(y[:, ::2].double().nan_to_num(0, 1, -1), want.nan_to_num(0, 1, -1))
    assert bool(torch.isfinite(y[:, 1::2]).all())
