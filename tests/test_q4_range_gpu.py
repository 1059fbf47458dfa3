"""4-bit decode products: scales and activations that are not finite, and every number of warps."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import vkblas_b200 as vk  # noqa: E402
from fused_util import TYPES, framed, rand  # noqa: E402
from test_q4_gpu import _check, _dense64, _weights  # noqa: E402


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


# 8, 12, 16 and 24 warps a CTA on 148 SMs, one token tile and two; K a whole number of steps and not
WARPS = [(1, 4096, 3584), (1, 2000, 4500), (9, 2000, 4500), (8, 2000, 4096), (1, 1000, 8200), (7, 2300, 6144), (9, 1000, 8200),
         (16, 2300, 6144), (16, 4096, 4096), (13, 4100, 4100), (16, 6000, 1100), (10, 40, 12300)]


@pytest.mark.parametrize("M,N,K", WARPS)
@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("group,zeros,pad", [(32, True, 0), (64, False, 4), (128, True, 1), (128, False, 0)])
def test_every_number_of_warps(cuda, M, N, K, kind, group, zeros, pad):
    gen = torch.Generator(device="cuda").manual_seed(M + N + K + group)
    t = TYPES[kind]
    q, s, z = _weights(gen, t, N, K, group, zeros)
    w = vk.q4_pack_tensors(q, s, z, K, group)
    x = framed(gen, t, M, K, pad + -K % 8, 0)[0]
    _check(x, _dense64(q, s, z, K, group), vk.gemv_q4_tensors(x, w))


def test_an_infinite_activation_reaches_every_output_of_its_row(cuda):
    """scale * (q - z) * inf is an infinity or, where q equals z, NaN; the other rows are as before."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    t = torch.bfloat16
    q, s, z = _weights(gen, t, 100, 256, 128, False)
    w = vk.q4_pack_tensors(q, s, z, 256, 128)
    x = rand(gen, t, 9, 256)
    clean = vk.gemv_q4_tensors(x, w)
    x[4, 17] = float("inf")
    y = vk.gemv_q4_tensors(x, w)
    n = (q[:, 8] >> 4).double() - 8
    assert torch.equal(torch.isnan(y[4]), n == 0)
    assert torch.equal(y[4][n != 0].double(), n[n != 0] * float("inf"))
    keep = [i for i in range(9) if i != 4]
    assert torch.equal(y[keep], clean[keep])
