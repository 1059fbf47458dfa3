"""The gated block's gradients over the range of its types, against 64-bit forms."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import vkblas_b200 as vk  # noqa: E402
from fused_util import TINY, TYPES, act64, framed, rand, rounded, sum_err, u, within  # noqa: E402
from gpu_util import check_status  # noqa: E402
from test_gated_gpu import _check_forward  # noqa: E402

ACTS = ["silu", "gelu", "gelu_tanh"]


def _grads(dh, g, up, x, wg, wu, act):
    a, d = act64(g.double(), act)
    dG, dU = dh.double() * up.double() * d, dh.double() * a
    return dG, dU


def _check(dh, g, up, x, wg, wu, act):
    """dx, dw_gate, dw_up within their roundings: dG and dU rounded once to the type, in fp16 after a
    power of two that brings the larger maximum into [2^14, 2^15)."""
    t = x.dtype
    got = vk.gated_backward_tensors(dh, g, up, x, wg, wu, act)
    dG, dU = _grads(dh, g, up, x, wg, wu, act)
    big = float(torch.maximum(dG.abs().max(), dU.abs().max()))
    step = big * 2.0 ** -14 * TINY[t] if t == torch.float16 else TINY[t]
    X, G, U = x.double(), wg.double(), wu.double()

    def err(a, b):
        return (u(t) + 2.0 ** -16) * (a.abs() @ b.abs()) + step * b.abs().sum(0) + sum_err(a, b.T.contiguous())

    for v, want, e, what in ((got[0], dG @ G + dU @ U, err(dG, G) + err(dU, U), "dx"),
                             (got[1], dG.T @ X, err(dG.T, X), "dw_gate"), (got[2], dU.T @ X, err(dU.T, X), "dw_up")):
        assert bool(torch.isfinite(v).all()), what
        within(v, want, e + rounded(want.abs() + e, t), what)
    check_status()
    return got


SIZES = [(5, 33, 40), (130, 264, 72), (300, 515, 264)]


@pytest.mark.parametrize("M,F,H", SIZES)
@pytest.mark.parametrize("pad", [0, 1])
def test_fp16_products_above_the_types_range(cuda, M, F, H, pad):
    """dh * u beyond 65504, weights and inputs small: the gradients are within the range."""
    gen = torch.Generator(device="cuda").manual_seed(M)
    t = torch.float16
    dh, up = (framed(gen, t, M, F, pad, 0, 300.0)[0] for _ in range(2))
    g = rand(gen, t, M, F, scale=3.0)
    x, wg, wu = (rand(gen, t, *s, scale=1e-3) for s in ((M, H), (F, H), (F, H)))
    assert float((dh.float() * up.float()).abs().max()) > 65504
    _check(dh, g, up, x, wg, wu, ACTS[M % 3])


@pytest.mark.parametrize("M,F,H", SIZES)
def test_fp16_products_below_the_types_range(cuda, M, F, H):
    """dh * u of 1e-8, weights and inputs large."""
    gen = torch.Generator(device="cuda").manual_seed(M)
    t = torch.float16
    dh = rand(gen, t, M, F, scale=1e-4)
    up, g = (rand(gen, t, M, F, scale=1e-4) for _ in range(2))
    x, wg, wu = (rand(gen, t, *s, scale=300.0) for s in ((M, H), (F, H), (F, H)))
    got = _check(dh, g, up, x, wg, wu, ACTS[M % 3])
    assert bool((got[0] != 0).any() & (got[1] != 0).any())


def test_fp16_scale_by_powers_of_two(cuda):
    """dh times a power of two gives the gradients times it, bit for bit, whatever its size."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    t, M, F, H = torch.float16, 150, 300, 128
    x, wg, wu = (rand(gen, t, *s, scale=0.05) for s in ((M, H), (F, H), (F, H)))
    g, up = rand(gen, t, M, F, scale=2.0), rand(gen, t, M, F)
    dh = ((rand(gen, t, M, F).float().clamp(-4, 4) * 2 ** 6).round() / 2 ** 6).to(t)     # exact over the shifts
    ref = vk.gated_backward_tensors(dh, g, up, x, wg, wu)
    for e in (-6, 9):
        got = vk.gated_backward_tensors(dh * 2.0 ** e, g, up, x, wg, wu)
        for a, b in zip(got, ref):
            want = b.float() * 2.0 ** e
            keep = (want.abs() >= 2.0 ** -14) & (b.float().abs() >= 2.0 ** -14)      # normal in both
            assert bool(keep.any()) and torch.equal(a.float()[keep], want[keep])


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
def test_gradient_of_zero_and_of_one_bad_row(cuda, kind):
    """No gradient at all; NaN and infinite gradients of single rows leave the others' dx alone."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    t, M, F, H = TYPES[kind], 140, 300, 128
    x, wg, wu = (rand(gen, t, *s) for s in ((M, H), (F, H), (F, H)))
    g, up, dh = (rand(gen, t, M, F) for _ in range(3))
    zero = vk.gated_backward_tensors(torch.zeros_like(dh), g, up, x, wg, wu)
    assert all(bool((v == 0).all()) for v in zero)
    clean = vk.gated_backward_tensors(dh, g, up, x, wg, wu, need_dw=False)[0]
    dh[3], dh[77] = float("nan"), float("inf")
    dx = vk.gated_backward_tensors(dh, g, up, x, wg, wu, need_dw=False)[0]
    keep = [i for i in range(M) if i not in (3, 77)]
    assert not bool(torch.isfinite(dx[[3, 77]]).any())
    # the bad rows take no part in the scale, but their own entries in it are gone: the others may
    # be rounded after another power of two
    a, b = dx[keep].double(), clean[keep].double()
    assert float((a - b).norm() / b.norm()) <= 2 * u(t)


@pytest.mark.parametrize("act", ACTS)
def test_bf16_projections_of_any_size(cuda, act):
    """Projections up to 1e30 on both sides: the derivative is 0 or 1 there, not NaN."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    t, M, F, H = torch.bfloat16, 50, 72, 64
    g = rand(gen, t, M, F) * (10.0 ** torch.arange(F, device="cuda").remainder(31)).to(t)
    dh, up = rand(gen, t, M, F, scale=1e-3), rand(gen, t, M, F)
    x, wg = rand(gen, t, M, H), rand(gen, t, F, H)
    _check(dh, g, up, x, wg, torch.zeros_like(wg), act)


@pytest.mark.parametrize("M", [1, 4, 9, 12, 16])
@pytest.mark.parametrize("F", [2400, 5461, 8192, 11008, 14336])
@pytest.mark.parametrize("kind,pad", [("fp16", 0), ("bf16", 0), ("bf16", 1)])
def test_every_number_of_warps_of_the_token_form(cuda, M, F, kind, pad):
    """F decides whether a CTA has 4, 5, 6 or 8 warps; H ends inside a warp's share."""
    gen = torch.Generator(device="cuda").manual_seed(M + F)
    t, H, act = TYPES[kind], 648, ACTS[F % 3]
    x = framed(gen, t, M, H, pad, 0)[0]
    wg, wu = (framed(gen, t, F, H, pad, pad, H ** -0.5)[0] for _ in range(2))
    h, g, up = vk.gated_tensors(x, wg, wu, act, save=True)
    assert torch.equal(vk.gated_tensors(x, wg, wu, act), h)
    _check_forward(x, wg, wu, act, h, g, up)
    check_status()


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("M,F,H", [(300, 2731, 1024), (1001, 2731, 1024), (70, 5000, 900)])
def test_weight_gradients_in_a_grid_each(cuda, M, F, H, kind):
    """Sizes whose two weight gradients take no fewer waves together than one after the other."""
    gen = torch.Generator(device="cuda").manual_seed(M + F)
    t = TYPES[kind]
    dh, g, up = rand(gen, t, M, F, scale=0.1), rand(gen, t, M, F, scale=2.0), rand(gen, t, M, F)
    x, wg, wu = rand(gen, t, M, H), rand(gen, t, F, H, scale=H ** -0.5), rand(gen, t, F, H, scale=H ** -0.5)
    _check(dh, g, up, x, wg, wu, ACTS[M % 3])


@pytest.mark.parametrize("M,pad,off,F,H", [(40, 3, 0, 133, 67), (300, 0, 1, 128, 64), (300, 5, 3, 65, 77), (17, 8, 8, 136, 72)])
@pytest.mark.parametrize("kind", ["fp16", "bf16"])
def test_layouts_bit_for_bit(cuda, M, pad, off, F, H, kind):
    """Strided and unaligned inputs give what compact ones give, forward and backward."""
    gen = torch.Generator(device="cuda").manual_seed(M + pad)
    t = TYPES[kind]
    x, wg, wu = (framed(gen, t, r, H, pad, off)[0] for r in (M, F, F))
    dh, g, up = (framed(gen, t, M, F, pad, off)[0] for _ in range(3))

    def compact(*ts):
        return [v.clone(memory_format=torch.contiguous_format) for v in ts]

    got = vk.gated_backward_tensors(dh, g, up, x, wg, wu, "gelu_tanh")
    want = vk.gated_backward_tensors(*compact(dh, g, up, x, wg, wu), "gelu_tanh")
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for m in (1, 13, M):
        assert torch.equal(vk.gated_tensors(x[:m], wg, wu), vk.gated_tensors(*compact(x[:m], wg, wu)))


def test_fp16_parts_and_replay(cuda):
    """One gradient alone is what both together give; a replayed capture scales by its new inputs."""
    gen = torch.Generator(device="cuda").manual_seed(8)
    t, M, F, H = torch.float16, 300, 515, 264
    x, wg, wu = (rand(gen, t, *s, scale=0.05) for s in ((M, H), (F, H), (F, H)))
    g, up, dh = rand(gen, t, M, F, scale=2.0), rand(gen, t, M, F), rand(gen, t, M, F, scale=0.01)
    full = vk.gated_backward_tensors(dh, g, up, x, wg, wu)
    assert torch.equal(vk.gated_backward_tensors(dh, g, up, x, wg, wu, need_dw=False)[0], full[0])
    for a, b in zip(vk.gated_backward_tensors(dh, g, up, x, wg, wu, need_dx=False)[1:], full[1:]):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = vk.gated_backward_tensors(dh, g, up, x, wg, wu)
    for size in (1.0, 2.0 ** 12, 2.0 ** -8):
        dh.copy_(rand(gen, t, M, F, scale=0.01 * size))
        graph.replay()
        want = vk.gated_backward_tensors(dh, g, up, x, wg, wu)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(bool(torch.isfinite(a).all()) for a in got)
    check_status()
