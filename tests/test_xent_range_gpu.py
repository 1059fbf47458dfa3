"""Cross entropy of a linear head where its gradients are small differences, its sums long and its
sizes take more than one piece or segment, against 64-bit forms."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import vkblas_b200 as vk  # noqa: E402
from fused_util import TYPES, rand, rounded, sum_err, u, within  # noqa: E402
from gpu_util import check_status  # noqa: E402
from test_xent_gpu import _check_forward, _check_grads, _grads64, _inputs  # noqa: E402


@pytest.fixture(autouse=True)
def _free():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("T", [40, 300])
@pytest.mark.parametrize("kind", ["fp16", "bf16"])
def test_gradients_of_well_predicted_tokens(cuda, T, kind):
    """Targets of probability 0.99 to 0.9999: their entry of D is p - 1, a small difference, and
    decides the row's gradient."""
    gen = torch.Generator(device="cuda").manual_seed(T)
    t, V, H = TYPES[kind], 1000, 4096
    w = rand(gen, t, V, H, scale=1.2 / 64)
    w[:, 0] = 1.0                       # column 0 of dx is the row sum of D
    targets = torch.randint(0, V, (T,), generator=gen, device="cuda")
    lean = torch.linspace(8.5, 11.5, T, device="cuda", dtype=torch.float64)[:, None]
    x = (torch.randn(T, H, generator=gen, device="cuda") + w[targets].float() * lean.float()).to(t)
    x[:, 0] = 0.0
    loss, lse = vk.linear_xent_tensors(x, w, targets)
    dloss = torch.full((T,), 1.0, device="cuda")
    dx, dw = vk.linear_xent_backward_tensors(dloss, lse, x, w, targets)
    X, W = x.double(), w.double()
    z = X @ W.T
    p = torch.softmax(z, 1)
    at = torch.arange(T, device="cuda"), targets
    rest = p.clone()
    rest[at] = 0
    q = rest.sum(1)                     # 1 - p of the target
    assert float(q.min()) < 3e-4 and float(q.max()) < 0.2 and float(q.median()) < 1e-2
    D = rest.clone()
    D[at] = -q
    # A logit is eight sums of 512 products and their sum in fp32; z and lse hold the same
    # computed logits, so D moves by twice that as a share of p, or of 1 - p at the target.
    ez = (512 + 16 + 8) * 2.0 ** -23 * (X.abs() @ W.abs().T).amax(1)[:, None]
    # lse: at most 100 additions in fp32 of a sum near 1, and its own rounding; the
    # exponential is 2^-22 off.
    el = 100 * 2.0 ** -24 + 2.0 ** -24 * lse.double().abs() + 2.0 ** -22
    eD = rest * (2 * ez + el[:, None]) + D.abs() * u(t)
    eD[at] += el + 2 * ez[:, 0] * q
    err = eD @ W.abs() + sum_err(D, W.T.contiguous())
    want = D @ W
    within(dx, want, err + rounded(want.abs() + err, t), "dx")
    # the row's gradient as a whole, where 1 - p is well above lse's own rounding
    rows = (dx.double() - want).norm(dim=1) / want.norm(dim=1)
    assert bool((rows <= el / q + 2 * ez[:, 0] + 2 * u(t)).all()), float(rows.max())
    err = eD.T @ X.abs() + sum_err(D.T.contiguous(), X.T.contiguous())
    want = D.T @ X
    within(dw, want, err + rounded(want.abs() + err, t), "dw")
    check_status()


@pytest.mark.parametrize("T,H", [(1023, 4096), (20, 200)])
def test_dx_of_a_long_vocabulary_has_no_bias(cuda, T, H):
    """Weights of one sign, so that dx sums 131072 terms of one sign.  Roundings to nearest leave a
    mean error of at most u / sqrt(elements compared) of the sum; what is left is a bias,
    which has to stay well below a single element's rounding: a quarter of u."""
    gen = torch.Generator(device="cuda").manual_seed(T)
    t, V = torch.float16, 131072
    x = rand(gen, t, T, H)
    x -= x.float().mean(1, keepdim=True).to(t)
    w = torch.empty(V, H, device="cuda", dtype=t)
    blocks = range(0, V, 16384)
    for i in blocks:
        w[i:i + 16384] = (torch.rand(16384, H, generator=gen, device="cuda") + 0.5) * H ** -0.5
    targets = torch.randint(0, V, (T,), generator=gen, device="cuda")
    _, lse = vk.linear_xent_tensors(x, w, targets)
    dx, dw = vk.linear_xent_backward_tensors(torch.ones(T, device="cuda"), lse, x, w, targets)
    rows = torch.arange(0, T, max(1, T // 5), device="cuda")
    z = torch.cat([x[rows].double() @ w[i:i + 16384].double().T for i in blocks], 1)
    p = torch.softmax(z, 1)
    total = sum(p[:, i:i + 16384] @ w[i:i + 16384].double() for i in blocks)
    want = total - w[targets[rows]].double()
    bias = float((dx[rows].double() - want).mean() / total.mean())
    assert abs(bias) <= u(t) / 4, bias
    assert bool(torch.isfinite(dw).all())
    check_status()


@pytest.mark.parametrize("T,V,H", [(100, 700, 1100), (300, 700, 1100), (257, 300, 2056)])
@pytest.mark.parametrize("kind", ["fp16", "bf16"])
def test_several_segments(cuda, T, V, H, kind):
    """K in more than one segment, the last one ragged, on single CTAs and on pairs."""
    gen = torch.Generator(device="cuda").manual_seed(T + H)
    x, w, targets = _inputs(gen, TYPES[kind], T, V, H)
    loss, lse = vk.linear_xent_tensors(x, w, targets)
    _check_forward(x, w, targets, loss, lse)
    dloss = torch.rand(T, generator=gen, device="cuda") / T
    dx, dw = vk.linear_xent_backward_tensors(dloss, lse, x, w, targets)
    _check_grads(x, w, targets, dloss, dx, dw, *_grads64(x, w, targets, dloss))
    check_status()


@pytest.mark.parametrize("T,V,H,kind", [(16400, 8500, 72, "fp16"), (16400, 8500, 72, "bf16"), (16400, 17001, 40, "bf16"),
                                        (1100, 20001, 2100, "fp16")])
def test_several_pieces(cuda, T, V, H, kind):
    """A vocabulary in more than one piece (16400 tokens), or a piece in more than one product for dx
    (1100 tokens, fp16): targets on both sides of every border, the last piece ragged."""
    gen = torch.Generator(device="cuda").manual_seed(T + V)
    x, w, targets = _inputs(gen, TYPES[kind], T, V, H)
    edges = torch.arange(0, V, 256, device="cuda")
    targets[:len(edges)] = edges
    targets[len(edges):2 * len(edges)] = (edges - 1).clamp(min=0)
    targets[-1] = V - 1
    loss, lse = vk.linear_xent_tensors(x, w, targets)
    _check_forward(x, w, targets, loss, lse)
    dloss = torch.rand(T, generator=gen, device="cuda") / T
    dx, dw = vk.linear_xent_backward_tensors(dloss, lse, x, w, targets)
    ref = _grads64(x, w, targets, dloss)
    _check_grads(x, w, targets, dloss, dx, dw, *ref)
    for got, want in ((dx, ref[1]), (dw, ref[2])):
        # D's rounding and the result's: rms u / sqrt 3 each, and fp16's half smallest step, which
        # a gradient of 1 / T may come near to
        floor = torch.finfo(got.dtype).smallest_normal * u(got.dtype) * want.numel() ** 0.5
        assert float((got.double() - want).norm()) <= 1.5 * u(got.dtype) * float(want.norm()) + floor
    part = vk.linear_xent_backward_tensors(dloss, lse, x, w, targets, need_dw=False)[0]
    assert torch.equal(part, dx)
    assert torch.equal(vk.linear_xent_backward_tensors(dloss, lse, x, w, targets, need_dx=False)[1], dw)
    check_status()


def test_dx_of_a_million_columns(cuda):
    """24 tokens, 1100000 x 4096: dx against the sum over blocks of the vocabulary."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    t, T, V, H = torch.bfloat16, 24, 1100000, 4096
    x = rand(gen, t, T, H)
    w = torch.empty(V, H, device="cuda", dtype=t)
    blocks = range(0, V, 100000)
    for i in blocks:
        w[i:i + 100000] = rand(gen, t, 100000, H, scale=1.5 / 64)
    targets = torch.randint(0, V, (T,), generator=gen, device="cuda")
    targets[:4] = torch.tensor([0, V - 1, 1048576, 1048575], device="cuda")
    _, lse = vk.linear_xent_tensors(x, w, targets)
    dx, _ = vk.linear_xent_backward_tensors(torch.ones(T, device="cuda"), lse, x, w, targets, need_dw=False)
    z = torch.cat([x.double() @ w[i:i + 100000].double().T for i in blocks], 1)
    D = torch.softmax(z, 1)
    D[torch.arange(T, device="cuda"), targets] -= 1
    want = sum(D[:, i:i + 100000] @ w[i:i + 100000].double() for i in blocks)
    # D's rounding, its error from the logits (1e-5 of p) and the sums' bias (1e-8 a column of at most
    # 65536, as a share of the sum of sizes) on every entry, then the result's rounding
    err = sum((D[:, i:i + 100000].abs() * (u(t) + 1e-5 + 6.6e-4)) @ w[i:i + 100000].double().abs() for i in blocks)
    within(dx, want, err + rounded(want.abs() + err, t), "dx")
    # as a whole: the roundings of D are independent, the bias is not
    assert float((dx.double() - want).norm() / want.norm()) <= 1.2 * u(t) + 6.6e-4
    check_status()


# fp16 has 2^30 between its smallest normal number and its largest, so -20 there
@pytest.mark.parametrize("kind,e", [("fp16", -20), ("fp16", 20), ("bf16", -30), ("bf16", 20)])
def test_dloss_far_from_one(cuda, kind, e):
    """dloss of 2^20 and 2^-30: a power of two goes through to the gradients bit for bit where both are in
    the type's normal range."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    t = TYPES[kind]
    # the gradients of dloss 1 are a few x resp. w: sized so that those of x stay in range
    scale = 1.0 if kind == "bf16" else 2.0 ** -12 if e > 0 else 2.0 ** 12
    x, w, targets = _inputs(gen, t, 130, 3000, 64)
    x, w = x * scale, w * (scale if e > 0 else 1 / scale)
    _, lse = vk.linear_xent_tensors(x, w, targets)
    ones = torch.ones(130, device="cuda")
    one = vk.linear_xent_backward_tensors(ones, lse, x, w, targets)
    got = vk.linear_xent_backward_tensors(ones * 2.0 ** e, lse, x, w, targets)
    low = torch.finfo(t).smallest_normal
    seen = 0
    for a, b in zip(got, one):
        want = b.double() * 2.0 ** e
        # the smallest normal number itself is what a little less rounds to in the coarser steps below it
        keep = (b.double().abs() > low) & (want.abs() > low) & (want.abs() < torch.finfo(t).max / 2)
        seen += int(keep.sum())
        assert torch.equal(a.double()[keep], want[keep])
    assert seen > 1000
