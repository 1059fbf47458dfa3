"""Cross entropy of a linear head where its gradients are small differences, its sums long and its
sizes take more than one piece or segment, against 64-bit forms."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import vkblas_b200 as vk  # noqa: E402
from fused_util import TYPES, rand, rounded, sum_err, u, within  # noqa: E402
from gpu_util import check_status  # noqa: E402


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
