"""Fused products whose offsets pass 32 bits, and a first call inside a capture."""
import os
import subprocess
import sys
import textwrap

import pytest
import torch

pytestmark = pytest.mark.gpu

import vkblas_b200 as vk  # noqa: E402
from fused_util import act64, rand, rounded, sum_err, u, within  # noqa: E402
from gpu_util import check_status  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(autouse=True)
def _free():
    yield
    torch.cuda.empty_cache()


def test_gated_output_past_32_bits(cuda):
    """330000 x 13104 outputs: 4.3e9 elements."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    t, M, F, H = torch.bfloat16, 330000, 13104, 64
    x, wg, wu = rand(gen, t, M, H), rand(gen, t, F, H, scale=0.25), rand(gen, t, F, H, scale=0.125)
    h = vk.gated_tensors(x, wg, wu, "silu")
    for r in (0, 1, 163840, 327680, 327807, M - 1):
        X, G, U = x[r:r + 1].double(), wg.double(), wu.double()
        zg, zu = X @ G.T, X @ U.T
        eg, eu = sum_err(X, G), sum_err(X, U)
        a = act64(zg, "silu")[0]
        err = (1.13 * eg + a.abs() * 2.0 ** -16) * (zu.abs() + eu) + a.abs() * eu
        within(h[r:r + 1], a * zu, err + rounded((a * zu).abs() + err, t), f"row {r}")
    check_status()


def test_xent_weights_past_32_bits(cuda):
    """A head of 1100000 x 4096 weights: 4.5e9 elements, read and as a gradient written."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    t, T, V, H = torch.bfloat16, 24, 1100000, 4096
    x = rand(gen, t, T, H)
    w = torch.empty(V, H, device="cuda", dtype=t)
    for i in range(0, V, 100000):
        w[i:i + 100000] = rand(gen, t, 100000, H, scale=1.5 / 64)
    targets = torch.randint(0, V, (T,), generator=gen, device="cuda")
    targets[:4] = torch.tensor([0, V - 1, 1048576, 1048575], device="cuda")
    loss, lse = vk.linear_xent_tensors(x, w, targets)
    parts, zt = [], torch.empty(T, device="cuda", dtype=torch.float64)
    for i in range(0, V, 100000):
        z = x.double() @ w[i:i + 100000].double().T
        parts.append(torch.logsumexp(z, 1))
        here = (targets >= i) & (targets < i + 100000)
        zt[here] = z[here, targets[here] - i]
    want = torch.logsumexp(torch.stack(parts), 0)
    # K = 4096 in segments of 512: 3.3e-7 of the logits' size (up to 10), the sum of V exponentials
    # in fp32 by pairs and blocks
    within(lse, want, 1e-5 + 0 * want, "lse")
    within(loss, want - zt, 1e-5 + 0 * want, "loss")
    dloss = torch.ones(T, device="cuda")
    dx, dw = vk.linear_xent_backward_tensors(dloss, lse, x, w, targets)
    rows = torch.cat((targets, torch.tensor([1, 1048577, V - 2], device="cuda")))
    z = x.double() @ w[rows].double().T
    D = torch.exp(z - want[:, None]) - (targets[:, None] == rows[None]).double()
    ref = D.T @ x.double()
    # D: its rounding, the logits' 3e-5 as a share of p
    err = (D.abs() * (u(t) + 1e-4)).T @ x.double().abs()
    within(dw[rows], ref, err + rounded(ref.abs() + err, t), "dw")
    assert bool(torch.isfinite(dx).all())
    check_status()


def test_q4_weights_past_32_bits(cuda):
    """1100000 x 8192 four-bit weights: 4.5e9 bytes."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    t, N, K, G = torch.float16, 1100000, 8192, 128
    q = torch.randint(0, 256, (N, K // 2), generator=gen, device="cuda", dtype=torch.uint8)
    s = (torch.rand(N, K // G, generator=gen, device="cuda") * 0.01 + 0.005).to(t)
    w = vk.q4_pack_tensors(q, s, None, K, G)
    x = rand(gen, t, 3, K)
    y = vk.gemv_q4_tensors(x, w)
    rows = torch.tensor([0, 15, 16, 524288, 1048575, 1048576, N - 17, N - 1], device="cuda")
    n = torch.stack((q[rows] & 15, q[rows] >> 4), -1).reshape(len(rows), -1).double() - 8
    W = n * s[rows].double().repeat_interleave(G, 1)
    want = x.double() @ W.T
    err = (K + 64) * 2.0 ** -23 * (x.double().abs() @ W.abs().T)
    within(y[:, rows], want, err + rounded(want.abs() + err, t), "y")


def test_first_call_inside_a_capture(cuda):
    """A process whose first use of the library is captured into a graph."""
    code = textwrap.dedent("""
        import torch, vkblas_b200 as vk
        t = torch.bfloat16
        x, w = torch.randn(300, 128, device="cuda").to(t), torch.randn(520, 128, device="cuda").to(t)
        tg = torch.arange(300, device="cuda")
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            h, a, b = vk.gated_tensors(x, w, w, save=True)
            s = vk.gated_tensors(x[:5], w, w)
            grads = vk.gated_backward_tensors(h, a, b, x, w, w)
            loss, lse = vk.linear_xent_tensors(x, w, tg)
            dx, dw = vk.linear_xent_backward_tensors(loss, lse, x, w, tg)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(h, vk.gated_tensors(x, w, w)) and torch.equal(s, vk.gated_tensors(x[:5], w, w))
        assert torch.equal(loss, vk.linear_xent_tensors(x, w, tg)[0])
        assert torch.equal(dw, vk.linear_xent_backward_tensors(loss, lse, x, w, tg)[1])
        assert vk.device_status() == 0
        print("ok")
    """)
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stderr[-2000:]


def test_calls_side_by_side(cuda):
    """The same products on four streams at once give what one alone gives."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    t = torch.float16
    x, wg, wu = rand(gen, t, 520, 256), rand(gen, t, 1032, 256, scale=0.1), rand(gen, t, 1032, 256, scale=0.1)
    w = rand(gen, t, 3001, 256, scale=0.1)
    tg = torch.randint(0, 3001, (520,), generator=gen, device="cuda")
    ones = torch.ones(520, device="cuda")

    def step(s=None):
        h, g, up = vk.gated_tensors(x, wg, wu, "gelu", save=True, stream=s)
        loss, lse = vk.linear_xent_tensors(x, w, tg, stream=s)
        return (h, *vk.gated_backward_tensors(h, g, up, x, wg, wu, "gelu", stream=s), loss,
                *vk.linear_xent_backward_tensors(ones, lse, x, w, tg, stream=s))

    want = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = [step(s) for _ in range(3) for s in streams]
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(a, b) for a, b in zip(want, r))
    check_status()
