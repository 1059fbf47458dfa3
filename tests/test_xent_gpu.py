"""Cross entropy of a linear head, forward and backward, against 64-bit forms."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import vkblas_b200 as vk  # noqa: E402
from fused_util import TYPES, framed, rand, rel, rounded, sum_err, u, within  # noqa: E402
from gpu_util import check_status  # noqa: E402


def _inputs(gen, t, T, V, H, pad=0, off=0, spread=1.5, ignored=0.2):
    x = framed(gen, t, T, H, pad, off)[0]
    w = framed(gen, t, V, H, pad, off, spread / H ** 0.5)[0]
    targets = torch.randint(0, V, (T,), generator=gen, device="cuda")
    targets[torch.rand(T, generator=gen, device="cuda") < ignored] = -100
    return x, w, targets


def _forward64(x, w, targets):
    z = x.double() @ w.double().T
    lse = torch.logsumexp(z, 1)
    keep = targets != -100
    zt = z.gather(1, targets.clamp(min=0)[:, None])[:, 0]
    return z, lse, torch.where(keep, lse - zt, torch.zeros_like(lse)), keep


def _check_forward(x, w, targets, loss, lse):
    z, e_lse, e_loss, keep = _forward64(x, w, targets)
    ez = sum_err(x.double(), w.double())
    # lse moves by at most the largest move of a logit; exp, sums and log in fp32
    # add (V + 64) 2^-23 of the sum, so as much to its logarithm, and roundings of lse.
    V = w.shape[0]
    el = ez.amax(1) + (V + 64) * 2.0 ** -23 + 4 * 2.0 ** -23 * z.abs().amax(1)
    within(lse, e_lse, el, "lse")
    within(loss, e_loss, torch.where(keep, 2 * el + 2.0 ** -23 * e_loss.abs(), torch.zeros_like(el)), "loss")


SIZES = [(1, 1, 1), (1, 1000, 64), (2, 33, 40), (7, 257, 200), (16, 500, 72), (33, 129, 256), (64, 3001, 128),
         (127, 512, 96), (128, 256, 64), (130, 4097, 88), (256, 777, 136), (300, 9000, 264), (515, 1031, 512)]


@pytest.mark.parametrize("T,V,H", SIZES)
@pytest.mark.parametrize("kind", ["fp16", "bf16"])
def test_forward(cuda, T, V, H, kind):
    gen = torch.Generator(device="cuda").manual_seed(T + V + H)
    x, w, targets = _inputs(gen, TYPES[kind], T, V, H)
    loss, lse = vk.linear_xent_tensors(x, w, targets)
    _check_forward(x, w, targets, loss, lse)
    check_status()


@pytest.mark.parametrize("T", [3, 140, 300])
@pytest.mark.parametrize("pad,off,V,H", [(3, 0, 300, 67), (0, 1, 256, 64), (8, 8, 301, 72)])
def test_forward_any_layout(cuda, T, pad, off, V, H):
    gen = torch.Generator(device="cuda").manual_seed(T + pad)
    x, w, targets = _inputs(gen, torch.bfloat16, T, V, H, pad, off)
    _check_forward(x, w, targets, *vk.linear_xent_tensors(x, w, targets))


@pytest.mark.parametrize("T", [5, 300])
def test_forward_peaked(cuda, T):
    """Logits of hundreds: exp would overflow without the maximum."""
    gen = torch.Generator(device="cuda").manual_seed(T)
    x, w, targets = _inputs(gen, torch.bfloat16, T, 1000, 128, spread=200.0)
    loss, lse = vk.linear_xent_tensors(x, w, targets)
    assert bool(torch.isfinite(loss).all() & torch.isfinite(lse).all())
    _check_forward(x, w, targets, loss, lse)


def test_targets(cuda):
    """Every row ignored; another ignore_index; targets outside the vocabulary."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, w, targets = _inputs(gen, torch.bfloat16, 150, 300, 64, ignored=0.0)
    none = torch.full_like(targets, -100)
    loss, lse = vk.linear_xent_tensors(x, w, none)
    assert bool((loss == 0).all()) and bool(torch.isfinite(lse).all())
    dx, dw = vk.linear_xent_backward_tensors(torch.ones(150, device="cuda"), lse, x, w, none)
    assert bool((dx == 0).all()) and bool((dw == 0).all())
    loss, _ = vk.linear_xent_tensors(x, w, targets, ignore_index=int(targets[3]))
    assert bool(((loss == 0) == (targets == targets[3])).all())
    targets[7], targets[9] = 300, -5
    loss, lse = vk.linear_xent_tensors(x, w, targets)
    bad = torch.zeros(150, device="cuda", dtype=torch.bool)
    bad[[7, 9]] = True
    assert torch.equal(torch.isnan(loss), bad) and bool(torch.isfinite(lse).all())
    dx, _ = vk.linear_xent_backward_tensors(torch.ones(150, device="cuda"), lse, x, w, targets, need_dw=False)
    assert torch.equal(torch.isnan(dx).all(1), bad) and torch.equal(torch.isnan(dx).any(1), bad)


def test_infinite_logits(cuda):
    """-inf logits (a masked vocabulary) drop out; a row of nothing else has lse -inf."""
    x = torch.zeros(4, 64, device="cuda", dtype=torch.float16)
    w = torch.zeros(600, 64, device="cuda", dtype=torch.float16)
    x[:, 0] = 1
    w[:500, 0] = float("-inf")
    x[:, 1] = torch.tensor([0.0, 1.0, 2.0, -1.0], device="cuda").half()
    w[500:, 1] = (torch.arange(100, device="cuda") % 7).half()
    targets = torch.tensor([500, 599, 520, 599], device="cuda")
    loss, lse = vk.linear_xent_tensors(x, w, targets)
    z = x[:, 1:].double() @ w[500:, 1:].double().T
    want = torch.logsumexp(z, 1)
    within(lse, want, 1e-5 + 0 * want)
    within(loss, want - z.gather(1, (targets - 500)[:, None])[:, 0], 1e-5 + 0 * want)
    w[:, 0] = float("-inf")
    _, lse = vk.linear_xent_tensors(x, w, targets)
    assert bool((lse == float("-inf")).all())


@pytest.mark.parametrize("T", [6, 300])
def test_nan_stays_in_its_row(cuda, T):
    gen = torch.Generator(device="cuda").manual_seed(T)
    x, w, targets = _inputs(gen, torch.bfloat16, T, 700, 64, ignored=0.0)
    clean, clean_lse = vk.linear_xent_tensors(x, w, targets)
    x[2] = float("nan")
    loss, lse = vk.linear_xent_tensors(x, w, targets)
    keep = [i for i in range(T) if i != 2]
    assert bool(torch.isnan(loss[2])) and bool(torch.isnan(lse[2]))
    assert torch.equal(loss[keep], clean[keep]) and torch.equal(lse[keep], clean_lse[keep])


def _grads64(x, w, targets, dloss):
    z, lse, _, keep = _forward64(x, w, targets)
    p = torch.exp(z - lse[:, None])
    p[keep, targets[keep]] -= 1
    D = p * torch.where(keep, dloss.double(), torch.zeros_like(lse))[:, None]
    return D, D @ w.double(), D.T @ x.double(), z


def _check_grads(x, w, targets, dloss, dx, dw, D, ex, ew, z):
    t = x.dtype
    # D: the logits' and lse's errors move exp by that share (p <= p - onehot in
    # size, but for the target, where it is 1), one rounding to t.
    k = sum_err(x.double(), w.double()) * 2 + (w.shape[0] + 64) * 2.0 ** -23 + 8 * 2.0 ** -23 * z.abs().amax(1)[:, None]
    eD = D.abs() * u(t) + dloss.abs().double()[:, None] * torch.softmax(z, 1) * k
    if t == torch.float16:
        eD = eD + float(dloss.abs().max()) * 2.0 ** -14 * 2.0 ** -25
    for got, want, err, what in (
            (dx, ex, eD @ w.double().abs() + sum_err(D, w.double().T.contiguous()), "dx"),
            (dw, ew, eD.T @ x.double().abs() + sum_err(D.T.contiguous(), x.double().T.contiguous()), "dw")):
        if got is not None:
            within(got, want, err + rounded(want.abs() + err, t), what)


@pytest.mark.parametrize("T,V,H", SIZES + [(40, 20000, 32)])
@pytest.mark.parametrize("kind", ["fp16", "bf16"])
def test_backward(cuda, T, V, H, kind):
    gen = torch.Generator(device="cuda").manual_seed(T + 2 * V + H)
    x, w, targets = _inputs(gen, TYPES[kind], T, V, H)
    dloss = torch.rand(T, generator=gen, device="cuda") / T
    _, lse = vk.linear_xent_tensors(x, w, targets)
    dx, dw = vk.linear_xent_backward_tensors(dloss, lse, x, w, targets)
    _check_grads(x, w, targets, dloss, dx, dw, *_grads64(x, w, targets, dloss))
    check_status()


@pytest.mark.parametrize("T,pad,off,V,H", [(3, 3, 0, 300, 67), (140, 0, 1, 256, 64), (300, 8, 8, 301, 72)])
def test_backward_any_layout(cuda, T, pad, off, V, H):
    gen = torch.Generator(device="cuda").manual_seed(T + pad)
    x, w, targets = _inputs(gen, torch.bfloat16, T, V, H, pad, off)
    dloss = torch.rand(T, generator=gen, device="cuda")
    _, lse = vk.linear_xent_tensors(x, w, targets)
    dx, dw = vk.linear_xent_backward_tensors(dloss, lse, x, w, targets)
    _check_grads(x, w, targets, dloss, dx, dw, *_grads64(x, w, targets, dloss))


@pytest.mark.parametrize("size", [1e-12, 1.0, 1e6])
def test_backward_scale(cuda, size):
    """Gradients of the losses far from 1 keep D's precision in fp16."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    x, w, targets = _inputs(gen, torch.float16, 64, 5000, 64)
    _, lse = vk.linear_xent_tensors(x, w, targets)
    one = vk.linear_xent_backward_tensors(torch.ones(64, device="cuda"), lse, x, w, targets)
    if size == 1e-12:     # below fp16: the result rounds to zero, not to garbage
        got = vk.linear_xent_backward_tensors(torch.full((64,), size, device="cuda"), lse, x, w, targets)
        assert all(bool((g == 0).all()) for g in got)
        return
    c = 0.25 * min(size, 8.0)
    got = vk.linear_xent_backward_tensors(torch.full((64,), c, device="cuda"), lse, x, w, targets)
    for a, b in zip(got, one):
        # c is a power of two, so both round the same number g but for its scale:
        # |a - c b| <= |a - c g| + c |g - b|, a rounding of a and c roundings of b.
        b = b.double()
        within(a, c * b, rounded(c * b * (1 + 2 * u(torch.float16)), torch.float16)
               + c * rounded(b * (1 + 2 * u(torch.float16)), torch.float16))


def test_backward_parts_and_broadcast(cuda):
    gen = torch.Generator(device="cuda").manual_seed(4)
    x, w, targets = _inputs(gen, torch.bfloat16, 80, 1000, 64)
    _, lse = vk.linear_xent_tensors(x, w, targets)
    dloss = torch.ones(80, device="cuda")
    dx, dw = vk.linear_xent_backward_tensors(dloss, lse, x, w, targets)
    a = vk.linear_xent_backward_tensors(dloss[:1].expand(80), lse, x, w, targets, need_dw=False)
    b = vk.linear_xent_backward_tensors(dloss, lse, x, w, targets, need_dx=False)
    assert torch.equal(a[0], dx) and a[1] is None and b[0] is None and torch.equal(b[1], dw)


@pytest.mark.parametrize("T", [20, 200])
def test_ignored_rows_may_hold_anything(cuda, T):
    """NaN in the rows of padding tokens reaches no gradient."""
    gen = torch.Generator(device="cuda").manual_seed(T)
    x, w, targets = _inputs(gen, torch.bfloat16, T, 600, 64, ignored=0.4)
    dloss = torch.rand(T, generator=gen, device="cuda")
    _, lse = vk.linear_xent_tensors(x, w, targets)
    want = vk.linear_xent_backward_tensors(dloss, lse, x, w, targets)
    x[targets == -100] = float("nan")
    dloss[targets == -100] = float("nan")
    loss, lse = vk.linear_xent_tensors(x, w, targets)
    assert bool((loss[targets == -100] == 0).all())
    got = vk.linear_xent_backward_tensors(dloss, lse, x, w, targets)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_backward_against_differences(cuda):
    gen = torch.Generator(device="cuda").manual_seed(12)
    t, T, V, H = torch.float16, 60, 400, 72
    x, w, targets = _inputs(gen, t, T, V, H)
    dloss = torch.rand(T, generator=gen, device="cuda")
    _, lse = vk.linear_xent_tensors(x, w, targets)
    grads = vk.linear_xent_backward_tensors(dloss, lse, x, w, targets)
    ins = [x.double(), w.double()]

    def loss(a, b):
        return (_forward64(a, b, targets)[2] * dloss.double()).sum()

    for i in range(2):
        v = torch.randn(ins[i].shape, generator=gen, device="cuda", dtype=torch.float64)
        lo, hi = ([q + s * 1e-5 * v if j == i else q for j, q in enumerate(ins)] for s in (-1, 1))
        want = float((loss(*hi) - loss(*lo)) / 2e-5)
        got = float((grads[i].double() * v).sum())
        # D and the result are rounded to t independently; differences err by 1e-10.
        assert abs(got - want) <= 8 * u(t) * float(torch.linalg.norm(grads[i].double())) + 1e-4 * abs(want)


def test_stream_and_capture(cuda):
    gen = torch.Generator(device="cuda").manual_seed(5)
    x, w, targets = _inputs(gen, torch.bfloat16, 300, 5000, 128)
    dloss = torch.rand(300, generator=gen, device="cuda")

    def step(stream=None):
        loss, lse = vk.linear_xent_tensors(x, w, targets, stream=stream)
        return (loss, lse, *vk.linear_xent_backward_tensors(dloss, lse, x, w, targets, stream=stream))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = step(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            graphs.append((gr, step()))
    x.copy_(rand(gen, torch.bfloat16, 300, 128))
    targets.copy_(targets.flip(0))
    want = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for s, (gr, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    for _, got in graphs:
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    check_status()


def test_block_head_and_step(cuda):
    """A training step of a block and its head as they are used together: the
    block, the down projection on the engine's GEMM, the loss, and back; the
    gradients against the whole step's in 64 bits."""
    gen = torch.Generator(device="cuda").manual_seed(21)
    t, T, H, F, V = torch.bfloat16, 200, 128, 384, 1500
    x = rand(gen, t, T, H)
    wg, wu = rand(gen, t, F, H, scale=H ** -0.5), rand(gen, t, F, H, scale=H ** -0.5)
    wd, wv = rand(gen, t, H, F, scale=2 * F ** -0.5), rand(gen, t, V, H, scale=H ** -0.5)
    targets = torch.randint(0, V, (T,), generator=gen, device="cuda")
    targets[::9] = -100
    n = int((targets != -100).sum())
    h, g, up = vk.gated_tensors(x, wg, wu, "silu", save=True)
    y = torch.empty(T, H, device="cuda", dtype=t)
    vk.gemm_tensors(vk.OP_N, vk.OP_T, T, H, F, 1.0, h, F, wd, F, 0.0, y, H)
    loss, lse = vk.linear_xent_tensors(y, wv, targets)
    dy, dwv = vk.linear_xent_backward_tensors(torch.full((T,), 1.0 / n, device="cuda"), lse, y, wv, targets)
    dh, dwd = torch.empty(T, F, device="cuda", dtype=t), torch.empty(H, F, device="cuda", dtype=t)
    vk.gemm_tensors(vk.OP_N, vk.OP_N, T, F, H, 1.0, dy, H, wd, F, 0.0, dh, F)
    vk.gemm_tensors(vk.OP_T, vk.OP_N, H, F, T, 1.0, dy, H, h, F, 0.0, dwd, F)
    dx, dwg, dwu = vk.gated_backward_tensors(dh, g, up, x, wg, wu, "silu")
    with torch.enable_grad():
        ref = [v.double().requires_grad_() for v in (x, wg, wu, wd, wv)]
        X, G, U, D, W = ref
        z = (torch.nn.functional.silu(X @ G.T) * (X @ U.T)) @ D.T @ W.T
        torch.nn.functional.cross_entropy(z, targets, ignore_index=-100).backward()
    # Every stage rounds to t: h, y, D, dy, dh, dG, dU, g, u and the result, each an
    # independent relative error of at most u; ten of them stay below 10 u.
    assert abs(float(loss.sum() / n) - float(torch.nn.functional.cross_entropy(z.detach(), targets))) < 10 * u(t)
    for got, want in zip((dx, dwg, dwu, dwd, dwv), ref):
        assert rel(got, want.grad) <= 10 * u(t)
    check_status()
