"""The gated feed-forward block and its backward pass against 64-bit forms."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import vkblas_b200 as vk  # noqa: E402
from fused_util import (TYPES, act64, framed, outside_untouched, rand, rel, rounded,  # noqa: E402
                        sum_err, u, within)
from gpu_util import check_status  # noqa: E402

ACTS = ["silu", "gelu", "gelu_tanh"]


def _inputs(gen, t, M, F, H, pad=0, off=0, scale=1.0):
    x = framed(gen, t, M, H, pad, off, scale)[0]
    wg = framed(gen, t, F, H, pad, off, 2.0 / H ** 0.5)[0]
    wu = framed(gen, t, F, H, 2 * pad, off, 1.0 / H ** 0.5)[0]
    return x, wg, wu


def _check_forward(x, wg, wu, act, h, g=None, up=None):
    t = x.dtype
    X, G, U = x.double(), wg.double(), wu.double()
    zg, zu = X @ G.T, X @ U.T
    eg, eu = sum_err(X, G), sum_err(X, U)
    a, _ = act64(zg, act)
    # |act'| <= 1.13; the activation itself is a few fp32 roundings (2^-20)
    ea = 1.13 * eg + a.abs() * 2.0 ** -20
    want = a * zu
    err = ea * (zu.abs() + eu) + a.abs() * eu
    within(h, want, err + rounded(want.abs() + err, t), "h")
    if g is not None:
        within(g, zg, eg + rounded(zg.abs() + eg, t), "g")
        within(up, zu, eu + rounded(zu.abs() + eu, t), "u")


# M through the token form (<= 16), its end, one tile, ragged tiles, two tiles and more
FORWARD = [
    (1, 1, 1), (1, 128, 64), (1, 300, 512), (3, 77, 200), (8, 136, 1024), (9, 5, 40), (16, 264, 96),
    (17, 128, 64), (33, 129, 72), (64, 257, 128), (128, 128, 256), (129, 384, 200), (255, 96, 88),
    (256, 256, 128), (257, 130, 136), (300, 1000, 264), (513, 520, 520),
]


@pytest.mark.parametrize("M,F,H", FORWARD)
@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("save", [False, True])
def test_forward(cuda, M, F, H, kind, save):
    gen = torch.Generator(device="cuda").manual_seed(M * 7 + F * 3 + H)
    act = ACTS[(M + F + H) % 3]
    x, wg, wu = _inputs(gen, TYPES[kind], M, F, H)
    r = vk.gated_tensors(x, wg, wu, act, save=save)
    h, g, up = r if save else (r, None, None)
    _check_forward(x, wg, wu, act, h, g, up)
    check_status()


# row padding and a start off the 16-byte grid, in elements; F and H odd
@pytest.mark.parametrize("M", [1, 5, 13, 40, 200, 300])
@pytest.mark.parametrize("pad,off,F,H", [(8, 0, 136, 128), (3, 0, 133, 67), (0, 1, 128, 64),
                                         (5, 3, 65, 77), (8, 8, 131, 72)])
def test_forward_any_layout(cuda, M, pad, off, F, H):
    gen = torch.Generator(device="cuda").manual_seed(M + pad + off)
    t = torch.bfloat16
    x, wg, wu = _inputs(gen, t, M, F, H, pad, off)
    out, buf = framed(gen, t, M, F, pad, off, fill=7.0)
    assert vk.gated_tensors(x, wg, wu, "gelu", out=out) is out
    _check_forward(x, wg, wu, "gelu", out)
    assert outside_untouched(out, buf, 7.0)
    check_status()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M", [2, 20, 260])
def test_forward_saturated(cuda, act, M):
    """Projections far out on both sides: no overflow in the activation."""
    gen = torch.Generator(device="cuda").manual_seed(M)
    x, wg, wu = _inputs(gen, torch.bfloat16, M, 128, 64, scale=60.0)
    h = vk.gated_tensors(x, wg, wu, act)
    assert bool(torch.isfinite(h).all())
    _check_forward(x, wg, wu, act, h)


@pytest.mark.parametrize("M", [4, 300])
def test_forward_keeps_nan_to_its_row(cuda, M):
    gen = torch.Generator(device="cuda").manual_seed(M)
    x, wg, wu = _inputs(gen, torch.float16, M, 200, 64)
    clean = vk.gated_tensors(x, wg, wu, "silu")
    x[1] = float("nan")
    x[2] = float("inf")
    h = vk.gated_tensors(x, wg, wu, "silu")
    assert bool(torch.isnan(h[1]).all())
    keep = [i for i in range(M) if i not in (1, 2)]
    assert torch.equal(h[keep], clean[keep])


def _grads64(dh, g, up, x, wg, wu, act):
    a, d = act64(g.double(), act)
    dG, dU = dh.double() * up.double() * d, dh.double() * a
    X = x.double()
    return dG, dU, dG @ wg.double() + dU @ wu.double(), dG.T @ X, dU.T @ X


BACKWARD = [(1, 1, 1), (1, 100, 64), (5, 33, 40), (16, 128, 128), (17, 130, 72), (64, 8, 136),
            (129, 264, 200), (256, 256, 256), (300, 515, 264), (520, 384, 512), (1000, 96, 88)]


@pytest.mark.parametrize("M,F,H", BACKWARD)
@pytest.mark.parametrize("kind", ["fp16", "bf16"])
def test_backward(cuda, M, F, H, kind):
    gen = torch.Generator(device="cuda").manual_seed(M + 5 * F + H)
    t, act = TYPES[kind], ACTS[(M + F) % 3]
    x, wg, wu = _inputs(gen, t, M, F, H)
    g, up, dh = rand(gen, t, M, F, scale=2.0), rand(gen, t, M, F), rand(gen, t, M, F, scale=0.1)
    dx, dwg, dwu = vk.gated_backward_tensors(dh, g, up, x, wg, wu, act)
    dG, dU, ex, eg, eu = _grads64(dh, g, up, x, wg, wu, act)
    # dG and dU carry a rounding to t (and 2^-19 of fp32 work), the sums theirs, the result one.
    def check(got, want, pairs, what):
        err = sum((u(t) + 2.0 ** -19) * (a.abs() @ b.abs()) + sum_err(a, b.T.contiguous())
                  + 2 * (rounded(torch.zeros(1, device="cuda"), t) * b.abs().sum(0)) for a, b in pairs)
        within(got, want, err + rounded(want.abs() + err, t), what)
    X = x.double()
    check(dx, ex, [(dG, wg.double()), (dU, wu.double())], "dx")
    check(dwg, eg, [(dG.T, X)], "dw_gate")
    check(dwu, eu, [(dU.T, X)], "dw_up")
    if M * F * H > 1e6 and kind == "bf16":
        # Two roundings of rms u / sqrt 3 each, independent from element to element.
        for got, want in ((dx, ex), (dwg, eg), (dwu, eu)):
            assert rel(got, want) <= 1.2 * u(t)
    check_status()


@pytest.mark.parametrize("M,pad,off,F,H", [(40, 3, 0, 133, 67), (300, 0, 1, 128, 64), (300, 5, 3, 65, 77),
                                           (17, 8, 8, 136, 72)])
def test_backward_any_layout(cuda, M, pad, off, F, H):
    """Strided and unaligned inputs give what compact ones give, bit for bit."""
    gen = torch.Generator(device="cuda").manual_seed(M + pad)
    t = torch.float16
    x, wg, wu = _inputs(gen, t, M, F, H, pad, off)
    dh, g, up = (framed(gen, t, M, F, pad, off)[0] for _ in range(3))
    got = vk.gated_backward_tensors(dh, g, up, x, wg, wu, "gelu_tanh")
    want = vk.gated_backward_tensors(*(v.clone(memory_format=torch.contiguous_format)
                                       for v in (dh, g, up, x, wg, wu)), "gelu_tanh")
    for a, b, f in zip(got, want, _grads64(dh, g, up, x, wg, wu, "gelu_tanh")[2:]):
        assert rel(a, f) <= 2 * u(t) and rel(b, f) <= 2 * u(t)
    check_status()


def test_backward_parts(cuda):
    """One gradient alone is what both calls together give."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    x, wg, wu = _inputs(gen, torch.bfloat16, 70, 96, 64)
    dh, g, up = (rand(gen, torch.bfloat16, 70, 96) for _ in range(3))
    dx, dwg, dwu = vk.gated_backward_tensors(dh, g, up, x, wg, wu)
    a = vk.gated_backward_tensors(dh, g, up, x, wg, wu, need_dw=False)
    b = vk.gated_backward_tensors(dh, g, up, x, wg, wu, need_dx=False)
    assert torch.equal(a[0], dx) and a[1] is None and a[2] is None
    assert b[0] is None and torch.equal(b[1], dwg) and torch.equal(b[2], dwu)


@pytest.mark.parametrize("act", ACTS)
def test_backward_against_differences(cuda, act):
    """<gradient, v> against central differences of the 64-bit loss sum(h dh)."""
    gen = torch.Generator(device="cuda").manual_seed(11)
    t, M, F, H = torch.float16, 48, 160, 72
    x, wg, wu = _inputs(gen, t, M, F, H)
    dh = rand(gen, t, M, F)
    _, g, up = vk.gated_tensors(x, wg, wu, act, save=True)
    grads = vk.gated_backward_tensors(dh, g, up, x, wg, wu, act)
    ins = [v.double() for v in (x, wg, wu)]

    def loss(a, b, c):
        return (act64(a @ b.T, act)[0] * (a @ c.T) * dh.double()).sum()

    for i in range(3):
        v = torch.randn(ins[i].shape, generator=gen, device="cuda", dtype=torch.float64)
        e = 1e-5
        lo, hi = ([w + s * e * v if j == i else w for j, w in enumerate(ins)] for s in (-1, 1))
        want = float((loss(*hi) - loss(*lo)) / (2 * e))
        got = float((grads[i].double() * v).sum())
        # g, u, dG, dU and the result are rounded to t, independently: rms error of a
        # random direction is a few u of |gradient|; differences err by e^2.
        assert abs(got - want) <= 8 * u(t) * float(torch.linalg.norm(grads[i].double())) + 1e-4 * abs(want)


def test_stream_and_capture(cuda):
    """A side stream, and forward with backward captured and replayed on new inputs."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    t, M, F, H = torch.bfloat16, 300, 264, 128
    x, wg, wu = _inputs(gen, t, M, F, H)
    dh = rand(gen, t, M, F)

    def step(stream=None):
        h, g, up = vk.gated_tensors(x, wg, wu, save=True, stream=stream)
        return (h, *vk.gated_backward_tensors(dh, g, up, x, wg, wu, stream=stream))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = step(side)
    raw = step(side.cuda_stream)
    torch.cuda.synchronize()
    for a, b, c in zip(want, got, raw):
        assert torch.equal(a, b) and torch.equal(a, c)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            graphs.append((gr, step()))
    x.copy_(rand(gen, t, M, H))
    dh.copy_(rand(gen, t, M, F))
    want = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for s, (gr, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    for _, got in graphs:
        for a, b in zip(want, got):
            assert torch.equal(a, b)
    check_status()


def test_repeats_bit_for_bit(cuda):
    gen = torch.Generator(device="cuda").manual_seed(6)
    x, wg, wu = _inputs(gen, torch.bfloat16, 520, 1032, 512)
    dh, g, up = (rand(gen, torch.bfloat16, 520, 1032) for _ in range(3))
    first = (vk.gated_tensors(x, wg, wu), *vk.gated_backward_tensors(dh, g, up, x, wg, wu))
    for _ in range(3):
        again = (vk.gated_tensors(x, wg, wu), *vk.gated_backward_tensors(dh, g, up, x, wg, wu))
        assert all(torch.equal(a, b) for a, b in zip(first, again))
