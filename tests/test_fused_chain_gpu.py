"""Fused products one after the other on buffers that are written and read again, as a decode loop
and a training step use them: the same results as with a wait for the GPU between the calls."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import vkblas_b200 as vk  # noqa: E402
from fused_util import TYPES, framed, rand  # noqa: E402
from gpu_util import check_status  # noqa: E402


def _compare(chain):
    """chain(wait) -> tensors, from the same start every time: waiting after each call, not
    waiting, and captured and replayed."""
    want = chain(torch.cuda.synchronize)
    for _ in range(5):
        got = chain(lambda: None)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain(lambda: None)
    for _ in range(5):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert all(bool(torch.isfinite(a).all() & (a != 0).any()) for a in want)
    check_status()


@pytest.mark.parametrize("M", [1, 5, 16])
@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("pad,off", [(0, 0), (3, 1)])
def test_decode_loop_on_two_buffers(cuda, M, kind, pad, off):
    """Layers read one of two buffers and write the other; every call's input was written by the call
    before it, and the buffer it writes was read by the call before that."""
    gen = torch.Generator(device="cuda").manual_seed(M)
    t, H, F = TYPES[kind], 256, 520
    wg, wu = (rand(gen, t, F, H, scale=H ** -0.5) for _ in range(2))
    q = torch.randint(0, 256, (H, F // 2), generator=gen, device="cuda", dtype=torch.uint8)
    s = ((torch.rand(H, (F + 31) // 32, generator=gen, device="cuda") + 0.5) * 0.25 * F ** -0.5).to(t)
    w = vk.q4_pack_tensors(q, s, None, F, 32)
    start = [rand(gen, t, M, H) for _ in range(2)]
    ab = [framed(gen, t, M, H, pad, off)[0] for _ in range(2)]
    h = framed(gen, t, M, F, pad, off)[0]

    def chain(wait):
        for v, x in zip(ab, start):
            v.copy_(x)
        wait()
        for i in range(40):
            vk.gated_tensors(ab[i % 2], wg, wu, out=h)
            wait()
            vk.gemv_q4_tensors(h, w, out=ab[1 - i % 2], alpha=0.5, beta=0.75)
            wait()
        return [ab[0].clone(), ab[1].clone(), h.clone()]

    _compare(chain)


@pytest.mark.parametrize("M", [40, 300])
def test_blocks_on_two_unaligned_buffers(cuda, M):
    """Inputs off the 16-byte grid are copied first: the copy sees what the block before wrote."""
    gen = torch.Generator(device="cuda").manual_seed(M)
    t, H = torch.bfloat16, 67
    wg, wu = (rand(gen, t, H, H, scale=1.25 * H ** -0.5) for _ in range(2))
    start = rand(gen, t, M, H)
    ab = [framed(gen, t, M, H, 2, 1)[0] for _ in range(2)]

    def chain(wait):
        ab[0].copy_(start)
        wait()
        for i in range(6):
            vk.gated_tensors(ab[i % 2], wg, wu, out=ab[1 - i % 2])
            wait()
        return [ab[0].clone(), ab[1].clone()]

    _compare(chain)


@pytest.mark.parametrize("T,H", [(24, 96), (300, 131)])
def test_steps_on_one_buffer(cuda, T, H):
    """A head's input is written by the block before it, step after step in the same buffer."""
    gen = torch.Generator(device="cuda").manual_seed(T)
    t, V = torch.bfloat16, 1000
    xs = [rand(gen, t, T, H) for _ in range(4)]
    wg, wu = (rand(gen, t, H, H, scale=H ** -0.5) for _ in range(2))
    w = rand(gen, t, V, H, scale=H ** -0.5)
    targets = torch.randint(0, V, (T,), generator=gen, device="cuda")
    targets[::5] = -100
    dloss = torch.rand(T, generator=gen, device="cuda")
    y = framed(gen, t, T, H, 1, 0)[0]

    def chain(wait):
        out = []
        for x in xs:
            vk.gated_tensors(x, wg, wu, out=y)
            wait()
            loss, lse = vk.linear_xent_tensors(y, w, targets)
            wait()
            out += [loss, *vk.linear_xent_backward_tensors(dloss, lse, y, w, targets)]
            wait()
        return out

    _compare(chain)
