"""Decode products with 4-bit weights and group scales against the 64-bit form."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu

import vkblas_b200 as vk  # noqa: E402
from fused_util import TYPES, framed, outside_untouched, rand, rounded, within  # noqa: E402


def _weights(gen, t, N, K, group, zeros, pad=0):
    ng = -(-K // group)
    q = torch.randint(0, 256, (N, (K + 1) // 2 + pad), generator=gen, device="cuda", dtype=torch.uint8)[:, :(K + 1) // 2]
    scales = ((torch.rand(N, ng + pad, generator=gen, device="cuda") + 0.5) * 0.25 * K ** -0.5).to(t)[:, :ng]
    z = torch.randint(0, 16, (N, ng + pad), generator=gen, device="cuda", dtype=torch.uint8)[:, :ng] if zeros else None
    return q, scales, z


def _dense64(q, scales, z, K, group):
    n = torch.stack((q & 15, q >> 4), -1).reshape(q.shape[0], -1)[:, :K].double()
    zz = 8.0 if z is None else z.double().repeat_interleave(group, 1)[:, :K]
    return (n - zz) * scales.double().repeat_interleave(group, 1)[:, :K]


def _check(x, W, y, alpha=1.0, beta=0.0, y0=None):
    t = x.dtype
    X = x.double()
    want = alpha * (X @ W.T)
    # products and group sums are exact or fp32; scales and partial sums fp32
    err = abs(alpha) * (x.shape[1] + 64) * 2.0 ** -23 * (X.abs() @ W.abs().T)
    if y0 is not None:
        want = want + beta * y0.double()
        err = err + 4 * 2.0 ** -24 * (want.abs() + (beta * y0.double()).abs())
    within(y, want, err + rounded(want.abs() + err, t), "y")


SIZES = [(1, 1, 1), (1, 16, 128), (1, 17, 32), (2, 100, 130), (3, 5, 33), (4, 333, 256), (7, 64, 1000), (8, 31, 4096),
         (9, 200, 96), (12, 48, 2049), (16, 129, 512), (1, 4096, 640), (5, 1000, 1100)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("group,zeros", [(32, False), (64, True), (128, False), (128, True), (96, True), (4096, False)])
def test_gemv(cuda, M, N, K, kind, group, zeros):
    gen = torch.Generator(device="cuda").manual_seed(M + N + K + group)
    t = TYPES[kind]
    q, s, z = _weights(gen, t, N, K, group, zeros)
    w = vk.q4_pack_tensors(q, s, z, K, group)
    x = rand(gen, t, M, K)
    _check(x, _dense64(q, s, z, K, group), vk.gemv_q4_tensors(x, w))


@pytest.mark.parametrize("M", [1, 6, 16])
@pytest.mark.parametrize("pad,off", [(1, 0), (2, 2), (4, 4), (8, 8), (3, 1)])
def test_layouts_and_scalars(cuda, M, pad, off):
    """Strided operands off the 16-byte grid, alpha and beta, an output inside a larger buffer."""
    gen = torch.Generator(device="cuda").manual_seed(M + pad)
    N, K, group, t = 77, 420, 64, torch.float16
    q, s, z = _weights(gen, t, N, K, group, True, pad=5)
    w = vk.q4_pack_tensors(q, s, z, K, group)
    W = _dense64(q, s, z, K, group)
    x = framed(gen, t, M, K, pad, off)[0]
    out, buf = framed(gen, t, M, N, pad, off, fill=3.0)
    assert vk.gemv_q4_tensors(x, w, out=out, alpha=-0.5, beta=2.0) is out
    _check(x, W, out, -0.5, 2.0, torch.full((M, N), 3.0, device="cuda"))
    assert outside_untouched(out, buf, 3.0)
    out.fill_(float("nan"))
    vk.gemv_q4_tensors(x, w, out=out)          # beta 0: not read
    _check(x, W, out)


def test_every_nibble_and_zero_point(cuda):
    """All 16 x 16 pairs of weight and zero point, one by one."""
    for t in TYPES.values():
        N, K, group = 256, 64, 32
        n = torch.arange(N, device="cuda")
        q = ((n % 16) | (n % 16) << 4).to(torch.uint8)[:, None].expand(N, K // 2).contiguous()
        z = (n // 16).to(torch.uint8)[:, None].expand(N, 2).contiguous()
        s = torch.ones(N, 2, device="cuda", dtype=t)
        w = vk.q4_pack_tensors(q, s, z, K, group)
        x = torch.zeros(16, K, device="cuda", dtype=t)
        x[torch.arange(16), torch.arange(16) * 4 + 1] = 1.0
        y = vk.gemv_q4_tensors(x, w)
        want = (n % 16 - n // 16).to(t)[None].expand(16, N)
        assert torch.equal(y, want)


def test_positions(cuda):
    """Each k alone reaches the output with its own weight."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    t, N, K, group = torch.float16, 40, 300, 32
    q, s, z = _weights(gen, t, N, K, group, True)
    w, W = vk.q4_pack_tensors(q, s, z, K, group), _dense64(q, s, z, K, group)
    for k0 in range(0, K, 16):
        m = min(16, K - k0)
        x = torch.zeros(m, K, device="cuda", dtype=t)
        x[torch.arange(m), k0 + torch.arange(m)] = 1.0
        assert torch.equal(vk.gemv_q4_tensors(x, w), W[:, k0:k0 + m].T.to(t))


def test_nan_stays_in_its_row(cuda):
    gen = torch.Generator(device="cuda").manual_seed(3)
    t = torch.bfloat16
    q, s, z = _weights(gen, t, 100, 256, 128, False)
    w = vk.q4_pack_tensors(q, s, z, 256, 128)
    x = rand(gen, t, 9, 256)
    clean = vk.gemv_q4_tensors(x, w)
    x[4, 17] = float("inf")
    x[5] = float("nan")
    y = vk.gemv_q4_tensors(x, w)
    keep = [0, 1, 2, 3, 6, 7, 8]
    assert torch.equal(y[keep], clean[keep]) and bool(torch.isnan(y[5]).all())
    assert not bool(torch.isfinite(y[4]).any() & (torch.isfinite(y[4]) & (y[4] != y[4])).any())


def test_pack_reads_only_the_low_zero_bits_and_keeps_its_buffer(cuda):
    gen = torch.Generator(device="cuda").manual_seed(4)
    t, N, K = torch.float16, 33, 200
    q, s, z = _weights(gen, t, N, K, 32, True)
    x = rand(gen, t, 2, K)
    a = vk.gemv_q4_tensors(x, vk.q4_pack_tensors(q, s, z, K, 32))
    b = vk.gemv_q4_tensors(x, vk.q4_pack_tensors(q, s, z | 0xA0, K, 32))
    assert torch.equal(a, b)
    # nothing past the packed size is written
    st = vk.fused.Q4(vk.DT_F16, N, K, 32, 1, None)
    n = vk.lib.vkblas_b200_q4_bytes(C.byref(st))
    buf = torch.full((n + 4096,), 0x5A, device="cuda", dtype=torch.uint8)
    assert vk.lib.vkblas_b200_q4_pack(C.byref(st), q.data_ptr(), q.stride(0), s.data_ptr(), s.stride(0), z.data_ptr(),
                                      z.stride(0), buf.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    assert bool((buf[n:] == 0x5A).all())


def test_stream_and_capture(cuda):
    gen = torch.Generator(device="cuda").manual_seed(6)
    t = torch.bfloat16
    q, s, z = _weights(gen, t, 520, 4096, 128, True)
    w = vk.q4_pack_tensors(q, s, z, 4096, 128)
    x = rand(gen, t, 4, 4096)
    want = vk.gemv_q4_tensors(x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = vk.gemv_q4_tensors(x, w, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        y = vk.gemv_q4_tensors(x, w)
    x.copy_(rand(gen, t, 4, 4096))
    gr.replay()
    assert torch.equal(y, vk.gemv_q4_tensors(x, w))


def test_q4_block_decode(cuda):
    """One token's block with 16-bit gate and up projections and a 4-bit down projection."""
    gen = torch.Generator(device="cuda").manual_seed(8)
    t, M, H, F = torch.float16, 3, 256, 1024
    x = rand(gen, t, M, H)
    wg, wu = rand(gen, t, F, H, scale=H ** -0.5), rand(gen, t, F, H, scale=H ** -0.5)
    q, s, z = _weights(gen, t, H, F, 128, True)
    y = vk.gemv_q4_tensors(vk.gated_tensors(x, wg, wu, "gelu"), vk.q4_pack_tensors(q, s, z, F, 128))
    h = torch.nn.functional.gelu(x.double() @ wg.double().T) * (x.double() @ wu.double().T)
    W = _dense64(q, s, z, F, 128)
    # h is rounded once, the result once: at most u of their sizes each
    err = (2.0 ** -11 + 2.0 ** -14) * (h.abs() @ W.abs().T)
    want = h @ W.T
    within(y, want, err + rounded(want.abs() + err, t), "y")
