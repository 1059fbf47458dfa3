"""Refusals of the fused products, before any device work (no GPU)."""
import ctypes as C

import pytest
import torch

import vkblas_b200 as vk
from vkblas_b200 import fused as F

P = 4096            # a non-null, 256-byte aligned address that nothing reads


def _gated(**kw):
    a = dict(dtype=vk.DT_BF16, act=0, M=4, F=24, H=16, x=P, ldx=16, w_gate=P, ldwg=16, w_up=P, ldwu=16, h=P, ldh=24)
    a.update(kw)
    return F.Gated(**a)


def _gated_bwd(**kw):
    a = dict(dtype=vk.DT_F16, act=2, M=4, F=24, H=16, dh=P, lddh=24, g=P, ldg=24, u=P, ldu=24, x=P, ldx=16,
             w_gate=P, ldwg=16, w_up=P, ldwu=16, dx=P, lddx=16, dw_gate=P, lddwg=16, dw_up=P, lddwu=16)
    a.update(kw)
    return F.GatedBackward(**a)


def _xent(**kw):
    a = dict(dtype=vk.DT_BF16, T=4, V=24, H=16, x=P, ldx=16, w=P, ldw=16, targets=P, ignore_index=-100, loss=P, lse=P)
    a.update(kw)
    return F.LinearXent(**a)


def _xent_bwd(**kw):
    a = dict(dtype=vk.DT_BF16, T=4, V=24, H=16, dloss=P, lse=P, x=P, ldx=16, w=P, ldw=16, targets=P, dx=P, lddx=16,
             dw=P, lddw=16)
    a.update(kw)
    return F.LinearXentBackward(**a)


def _call(name, a, ws=1 << 20, nbytes=1 << 40):
    return getattr(vk.lib, f"vkblas_b200_{name}")(C.byref(a), ws, nbytes, None)


@pytest.mark.parametrize("name,make,bad", [
    (n, m, b) for n, m, bads in (
        ("gated", _gated, [dict(dtype=vk.DT_F32), dict(dtype=9), dict(act=3), dict(act=-1), dict(M=0), dict(F=0),
                           dict(H=0), dict(x=None), dict(w_gate=None), dict(w_up=None), dict(h=None), dict(ldx=15),
                           dict(ldwg=15), dict(ldwu=15), dict(ldh=23), dict(x=P + 1), dict(g=P, ldg=24),
                           dict(u=P, ldu=24), dict(g=P, ldg=23, u=P, ldu=24)]),
        ("gated_backward", _gated_bwd, [dict(dtype=vk.DT_F32), dict(act=7), dict(M=0), dict(dh=None), dict(g=None),
                                        dict(u=None), dict(lddh=23), dict(dx=None, dw_gate=None, dw_up=None),
                                        dict(w_gate=None), dict(w_up=None), dict(x=None), dict(lddx=15),
                                        dict(lddwg=15), dict(lddwu=1), dict(dx=P + 1)]),
        ("linear_xent", _xent, [dict(dtype=vk.DT_F32), dict(T=0), dict(V=0), dict(H=0), dict(x=None), dict(w=None),
                                dict(targets=None), dict(loss=None), dict(ldx=3), dict(ldw=15), dict(targets=P + 4),
                                dict(loss=P + 2)]),
        ("linear_xent_backward", _xent_bwd, [dict(dtype=vk.DT_F32), dict(T=0), dict(V=0), dict(H=0), dict(dloss=None),
                                             dict(lse=None), dict(dx=None, dw=None), dict(lddx=15), dict(lddw=15),
                                             dict(targets=None), dict(dw=P + 1)]),
    ) for b in bads])
def test_bad_structs(name, make, bad):
    assert _call(name, make(**bad)) == vk.VKBLAS_ERR_PARAM


@pytest.mark.parametrize("name,make", [("gated", _gated), ("gated_backward", _gated_bwd), ("linear_xent", _xent),
                                       ("linear_xent_backward", _xent_bwd)])
def test_good_structs_reach_the_device(name, make):
    """Sound arguments get as far as the device; a null struct does not."""
    a = make()
    lib = vk.lib
    assert getattr(lib, f"vkblas_b200_{name}")(None, None, 0, None) == vk.VKBLAS_ERR_PARAM
    assert getattr(lib, f"vkblas_b200_{name}_workspace")(None) == 0
    need = getattr(lib, f"vkblas_b200_{name}_workspace")(C.byref(a))
    if need:
        assert _call(name, a, None, 0) == vk.VKBLAS_ERR_PARAM
        assert _call(name, a, 1 << 20, need - 1) == vk.VKBLAS_ERR_PARAM
        assert _call(name, a, (1 << 20) + 16, need) == vk.VKBLAS_ERR_PARAM
    if not torch.cuda.is_available():
        assert _call(name, a, 1 << 20, need) == vk.VKBLAS_ERR_INIT


def test_workspace_does_not_shrink_with_size():
    """Workspaces of larger problems are no smaller, and their sizes do not wrap."""
    for T in (1, 100, 5000, 100000):
        a, b = (vk.lib.vkblas_b200_gated_backward_workspace(C.byref(_gated_bwd(M=T * k, F=14336, lddh=14336, ldg=14336,
                                                                                ldu=14336))) for k in (1, 2))
        assert a <= b and a >= 2 * T * 14336 * 2
        a, b = (vk.lib.vkblas_b200_linear_xent_backward_workspace(
            C.byref(_xent_bwd(T=T * k, V=128000, H=4096, ldx=4096, ldw=4096, lddx=4096, lddw=4096))) for k in (1, 2))
        assert 0 < a <= b


Q = dict(dtype=vk.DT_F16, N=20, K=100, group=32, has_zeros=1, packed=P)


@pytest.mark.parametrize("bad", [dict(dtype=vk.DT_F32), dict(N=0), dict(K=0), dict(group=0), dict(group=48),
                                 dict(group=16)])
def test_bad_q4(bad):
    w = F.Q4(**{**Q, **bad})
    assert vk.lib.vkblas_b200_q4_bytes(C.byref(w)) == 0
    assert vk.lib.vkblas_b200_q4_pack(C.byref(w), P, 64, P, 8, P, 8, P, None) == vk.VKBLAS_ERR_PARAM
    assert vk.lib.vkblas_b200_gemv_q4(C.byref(w), 1, 1.0, P, 128, 0.0, P, 32, None) == vk.VKBLAS_ERR_PARAM


def test_bad_q4_calls():
    w = F.Q4(**Q)
    assert vk.lib.vkblas_b200_q4_bytes(C.byref(w)) >= 20 * 50 + 20 * 4 * 3
    for a in ((None, 64, P, 8, P, 8, P), (P, 49, P, 8, P, 8, P), (P, 64, None, 8, P, 8, P), (P, 64, P, 3, P, 8, P),
              (P, 64, P, 8, None, 8, P), (P, 64, P, 8, P, 3, P), (P, 64, P, 8, P, 8, None), (P, 64, P, 8, P, 8, P + 16),
              (P, 64, P + 1, 8, P, 8, P)):
        assert vk.lib.vkblas_b200_q4_pack(C.byref(w), *a, None) == vk.VKBLAS_ERR_PARAM
    for a in ((0, 1.0, P, 128, 0.0, P, 32), (17, 1.0, P, 128, 0.0, P, 32), (1, 1.0, None, 128, 0.0, P, 32),
              (1, 1.0, P, 99, 0.0, P, 32), (1, 1.0, P, 128, 0.0, None, 32), (1, 1.0, P, 128, 0.0, P, 19),
              (1, 1.0, P + 1, 128, 0.0, P, 32)):
        assert vk.lib.vkblas_b200_gemv_q4(C.byref(w), *a, None) == vk.VKBLAS_ERR_PARAM
    assert vk.lib.vkblas_b200_gemv_q4(C.byref(F.Q4(**{**Q, "packed": None})), 1, 1.0, P, 128, 0.0, P, 32,
                                      None) == vk.VKBLAS_ERR_PARAM
    assert vk.lib.vkblas_b200_gemv_q4(None, 1, 1.0, P, 128, 0.0, P, 32, None) == vk.VKBLAS_ERR_PARAM


# ---------------------------------------------------------------- the tensor helpers
class Fake:
    """Stands in for a CUDA tensor: only what the checks read."""

    def __init__(self, *shape, dtype=torch.bfloat16, device="cuda:0", stride=None):
        self.shape, self.dtype, self.device, self.is_cuda = shape, dtype, torch.device(device), True
        self._stride = stride or (shape[-1], 1)

    def dim(self):
        return len(self.shape)

    def stride(self, i):
        return self._stride[i]

    def data_ptr(self):
        return P

    def get_device(self):
        return self.device.index


def _x(*s, **k):
    return Fake(*s, **k)


@pytest.mark.parametrize("call,msg", [
    (lambda: vk.gated_tensors(torch.zeros(2, 8, dtype=torch.bfloat16), _x(4, 8), _x(4, 8)), "CUDA tensor"),
    (lambda: vk.gated_tensors(_x(2, 8, dtype=torch.float32), _x(4, 8), _x(4, 8)), "float16 or bfloat16"),
    (lambda: vk.gated_tensors(_x(2, 8), _x(4, 8, dtype=torch.float16), _x(4, 8)), "dtypes differ"),
    (lambda: vk.gated_tensors(_x(2, 8), _x(4, 8, device="cuda:1"), _x(4, 8)), "devices differ"),
    (lambda: vk.gated_tensors(_x(2, 8), _x(4, 9), _x(4, 8)), "not"),
    (lambda: vk.gated_tensors(_x(2, 8), _x(4, 8), _x(5, 8)), "not"),
    (lambda: vk.gated_tensors(_x(2, 8), _x(4, 8, stride=(1, 4)), _x(4, 8)), "contiguous"),
    (lambda: vk.gated_tensors(_x(2, 8, stride=(0, 1)), _x(4, 8), _x(4, 8)), "row stride"),
    (lambda: vk.gated_tensors(_x(0, 8), _x(4, 8), _x(4, 8)), "positive"),
    (lambda: vk.gated_tensors(_x(2, 2, 8), _x(4, 8), _x(4, 8)), "2-D"),
    (lambda: vk.gated_tensors(_x(2, 8), _x(4, 8), _x(4, 8), act="relu"), "act is one of"),
    (lambda: vk.gated_backward_tensors(_x(2, 4), _x(2, 4), _x(2, 5), _x(2, 8), _x(4, 8), _x(4, 8)), "not"),
    (lambda: vk.gated_backward_tensors(_x(2, 4), _x(2, 4), _x(2, 4), _x(2, 8), _x(4, 8), _x(4, 8), need_dx=False,
                                       need_dw=False), "no gradient"),
    (lambda: vk.linear_xent_tensors(_x(2, 8), _x(4, 8), _x(2, dtype=torch.int32, stride=(1,))), "int64"),
    (lambda: vk.linear_xent_tensors(_x(2, 8), _x(4, 8), _x(3, dtype=torch.int64, stride=(1,))), "shape"),
    (lambda: vk.linear_xent_tensors(_x(2, 8), _x(0, 8), _x(2, dtype=torch.int64, stride=(1,))), "positive"),
    (lambda: vk.linear_xent_backward_tensors(_x(2, stride=(1,)), _x(2, dtype=torch.float32, stride=(1,)), _x(2, 8),
                                             _x(4, 8), _x(2, dtype=torch.int64, stride=(1,))), "dloss"),
    (lambda: vk.q4_pack_tensors(_x(4, 8, dtype=torch.uint8), _x(4, 1), None, 16, 24), "multiple of 32"),
    (lambda: vk.q4_pack_tensors(_x(4, 9, dtype=torch.uint8), _x(4, 1), None, 16, 32), "not"),
    (lambda: vk.q4_pack_tensors(_x(4, 8, dtype=torch.int8), _x(4, 1), None, 16, 32), "dtypes differ"),
    (lambda: vk.q4_pack_tensors(_x(4, 8, dtype=torch.uint8), _x(4, 1), _x(4, 2, dtype=torch.uint8), 16, 32), "not"),
    (lambda: vk.gemv_q4_tensors(_x(17, 16), F.Q4Weight(torch.bfloat16, 4, 16, 32, False, _x(256))), "at most 16"),
    (lambda: vk.gemv_q4_tensors(_x(1, 15), F.Q4Weight(torch.bfloat16, 4, 16, 32, False, _x(256))), "not"),
    (lambda: vk.gemv_q4_tensors(_x(1, 16), F.Q4Weight(torch.float16, 4, 16, 32, False, _x(256))), "dtypes differ"),
    (lambda: vk.gemv_q4_tensors(_x(1, 16), F.Q4Weight(torch.bfloat16, 4, 16, 32, False, _x(256)), beta=1.0), "beta"),
])
def test_misfits_raise(call, msg):
    with pytest.raises(ValueError, match=msg):
        call()
