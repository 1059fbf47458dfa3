"""An output that overlaps an input is refused before anything is launched; neighbours in one buffer
are not (no GPU)."""
import pytest
import torch

import vkblas_b200 as vk
from vkblas_b200 import fused as F


class At:
    """Stands in for a CUDA tensor at an address: only what the checks read."""

    def __init__(self, base, rows, cols, ld=None, dtype=torch.bfloat16):
        self.shape, self.dtype, self.is_cuda, self.device = (rows, cols), dtype, True, torch.device("cuda:0")
        self._p, self._ld = (1 << 20) + 2 * base, ld or cols

    def dim(self):
        return 2

    def stride(self, i):
        return (self._ld, 1)[i]

    def data_ptr(self):
        return self._p

    def element_size(self):
        return 2

    def get_device(self):
        return 0


FAR = 1 << 16


@pytest.mark.parametrize("x,out", [
    (At(0, 4, 64), At(0, 4, 64)),                          # in place
    (At(0, 4, 64), At(192, 4, 64)),                        # the last row
    (At(0, 4, 64), At(255, 4, 64)),                        # one element
    (At(0, 4, 64, 128), At(32, 4, 64, 128)),               # columns 0-63 and 32-95 of one buffer
    (At(100, 4, 64, 128), At(0, 4, 64, 128)),              # columns 100-163: into the next row
    (At(0, 1, 64), At(63, 1, 64)),                         # single rows
    (At(64, 1, 64), At(0, 4, 65)),                         # a row across another buffer's rows
    (At(0, 4, 64), At(0, 4, 64, 128)),                     # different row strides in one place
])
def test_overlapping_outputs_are_refused(x, out):
    with pytest.raises(ValueError, match="overlaps x"):
        F._given(out, *out.shape, out, x=x)


def test_every_input_counts():
    x, wg, wu = At(0, 4, 64), At(FAR, 64, 64), At(2 * FAR, 64, 64)
    for name, at in (("w_gate", FAR), ("w_up", 2 * FAR + 4000)):
        with pytest.raises(ValueError, match=f"overlaps {name}"):
            vk.gated_tensors(x, wg, wu, out=At(at, 4, 64))
    q4 = F.Q4Weight(torch.bfloat16, 64, 64, 32, False, At(FAR, 1, 4096))
    with pytest.raises(ValueError, match="overlaps x"):
        vk.gemv_q4_tensors(x, q4, out=At(128, 4, 64), beta=1.0)


@pytest.mark.parametrize("x,out", [
    (At(0, 4, 64), At(256, 4, 64)), (At(256, 4, 64), At(0, 4, 64)),
    (At(0, 4, 64, 128), At(64, 4, 64, 128)),               # two column blocks of one buffer
    (At(64, 4, 64, 128), At(0, 4, 64, 128)),
    (At(128, 4, 64, 256), At(16, 4, 64, 256)),
    (At(64, 1, 64), At(0, 4, 64, 128)),                    # a row between another's
    (At(0, 4, 64, 128), At(64, 1, 64)),
])
def test_neighbours_pass(x, out):
    assert F._given(out, *out.shape, out, x=x) == (out.data_ptr(), out._ld if out.shape[0] > 1 else 64)
