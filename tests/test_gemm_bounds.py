"""CPU: ops.gemm takes segment bounds of any type that int() takes, and refuses those that fit no call with the library's error."""
import pytest
import torch

from segquant_b200 import _lib as L
from segquant_b200 import ops


class _Tensor:
    """What ops.gemm asks a tensor, without a device."""
    def __init__(self, *shape, dtype=torch.uint8):
        self.shape, self.dtype, self.is_cuda = shape, dtype, True

    def data_ptr(self):
        return 4096

    def get_device(self):
        return 0

    def new_empty(self, shape, dtype):
        return _Tensor(*shape, dtype=dtype)


def _gemm_block(monkeypatch, bounds, **kw):
    seen = {}
    monkeypatch.setattr(ops, "_run", lambda fn, what, dev, a: seen.update(block=a))
    f = torch.float32
    ops.gemm(L.SQ_GEMM_W8A8_I8, _Tensor(1, 4, 64), _Tensor(1, 32, 64), 32, bounds, _Tensor(2, dtype=f), _Tensor(32, dtype=f), **kw)
    return L.GemmArgs.from_buffer_copy(seen["block"])


@pytest.mark.parametrize("bounds", [[0, 32, 64], (0.0, 32.0, 64.0), torch.tensor([0, 32, 64]), [0, 32, 64.0]], ids=["int", "float", "tensor", "mixed"])
def test_bounds_of_any_whole_number_type(native_lib, monkeypatch, bounds):
    a = _gemm_block(monkeypatch, bounds)
    assert a.num_segs == 2 and list(a.seg_bounds) == [0, 32, 64] + [0] * (L.SQ_MAX_SEGS - 2)


def test_bounds_that_fit_no_call(native_lib, monkeypatch):
    with pytest.raises(L.SegQuantError):
        _gemm_block(monkeypatch, list(range(0, 32 * 67, 32)))
    with pytest.raises(L.SegQuantError):
        _gemm_block(monkeypatch, [0, 1 << 40])
