"""CPU tests: sizes that the C structures hold in 32 bits are refused by the Python entry points
before they would come out small. The tensors are stand-ins with sizes only."""

import pytest
import torch

from rpfq_review_b200 import _lib, ops

BIG = 2 ** 32 + 16  # 16 in 32 bits


class Sizes:
    """A CUDA tensor as far as the checks look at it: a shape, a type, row-major strides."""
    is_cuda, requires_grad, device = True, False, "cuda:0"

    def __init__(self, *shape, dtype=torch.float32):
        self.shape, self.dtype = torch.Size(shape), dtype

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()

    def get_device(self):
        return 0

    def is_contiguous(self):
        return True

    def contiguous(self):
        return self

    def stride(self, i=None):
        s = [1]
        for n in self.shape[:0:-1]:
            s.insert(0, s[0] * n)
        return tuple(s) if i is None else s[i]

    def data_ptr(self):
        return 1 << 20

    def new_empty(self, shape, dtype=None):
        return Sizes(*shape, dtype=dtype or self.dtype)


@pytest.fixture
def no_launch(monkeypatch):
    class Library:
        def __getattr__(self, name):
            raise AssertionError(f"{name} was called")
    monkeypatch.setattr(_lib, "lib", lambda: Library())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)


def test_wide_sizes_are_refused(no_launch):
    q8 = lambda *s: Sizes(*s, dtype=torch.int8)  # noqa: E731
    half = lambda *s: Sizes(*s, dtype=torch.float16)  # noqa: E731
    f64 = lambda n: Sizes(n, dtype=torch.float64)  # noqa: E731
    for call in (lambda: ops.quantize_rows(half(2, BIG)), lambda: ops.quantize_rows(half(2, 2 ** 30 + 1)),
                 lambda: ops.gemm_int8(q8(2, BIG), Sizes(2), q8(3, BIG), Sizes(3)),
                 lambda: ops.gemm_int8(q8(2, 131072), Sizes(2), q8(3, 131072), Sizes(3)),
                 lambda: ops.gemm_int8(q8(2, 16), Sizes(2), q8(BIG, 16), Sizes(BIG)),
                 lambda: ops.gemm_int8(q8(2, 16), Sizes(2), q8(2 ** 31 - 256, 16), Sizes(2 ** 31 - 256)),
                 lambda: ops.linear_int8(half(2, BIG), q8(3, BIG), Sizes(3)),
                 lambda: ops.linear_int8(half(2, 16), q8(BIG, 16), Sizes(BIG)),
                 lambda: ops.rotary(half(1, BIG, 16), Sizes(1, dtype=torch.int32), f64(8)),
                 lambda: ops.rotary(half(1, 2 ** 24 + 1, 16), Sizes(1, dtype=torch.int32), f64(8)),
                 lambda: ops.rotary(half(1, 1, BIG), Sizes(1, dtype=torch.int32), f64(8)),
                 lambda: ops.rotary(half(1, 1, 2 * BIG), Sizes(1, dtype=torch.int32), f64(BIG))):
        with pytest.raises(NotImplementedError, match="at most"):
            call()
