"""heads_16bit: a tensor's rows as the serving calls hand them to a kernel (address and strides; nothing here touches a device)."""
import pytest
import torch

from heimdall_b200.functional import heads_16bit

bf = torch.bfloat16


@pytest.mark.parametrize("cut,strides", [
    (lambda: torch.empty(1, 1, 14342, dtype=bf)[0, :, :5120], [0]),                                     # one token of a fused projection
    (lambda: torch.empty(4, 217, dtype=bf)[0:1, :136], [0]),
    (lambda: torch.empty(1, 1, 1003, dtype=bf)[..., :512].unflatten(2, (2, 256)), [0, 0, 256]),         # one sequence, one token
    (lambda: torch.empty(1, 3, 1003, dtype=bf)[:, 0:1, :512].unflatten(2, (1, 512)), [0, 0, 0]),
    (lambda: torch.empty_strided((1, 1, 2, 256), (3, 5, 256, 1), dtype=torch.float16), [0, 0, 256]),
    (lambda: torch.empty(3, 2, 4, 256, dtype=bf), [2048, 1024, 256]),
    (lambda: torch.empty(3, 1, 4, 256, dtype=bf), [1024, 0, 256]),
    (lambda: torch.empty(0, 1, 4, 256, dtype=bf), [0, 0, 256])])
def test_the_stride_of_a_dimension_of_one_is_given_as_0(cut, strides):
    t = cut()
    kept, at, got = heads_16bit("t", t)
    assert kept is t and at == t.data_ptr() and got == strides


def test_rows_that_a_kernel_cannot_take_are_copied():
    for t in (torch.randn(3, 217).to(bf)[:, :136], torch.randn(2 * 136 + 1).to(bf)[1:].view(2, 136), torch.randn(1, 136).to(bf).expand(4, 136)):
        kept, at, strides = heads_16bit("t", t)
        assert kept is not t and torch.equal(kept, t) and at == kept.data_ptr() and at % 16 == 0 and strides == [136]
