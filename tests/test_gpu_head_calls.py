"""Calls of alphazero_amd.head that other code makes of it: modules that are cast, padded weights, several pieces, values far apart."""
import math

import pytest
import torch

import head_ref as R

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DTYPES = [F32, BF16, F16]
ids = lambda v: str(v).replace("torch.", "").replace(" ", "")  # noqa: E731


def _head():
    from alphazero_amd import head
    return head


@pytest.mark.parametrize("dtype", [BF16, F16], ids=ids)
@pytest.mark.parametrize("tokens", [1, 40])
def test_int8_layer_cast_with_its_module(dtype, tokens):
    head = _head()
    torch.manual_seed(1)
    lin = torch.nn.Linear(162, 82).cuda()
    x = torch.randn(tokens, 162, device="cuda").to(dtype)
    one = head.Int8Linear(lin)
    want = head.int8_linear(x, one.qweight[:, :162], one.weight_scale, one.bias.to(dtype))
    cast = torch.nn.Sequential(head.Int8Linear(lin)).to(dtype)
    with torch.no_grad():
        y = cast(x)
    assert y.dtype == dtype and torch.equal(y, want)
