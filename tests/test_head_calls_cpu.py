"""Calls of alphazero_amd.head that have to be refused rather than answered wrongly, on stand-ins for GPU tensors."""
import ctypes as C

import pytest
import torch
from torch.autograd import forward_ad

from alphazero_amd import _native as N
from alphazero_amd import head
from test_head_cpu import _fake


def test_forward_mode_is_refused():
    """A tangent that the kernels do not carry would come back as a derivative of zero."""
    with forward_ad.dual_level():
        def dual(*shape):
            return forward_ad.make_dual(_fake(*shape), torch.ones(shape))
        x, w8, ones = _fake(3, 8), _fake(5, 8, dtype=torch.int8), _fake(5)
        t = _fake(3, dtype=torch.int64)
        for call in (lambda: head.dropout(dual(3, 8), 0.5, 1), lambda: head.dropout(x, 0.5, 1, residual=dual(3, 8)), lambda: head.quantize_rows(dual(3, 8)),
                     lambda: head.int8_linear(dual(3, 8), w8, ones), lambda: head.int8_linear(x, w8, dual(5)), lambda: head.int8_linear(x, w8, ones, dual(5)),
                     lambda: head.int8_linear(_fake(3, 8, dtype=torch.int8), w8, ones, x_scale=dual(3)),
                     lambda: head.linear_cross_entropy(dual(3, 8), _fake(5, 8), t), lambda: head.linear_cross_entropy(x, dual(5, 8), t),
                     lambda: head.linear_cross_entropy(x, _fake(5, 8), t, dual(5)), lambda: head.linear_cross_entropy(x, _fake(5, 8), dual(3, 5))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        with pytest.raises(ValueError, match="probability"):        # without a tangent the call goes on, to its next check
            head.dropout(x, 2.0, 1)


@pytest.mark.filterwarnings("ignore")
def test_recording_is_refused():
    """torch.jit.trace and make_fx record torch operations: the result's allocation, and none of the kernels."""
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w8, ones, t = _fake(3, 8), _fake(5, 8, dtype=torch.int8), _fake(5), _fake(3, dtype=torch.int64)
    layer = head.Int8Linear.__new__(head.Int8Linear)
    torch.nn.Module.__init__(layer)
    layer.in_features, layer.out_features = 8, 5
    for name, v in (("qweight", w8), ("weight_scale", ones), ("bias", None)):
        layer.register_buffer(name, v)
    calls = (lambda: head.dropout(x, 0.5, 1), lambda: head.quantize_rows(x)[1], lambda: head.int8_linear(x, w8, ones), lambda: layer(x),
             lambda: head.linear_cross_entropy(x, _fake(5, 8), t))
    for call in calls:
        def one(v):
            return v + call()
        with pytest.raises(NotImplementedError, match="cannot be traced"):
            torch.jit.trace(one, torch.zeros(()), check_trace=False)
    for call in calls[:3] + calls[4:]:
        with pytest.raises(NotImplementedError, match="cannot be traced"):
            make_fx(lambda v: v + call())(torch.zeros(()))


def _layer(bias=True):
    """An Int8Linear as its constructor leaves it, on the CPU."""
    layer = head.Int8Linear.__new__(head.Int8Linear)
    torch.nn.Module.__init__(layer)
    layer.in_features, layer.out_features = 18, 5
    layer.register_buffer("qweight", torch.randint(-127, 128, (5, 32)).to(torch.int8))
    layer.register_buffer("weight_scale", torch.rand(5))
    layer.register_buffer("bias", torch.rand(5) if bias else None)
    return layer


@pytest.mark.parametrize("bias", [False, True])
def test_int8_layer_keeps_its_weights_under_casts(bias):
    for cast, kind in ((lambda m: m.half(), torch.float16), (lambda m: m.bfloat16(), torch.bfloat16), (lambda m: m.to(torch.float16), torch.float16),
                       (lambda m: m.to("cpu", torch.bfloat16), torch.bfloat16), (lambda m: m.type(torch.float16), torch.float16),
                       (lambda m: torch.nn.Sequential(m).half()[0], torch.float16), (lambda m: m.half().float(), torch.float32),
                       (lambda m: m.to("cpu"), torch.float32)):
        layer = _layer(bias)
        q, s = layer.qweight.clone(), layer.weight_scale.clone()
        m = cast(layer)
        assert m is layer and m.qweight.dtype == torch.int8 and torch.equal(m.qweight, q)
        assert m.weight_scale.dtype == torch.float32 and torch.equal(m.weight_scale, s)
        assert set(m.state_dict()) == {"qweight", "weight_scale"} | ({"bias"} if bias else set())
        if bias:
            assert m.bias.dtype == kind
    there = _layer(bias).to("meta", torch.float16)
    assert there.qweight.is_meta and there.weight_scale.is_meta and there.weight_scale.dtype == torch.float32


def test_int8_layer_has_no_gradient_and_says_so():
    layer = _layer()
    for name in ("qweight", "weight_scale", "bias"):
        setattr(layer, name, getattr(layer, name).as_subclass(_fake(1).__class__))
    with pytest.raises(ValueError, match="no gradient"):
        layer(_fake(3, 18).requires_grad_(True))
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        layer(forward_ad.make_dual(_fake(3, 18), torch.ones(3, 18)))


def test_padded_int8_weights_are_read_in_place():
    """The layout of Int8Linear, rows at multiples of 16 bytes: no scratch memory for a copy, whatever the number of features."""
    L = N.lib()
    for tokens, features, channels in ((256, 722, 362), (60, 162, 82), (32, 4095, 4096), (300, 17, 5000)):
        pitch = (features + 15) // 16 * 16

        def size(**change):
            good = dict(x=256, weight=512, x_scale=None, weight_scale=768, bias=None, y=1024, tokens=tokens, features=features, channels=channels, x_pitch=pitch,
                        weight_pitch=pitch, x_dtype=N.AZ_DT_F32, bias_dtype=0, y_dtype=N.AZ_DT_F32)
            return L.az_int8_workspace(C.byref(N.AzInt8Args(**(good | change))))
        assert size() == size(features=pitch)
        assert size(weight=513) >= size() + channels * pitch and size(weight_pitch=pitch + 1) >= size() + channels * pitch
        eight = dict(x_dtype=N.AZ_DT_I8, x_scale=256)      # 8-bit tokens: they are copied instead, with zeros behind their last feature
        assert size(**eight) >= size(features=pitch, **eight) + tokens * pitch


def test_one_floating_token_needs_no_scratch_memory():
    """One or two floating tokens are quantised in the product's own launch whatever the number of channels."""
    L = N.lib()
    for tokens, features, channels in ((1, 162, 82), (1, 4096, 4096), (1, 1024, 32000), (2, 3584, 18944), (1, 4096, 20480), (2, 2048, 131072), (1, 32768, 64)):
        a = N.AzInt8Args(x=256, weight=512, weight_scale=768, y=1024, tokens=tokens, features=features, channels=channels, x_pitch=features,
                         weight_pitch=features, x_dtype=N.AZ_DT_BF16, y_dtype=N.AZ_DT_BF16)
        assert L.az_int8_workspace(C.byref(a)) == 0, (tokens, features, channels)


def test_scratch_memory_of_the_loss_is_bounded():
    """What linear_cross_entropy says of its scratch memory, over many classes, many rows and long features."""
    L = N.lib()
    for dtype, size in ((N.AZ_DT_F32, 4), (N.AZ_DT_BF16, 2), (N.AZ_DT_F16, 2)):
        for rows, features, classes in ((256, 4096, 1 << 20), (64, 4096, 1 << 20), (64, 8192, 270001), (262144, 4096, 32000), (1 << 20, 4096, 50021), (8192, 4096, 131072),
                                        (17, 16384, 1 << 20), (129, 100000, 100000), (1, 4096, 1 << 24), (40, 8, 1 << 28), (200000, 8, 4000), (1 << 20, 64, 1000), (500, 1 << 20, 900)):
            for pitch in (features, features + 1):        # a weight that is read in place, and one that is copied
                a = N.AzLinearCeArgs(x=256, weight=512, target=768, rows=rows, features=features, classes=classes, x_pitch=pitch, weight_pitch=pitch,
                                     ignore_index=-100, dtype=dtype, reduction=N.AZ_REDUCE_MEAN)
                back, ahead = (L.az_linear_ce_workspace(C.byref(a), b) for b in (1, 0))
                x = rows * features * size
                weight = max(2 ** 29, 256 * features * size)        # of a piece of the classes, which has 256 at least
                assert 0 < back <= 1.25 * 2 ** 30 + 2 * weight + 4 * x + 70 * classes, (dtype, rows, features, classes, pitch, back / 2 ** 30)
                assert 0 < ahead <= 2 ** 25 + weight + 1.01 * x + 16 * (rows * classes / 32 + rows + classes), (dtype, rows, features, classes, pitch, ahead / 2 ** 30)


def test_precise_gradient_of_the_c_entry_points():
    """The flag goes with every reduction, and with nothing else; it takes the memory of a second plane."""
    L = N.lib()
    good = dict(x=256, weight=512, target=768, rows=4000, features=64, classes=3000, x_pitch=64, weight_pitch=64, ignore_index=-100, dtype=N.AZ_DT_BF16)
    for reduction in (N.AZ_REDUCE_NONE, N.AZ_REDUCE_MEAN, N.AZ_REDUCE_SUM):
        plain, precise = (N.AzLinearCeArgs(reduction=reduction | flag, **good) for flag in (0, N.AZ_PRECISE_GRADIENT))
        assert L.az_linear_ce_workspace(C.byref(plain), 0) == L.az_linear_ce_workspace(C.byref(precise), 0) > 0
        more = L.az_linear_ce_workspace(C.byref(precise), 1) - L.az_linear_ce_workspace(C.byref(plain), 1)
        assert more >= 4 * 4000 * 3000 * 0.99       # G and its transpose
    for reduction in (3, 3 | N.AZ_PRECISE_GRADIENT, 8, -1, 8 | N.AZ_PRECISE_GRADIENT):
        assert L.az_linear_ce_workspace(C.byref(N.AzLinearCeArgs(reduction=reduction, **good)), 0) == N.AZ_ERR_ARG
