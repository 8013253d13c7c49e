"""What alphazero_amd.head refuses before anything runs, the C entry points' own checks, and the plain forms' generator."""
import ctypes as C

import pytest
import torch

import head_ref as R
from alphazero_amd import _native as N
from alphazero_amd import head


class _Fake(torch.Tensor):
    """A CPU tensor that says it is on the GPU: argument checks run on it, nothing else is reached."""

    @property
    def is_cuda(self):
        return True


def _fake(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype).as_subclass(_Fake)


def test_no_cpu_fallback():
    x, w = torch.zeros(2, 3), torch.zeros(4, 3)
    for call in (lambda: head.linear_cross_entropy(x, w, torch.zeros(2, dtype=torch.int64)), lambda: head.dropout(x, 0.5, 1),
                 lambda: head.quantize_rows(x), lambda: head.int8_linear(x, w.to(torch.int8), torch.ones(4)),
                 lambda: head.Int8Linear(torch.nn.Linear(3, 4))):
        with pytest.raises(N.NativeError, match="no CPU fallback"):
            call()
    from alphazero_amd.model import AlphaZeroNet
    from alphazero_amd.train_step import DataParallelTrainer
    net = AlphaZeroNet(board_size=5, channels=32, num_blocks=1)
    for kw in (dict(fused_policy_loss=True), dict(head_dropout=0.1)):
        with pytest.raises(N.NativeError, match="GPU"):
            DataParallelTrainer(net, **kw)
    with pytest.raises(ValueError):
        DataParallelTrainer(net, head_dropout=1.0)
    with pytest.raises(N.NativeError):
        net.int8_heads()
    assert isinstance(net.policy_fc, torch.nn.Linear)


def test_loss_refuses():
    x, w, t = _fake(6, 8), _fake(5, 8), _fake(6, dtype=torch.int64)
    bad = [
        (dict(x=_fake(6, 7)), "do not fit"), (dict(w=_fake(8)), "do not fit"), (dict(t=_fake(5, dtype=torch.int64)), "does not fit"),
        (dict(t=_fake(6, dtype=torch.int32)), "int64"), (dict(t=_fake(6, 4)), "do not fit"), (dict(b=_fake(6)), "one value per class"),
        (dict(w=_fake(5, 8, dtype=torch.bfloat16)), "one dtype"), (dict(x=_fake(6, 8, dtype=torch.float64)), "float32"),
        (dict(reduction="avg"), "reduction"), (dict(w=_fake(0, 8)), "at least 1"), (dict(b=_fake(5, dtype=torch.float16)), "one dtype"),
    ]
    for change, says in bad:
        a = dict(x=x, w=w, t=t, b=None, reduction="mean") | change
        with pytest.raises(ValueError, match=says):
            head.linear_cross_entropy(a["x"], a["w"], a["t"], a["b"], reduction=a["reduction"])
    soft = _fake(6, 5).requires_grad_(True)
    with pytest.raises(ValueError, match="no gradient"):
        head.linear_cross_entropy(x, w, soft)


def test_dropout_refuses():
    x = _fake(4, 4)
    for kw, says in ((dict(p=1.5), "probability"), (dict(p=-0.1), "probability"), (dict(p=float("nan")), "probability"), (dict(seed=-1), "seed"),
                     (dict(seed=1 << 64), "seed"), (dict(offset=-1), "offset"), (dict(residual=_fake(4, 3)), "residual"),
                     (dict(residual=_fake(4, 4, dtype=torch.float16)), "residual"), (dict(seed=_fake(2, dtype=torch.int64)), "seed tensor"),
                     (dict(seed=_fake(1)), "seed tensor"), (dict(x=_fake(4, dtype=torch.float64)), "float32")):
        a = dict(x=x, p=0.5, seed=1, offset=0, residual=None) | kw
        with pytest.raises(ValueError, match=says):
            head.dropout(a["x"], a["p"], a["seed"], a["offset"], residual=a["residual"])


def test_int8_refuses():
    x, w, s = _fake(3, 8), _fake(5, 8, dtype=torch.int8), _fake(5)
    for kw, says in ((dict(w=_fake(5, 8)), "int8 matrix"), (dict(w=_fake(5, 9, dtype=torch.int8)), "do not fit"), (dict(s=_fake(4)), "one float32 per channel"),
                     (dict(s=_fake(5, dtype=torch.float16)), "one float32 per channel"), (dict(b=_fake(4)), "bias"), (dict(xs=_fake(3)), "x_scale comes"),
                     (dict(x=_fake(3, 8, dtype=torch.int8)), "x_scale comes"), (dict(x=_fake(3, 8, dtype=torch.int8), xs=_fake(4)), "one float32 per row"),
                     (dict(out=torch.float64), "out_dtype"), (dict(x=_fake(3, 8, dtype=torch.float64)), "float32"),
                     (dict(x=_fake(1, 131072), w=_fake(1, 131072, dtype=torch.int8), s=_fake(1)), "131071"),
                     (dict(x=_fake(3, 8).requires_grad_(True)), "no gradient")):
        a = dict(x=x, w=w, s=s, b=None, xs=None, out=None) | kw
        with pytest.raises(ValueError, match=says):
            head.int8_linear(a["x"], a["w"], a["s"], a["b"], x_scale=a["xs"], out_dtype=a["out"])
    with pytest.raises(ValueError, match="at least one"):
        head.quantize_rows(_fake(3, 0))


def test_c_entry_points_refuse():
    """The C ABI's own checks, with pointers that nothing may follow: every call returns before it would."""
    L = N.lib()
    good = dict(x=256, weight=512, bias=None, target=768, rows=4, features=8, classes=3, x_pitch=8, weight_pitch=8, target_pitch=0, ignore_index=-100,
                dtype=N.AZ_DT_BF16, target_dense=0, reduction=N.AZ_REDUCE_MEAN, entropy_coeff=0.0)
    ws = C.c_int64(L.az_linear_ce_workspace(C.byref(N.AzLinearCeArgs(**good)), 0)).value
    assert ws > 0
    for change in (dict(x=None), dict(weight=None), dict(target=None), dict(rows=0), dict(features=0), dict(classes=0), dict(x_pitch=7), dict(weight_pitch=7),
                   dict(dtype=3), dict(dtype=-1), dict(reduction=3), dict(target_dense=1), dict(rows=1 << 31), dict(classes=1 << 31), dict(features=1 << 23)):
        a = N.AzLinearCeArgs(**(good | change))
        assert L.az_linear_ce_workspace(C.byref(a), 0) == N.AZ_ERR_ARG and L.az_linear_ce_workspace(C.byref(a), 1) == N.AZ_ERR_ARG, change
        assert L.az_linear_ce_forward(C.byref(a), 256, 256, None, None, 256, 1 << 40, None) == N.AZ_ERR_ARG
    a = N.AzLinearCeArgs(**good)
    assert L.az_linear_ce_workspace(None, 0) == N.AZ_ERR_ARG
    for args in ((None, 256, 256, ws), (256, None, 256, ws), (256, 256, None, ws), (256, 256, 256, ws - 1), (256, 256, 257, ws)):
        assert L.az_linear_ce_forward(C.byref(a), args[0], args[1], None, None, args[2], args[3], None) == N.AZ_ERR_ARG
    wb = L.az_linear_ce_workspace(C.byref(a), 1)
    for args in ((None, 256, 256, 256, wb), (256, None, 256, 256, wb), (256, 256, 264, 256, wb), (256, 256, 256, 256, wb - 1)):
        assert L.az_linear_ce_backward(C.byref(a), args[0], args[1], args[2], None, None, args[3], args[4], None) == N.AZ_ERR_ARG
    assert L.az_linear_ce_backward(C.byref(a), 256, 256, None, None, None, 256, wb, None) == N.AZ_OK      # nothing asked for
    assert L.az_dropout(256, None, 256, 8, 9, 0, 0, None, 0, None) == N.AZ_ERR_ARG
    assert L.az_dropout(256, None, 256, 8, 0, 65537, 0, None, 0, None) == N.AZ_ERR_ARG
    assert L.az_dropout(256, None, 256, -1, 0, 0, 0, None, 0, None) == N.AZ_ERR_ARG
    assert L.az_dropout(None, None, 256, 8, 0, 0, 0, None, 0, None) == N.AZ_ERR_ARG
    assert L.az_dropout(None, None, None, 0, 0, 0, 0, None, 0, None) == N.AZ_OK
    assert L.az_quantize_rows(256, 0, 4, 8, 7, 256, 8, 256, None) == N.AZ_ERR_ARG
    assert L.az_quantize_rows(256, 0, 4, 8, 8, 256, 7, 256, None) == N.AZ_ERR_ARG
    assert L.az_quantize_rows(None, 0, 4, 8, 8, 256, 8, 256, None) == N.AZ_ERR_ARG
    assert L.az_quantize_rows(None, 0, 0, 8, 8, None, 8, None, None) == N.AZ_OK
    good = dict(x=256, weight=512, x_scale=None, weight_scale=768, bias=None, y=1024, tokens=8, features=16, channels=4, x_pitch=16, weight_pitch=16,
                x_dtype=N.AZ_DT_F32, bias_dtype=0, y_dtype=N.AZ_DT_F32)
    size = L.az_int8_workspace(C.byref(N.AzInt8Args(**good)))
    assert size > 0
    for change in (dict(x=None), dict(weight=None), dict(weight_scale=None), dict(y=None), dict(y=1028), dict(x_dtype=4), dict(x_dtype=N.AZ_DT_I8), dict(y_dtype=3),
                   dict(bias=4, bias_dtype=3), dict(tokens=0), dict(features=0), dict(channels=0), dict(features=131072, x_pitch=131072, weight_pitch=131072),
                   dict(x_pitch=15), dict(weight_pitch=15)):
        a = N.AzInt8Args(**(good | change))
        assert L.az_int8_workspace(C.byref(a)) == N.AZ_ERR_ARG and L.az_int8_linear(C.byref(a), 256, 1 << 40, None) == N.AZ_ERR_ARG, change
    a = N.AzInt8Args(**good)
    assert L.az_int8_linear(C.byref(a), None, size, None) == N.AZ_ERR_ARG and L.az_int8_linear(C.byref(a), 256, size - 1, None) == N.AZ_ERR_ARG


def test_c_entry_points_refuse_what_no_launch_holds():
    L = N.lib()
    good = dict(x=256, weight=512, bias=None, target=768, rows=1 << 20, features=1 << 14, classes=3, x_pitch=1 << 15, weight_pitch=1 << 15, target_pitch=0,
                ignore_index=-100, dtype=N.AZ_DT_BF16, target_dense=0, reduction=N.AZ_REDUCE_MEAN, entropy_coeff=0.0)
    assert L.az_linear_ce_workspace(C.byref(N.AzLinearCeArgs(**good)), 0) > 0
    assert L.az_linear_ce_workspace(C.byref(N.AzLinearCeArgs(**(good | dict(features=(1 << 14) + 1)))), 0) == N.AZ_ERR_ARG
    good = dict(x=256, weight=512, x_scale=None, weight_scale=768, bias=None, y=1024, tokens=1 << 30, features=16, channels=1 << 27, x_pitch=16,
                weight_pitch=16, x_dtype=N.AZ_DT_F32, bias_dtype=0, y_dtype=N.AZ_DT_F32)
    assert L.az_int8_workspace(C.byref(N.AzInt8Args(**good))) > 0
    for change in (dict(tokens=(1 << 30) + 1), dict(channels=(1 << 27) + 1)):
        assert L.az_int8_workspace(C.byref(N.AzInt8Args(**(good | change)))) == N.AZ_ERR_ARG, change


def test_generator_known_answers():
    """The published known answers of Philox4x32-10 (counters and keys of zeros, of ones, and of the digits of pi)."""
    def words(c, k):
        return [int(v) for v in R.philox_block(c, k)]
    assert words((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    f = 0xFFFFFFFF
    assert words((f, f, f, f), (f, f)) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert words((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0)) == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]
    kept, w = R.philox_kept(16, 0.5, 0, 0)
    assert [int(v) for v in w[0]] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert kept[:4].tolist() == [0xE8D5 >= 32768, 0x6627 >= 32768, 0xC58D >= 32768, 0xE169 >= 32768]


def test_loss_reference_against_autograd():
    g = torch.Generator().manual_seed(0)
    x, w, b = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((9, 6), (7, 6), (7,)))
    for t in (torch.tensor([0, 6, -100, 3, 2, 1, 1, -100, 5]), torch.rand((9, 7), generator=g)):
        leaves = [v.clone().requires_grad_(True) for v in (x, w, b)]
        logp = torch.log_softmax(leaves[0] @ leaves[1].t() + leaves[2], 1)
        rows = -(t * logp).sum(1) if t.is_floating_point() else torch.where(t == -100, 0.0, -logp.gather(1, t.clamp(min=0)[:, None])[:, 0])
        n = 9 if t.is_floating_point() else 7
        ent = -(logp.exp() * logp).sum(1) * (1.0 if t.is_floating_point() else (t != -100).double())
        loss = (rows - 0.3 * ent).sum() / n
        loss.backward()
        ref = R.loss_reference(x, w, t, b, c=0.3, grad=torch.ones(()))
        for name, want in (("loss", loss.detach()), ("gx", leaves[0].grad), ("gw", leaves[1].grad), ("gb", leaves[2].grad)):
            assert torch.allclose(ref[name][0], want, rtol=0, atol=1e-12), name


def test_quantize_reference_rounds_to_even():
    q, s = R.quantize_reference(torch.tensor([[127.0, 0.5, 1.5, -2.5, 2.5000002], [0.0, 0, 0, 0, 0]]))
    assert q.tolist() == [[127, 0, 2, -2, 3], [0, 0, 0, 0, 0]] and s.tolist() == [1.0, 0.0]
