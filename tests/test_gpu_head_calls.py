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


# ragged and whole pieces of 16 bytes; few tokens, tiles of each size, walks in pieces
PADDED = [(40, 162, 82), (70, 722, 362), (256, 722, 362), (100, 17, 33), (64, 4095, 300), (300, 129, 517), (2304, 250, 5632), (20, 8201, 70), (65, 3, 65), (49, 15, 1), (1, 162, 82),
          (2, 2047, 600), (3, 722, 362), (4, 162, 82), (5, 4095, 300), (16, 2047, 600), (4, 4095, 16500)]


@pytest.mark.parametrize("size", PADDED, ids=ids)
def test_int8_rows_that_end_inside_16_bytes(size):
    """Rows at multiples of 16 bytes with anything between them, the last one at the end of its memory, against a dense weight."""
    head = _head()
    m, k, n = size
    g = torch.Generator(device="cuda").manual_seed(m + k + n)
    x = torch.randn((m, k), generator=g, device="cuda")
    w = torch.randint(-127, 128, (n, k), generator=g, device="cuda").to(torch.int8)
    ws = torch.rand(n, generator=g, device="cuda") / 127
    q, s = head.quantize_rows(x)
    want = ((q.double() @ w.double().t()).float() * s[:, None]) * ws      # the sum is exact, then two roundings
    pitch = (k + 15) // 16 * 16
    for fill in (77, -128):
        for extra in (0, 16, 48):
            store = torch.full(((n - 1) * (pitch + extra) + k,), fill, dtype=torch.int8, device="cuda")
            rows = store.as_strided((n, k), (pitch + extra, 1))
            rows.copy_(w)
            assert torch.equal(head.int8_linear(x, rows, ws), want)
            q8 = torch.full((m, pitch + extra), fill, dtype=torch.int8, device="cuda")
            q8[:, :k] = q
            assert torch.equal(head.int8_linear(q8[:, :k], rows, ws, x_scale=s), want)
            assert torch.equal(head.int8_linear(q8[:, :k], w, ws, x_scale=s), want)


# around one round of workgroups, and several
@pytest.mark.parametrize("size", [(1, 256, 4080), (2, 256, 4112), (1, 130, 6000), (1, 256, 16400), (2, 1024, 20480), (1, 64, 70001), (12, 128, 8200), (16, 256, 12000), (40, 96, 16000)],
                         ids=ids)
def test_int8_few_tokens_of_many_channels(size):
    head = _head()
    m, k, n = size
    g = torch.Generator(device="cuda").manual_seed(m + k + n)
    x = torch.randn((m, k), generator=g, device="cuda")
    w = torch.randint(-127, 128, (n, k), generator=g, device="cuda").to(torch.int8)
    ws = torch.rand(n, generator=g, device="cuda") / 127
    q, s = head.quantize_rows(x)
    want = ((q.double() @ w.double().t()).float() * s[:, None]) * ws
    assert torch.equal(head.int8_linear(x, w, ws), want)
    assert torch.equal(head.int8_linear(q, w, ws, x_scale=s), want)


def _loss_inputs(rows, feats, classes, dtype, dense, bias, seed=0):
    from test_gpu_head import _inputs
    return _inputs(rows, feats, classes, dtype, dense, bias, seed)


def _loss_run(x, w, b, t, grad=None, **kw):
    from test_gpu_head import _run
    return _run(x, w, b, t, grad, **kw)


@pytest.mark.parametrize("size", [(20, 64, 300), (10, 64, 300), (9, 1032, 33000), (30, 300, 2000), (200, 64, 300), (100, 5000, 60)], ids=ids)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=ids)
@pytest.mark.parametrize("factor", [1e6, 1e9, 1e12, 1e16])
def test_a_row_of_huge_logits_has_a_finite_gradient(size, dtype, factor):
    """The passes may make the logits by different kernels; what their roundings differ by must not become a p of infinity."""
    x, w, b, t = _loss_inputs(*size, dtype, False, True)
    x[3] *= factor
    t[3] = 5
    loss, ce, ent, gx, gw, gb = _loss_run(x, w, b, t, reduction="sum", entropy_coeff=0.01)
    for v in (loss, ce, ent, gx, gw, gb):
        assert torch.isfinite(v).all()
    # |G| of a row sums to twice its weights' sum and the entropy's part at most, with every p at most one; roundings beside it
    most = (2 + 0.01 * (0.4 + math.log(size[2]))) * 1.02
    assert float(gx[3].abs().max()) <= most * float(w.abs().max())


@pytest.mark.parametrize("rows", [10, 20, 50, 200, 300])
@pytest.mark.parametrize("dense", [False, True], ids=["index", "dense"])
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("factor", [1e6, 1e12, 1e16])
def test_float32_rows_of_very_different_size(rows, dense, reduction, factor):
    """One counted row of x, then one class of the weight, far larger than the others: every row has its own softmax and gradient. The sums of
    the gradients hold their operand to 2^-49 of its largest value (2^-35 in planes whose largest is 2^13 or more, rounded)."""
    for large in ("row", "class"):
        x, w, b, t = _loss_inputs(rows, 64, 300, F32, dense, True)
        if large == "row":
            x[3] *= factor
            if not dense:
                t[3] = 5
        else:
            w[7] *= factor
        grad = torch.ones((rows,) if reduction == "none" else (), device="cuda")
        got = _loss_run(x, w, b, t, grad, reduction=reduction)
        ref = R.loss_reference(x, w, t, b, reduction=reduction, grad=grad)
        ref = {k: (v.clone(), tol.clone()) for k, (v, tol) in ref.items()}
        counts = torch.ones(rows, dtype=torch.bool, device="cuda") if dense else t != -100
        each = 1.0 if reduction == "none" else 1.0 / float(counts.sum())
        total = t.double().sum(1) if dense else counts.double()
        # each row of G sums to twice its weights' sum at most, each column to that over the rows
        ref["gx"][1].add_((2.0 ** -49 * float(w.abs().max()) * 2 * each * total)[:, None])
        ref["gw"][1].add_(2.0 ** -49 * float(x[counts].abs().max()) * 2 * each * float(total.sum()))
        for name, v in zip(("loss", "ce", "ent", "gx", "gw", "gb"), got):
            R.close(name, v[counts] if name in ("loss", "ce", "ent") and v.dim() else v, ref[name] if name in ("gx", "gw", "gb") or not v.dim() else
                    (ref[name][0][counts], ref[name][1][counts]))


def _loss_gradients(x, w, b, t, f):
    """gx and gw in 64 bits, for the factor f of each row."""
    z = x.double() @ w.double().t() + (0 if b is None else b.double())
    if t.is_floating_point():
        pi = t.double()
    else:
        pi = torch.zeros_like(z)
        live = t != -100
        pi[live, t[live]] = 1.0
    g = f[:, None] * (pi.sum(1, keepdim=True) * torch.softmax(z, 1) - pi)
    return g @ w.double(), g.t() @ x.double()


# (rows, features, classes, the caller asks for it)
KEPT = [(129, 722, 362, False), (256, 162, 82, False), (1030, 722, 362, False), (4096, 722, 362, False), (2000, 100, 512, False), (40, 256, 3000, False),
        (200, 100, 513, True), (1024, 512, 4096, True), (700, 65, 20000, True), (9000, 64, 33000, True), (300, 64, 40, True)]


@pytest.mark.parametrize("size", KEPT, ids=ids)
@pytest.mark.parametrize("dtype", [BF16, F16], ids=ids)
@pytest.mark.parametrize("dense", [False, True], ids=["index", "dense"])
@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_gradients_as_near_as_their_type(size, dtype, dense, reduction):
    """With G in 16 bits or more, the error of a gradient is what rounding it to its own type makes. G's rounding (2^-17 of a value against
    2^-9 in bfloat16) and float32's sums add less than 3 % to its size; G in the type's own bits adds up to 60 %."""
    rows, feats, classes, asked = size
    if dense and rows * classes > 1 << 25:
        pytest.skip("64-bit target weights of this size")
    x, w, b, t = _loss_inputs(rows, feats, classes, dtype, dense, True)
    f = torch.full((rows,), 64.0, device="cuda")
    if reduction == "none":
        f *= 0.5 + torch.rand(rows, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    got = _loss_run(x, w, b, t, f if reduction == "none" else f[0], reduction=reduction, precise_gradient=asked)
    for name, v, want in zip(("gx", "gw"), got[3:5], _loss_gradients(x, w, b, t, f)):
        fine = want.abs() >= 2.0 ** -14 if dtype == F16 else torch.ones_like(want, dtype=torch.bool)     # below, float16 has fewer bits
        own = float((want.to(dtype).double() - want)[fine].norm())
        assert float((v.double() - want)[fine].norm()) <= 1.03 * own, (name, float((v.double() - want)[fine].norm()) / own)


def test_precise_gradient_changes_nothing_else():
    for dtype in DTYPES:
        x, w, b, t = _loss_inputs(300, 96, 2000, dtype, False, True)
        one, two = (_loss_run(x, w, b, t, entropy_coeff=0.01, precise_gradient=p) for p in (False, True))
        for k in (0, 1, 2) if dtype != F32 else range(6):
            assert torch.equal(one[k], two[k])
        ref = R.loss_reference(x, w, t, b, c=0.01, grad=torch.ones((), device="cuda"))
        for name, v in zip(("gx", "gw", "gb"), two[3:]):
            R.close(name, v, ref[name])


# ------------------------------------------------------------------------------------------------ several pieces of the classes
def _scratch(rows, feats, classes, dtype, dense, reduction, precise=False):
    """Bytes of scratch memory of the forward and of the backward pass."""
    import ctypes as C
    from alphazero_amd import _native as N
    code = {"none": N.AZ_REDUCE_NONE, "mean": N.AZ_REDUCE_MEAN, "sum": N.AZ_REDUCE_SUM}[reduction] | (N.AZ_PRECISE_GRADIENT if precise else 0)
    a = N.AzLinearCeArgs(x=256, weight=512, target=768, rows=rows, features=feats, classes=classes, x_pitch=feats, weight_pitch=feats, target_pitch=classes,
                         ignore_index=-100, dtype={F32: N.AZ_DT_F32, BF16: N.AZ_DT_BF16, F16: N.AZ_DT_F16}[dtype], target_dense=dense, reduction=code)
    return [N.lib().az_linear_ce_workspace(C.byref(a), k) for k in (0, 1)]


def _pieces(rows, feats, classes, dtype, dense, reduction, precise=False):
    """(forward, backward): at least so many pieces of the classes, from the scratch memory, which would hold the copies of the weight (forward) or
    G and its transpose (backward) of all classes were there one piece."""
    ahead, back = _scratch(rows, feats, classes, dtype, dense, reduction, precise)
    planes = 2 if dtype == F32 else 1
    copied = classes * feats * 2 * planes if dtype == F32 or feats % 8 else 0
    g = classes * rows * 4 * (2 if dtype == F32 or rows <= 128 or precise else 1)
    return math.ceil(copied / ahead), math.ceil((g + classes * feats * 2 * planes + copied) / back)


# G's bytes make the pieces, with one and two planes; the weight's copies do, in both passes, with few and many rows
PIECES = [(2800, 16, 100003, F32, False, "mean", False, 1, 3), (2800, 24, 60001, F32, True, "none", False, 1, 2), (8200, 16, 70001, BF16, False, "none", False, 0, 3),
          (8200, 16, 40001, F16, False, "sum", False, 0, 2), (4200, 40, 70000, BF16, False, "mean", True, 0, 3), (9000, 33, 33001, F16, True, "none", False, 1, 2),
          (50, 8192, 33001, F32, False, "none", False, 3, 2), (50, 8192, 20001, F32, True, "mean", False, 2, 2), (200, 4100, 40001, F32, False, "mean", False, 2, 2),
          (70, 8191, 40001, BF16, False, "mean", False, 2, 2), (300, 8191, 40001, F16, True, "none", False, 2, 2), (100, 4095, 70001, BF16, True, "none", False, 2, 2),
          (60, 4096, 140001, F16, False, "none", False, 0, 2), (300, 4096, 140001, BF16, False, "none", False, 0, 2)]


@pytest.mark.parametrize("case", PIECES, ids=ids)
def test_several_pieces_of_the_classes(case):
    """Against the 64-bit form: packed weights and in-place ones, per-row gradients, target weights with entropy and bias, split sums that go on
    from the piece before."""
    rows, feats, classes, dtype, dense, reduction, precise, ahead, back = case
    got = _pieces(rows, feats, classes, dtype, dense, reduction, precise)
    assert got[0] >= ahead and got[1] >= back, got
    _check_pieces(rows, feats, classes, dtype, dense, reduction, precise)


# a weight that is read in place, one that is copied, and planes of float32: pieces of 131072, 65536 and 16384 classes
@pytest.mark.parametrize("case", [(300, 4096, 131072, F16, False, "mean"), (100, 4095, 65536, BF16, True, "none"), (50, 8192, 16384, F32, False, "none")], ids=ids)
@pytest.mark.parametrize("more", [0, 1])
def test_one_class_more_than_a_piece(case, more):
    rows, feats, classes, *rest = case
    sums = rows * feats * 4        # of dx, which go from piece to piece: that is what one class more has to bring
    assert _scratch(rows, feats, classes + 1, *rest)[1] - _scratch(rows, feats, classes, *rest)[1] >= sums
    assert _scratch(rows, feats, classes, *rest)[1] - _scratch(rows, feats, classes - 1, *rest)[1] < sums
    _check_pieces(rows, feats, classes + more, *rest)


def _check_pieces(rows, feats, classes, dtype, dense, reduction, precise=False):
    x, w, b, t = _loss_inputs(rows, feats, classes, dtype, dense, True)
    g = torch.Generator(device="cuda").manual_seed(5)
    grad = (0.5 + torch.rand(rows, generator=g, device="cuda")) * 64 if reduction == "none" else torch.tensor(64.0, device="cuda")
    c = 0.01 if dense else 0.0
    out = _loss_run(x, w, b, t, grad, reduction=reduction, entropy_coeff=c, precise_gradient=precise)
    ref = R.loss_reference(x, w, t, b, c=c, reduction=reduction, grad=grad)
    counts = torch.ones(rows, dtype=torch.bool, device="cuda") if dense else t != -100
    for name, v in zip(("loss", "ce", "ent", "gx", "gw", "gb"), out):
        if name in ("loss", "ce", "ent") and v.dim():
            R.close(name, v[counts], (ref[name][0][counts], ref[name][1][counts]))
        else:
            R.close(name, v, ref[name])


# ------------------------------------------------------------------------------------------------ derivatives of derivatives
@pytest.mark.parametrize("dense", [False, True], ids=["index", "dense"])
def test_a_second_derivative_is_refused(dense):
    """create_graph gives the first derivatives; what is differentiated again raises, where it would be taken for a constant."""
    head = _head()
    x, w, b, t = _loss_inputs(40, 64, 90, F32, dense, True)
    want = _loss_run(x, w, b, t)[3:]
    for k in range(3):
        leaves = [v.clone().requires_grad_(True) for v in (x, w, b)]
        loss = head.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2])
        grads = torch.autograd.grad(loss, leaves, create_graph=True)
        for g, v in zip(grads, want):
            assert torch.equal(g, v)
        with pytest.raises(NotImplementedError, match="second derivative"):
            (loss + grads[k].square().sum()).backward()
        with torch.no_grad():                       # clipping, say
            assert torch.equal(grads[k].mul_(0.5), 0.5 * want[k])
        assert torch.equal((grads[k] * 2).detach(), want[k])
        other = (leaves[0] ** 3).sum()              # a second derivative of something else in the same graph
        loss = head.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2])
        g, = torch.autograd.grad(other + loss, leaves[1 - k % 2], create_graph=True)
        assert g.requires_grad
        g.mul_(2.0)
    xs = x.clone().requires_grad_(True)
    factor = torch.ones((), device="cuda", requires_grad=True)
    y = head.dropout(xs, 0.25, 3)
    g, = torch.autograd.grad(y.sum() * factor, xs, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
