"""The operators of alphazero_amd.head on the GPU against plain forms in 64 bits (head_ref.py)."""
import math

import numpy as np
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


def _inputs(rows, feats, classes, dtype, dense, bias, seed=0, device="cuda"):
    g = torch.Generator(device=device).manual_seed(1000 * rows + 10 * feats + classes + seed)
    x = torch.randn((rows, feats), generator=g, device=device).to(dtype)
    w = (torch.randn((classes, feats), generator=g, device=device) * (2.0 / math.sqrt(feats))).to(dtype)
    b = (torch.randn(classes, generator=g, device=device) * 0.3).to(dtype) if bias else None
    if dense:
        t = torch.rand((rows, classes), generator=g, device=device) ** 4
        t = torch.where(t < 0.3, 0.0, t) + 1e-3
        t = t / t.sum(1, keepdim=True) * (0.5 + torch.rand((rows, 1), generator=g, device=device))      # need not sum to one
    else:
        t = torch.randint(classes, (rows,), generator=g, device=device)
        if rows > 2:
            t[torch.rand(rows, generator=g, device=device) < 0.2] = -100
            t[0] = classes - 1
    return x, w, b, t


def _run(x, w, b, t, grad=None, **kw):
    """(loss, ce, ent, gx, gw, gb) of the operator with fresh leaves."""
    leaves = [v.detach().clone().requires_grad_(True) if v is not None else None for v in (x, w, b)]
    loss, ce, ent = _head().linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], parts=True, **kw)
    loss.backward(torch.ones_like(loss) if grad is None else grad)
    return (loss.detach(), ce, ent, *(v.grad if v is not None else None for v in leaves))


def _check(x, w, b, t, c=0.0, reduction="mean", grad=None, ignore=-100):
    got = _run(x, w, b, t, grad, entropy_coeff=c, reduction=reduction, ignore_index=ignore)
    ref = R.loss_reference(x, w, t, b, ignore, c, reduction, torch.ones((), device=x.device) if grad is None else grad)
    counts = slice(None) if t.is_floating_point() or reduction != "none" else t != ignore
    for name, v in zip(("loss", "ce", "ent"), got):
        pick = counts if v.dim() else ()
        R.close(name, v[pick], (ref[name][0][pick], ref[name][1][pick]))
    for name, v in zip(("gx", "gw", "gb"), got[3:]):
        if v is not None:
            R.close(name, v, ref[name])
    return got


# up to 16 rows, up to 64 and more take other kernels
SIZES = [(2, 4100, 40), (5, 1111, 1000), (9, 31, 700), (16, 2050, 70), (12, 70, 20000), (33, 257, 600), (48, 96, 3000),
         (1, 1, 1), (1, 8, 2), (3, 5, 7), (64, 64, 64), (65, 72, 130), (256, 162, 82), (17, 1000, 300), (300, 200, 513), (130, 722, 362)]


@pytest.mark.parametrize("size", SIZES, ids=ids)
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("dense", [False, True], ids=["index", "dense"])
def test_loss_and_gradients(size, dtype, dense):
    x, w, b, t = _inputs(*size, dtype, dense, bias=size[0] % 2 == 1 or size[0] == 256)
    scale = 256.0 if dtype == F16 else 1.0
    _check(x, w, b, t, grad=torch.tensor(scale, device="cuda"))


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("dense", [False, True], ids=["index", "dense"])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("rows", [11, 40, 200])
def test_entropy_and_reductions(dtype, dense, reduction, rows):
    x, w, b, t = _inputs(rows, 96, 150, dtype, dense, True)
    g = torch.linspace(-3, 5, rows, device="cuda") if reduction == "none" else torch.tensor(7.0, device="cuda")
    _check(x, w, b, t, c=0.05, reduction=reduction, grad=g)


@pytest.mark.parametrize("size", [(20, 5000, 90), (70, 8200, 60), (33, 4096, 1100), (130, 2999, 70), (257, 1999, 33), (65, 20001, 3)], ids=ids)
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("dense", [False, True], ids=["index", "dense"])
def test_long_features(size, dtype, dense):
    """Few rows and classes: the walk over the features is split."""
    x, w, b, t = _inputs(*size, dtype, dense, size[0] & 1 == 0)
    _check(x, w, b, t, c=0.01 if size[0] > 100 else 0.0, reduction="sum" if size[0] == 70 else "mean")


@pytest.mark.parametrize("rows", [1, 3, 17, 40, 128])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=ids)
@pytest.mark.parametrize("dense", [False, True], ids=["index", "dense"])
@pytest.mark.parametrize("size", [(759, 369), (72, 2000), (4096, 130)], ids=ids)
def test_gradients_of_few_rows_keep_their_type(size, dtype, dense, rows):
    """With few rows the gradient of the logits is held in more than 16 bits: what is left is the rounding of the results (half a step) and
    16 bits or more of each term of their sums, 2^-15 with the float32 sums' own."""
    x, w, b, t = _inputs(rows, *size, dtype, dense, True)
    got = _run(x, w, b, t, torch.tensor(64.0, device="cuda"), reduction="sum")
    z = x.double() @ w.double().t() + b.double()
    if dense:
        pi = t.double()
    else:
        pi = torch.zeros_like(z)
        live = t != -100
        pi[live, t[live]] = 1.0
    g = 64.0 * (pi.sum(1, keepdim=True) * torch.softmax(z, 1) - pi)
    size_g = 64.0 * (pi.sum(1, keepdim=True) * torch.softmax(z, 1) + pi)      # of what g is the difference of, for its softmax' float32
    for name, v, want, terms in (("gx", got[3], g @ w.double(), size_g @ w.double().abs()), ("gw", got[4], g.t() @ x.double(), size_g.t() @ x.double().abs())):
        half = torch.finfo(dtype).eps / 2
        R.close(name, v, (want, half * want.abs() + 2.0 ** -15 * terms + R.TINY[dtype]))


# a few rows of a large weight take the kernels that stream it: both passes, only the backward one (16 bits, read in place)
@pytest.mark.parametrize("size", [(1, 1032, 33000), (2, 1032, 33000), (4, 1032, 33000), (7, 2056, 17000), (16, 1032, 33000), (16, 1025, 66000), (3, 1025, 66001),
                                  (30, 1025, 66001), (9, 72, 66001)], ids=ids)
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("dense", [False, True], ids=["index", "dense"])
def test_few_rows_of_a_large_weight(size, dtype, dense):
    x, w, b, t = _inputs(*size, dtype, dense, size[0] != 4)
    _check(x, w, b, t, c=0.01 if size[0] in (7, 16) else 0.0, grad=torch.tensor(256.0 if dtype == F16 else 1.0, device="cuda"))


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("size", [(13, 1032, 33000), (11, 1025, 66001)], ids=ids)
def test_few_rows_of_a_large_weight_special_values(dtype, size):
    rows, feats, classes = size
    x, w, b, t = _inputs(*size, dtype, False, True)
    t[4], t[6] = -100, 7
    shut = torch.arange(classes, device="cuda") % 3 == 0
    shut[64:4096] = True
    b[shut] = -float("inf")
    t = torch.where(t == -100, t, torch.where(shut[t.clamp(min=0)], 1, t))
    g = torch.linspace(0.5, 2.0, rows, device="cuda")
    good = _check(x, w, b, t, c=0.05, reduction="none", grad=g)
    assert not good[5][shut].any() and not good[4][shut].any()
    y = x.clone()
    y[4] = float("nan")                                  # a row that does not count holds anything
    h = g.clone()
    h[4] = float("inf")
    for a, v in zip(good, _run(y, w, b, t, h, entropy_coeff=0.05, reduction="none")):
        assert torch.equal(a, v)
    for wrong in (classes, -1, 1 << 40):
        u = t.clone()
        u[6] = wrong
        each, _, _, gx, gw, gb = _run(x, w, b, u, g, reduction="none")
        keep = torch.arange(rows) != 6
        assert math.isnan(float(each[6])) and torch.isfinite(each[keep]).all()
        assert torch.isnan(gx[6]).all() and torch.isnan(gw).any() and torch.isnan(gb).any()


@pytest.mark.parametrize("size", [(520, 64, 20000), (2048, 128, 3000), (5000, 40, 700)], ids=ids)
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
def test_large_and_middle_tiles(size, dtype):
    x, w, b, t = _inputs(*size, dtype, False, True)
    _check(x, w, b, t, c=0.01, grad=torch.tensor(512.0 if dtype == F16 else 1.0, device="cuda"))


@pytest.mark.parametrize("dtype", [F32, F16], ids=ids)
def test_dense_large_tiles(dtype):
    x, w, b, t = _inputs(4096, 48, 3300, dtype, True, True)
    _check(x, w, b, t, c=0.01, grad=torch.tensor(512.0, device="cuda"))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=ids)
def test_pieces_of_the_classes(dtype):
    rows, classes = (2800, 33000) if dtype == F32 else (8200, 33000)     # more than one piece: 1 GB / (4 bytes x planes x rows)
    x, w, b, t = _inputs(rows, 16, classes, dtype, False, True)
    _check(x, w, b, t)


def test_gradient_by_differences():
    """Float32 gradients against central differences of the 64-bit loss along random directions."""
    x, w, b, t = _inputs(40, 33, 57, F32, True, True)
    _, _, _, gx, gw, gb = _run(x, w, b, t, entropy_coeff=0.1)

    def f(dx, dw, db, h):
        logp = torch.log_softmax((x.double() + h * dx) @ (w.double() + h * dw).t() + b.double() + h * db, 1)
        return (-(t.double() * logp).sum(1) + 0.1 * (logp.exp() * logp).sum(1)).mean()

    for seed in range(3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        d = [torch.randn(v.shape, generator=g, device="cuda", dtype=torch.float64) for v in (x, w, b)]
        h = 1e-5
        want = (f(*d, h) - f(*d, -h)) / (2 * h)
        have = sum((a.double() * v).sum() for a, v in zip((gx, gw, gb), d))
        # differences are off by h^2 times the third derivative (~1e-8 here), the gradients by 2^-20 of their magnitude
        size = sum((a.double().abs() * v.abs()).sum() for a, v in zip((gx, gw, gb), d))
        assert abs(float(want - have)) <= 2.0 ** -18 * float(size) + 1e-7


@pytest.mark.parametrize("rows", [9, 50, 70])
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
def test_rows_that_do_not_count_may_hold_anything(dtype, rows):
    x, w, b, t = _inputs(rows, 40, 90, dtype, False, True)
    t[torch.arange(1, 8, 3)] = -100
    out = (t == -100).nonzero()[:, 0]
    assert len(out) >= 3
    x[out[0]], x[out[1]], x[out[2], 3] = float("nan"), float("inf"), -float("inf")
    got = _check(x, w, b, t, c=0.01)
    assert (got[3][out] == 0).all()
    g = torch.linspace(0.5, 1.5, rows, device="cuda")
    g[out] = float("nan")                                # nor may their gradients matter
    none = _run(x, w, b, t, g, reduction="none")
    assert (none[0][out] == 0).all() and (none[3][out] == 0).all()
    assert all(torch.isfinite(v).all() for v in none[3:])
    g[out] = 0.0
    for a, v in zip(none, _run(x, w, b, t, g, reduction="none")):
        assert torch.equal(a, v)


def test_no_row_counts():
    x, w, b, t = _inputs(20, 16, 30, BF16, False, True)
    t[:] = -100
    loss, _, _, gx, gw, gb = _run(x, w, b, t)
    assert math.isnan(float(loss))                      # a mean of nothing, as in torch
    assert not gx.any() and not gw.any() and not gb.any()
    assert float(_run(x, w, b, t, reduction="sum")[0]) == 0.0


def test_other_ignore_index_and_last_row():
    x, w, b, t = _inputs(33, 16, 30, F32, False, True)
    t[t == -100] = 5
    t[32] = 7
    _check(x, w, b, t, ignore=5)


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("dense", [False, True], ids=["index", "dense"])
@pytest.mark.parametrize("rows", [13, 50, 90])
def test_classes_that_cannot_be(dtype, dense, rows):
    x, w, b, t = _inputs(rows, 24, 200, dtype, dense, True)
    shut = torch.arange(200, device="cuda") % 3 == 0
    shut[64:192] = True                                  # whole tiles of them
    b[shut] = -float("inf")
    if dense:
        t = torch.where(shut, 0.0, t)
    else:
        t = torch.where(t == -100, t, torch.where(shut[t.clamp(min=0)], 1, t))
    got = _check(x, w, b, t, c=0.05)
    assert not got[5][shut].any() and not got[4][shut].any()
    b[:] = torch.finfo(dtype).min                        # the type's lowest value everywhere is still a softmax
    loss = _run(x * 0, w, b, t, reduction="none")[1]
    live = slice(None) if dense else t != -100
    total = t.sum(1) if dense else 1.0
    # equal logits, whatever they are: log(classes) from a sum of ones, to the rounding of a logarithm and two products
    assert ((loss - total * math.log(200)).abs()[live] <= 8 * 2.0 ** -23 * 6).all()


@pytest.mark.parametrize("rows", [5, 30, 100])
def test_row_without_a_softmax(rows):
    x, w, b, t = _inputs(rows, 8, 12, F32, False, True)
    t[:5] = torch.tensor([1, 2, 3, 4, -100], device="cuda")
    b[:] = -float("inf")
    loss = _run(x, w, b, t, reduction="none")[0]
    assert torch.isnan(loss[:4]).all() and float(loss[4]) == 0.0
    b[:] = 0
    b[3] = -float("inf")                                 # the target itself cannot be: an infinite loss, the others stay
    loss = _run(x, w, b, t, reduction="none")[0]
    assert float(loss[2]) == float("inf") and torch.isfinite(loss[:2]).all()


@pytest.mark.parametrize("rows", [10, 40, 80])
def test_index_outside_the_classes(rows):
    x, w, b, t = _inputs(rows, 16, 30, BF16, False, True)
    for wrong in (30, -1, 1 << 40, -(1 << 62)):
        u = t.clone()
        u[3] = wrong
        each = _run(x, w, b, u, reduction="none")[0]
        assert math.isnan(float(each[3])) and torch.isfinite(each[torch.arange(rows) != 3]).all()
        loss, _, _, gx, gw, gb = _run(x, w, b, u)
        assert math.isnan(float(loss)) and torch.isnan(gx[3]).all() and torch.isnan(gw).any() and torch.isnan(gb).all()


@pytest.mark.parametrize("rows", [12, 60, 80])
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
def test_layouts(dtype, rows):
    head = _head()
    x, w, b, t = _inputs(rows, 40, 70, dtype, True, True)
    want = _run(x, w, b, t, entropy_coeff=0.01)
    big = torch.full((rows + 20, 64), float("nan"), device="cuda", dtype=dtype)
    wide = torch.full((90, 56), float("nan"), device="cuda", dtype=dtype)
    tt = torch.full((rows, 99), float("nan"), device="cuda")
    for dr, dc in ((0, 0), (3, 8), (5, 1)):              # aligned rows of a larger matrix, and rows that start anywhere
        big[dr:dr + rows, dc:dc + 40] = x
        wide[dr:dr + 70, dc:dc + 40] = w
        tt[:, dc:dc + 70] = t
        got = _run_views(big[dr:dr + rows, dc:dc + 40], wide[dr:dr + 70, dc:dc + 40], b, tt[:, dc:dc + 70])
        for a, v in zip(want, got):
            assert torch.equal(a, v)
        for a, v in zip(want, _run_views(x, wide[dr:dr + 70, dc:dc + 40], b, t)):      # one operand in place, the other not
            assert torch.equal(a, v)
        for a, v in zip(want, _run_views(big[dr:dr + rows, dc:dc + 40], w, b, t)):
            assert torch.equal(a, v)
    xt = x.t().contiguous().t()                          # columns first
    assert torch.equal(head.linear_cross_entropy(xt, w, t, b, entropy_coeff=0.01), want[0])
    x3 = x.reshape(2, rows // 2, 40)
    assert torch.equal(head.linear_cross_entropy(x3, w, t.reshape(2, rows // 2, 70), b, entropy_coeff=0.01), want[0])
    each = head.linear_cross_entropy(x3, w, t.reshape(2, rows // 2, 70), b, reduction="none")
    assert each.shape == (2, rows // 2)
    one = x[:1].expand(rows, 40)                           # a row many times: stride 0
    assert torch.equal(head.linear_cross_entropy(one, w, t, b), head.linear_cross_entropy(one.contiguous(), w, t, b))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=ids)
def test_rows_far_apart(dtype):
    """Rows of a very wide matrix (beyond what the tiles address in place), and features that start past 2^31 bytes of a tensor."""
    x, w, b, t = _inputs(70, 64, 300, dtype, False, True)
    want = _run(x, w, b, t)
    far = torch.zeros((300, 4_200_008), device="cuda", dtype=dtype)
    far[:, 4_200_000 - 64:4_200_000] = w
    got = _run_views(x, far[:, 4_200_000 - 64:4_200_000], b, t, 0.0)
    for a, v in zip(want, got):
        assert torch.equal(a, v)


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("rows", [8, 80])
def test_a_row_of_infinite_weights_spoils_itself_only(dtype, rows):
    x, w, b, t = _inputs(rows, 32, 50, dtype, True, False)
    bad = t.clone()
    bad[3, 7] = float("inf")
    good, got = _run(x, w, None, t, reduction="sum"), _run(x, w, None, bad, reduction="sum")
    keep = torch.arange(rows) != 3
    assert torch.equal(got[3][keep], good[3][keep]) and not torch.isfinite(got[3][3]).any()
    big = t.clone()
    big[3] *= 1e4                                        # weights of very different sums
    _check(x, w, None, big, reduction="sum")


def _run_views(x, w, b, t, c=0.01):
    x, w, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True), b.detach().clone().requires_grad_(True)
    loss, ce, ent = _head().linear_cross_entropy(x, w, t, b, entropy_coeff=c, parts=True)
    gx, gw, gb = torch.autograd.grad(loss, (x, w, b))
    return loss.detach(), ce, ent, gx, gw, gb


def test_some_gradients_only():
    x, w, b, t = _inputs(100, 48, 77, BF16, False, True)
    full = _run(x, w, b, t)
    for k in range(3):
        leaves = [v.detach().clone().requires_grad_(i == k) for i, v in enumerate((x, w, b))]
        loss = _head().linear_cross_entropy(leaves[0], leaves[1], t, leaves[2])
        (g,) = torch.autograd.grad(loss, leaves[k])
        assert torch.equal(g, full[3 + k])


def test_same_bits_every_time_and_broadcast_gradient():
    x, w, b, t = _inputs(500, 100, 3000, F16, False, True)
    first = _run(x, w, b, t, entropy_coeff=0.01)
    for a, v in zip(first, _run(x, w, b, t, entropy_coeff=0.01)):
        assert torch.equal(a, v)
    xs = x.clone().requires_grad_(True)
    rows = _head().linear_cross_entropy(xs, w, t, b, reduction="none")
    rows.sum().backward()                                # the gradient of a sum is one value with stride 0
    ref = R.loss_reference(x, w, t, b, grad=torch.ones(500, device="cuda"), reduction="none")
    R.close("gx", xs.grad, ref["gx"])


def test_autocast_like_a_linear_layer():
    x, w, b, t = _inputs(64, 32, 50, F32, True, True)
    w.requires_grad_(True)
    with torch.autocast("cuda", dtype=BF16):
        loss = _head().linear_cross_entropy(x, w, t, b)
    loss.backward()
    assert w.grad.dtype == F32
    assert torch.equal(loss, _head().linear_cross_entropy(x.bfloat16(), w.bfloat16(), t, b.bfloat16()))


def test_no_rows():
    head = _head()
    w = torch.randn(5, 4, device="cuda", requires_grad=True)
    x = torch.empty(0, 4, device="cuda", requires_grad=True)
    t = torch.empty(0, dtype=torch.int64, device="cuda")
    assert math.isnan(float(head.linear_cross_entropy(x, w, t).detach()))
    s = head.linear_cross_entropy(x, w, t, reduction="sum")
    s.backward()
    assert float(s.detach()) == 0.0 and not w.grad.any() and x.grad.shape == (0, 4)
    assert head.linear_cross_entropy(x, w, t, reduction="none").shape == (0,)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("dense", [False, True], ids=["index", "dense"])
def test_no_rows_look_at_no_weights(reduction, dense):
    """Without rows the weights have no part in the result, whatever they hold: infinities, or values whose sum leaves float16."""
    head = _head()
    for fill in (float("inf"), 65504.0):
        x = torch.empty(0, 9, dtype=F16, device="cuda", requires_grad=True)
        w = torch.full((50, 9), fill, dtype=F16, device="cuda", requires_grad=True)
        b = torch.full((50,), fill, dtype=F16, device="cuda", requires_grad=True)
        t = torch.empty(0, 50, device="cuda") if dense else torch.empty(0, dtype=torch.int64, device="cuda")
        loss, ce, ent = head.linear_cross_entropy(x, w, t, b, reduction=reduction, parts=True)
        for v in (loss, ce, ent):
            assert v.shape == ((0,) if reduction == "none" else ()) and v.dtype == F32
            assert torch.isnan(v).all() if reduction == "mean" else not v.any()
        assert not ce.requires_grad
        loss.sum().backward()
        assert x.grad.shape == (0, 9) and not w.grad.any() and not b.grad.any()


# ------------------------------------------------------------------------------------------------ dropout
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("count", [1, 7, 8, 9, 255, 2048, 2049, 100003])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_dropout(dtype, count, p):
    head = _head()
    g = torch.Generator(device="cuda").manual_seed(count)
    x, r, gy = (torch.randn(count, generator=g, device="cuda").to(dtype) for _ in range(3))
    seed, offset = 0x0123456789ABCDEF ^ (count << 33), count * 977 + (1 << 40)
    kept = torch.from_numpy(R.philox_kept(count, p, seed, offset)[0]).cuda()
    t = round(65536 * p)
    scale = 65536 / (65536 - t) if t < 65536 else 0.0
    for residual in (None, r):
        xs = x.clone().requires_grad_(True)
        rs = None if residual is None else residual.clone().requires_grad_(True)
        y = head.dropout(xs, p, seed, offset, residual=rs)
        want = torch.where(kept, x.double() * scale, 0.0) + (0 if residual is None else r.double())
        mag = torch.where(kept, (x.double() * scale).abs(), 0.0) + (0 if residual is None else r.double().abs())
        R.close("y", y.detach(), (want, R.U[dtype] * want.abs() + 4 * R.F32 * mag + R.TINY[dtype]))
        y.backward(gy)
        gw = torch.where(kept, gy.double() * scale, 0.0)
        R.close("gx", xs.grad, (gw, R.U[dtype] * gw.abs() + 4 * R.F32 * gw.abs() + R.TINY[dtype]))
        assert not xs.grad[~kept].any()
        if rs is not None:
            assert torch.equal(rs.grad, gy)


def test_dropout_layouts_and_masks():
    head = _head()
    x = torch.randn(64, 37, device="cuda")
    y = head.dropout(x, 0.3, 5)
    assert torch.equal(head.dropout(x.t().contiguous().t(), 0.3, 5), y)                    # by position, not by address
    buf = torch.zeros(64 * 37 + 1, device="cuda")
    buf[1:] = x.reshape(-1)
    assert torch.equal(head.dropout(buf[1:].view(64, 37), 0.3, 5), y)                      # not at a multiple of 16 bytes
    assert not torch.equal(head.dropout(x, 0.3, 6), y) and not torch.equal(head.dropout(x, 0.3, 5, 1), y)
    seed = torch.tensor([5], device="cuda")
    assert torch.equal(head.dropout(x, 0.3, seed), y)
    negative = torch.tensor(-1, device="cuda")
    assert torch.equal(head.dropout(x, 0.3, negative), head.dropout(x, 0.3, (1 << 64) - 1))
    bad = x.clone()
    dropped = y == 0
    bad[dropped] = float("nan")
    assert torch.equal(head.dropout(bad, 0.3, 5), y)
    xs = x.clone().requires_grad_(True)
    head.dropout(xs, 0.3, 5).sum().backward()                                              # a gradient with stride 0
    assert torch.equal(xs.grad == 0, dropped)
    assert head.dropout(torch.empty(0, 3, device="cuda"), 0.3, 5).shape == (0, 3)
    share = float((head.dropout(torch.ones(1 << 20, device="cuda"), 0.1, 3) == 0).float().mean())
    assert abs(share - 0.1) < 6 * math.sqrt(0.09 / (1 << 20))                              # six standard deviations


# ------------------------------------------------------------------------------------------------ 8-bit integers
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("size", [(1, 1), (3, 15), (5, 16), (4, 162), (2, 4097), (3, 23104)], ids=ids)
def test_quantize_rows(dtype, size):
    g = torch.Generator(device="cuda").manual_seed(size[1])
    x = torch.randn(size, generator=g, device="cuda").to(dtype)
    if size[1] > 8:
        x[-1] = 0
        x[0, :4] = torch.tensor([127.0, 0.5, 1.5, -2.5])                                   # ties, with max 127 at least
        x[0, 4:] = x[0, 4:].clamp(-100, 100)
    q, s = _head().quantize_rows(x)
    rq, rs = R.quantize_reference(x)
    assert torch.equal(q.cpu(), rq) and torch.equal(s.cpu(), rs)


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("size", [(2051, 1), (2048, 63), (2049, 129), (2050, 361), (3001, 513), (2053, 1025), (2047, 2048), (2055, 2047),
                                  (100, 6001), (70, 14333), (60, 23105), (50, 33001), (40, 70003)], ids=ids)
def test_quantize_many_short_rows(dtype, size):
    """Rows that share a workgroup, of odd lengths and far apart; a row that is not finite and one of zeros stay their own affair."""
    rows, cols = size
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    wide = (torch.randn((rows, cols + 3), generator=g, device="cuda") * 3).to(dtype)
    x = wide[:, 1:cols + 1]
    x[5], x[7, cols // 2], x[rows - 2, cols - 1] = 0.0, float("nan"), float("-inf")
    q, scale = _head().quantize_rows(x)
    v = x.double()
    top = v.abs().amax(1)
    good = torch.isfinite(top) & (top > 0)
    assert torch.equal(scale[good], (top[good] / 127).float()) and scale[5] == 0 and torch.isnan(scale[[7, rows - 2]]).all()
    assert not q[~good].any()
    exact = torch.round(127 * v[good] / top[good, None])
    assert torch.equal(q[good].double(), exact)


def test_quantize_rows_near_halves_and_odd_values():
    head = _head()
    g = torch.Generator(device="cuda").manual_seed(2)
    top = torch.rand(64, 1, generator=g, device="cuda") * 3 + 0.1
    x = (top.double() * (torch.randint(-127, 127, (64, 200), generator=g, device="cuda") + 0.5) / 127).float()    # as near to a half as float32 gets
    x[:, :1] = top
    q, s = head.quantize_rows(x)
    rq, rs = R.quantize_reference(x)
    assert torch.equal(q.cpu(), rq) and torch.equal(s.cpu(), rs)
    x = torch.tensor([[1e-40, -2e-40, 0.0], [3e38, -1e38, 0.0], [float("inf"), 1.0, 2.0], [float("nan"), 1.0, 2.0], [0.0, -0.0, 0.0]], device="cuda")
    q, s = head.quantize_rows(x)
    # 1e-40 and 2e-40 are 71362 and 142725 of float32's smallest steps: 127 * 71362 / 142725 = 63.49956
    assert q.cpu().tolist() == [[63, -127, 0], [127, -42, 0], [0, 0, 0], [0, 0, 0], [0, 0, 0]]
    assert torch.isnan(s[2:4]).all() and float(s[4]) == 0.0
    y = head.int8_linear(x, torch.ones(4, 3, dtype=torch.int8, device="cuda"), torch.ones(4, device="cuda"))
    assert torch.isnan(y[2:4]).all() and torch.isfinite(y[[0, 1, 4]]).all()


def _int8_check(x, qw, ws, b, y, q, s):
    dt = y.dtype
    sums = q.double() @ qw.double().t()
    want = sums * s.double()[..., None] * ws.double() + (0 if b is None else b.double())
    mag = (sums * s.double()[..., None] * ws.double()).abs() + (0 if b is None else b.double().abs())
    R.close("y", y, (want, R.U[dt] * want.abs() + 8 * R.F32 * mag + R.TINY[dt]))


INT8 = [(1, 1, 1), (1, 64, 16), (1, 4096, 1024), (5, 100, 33), (16, 130, 50), (17, 2000, 83), (33, 77, 300), (64, 512, 128), (65, 64, 64), (70, 1000, 90),
        (256, 3000, 256), (300, 129, 517), (1024, 200, 2500), (2304, 256, 5632),
        # few tokens of aligned weights, of crooked ones, of many channels; walks over the features in pieces
        (3, 256, 100), (9, 1024, 500), (16, 4096, 333), (20, 2048, 31), (40, 2048, 100), (48, 512, 128), (49, 512, 128), (2, 4095, 300), (4, 131, 50), (1, 128, 16500),
        (3, 130, 16400), (20, 8208, 70), (64, 23104, 256), (90, 14336, 1000), (200, 5000, 65)]


@pytest.mark.parametrize("size", INT8, ids=ids)
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
def test_int8_linear(size, dtype):
    head = _head()
    m, k, n = size
    g = torch.Generator(device="cuda").manual_seed(m + k + n)
    x = torch.randn((m, k), generator=g, device="cuda").to(dtype)
    qw = torch.randint(-127, 128, (n, k), generator=g, device="cuda").to(torch.int8)
    ws = torch.rand(n, generator=g, device="cuda") / 127
    b = torch.randn(n, generator=g, device="cuda").to(dtype) if n % 2 else None
    q, s = head.quantize_rows(x)
    y = head.int8_linear(x, qw, ws, b)
    assert y.dtype == dtype
    _int8_check(x, qw, ws, b, y, q, s)
    y8 = head.int8_linear(q, qw, ws, b, x_scale=s, out_dtype=dtype)
    assert torch.equal(y8, y)                                                              # the sum is exact on every path
    assert head.int8_linear(q, qw, ws, x_scale=s).dtype == F32


def test_int8_extremes_and_layouts():
    head = _head()
    k = 131071
    for m in (1, 100):
        x = torch.full((m, k), -128, dtype=torch.int8, device="cuda")
        w = torch.full((70, k), -128, dtype=torch.int8, device="cuda")
        y = head.int8_linear(x, w, torch.ones(70, device="cuda"), x_scale=torch.ones(m, device="cuda"))
        assert (y.double() == float(np.float32(k * 16384))).all()
    g = torch.Generator(device="cuda").manual_seed(4)
    for m in (3, 100):
        x = torch.randn((m, 200), generator=g, device="cuda")
        w = torch.randint(-127, 128, (90, 200), generator=g, device="cuda").to(torch.int8)
        ws = torch.rand(90, generator=g, device="cuda")
        want = head.int8_linear(x, w, ws)
        for dc, width in ((0, 208), (16, 256), (5, 233), (1, 201)):
            big = torch.full((90, width), 77, dtype=torch.int8, device="cuda")
            big[:, dc:dc + 200] = w
            xb = torch.full((m, 300), float("nan"), device="cuda")
            xb[:, dc:dc + 200] = x
            assert torch.equal(head.int8_linear(xb[:, dc:dc + 200], big[:, dc:dc + 200], ws), want)
        assert torch.equal(head.int8_linear(x.reshape(m, 1, 200), w, ws), want.reshape(m, 1, 90))
        assert torch.equal(head.int8_linear(x, w.t().contiguous().t(), ws), want)
    assert head.int8_linear(torch.empty(0, 200, device="cuda"), w, ws).shape == (0, 90)


def test_int8_layer():
    head = _head()
    torch.manual_seed(0)
    lin = torch.nn.Linear(163, 83).cuda()
    q = head.Int8Linear(lin)
    x = torch.randn(40, 163, device="cuda")
    y = q(x)
    # each product is off by half a step of both operands: |x| w_step / 2 + |w| x_step / 2 + a quarter of their product
    xs, wsc = x.abs().amax(1, keepdim=True) / 127, lin.weight.abs().amax(1) / 127
    tol = x.abs().sum(1, keepdim=True) * wsc / 2 + xs * lin.weight.abs().sum(1) / 2 + 163 * xs * wsc / 4
    assert ((y - lin(x)).abs() <= tol * 1.0001 + 1e-5).all()
    other = head.Int8Linear(torch.nn.Linear(163, 83).cuda())
    other.load_state_dict(q.state_dict())
    assert torch.equal(other(x), y)


# ------------------------------------------------------------------------------------------------ together, streams, graphs
def test_training_step_of_a_head():
    """Dropout with a residual, then the loss, and back: against the same in 64 bits with the operator's own mask."""
    head = _head()
    x, w, b, t = _inputs(128, 64, 90, F32, True, True)
    r = torch.randn(128, 64, device="cuda")
    leaves = [v.clone().requires_grad_(True) for v in (x, r, w, b)]
    h = head.dropout(leaves[0], 0.25, 11, 4, residual=leaves[1])
    loss = head.linear_cross_entropy(h, leaves[2], t, leaves[3], entropy_coeff=0.01)
    loss.backward()
    ref = R.loss_reference(h.detach(), w, t, b, c=0.01, grad=torch.ones((), device="cuda"))
    R.close("loss", loss.detach(), ref["loss"])
    kept = torch.from_numpy(R.philox_kept(128 * 64, 0.25, 11, 4)[0]).cuda().view(128, 64)
    gx, tol = ref["gx"]
    R.close("residual", leaves[1].grad, (gx, tol))
    scale = 65536 / (65536 - round(65536 * 0.25))
    R.close("x", leaves[0].grad, (torch.where(kept, gx * scale, 0.0), torch.where(kept, tol * scale + 4 * R.F32 * gx.abs(), 0.0)))
    R.close("w", leaves[2].grad, ref["gw"])
    with torch.no_grad():        # the served form of the same layer
        lin = torch.nn.Linear(64, 90).cuda()
        lin.weight.copy_(w)
        lin.bias.copy_(b)
        y = head.Int8Linear(lin)(h)
    assert y.shape == (128, 90)


def test_other_streams_at_once():
    head = _head()
    x, w, b, t = _inputs(600, 96, 2000, BF16, False, True)
    want = _run(x, w, b, t)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(_run(x, w, b, t))
    torch.cuda.synchronize()
    for g in got:
        for a, v in zip(want, g):
            assert torch.equal(a, v)


def test_captured_and_replayed():
    """Forward and backward of dropout + loss in one graph, replayed with other inputs and seeds, eager work between."""
    head = _head()
    x, w, b, t = _inputs(300, 72, 500, F16, False, True)
    x.requires_grad_(True)
    w.requires_grad_(True)
    seed = torch.tensor([1], device="cuda")
    g1 = torch.tensor(64.0, device="cuda")

    def step():
        h = head.dropout(x, 0.2, seed)
        loss = head.linear_cross_entropy(h, w, t, b, entropy_coeff=0.01)
        gx, gw = torch.autograd.grad(loss, (x, w), g1)
        with torch.no_grad():
            y = head.int8_linear(h.detach(), q, ws)
        return loss.detach(), gx, gw, y

    q, ws = head.quantize_rows(w.detach())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.cuda.graph(second):      # another one, with scratch memory of its own pool
        out2 = step()
    for k in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(300, 72, device="cuda") + k)
        seed.fill_(100 + k)
        want = [v.clone() for v in step()]
        torch.cuda.synchronize()
        graph.replay()
        second.replay()
        torch.cuda.synchronize()
        for a, v, u in zip(want, out, out2):
            assert torch.equal(a, v) and torch.equal(a, u)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=ids)
def test_split_walks_captured_and_at_once(dtype):
    """Products whose walk is in pieces, in one graph and on two streams at once: each call has its own scratch memory."""
    head = _head()
    x, w, b, t = _inputs(70, 6000, 90, dtype, False, True)
    x.requires_grad_(True)
    w.requires_grad_(True)
    q, ws = head.quantize_rows(w.detach())
    one = torch.ones((), device="cuda")

    def step():
        loss = head.linear_cross_entropy(x, w, t, b, entropy_coeff=0.01)
        gx, gw = torch.autograd.grad(loss, (x, w), one)
        return loss.detach(), gx, gw, head.int8_linear(x.detach(), q, ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(70, 6000, device="cuda") * (k + 1))
        want = [v.clone() for v in step()]
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            there = step()
        here = step()
        torch.cuda.synchronize()
        for a, v, u, h in zip(want, out, there, here):
            assert torch.equal(a, v) and torch.equal(a, u) and torch.equal(a, h)


# ------------------------------------------------------------------------------------------------ the framework's own callers
def _net_and_batch(seed=0, n=5, rows=48):
    import stubnets
    from alphazero_amd.model import AlphaZeroNet
    torch.manual_seed(seed)
    net = AlphaZeroNet(board_size=n, channels=32, num_blocks=1).cuda()
    x = torch.from_numpy(stubnets.synthetic_planes(rows, 21, n, seed=seed + 1)).cuda()
    pi = torch.softmax(2 * torch.randn(rows, n * n + 1, device="cuda"), 1)
    z = torch.rand(rows, device="cuda") * 2 - 1
    return net, x, pi, z


@pytest.mark.parametrize("amp", [False, True])
def test_training_step_with_the_fused_policy_loss(amp):
    import copy
    from alphazero_amd.train_step import DataParallelTrainer, head_loss_terms, loss_terms
    net, x, pi, z = _net_and_batch()
    net.train()
    with torch.autocast("cuda", enabled=amp):
        feats, v = net.policy_features(x)
        feats, v = feats.detach(), v.detach()
        fused = head_loss_terms(feats, net.policy_fc, v, pi, z)
        plain = loss_terms(net.policy_fc(feats), v, pi, z)
    ref = R.loss_reference(feats, net.policy_fc.weight.to(feats.dtype), pi, net.policy_fc.bias.to(feats.dtype), c=1e-3)
    R.close("policy loss", fused[1].detach(), ref["ce"])
    assert torch.equal(fused[2], plain[2])
    # under autocast the stored logits are rounded to float16: half a step of the largest, twice (logit and normaliser)
    step = 2 * 2.0 ** -11 * 8 if amp else 1e-5
    assert abs(float(fused[0].detach() - plain[0].detach())) <= step
    runs = []
    for kw in (dict(fused_policy_loss=True), dict(fused_policy_loss=True), dict(fused_policy_loss=True, head_dropout=0.2, dropout_seed=3),
               dict(fused_policy_loss=True, head_dropout=0.2, dropout_seed=3), dict(head_dropout=0.2, dropout_seed=4)):
        m = copy.deepcopy(net)
        t = DataParallelTrainer(m, use_amp=amp, **kw)
        losses = [t.step(x, pi, z) for _ in range(3)]
        assert all(np.isfinite(v).all() for v in losses)
        assert any(not torch.equal(a, b) for a, b in zip(m.parameters(), net.parameters()))
        runs.append(losses)
    assert abs(runs[0][0][1] - float(ref["ce"][0])) <= 1e-2 and runs[2][0] != runs[0][0] and runs[4][0] != runs[2][0]
    assert runs[0][0] == runs[1][0] and runs[2][0] == runs[3][0]


def test_command_line_knobs_reach_the_step():
    from alphazero_amd import train as T
    cfg = T.parse_args(["--device", "cuda", "--board-size", "5", "--channels", "32", "--num-blocks", "1", "--train-steps-per-iter", "2", "--batch-size", "16",
                        "--fused-policy-loss", "--head-dropout", "0.1"])
    assert cfg.fused_policy_loss and cfg.head_dropout == 0.1
    import stubnets
    buf = T.ReplayBuffer(64)
    planes = stubnets.synthetic_planes(32, 21, 5, seed=3)
    rng = np.random.RandomState(0)
    buf.extend([(planes[i], rng.dirichlet(np.ones(26)).astype(np.float32), float(rng.uniform(-1, 1)), 1.0) for i in range(32)])
    T.set_seed(1)
    model = T.build_model(cfg).to("cuda")
    loss = T.train_candidate(model, buf, cfg)
    assert np.isfinite(loss).all()


def test_network_with_int8_heads():
    net, x, _, _ = _net_and_batch(n=9, rows=70)
    net.eval()
    q = net.int8_heads()
    with torch.no_grad():
        feats, _ = net.policy_features(x)
        lg, v = net(x)
        lq, vq = q(x)
    w = net.policy_fc.weight.detach()
    xs, ws = feats.abs().amax(1, keepdim=True) / 127, w.abs().amax(1) / 127
    tol = feats.abs().sum(1, keepdim=True) * ws / 2 + xs * w.abs().sum(1) / 2 + w.shape[1] * xs * ws / 4
    assert ((lq - lg).abs() <= tol * 1.001 + 1e-5).all()
    assert vq.shape == v.shape and torch.isfinite(vq).all() and (vq.abs() <= 1).all()
    net.native("f32")
    assert torch.equal(net.int8_heads()(x)[0], lq)        # also from a network with native handles
    from alphazero_amd.go import GoState
    from alphazero_amd.mcts import MCTS
    pi, action = MCTS(model=q, device="cuda", num_simulations=16, inference_batch_size=4).run(GoState.new_game(9), temperature=1e-6, add_exploration_noise=False)[:2]
    assert abs(float(np.sum(pi)) - 1) < 1e-6


# ------------------------------------------------------------------------------------------------ beyond 4 GB
def _large(shape, seed, std=1.0):
    out = torch.empty(shape, dtype=BF16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(seed)
    for i in range(0, shape[0], 1 << 16):
        out[i:i + (1 << 16)] = torch.randn((min(1 << 16, shape[0] - i), shape[1]), generator=g, device="cuda") * std
    return out


def test_loss_with_features_beyond_4_gigabytes():
    rows, feats, classes = 560_003, 4096, 40
    x, w = _large((rows, feats), 1).requires_grad_(True), _large((classes, feats), 2, 2.0 / 64).requires_grad_(True)
    t = torch.randint(classes, (rows,), device="cuda")
    loss = _head().linear_cross_entropy(x, w, t, reduction="sum")
    gx, gw = torch.autograd.grad(loss, (x, w))
    total, want_w = 0.0, torch.zeros(classes, feats, dtype=torch.float64, device="cuda")
    with torch.no_grad():
        for i in range(0, rows, 1 << 15):
            part = R.loss_reference(x[i:i + (1 << 15)], w, t[i:i + (1 << 15)], None, reduction="sum", grad=torch.ones((), device="cuda"))
            total += float(part["loss"][0])
            want_w += part["gw"][0]
            R.close(f"gx from row {i}", gx[i:i + (1 << 15)], part["gx"])
    # a row's loss is off by 1e-5 at most (its bound above), a gradient of the weight by half a step of its own and G's roundings, which
    # average out over 560003 rows: 2^-9 relative to the largest is four of them
    assert abs(float(loss.detach()) - total) <= 1e-5 * rows + 2.0 ** -22 * total
    assert (gw.double() - want_w).abs().max() <= 2.0 ** -8 * want_w.abs().max()


@pytest.mark.parametrize("rows", [3, 70])
def test_loss_with_weights_beyond_4_gigabytes(rows):
    feats, classes = 8192, 270_001
    w = _large((classes, feats), 3, 2.0 / 90).requires_grad_(True)
    x = _large((rows, feats), 4).requires_grad_(True)
    t = torch.randint(classes, (rows,), device="cuda")
    t[0], t[-1] = classes - 1, classes - 2
    rows_loss = _head().linear_cross_entropy(x, w, t, reduction="none")
    gx, gw = torch.autograd.grad(rows_loss.sum(), (x, w))
    with torch.no_grad():
        z = torch.cat([x.double() @ w[i:i + 8192].double().t() for i in range(0, classes, 8192)], 1)
        p = torch.softmax(z, 1)
        want = torch.logsumexp(z, 1) - z[torch.arange(rows), t]
        assert (rows_loss.detach().double() - want).abs().max() <= 1e-4       # 8192 products in float32 on logits of up to 12
        g = p.clone()
        g[torch.arange(rows), t] -= 1.0
        want_x = sum(g[:, i:i + 8192] @ w[i:i + 8192].double() for i in range(0, classes, 8192))
        assert (gx.double() - want_x).abs().max() <= 2.0 ** -7 * want_x.abs().max()      # G's rounding and the result's
        for i in (0, 131_072, classes - 300):
            part = g[:, i:i + 300].t() @ x.double()
            size = g[:, i:i + 300].abs().t() @ x.double().abs()
            assert ((gw[i:i + 300].double() - part).abs() <= 2.0 ** -7 * size + 1e-6 * size.max()).all()


def test_dropout_beyond_4_gigabytes():
    head = _head()
    n = (1 << 32) + 12_345
    x = torch.ones(n, dtype=BF16, device="cuda")
    y = head.dropout(x, 0.25, 9, 2)
    group = (n // 8 - 100)
    c = np.arange(group, (n + 7) // 8, dtype=np.uint64)
    words = np.stack(R.philox_block((c & np.uint64(0xFFFFFFFF), c >> np.uint64(32), np.full_like(c, 2), np.zeros_like(c)), (9, 0)), 1)
    bits = np.stack((words & np.uint64(0xFFFF), words >> np.uint64(16)), 2).reshape(-1)[:n - group * 8]
    assert torch.equal(y[group * 8:].cpu() != 0, torch.from_numpy(bits >= 16384))
    assert float(y[:1 << 20].float().sum()) > 0


@pytest.mark.parametrize("tokens", [2, 90])
def test_int8_weights_beyond_4_gigabytes(tokens):
    head = _head()
    channels, feats = 540_001, 8192
    w = torch.randint(-127, 128, (channels, feats), dtype=torch.int8, device="cuda")
    ws = torch.rand(channels, device="cuda")
    x = torch.randn(tokens, feats, device="cuda")
    q, s = head.quantize_rows(x)
    y = head.int8_linear(x, w, ws)
    for i in (0, 262_144, 524_288, channels - 500):
        _int8_check(x, w[i:i + 500], ws[i:i + 500], None, y[:, i:i + 500], q, s)


# ------------------------------------------------------------------------------------------------ more than one launch holds
def test_dropout_of_more_than_one_launch():
    """2^35 + 12345 elements in place: more threads than a launch holds."""
    from alphazero_amd import _native as N
    n, seed, offset, threshold = (1 << 35) + 12_345, 5, 3, 40_000
    x = torch.ones(n, dtype=BF16, device="cuda")
    N.check(N.lib().az_dropout(x.data_ptr(), None, x.data_ptr(), n, N.AZ_DT_BF16, threshold, seed, None, offset, torch.cuda.current_stream().cuda_stream),
            "az_dropout")
    scale = torch.tensor(65536.0 / (65536 - threshold), dtype=BF16)
    for at in (0, (1 << 34) - 4096, (1 << 35) - 4096, n - 8000 - n % 8):
        end = min(n, at + 8192)
        c = np.arange(at // 8, (end + 7) // 8, dtype=np.uint64)
        words = np.stack(R.philox_block((c & np.uint64(0xFFFFFFFF), c >> np.uint64(32), np.full_like(c, offset), np.zeros_like(c)), (seed, 0)), 1)
        bits = np.stack((words & np.uint64(0xFFFF), words >> np.uint64(16)), 2).reshape(-1)[:end - at]
        want = torch.where(torch.from_numpy(bits >= threshold), scale, torch.zeros((), dtype=BF16))
        assert torch.equal(x[at:end].cpu(), want), at


def test_quantize_rows_of_more_than_one_launch():
    rows = (1 << 24) + 5
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((rows, 8), generator=g, device="cuda").to(BF16)
    q, scale = _head().quantize_rows(x)
    for i in range(0, rows, 1 << 22):
        v = x[i:i + (1 << 22)].double()
        top = v.abs().amax(1)
        assert torch.equal(scale[i:i + (1 << 22)], (top / 127).float())      # torch's float32 division by a number is a product with 1 / 127
        assert torch.equal(q[i:i + (1 << 22)].double(), torch.round(127 * v / top[:, None]))      # 127 v is exact; ties to even


def test_int8_tokens_of_more_than_one_launch():
    tokens, feats, channels = (1 << 28) + 77, 16, 3
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randint(-127, 128, (tokens, feats), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(-127, 128, (channels, feats), generator=g, device="cuda", dtype=torch.int8)
    xs = torch.rand(tokens, generator=g, device="cuda") + 0.5
    ws = torch.tensor([1.0, 0.5, 2.0], device="cuda")
    y = _head().int8_linear(x, w, ws, x_scale=xs)
    for i in list(range(0, tokens, 1 << 24)):
        sums = x[i:i + (1 << 24)].float() @ w.float().t()        # whole numbers below 2^24: exact
        assert torch.equal(y[i:i + (1 << 24)], sums * xs[i:i + (1 << 24), None] * ws), i      # powers of two: one rounding


def test_int8_weights_copied_in_more_than_one_launch():
    channels, feats, tokens = (1 << 18) + 3, 131_057, 65
    w = torch.empty((channels, feats), dtype=torch.int8, device="cuda")
    w.random_(-127, 128, generator=torch.Generator(device="cuda").manual_seed(3))
    x = torch.randint(-127, 128, (tokens, feats), device="cuda", dtype=torch.int8)
    y = _head().int8_linear(x, w, torch.ones(channels, device="cuda"), x_scale=torch.ones(tokens, device="cuda"))
    for i in (0, 131_072, channels - 259):
        want = x.double() @ w[i:i + 259].double().t()
        assert torch.equal(y[:, i:i + 259], want.float()), i


def test_loss_of_more_tiles_than_one_launch():
    """20000 x 13.6 million logits: more tiles than a launch holds."""
    rows, feats, classes = 20_000, 8, 13_600_003
    x, w = _large((rows, feats), 5, 1.5), _large((classes, feats), 6)
    t = torch.randint(classes, (rows,), device="cuda")
    t[0], t[1], t[-1] = classes - 1, 0, 13_591_552
    with torch.no_grad():
        loss = _head().linear_cross_entropy(x, w, t, reduction="none")
        at = torch.cat([torch.arange(8, device="cuda"), torch.randint(rows, (48,), device="cuda"), torch.arange(rows - 8, rows, device="cuda")])
        z = x[at].double() @ w.double().t()
        want = torch.logsumexp(z, 1) - z[torch.arange(64), t[at]]
    # logits of up to 60 in float32 and sums of 53125 parts: 60 * 2^-22 + 2^-20 of the loss
    assert torch.isfinite(loss).all()
    assert ((loss[at].double() - want).abs() <= 60 * 2.0 ** -22 + 2.0 ** -20 * want.abs()).all()
