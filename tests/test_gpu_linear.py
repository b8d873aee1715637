"""Products of a layer with their epilogues, by group and alone, their backward pass and the per-example gradients, against
the formulas in 64 bits.

A result is a sum of k products of exact operands in fp32, in some order, then a few fp32 operations and one rounding:
off by at most (k + 40) 2^-24 times the sum of the products' sizes, carried through the epilogue (slopes of the activations
are at most 1.13; the 40 covers the epilogue's own operations), and half a unit in the last place of the result.  dZ is rounded to
the type before its products: another half unit of each term."""

import ctypes as C

import numpy as np
import pytest
import torch

import npeff_ref_amd as d

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {k: torch.finfo(t).eps / 2 for k, t in DTYPES.items()}  # relative half unit in the last place
TINY = {"f32": 0.0, "f16": 2.0**-25, "bf16": 0.0}  # absolute, where results are subnormal
EPS32 = 2.0**-24
ACTS = {
    "none": lambda z: z,
    "relu": torch.relu,
    "silu": torch.nn.functional.silu,
    "gelu": torch.nn.functional.gelu,
    "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh"),
}


def rand(shape, dt, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(DTYPES[dt]).cuda()


def wide(t, extra, shift):
    """The same values in rows that are `extra` elements further apart and begin `shift` elements late."""
    shape = t.shape[:-1] + (t.shape[-1] + extra,)
    big = torch.full((int(np.prod(shape)) + shift,), 7.0, dtype=t.dtype, device="cuda")
    v = big[shift:].view(shape)[..., : t.shape[-1]]
    v.copy_(t)
    return v


def ends_of(sizes):
    return torch.tensor([0] + list(np.cumsum(sizes)), dtype=torch.int64).cuda()


def close(got, want, sums, k, dt, more=0.0):
    """sums: of the sizes of the products behind each result; more: a further error of each."""
    got, want = got.double().cpu(), want.double().cpu()
    bound = HALF[dt] * 1.01 * want.abs() + (k + 40) * EPS32 * 1.2 * sums.double().cpu() + more + TINY[dt]
    off = (got - want).abs() - bound
    assert torch.isfinite(got).all()
    assert (off <= 0).all(), f"worst {off.max().item():g} past its bound, at {np.unravel_index(int(off.argmax()), off.shape)}"


def segments(rows, sizes):
    ends = [0] + list(np.cumsum(sizes))
    return [(g, a, b) for g, (a, b) in enumerate(zip(ends, ends[1:]))]


def reference(X, W, b, act, R, sizes):
    """(Y, Z, sums of sizes) in 64 bits on the host; sizes: rows of each group, or None."""
    X, W = X.double().cpu(), W.double().cpu()
    rows, n_out = X.shape[0], W.shape[-2]
    Z, S = torch.zeros(rows, n_out, dtype=torch.float64), torch.zeros(rows, n_out, dtype=torch.float64)
    Y = torch.zeros_like(Z)
    for g, i, j in [(None, 0, rows)] if sizes is None else segments(rows, sizes):
        w, bias = (W, b) if g is None else (W[g], None if b is None else b[g])
        Z[i:j], S[i:j] = X[i:j] @ w.T, X[i:j].abs() @ w.T.abs()
        if bias is not None:
            Z[i:j] += bias.double().cpu()
            S[i:j] += bias.double().cpu().abs()
        Y[i:j] = ACTS[act](Z[i:j])
    if R is not None:
        Y, S = Y + R.double().cpu(), S + R.double().cpu().abs()
    return Y, Z, S


def check_forward(rows, n_in, n_out, dt, act="none", bias=False, residual=False, sizes=None, lay=(0, 0), seed=0):
    lead = () if sizes is None else (len(sizes),)
    X = rand((rows, n_in), dt, seed)
    W = rand(lead + (n_out, n_in), dt, seed + 1, n_in**-0.5)
    b = rand(lead + (n_out,), dt, seed + 2) if bias else None
    R = rand((rows, n_out), dt, seed + 3) if residual else None
    Y, Z, S = reference(X, W, b, act, R, sizes)
    put = lambda t: None if t is None else wide(t, *lay)  # noqa: E731
    y, pre = put(torch.zeros(rows, n_out, dtype=DTYPES[dt], device="cuda")), put(torch.zeros(rows, n_out, dtype=DTYPES[dt], device="cuda"))
    d.op_linear(put(X), put(W), y, bias=b, act=act, residual=put(R), pre=pre, groups=None if sizes is None else ends_of(sizes))
    close(y, Y, S, n_in, dt)
    close(pre, Z, S, n_in, dt)


def check_backward(rows, n_in, n_out, dt, act="none", sizes=None, lay=(0, 0), seed=0, bias=True):
    lead = () if sizes is None else (len(sizes),)
    X, W = rand((rows, n_in), dt, seed), rand(lead + (n_out, n_in), dt, seed + 1, n_in**-0.5)
    dY, pre = rand((rows, n_out), dt, seed + 2), rand((rows, n_out), dt, seed + 3)
    # the formula: act' from autograd in 64 bits at the given pre
    z = pre.double().cpu().requires_grad_(True)
    ACTS[act](z).sum().backward()
    dZ = dY.double().cpu() * z.grad
    x, w = X.double().cpu(), W.double().cpu()
    dX, sX = torch.zeros(rows, n_in, dtype=torch.float64), torch.zeros(rows, n_in, dtype=torch.float64)
    dW, sW = torch.zeros(W.shape, dtype=torch.float64), torch.zeros(W.shape, dtype=torch.float64)
    db, sb = torch.zeros(lead + (n_out,), dtype=torch.float64), torch.zeros(lead + (n_out,), dtype=torch.float64)
    for g, i, j in [((), 0, rows)] if sizes is None else segments(rows, sizes):
        dX[i:j], sX[i:j] = dZ[i:j] @ w[g], dZ[i:j].abs() @ w[g].abs()
        dW[g], sW[g] = dZ[i:j].T @ x[i:j], dZ[i:j].abs().T @ x[i:j].abs()
        db[g], sb[g] = dZ[i:j].sum(0), dZ[i:j].abs().sum(0)
    zX, zW = sX.clone(), sW.clone()
    put = lambda t: None if t is None else wide(t, *lay)  # noqa: E731
    gx, gw = put(torch.zeros_like(X)), put(torch.zeros_like(W))
    gb = torch.zeros(lead + (n_out,), dtype=DTYPES[dt], device="cuda") if bias else None
    d.op_linear_backward(put(dY), put(X), put(W), pre=put(pre), act=act, dX=gx, dW=gw, dbias=gb,
                         groups=None if sizes is None else ends_of(sizes))
    rounded = 0.0 if act == "none" else HALF[dt] * 1.01
    # a slope's own error: four units of fp32 of terms that are at most 3 in size (it crosses zero, they do not)
    slope = 0.0 if act in ("none", "relu") else 12 * EPS32
    sub = TINY[dt] * 4
    a, one = dY.double().cpu().abs(), torch.ones(rows, 1, dtype=torch.float64)
    for g, i, j in [((), 0, rows)] if sizes is None else segments(rows, sizes):
        sX[i:j] = sX[i:j] * rounded + slope * a[i:j] @ w[g].abs()
        sW[g] = sW[g] * rounded + slope * a[i:j].T @ x[i:j].abs()
        sb[g] = (rows + 40) * EPS32 * sb[g] + slope * (a[i:j].T @ one[i:j])[:, 0]
    close(gx, dX, zX, n_out, dt, sX + sub * n_out)
    close(gw, dW, zW, rows, dt, sW + sub * rows)
    if bias:
        close(gb, db, sb * 0, 0, dt, sb)


SHAPES = [(1, 1, 1), (1, 64, 16), (2, 200, 65), (16, 512, 256), (17, 63, 129), (127, 65, 127), (128, 128, 128), (129, 136, 200), (300, 1003, 77)]


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_sizes(shape, dt):
    check_forward(*shape, dt, act="gelu", bias=True, residual=True, seed=sum(shape))


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("shape", SHAPES)
def test_backward_sizes(shape, dt):
    check_backward(*shape, dt, act="silu", seed=sum(shape))


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("act", list(ACTS))
def test_activations(act, dt):
    check_forward(130, 96, 72, dt, act=act, bias=True)
    check_backward(130, 96, 72, dt, act=act)


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("rows", [16, 200])
def test_left_tail_of_activations(rows, act, dt):
    """z s(w) and its slope, s the logistic function and w = z or sqrt(8 / pi) (z + 0.044715 z^3), by their own size at z from -8 to -3: w is
    off by 9 units of 2^-24 with the exponential's argument, s and what is made of it by a few more."""
    z = torch.linspace(-8, -3, rows).to(DTYPES[dt])
    one = torch.ones(24, 1, dtype=DTYPES[dt], device="cuda")
    X = z[:, None].cuda()
    Y = torch.zeros(rows, 24, dtype=DTYPES[dt], device="cuda")
    d.op_linear(X, one, Y, act=act)
    z64 = z.double().requires_grad_(True)
    w = z64 if act == "silu" else (8 / np.pi) ** 0.5 * (z64 + 0.044715 * z64**3)
    want = z64 * torch.sigmoid(w)  # (1 + tanh in 64 bits has nothing left at -8 either)
    want.sum().backward()
    w = w.detach()
    near = (9 * w.abs() + 30) * EPS32
    s = torch.sigmoid(w)
    for got in Y.double().cpu().T:
        assert ((got - want.detach()).abs() <= want.detach().abs() * (near + 1.01 * HALF[dt]) + TINY[dt]).all()
    dX = torch.zeros_like(X)
    d.op_linear_backward(torch.ones(rows, 1, dtype=DTYPES[dt], device="cuda"), X, one[:1], pre=X, act=act, dX=dX)
    terms = s + (z64.grad - s).abs()  # (the slope is the difference of two such)
    off = (dX[:, 0].double().cpu() - z64.grad).abs()
    assert (off <= terms * near + z64.grad.abs() * 2.1 * HALF[dt] + 2 * TINY[dt]).all()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_slopes_far_out(dt):
    z = torch.tensor([-3e38, -1e25, -1e19, 1e13, 1e25, 3e38]).to(DTYPES[dt]).cuda()[:, None]
    one = torch.ones(1, 1, dtype=DTYPES[dt], device="cuda")
    for act in ("silu", "gelu", "gelu_tanh"):
        dX = torch.zeros_like(z)
        d.op_linear_backward(torch.ones_like(z), z, one, pre=z, act=act, dX=dX)
        assert dX[:, 0].tolist() == [0, 0, 0, 1, 1, 1]


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("lay", [(8, 0), (8, 8), (1, 0), (3, 1), (4, 4)])
def test_strides_and_alignments(lay, dt):
    check_forward(140, 144, 136, dt, act="relu", bias=True, residual=True, lay=lay)
    check_backward(140, 144, 136, dt, act="gelu_tanh", lay=lay)


# enough tiles of 256 x 256 for the large kernel, rests in every direction; reductions that are split
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_large_tiles(dt):
    check_forward(3601, 200, 3848, dt, act="silu", bias=True)
    check_backward(3601, 3848, 200, dt, act="none", bias=False)
    check_backward(200, 3600, 3848, dt, act="gelu")


@pytest.mark.parametrize("dt", list(DTYPES))
def test_split_reductions(dt):
    check_forward(100, 5000, 96, dt, act="gelu", bias=True, residual=True)
    check_backward(2500, 90, 100, dt, act="relu")
    check_backward(64, 72, 4111, dt, act="none")


GROUPS = [[5, 0, 130, 1, 0, 0, 64], [0, 0, 3], [300], [0, 0], [1] * 70 + [0] * 9 + [200], [128, 256, 127, 129]]


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("sizes", GROUPS, ids=lambda s: f"{len(s)}_{sum(s)}")
@pytest.mark.parametrize("padding", [0, 7])
def test_groups(sizes, padding, dt):
    rows = sum(sizes) + padding
    check_forward(rows, 72, 136, dt, act="silu", bias=True, residual=True, sizes=sizes)
    check_backward(rows, 72, 136, dt, act="gelu", sizes=sizes)


def check_strided_groups(rows_of, n_in, n_out, dt, lay, beside=False):
    """Forward, backward and per-example gradients of groups whose arrays are wider than their rows, all of them."""
    sizes, n = rows_of, len(rows_of)
    rows = sum(sizes) + 4
    X, W = rand((rows, n_in), dt, 1), rand((n, n_out, n_in), dt, 2, n_in**-0.5)
    b, R, dY, pre = rand((n, n_out), dt, 3), rand((rows, n_out), dt, 4), rand((rows, n_out), dt, 5), rand((rows, n_out), dt, 6)
    put = lambda t: wide(t, *lay)  # noqa: E731
    weights = (lambda t: wide(t.transpose(0, 1), *lay).transpose(0, 1)) if beside else put
    dense = {}
    for name, f, w in (("dense", lambda t: t.clone(), lambda t: t.clone()), ("wide", put, weights)):
        y, z, gx, gw = f(torch.zeros_like(R)), f(torch.zeros_like(R)), f(torch.zeros_like(X)), w(torch.zeros_like(W))
        gb, out = torch.zeros_like(b), torch.zeros(n, n_out, n_in, device="cuda")
        d.op_linear(f(X), w(W), y, bias=b, act="silu", residual=f(R), pre=z, groups=ends_of(sizes))
        d.op_linear_backward(f(dY), f(X), w(W), pre=f(pre), act="gelu", dX=gx, dW=gw, dbias=gb, groups=ends_of(sizes))
        d.op_example_grads(f(dY), f(X), ends_of(sizes), out, square=True)
        dense[name] = (y, z, gx, gw, gb, out)
        if name == "wide":  # what lies between the rows is as it was
            for t in (y, z, gx, gw):
                gap = t.as_strided(t.shape[:-1] + (lay[0],), t.stride(), t.storage_offset() + t.shape[-1])
                assert (gap == 7).all()
    for a, b in zip(dense["dense"], dense["wide"]):
        assert torch.equal(a, b)  # the same sums in the same order


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("beside", [False, True])
@pytest.mark.parametrize("lay", [(8, 0), (8, 8), (1, 0), (3, 1)])
def test_groups_of_strided_arrays(lay, beside, dt):
    check_strided_groups([5, 0, 130, 1, 64], 72, 136, dt, lay, beside)
    check_strided_groups([3, 0, 5], 33, 65, dt, lay, beside)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_groups_on_large_tiles(dt):
    sizes = [700, 0, 256, 1300, 3, 1741]
    check_forward(sum(sizes) + 9, 136, 3000, dt, act="gelu_tanh", sizes=sizes)
    check_backward(sum(sizes) + 9, 3000, 136, dt, sizes=sizes, bias=False)
    check_backward(sum(sizes) + 9, 1000, 2000, dt, sizes=sizes, act="silu")


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("n_in,n_out", [(64, 128), (77, 33), (1, 1), (136, 264)])
@pytest.mark.parametrize("square", [False, True])
def test_example_grads(n_in, n_out, square, dt):
    sizes = [1, 0, 200, 33, 64, 65]
    rows = sum(sizes) + 2
    dY, X = rand((rows, n_out), dt, 1), rand((rows, n_in), dt, 2)
    out = torch.full((len(sizes), n_out, n_in), 9.0, device="cuda")
    d.op_example_grads(dY, X, ends_of(sizes), out, square=square)
    for e, i, j in segments(rows, sizes):
        a, b = dY[i:j].double().cpu(), X[i:j].double().cpu()
        want, sums = a.T @ b, a.T.abs() @ b.abs()
        if square:
            want, sums = want**2, 2 * want.abs() * sums + (j - i + 40) * EPS32 * 1.2 * sums**2
        close(out[e], want, sums, j - i, "f32")


@pytest.mark.parametrize("dt", list(DTYPES))
def test_gradient_against_differences(dt):
    """Of the formulas above in 64 bits: the slope that the gradients are held to is that of the forward pass."""
    rows, n_in, n_out = 6, 9, 7
    X, W, b, R = rand((rows, n_in), dt, 1), rand((n_out, n_in), dt, 2, 0.3), rand((n_out,), dt, 3), rand((rows, n_out), dt, 4)
    dY = rand((rows, n_out), dt, 5)
    for act in ("silu", "gelu", "gelu_tanh"):
        _, Z, _ = reference(X, W, b, act, R, None)
        pre = Z.to(DTYPES[dt]).cuda()
        gx = torch.zeros_like(X)
        d.op_linear_backward(dY, X, W, pre=pre, act=act, dX=gx)
        h, gX = 1e-5, torch.zeros(rows, n_in, dtype=torch.float64)
        for i in range(rows):
            for j in range(n_in):
                lo, hi = X.double().cpu().clone(), X.double().cpu().clone()
                lo[i, j] -= h
                hi[i, j] += h
                f = [(reference(t, W, b, act, R, None)[0] * dY.double().cpu()).sum() for t in (lo, hi)]
                gX[i, j] = (f[1] - f[0]) / (2 * h)
        size = dY.double().cpu().abs() @ W.double().cpu().abs()
        # pre is rounded (slopes change by at most 1.2 times that), dZ is, the result is; differences: h^2 and 1e-16 / h
        bound = size * (HALF[dt] * (1.2 * Z.abs().max() + 1.13) + 1e-5) + HALF[dt] * gX.abs() + 1e-8 + 32 * TINY[dt]
        assert ((gx.double().cpu() - gX).abs() <= bound).all()


def test_no_rows():
    X, W, Y = (torch.zeros(s, device="cuda") for s in ((0, 8), (4, 8), (0, 4)))
    d.op_linear(X, W, Y)
    dW, db = torch.ones(4, 8, device="cuda"), torch.ones(4, device="cuda")
    d.op_linear_backward(Y, X, W, dX=torch.zeros_like(X), dW=dW, dbias=db)
    assert not dW.any() and not db.any()
    out = torch.ones(2, 4, 8, device="cuda")
    d.op_example_grads(Y, X, ends_of([0, 0]), out)
    assert not out.any()


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("lay", [(8, 8), (3, 1)])
def test_strided_arrays_on_large_tiles_and_split_reductions(lay, dt):
    check_forward(3601, 200, 3848, dt, act="silu", bias=True, residual=True, lay=lay)
    check_backward(3601, 3848, 200, dt, act="silu", lay=lay)
    check_forward(100, 5000, 96, dt, act="gelu", bias=True, residual=True, lay=lay)
    check_backward(2500, 90, 100, dt, act="relu", lay=lay)


def test_fp32_groups_on_large_tiles():
    sizes = [700, 0, 256, 1300, 3, 1741]
    check_forward(sum(sizes) + 9, 136, 3000, "f32", act="gelu_tanh", sizes=sizes)
    check_backward(sum(sizes) + 9, 3000, 136, "f32", sizes=sizes, bias=False)
    check_backward(sum(sizes) + 9, 1000, 2000, "f32", sizes=sizes, act="silu")


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("rows, n_in, n_out, sizes", [(12, 40, 77, None), (12, 40, 77, [5, 0, 4]), (300, 64, 133, None), (300, 64, 133, [100, 0, 190]),
                                                      (100, 5000, 99, None), (3601, 200, 3843, None)])
def test_the_residual_may_be_the_result(rows, n_in, n_out, sizes, dt):
    X, W = rand((rows, n_in), dt, 1), rand((() if sizes is None else (len(sizes),)) + (n_out, n_in), dt, 2, n_in**-0.5)
    R, groups = rand((rows, n_out), dt, 3), None if sizes is None else ends_of(sizes)
    Y = torch.zeros_like(R)
    d.op_linear(X, W, Y, act="silu", residual=R, groups=groups)
    d.op_linear(X, W, R, act="silu", residual=R, groups=groups)
    assert torch.equal(Y, R)


def test_infinities_and_nan_stay_in_their_rows():
    X, W = rand((300, 64), "bf16", 1), rand((200, 64), "bf16", 2)
    Y, clean = torch.zeros(300, 200, dtype=torch.bfloat16, device="cuda"), torch.zeros(300, 200, dtype=torch.bfloat16, device="cuda")
    d.op_linear(X, W, clean, act="relu")
    X[5, 3], X[200, 0] = float("nan"), float("inf")
    d.op_linear(X, W, Y, act="relu")
    assert Y[5].isnan().all()
    rest = torch.ones(300, dtype=torch.bool)
    rest[[5, 200]] = False
    assert torch.equal(Y[rest], clean[rest])


def same_where_not_finite(got, want, bound):
    got, want = got.double().cpu(), want.double()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isposinf(), want.isposinf())
    assert torch.equal(got.isneginf(), want.isneginf())
    ok = torch.isfinite(want)
    assert ((got - want).abs()[ok] <= bound[ok]).all()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("rows, n_in, n_out", [(12, 40, 24), (50, 96, 200), (300, 64, 200), (100, 5000, 96)])
def test_infinities_and_large_numbers(rows, n_in, n_out, dt):
    """Infinities give infinities of the product's sign (NaN where they meet zeros or each other), and numbers up to the type's
    largest what they are worth, however many rows there are."""
    X, W = rand((rows, n_in), dt, 1), rand((n_out, n_in), dt, 2, 1e-3)
    inf, most = float("inf"), torch.finfo(DTYPES[dt]).max
    X[1, 3], X[2, 5], X[3, 7], X[3, 9], X[4, 11], X[5, 0], X[6, 1], X[7, 2] = inf, -inf, inf, inf, float("nan"), most, -most, most * 0.999
    X[8, 4] = inf
    W[5, 4], W[6, 6], W[7, 8] = 0.0, inf, -inf
    X[9, 6] = -inf
    x, w = X.double().cpu(), W.double().cpu()
    bound = (n_in + 40) * EPS32 * 1.2 * (x.abs() @ w.abs().T) + HALF[dt] * 1.01 * (x @ w.T).abs()
    Y = torch.zeros(rows, n_out, dtype=DTYPES[dt], device="cuda")
    d.op_linear(X, W, Y)
    same_where_not_finite(Y, x @ w.T, bound)
    # dX of such W, dW of such X, for dY with the same
    dY = rand((rows, n_out), dt, 3, 1e-3)
    dY[0, 3], dY[1, 2], dY[9, 1] = inf, -inf, 0.0
    g = dY.double().cpu()
    dX, dW = torch.zeros_like(X), torch.zeros_like(W)
    d.op_linear_backward(dY, X, W, dX=dX, dW=dW)
    for got, a, b in ((dX, g, w), (dW, g.T, x)):
        want = a @ b
        k = a.shape[1]
        same_where_not_finite(got, want, (k + 40) * EPS32 * 1.2 * (a.abs() @ b.abs()) + HALF[dt] * 1.01 * want.abs())


def test_falling_and_wild_ends_stay_inside():
    """No promise of values, but every access is inside the arrays: guards around the outputs keep theirs."""
    X, W = rand((64, 64), "bf16", 1), rand((4, 128, 64), "bf16", 2)
    for ends in ([0, 50, 20, 64, 10], [0, 1 << 40, -5, 3, 64], [7, 7, 7, 7, 7]):
        e = torch.tensor(ends, dtype=torch.int64, device="cuda")
        guard = torch.full((66, 128), 3.0, dtype=torch.bfloat16, device="cuda")
        dW = torch.full((6, 128, 64), 3.0, dtype=torch.bfloat16, device="cuda")
        db = torch.full((6, 128), 3.0, dtype=torch.bfloat16, device="cuda")
        d.op_linear(X, W, guard[1:65], groups=e)
        d.op_linear_backward(guard[1:65], X, W, dW=dW[1:5], dbias=db[1:5], groups=e)
        assert (guard[[0, 65]] == 3).all() and (dW[[0, 5]] == 3).all() and (db[[0, 5]] == 3).all()


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("rows", [5, 16])
def test_falling_and_wild_ends_of_few_rows_stay_inside(rows, dt):
    X, W = rand((rows, 64), dt, 1), rand((4, 40, 64), dt, 2)
    for ends in ([0, 5, 2, 16, 1], [0, 1 << 40, -5, 3, 64], [7, 7, 7, 7, 7], [0, 3, 3, 3, 4]):
        e = torch.tensor(ends, dtype=torch.int64, device="cuda")
        Y, pre = [torch.full((rows + 2, 40), 3.0, dtype=DTYPES[dt], device="cuda") for _ in range(2)]
        d.op_linear(X, W, Y[1:-1], pre=pre[1:-1], groups=e)
        assert (Y[[0, -1]] == 3).all() and (pre[[0, -1]] == 3).all()


def test_overlapping_groups_of_more_tiles_than_32_bits_count():
    """65534 groups whose ends go up to all rows and down again: 2.3e9 tiles of 128 rows by their counts.  As above, every access is
    inside the arrays."""
    rows, groups = 9_000_000, 65_534
    ends = torch.zeros(groups + 1, dtype=torch.int64)
    ends[1::2] = rows
    ends = ends.cuda()
    X = torch.ones(rows, 8, dtype=torch.bfloat16, device="cuda")
    W = torch.ones(groups, 8, 8, dtype=torch.bfloat16, device="cuda")
    Y, dX = [torch.full((rows + 2, 8), 3.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    db = torch.full((groups + 2, 8), 3.0, dtype=torch.bfloat16, device="cuda")
    d.op_linear(X, W, Y[1:-1], groups=ends)
    d.op_linear_backward(X, X, W, pre=X, act="relu", dX=dX[1:-1], dbias=db[1:-1], groups=ends)
    torch.cuda.synchronize()
    assert (Y[[0, -1]] == 3).all() and (dX[[0, -1]] == 3).all() and (db[[0, -1]] == 3).all()


def test_same_bits_again_and_on_another_stream():
    X, W = rand((500, 1000), "bf16", 1), rand((300, 1000), "bf16", 2)
    Y = [torch.zeros(500, 300, dtype=torch.bfloat16, device="cuda") for _ in range(3)]
    d.op_linear(X, W, Y[0], act="gelu")
    d.op_linear(X, W, Y[1], act="gelu")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        slow = torch.randn(2000, 2000, device="cuda")
        for _ in range(10):
            slow = slow @ slow * 1e-3
        X2 = X + slow[:500, :1000].to(X.dtype) * 0  # ready only after the work before it
        d.op_linear(X2, W, Y[2], act="gelu")
    side.synchronize()
    assert torch.equal(Y[0], Y[1]) and torch.equal(Y[0], Y[2])


def test_graph_capture_with_a_workspace_of_the_callers():
    X, W = rand((100, 4096), "bf16", 1), rand((64, 4096), "bf16", 2)
    Y = torch.zeros(100, 64, dtype=torch.bfloat16, device="cuda")
    ws = torch.empty(max(1, d.linear_workspace(100, 4096, 64, "torch.bfloat16")[0]), dtype=torch.uint8, device="cuda")
    d.op_linear(X, W, Y, workspace=ws)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        d.op_linear(X, W, Y, workspace=ws)
    for k in range(3):
        X.copy_(rand((100, 4096), "bf16", 10 + k))
        want = torch.zeros_like(Y)
        g.replay()
        torch.cuda.synchronize()
        d.op_linear(X, W, want, workspace=torch.empty_like(ws))
        torch.cuda.synchronize()
        assert torch.equal(Y, want)


def test_device_arrays():
    rng = np.random.default_rng(0)
    x, w = rng.standard_normal((33, 40), dtype=np.float32), rng.standard_normal((20, 40), dtype=np.float32)
    X, W, Y = d.DeviceArray.from_numpy(x), d.DeviceArray.from_numpy(w), d.DeviceArray((33, 20))
    d.op_linear(X, W, Y, act="relu")
    d.sync()
    want = np.maximum(x.astype(np.float64) @ w.T.astype(np.float64), 0)
    assert np.abs(Y.numpy() - want).max() <= 80 * EPS32 * (np.abs(x) @ np.abs(w).T).max()
    bits = d.DeviceArray.from_numpy((x.view(np.uint32) >> 16).astype(np.uint16), dtype=np.uint16)
    wb = d.DeviceArray.from_numpy((w.view(np.uint32) >> 16).astype(np.uint16), dtype=np.uint16)
    ends = d.DeviceArray.from_numpy(np.array([0, 10, 10, 33]), dtype=np.int64)
    out, dY = d.DeviceArray((3, 40, 40)), bits
    d.op_example_grads(dY, bits, ends, out)
    d.sync()
    xb = ((x.view(np.uint32) >> 16) << 16).view(np.float32).astype(np.float64)
    for e, (i, j) in enumerate(((0, 10), (10, 10), (10, 33))):
        assert np.abs(out.numpy()[e] - xb[i:j].T @ xb[i:j]).max() <= 1e-4
    del wb


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("rows, n_out", [(4200, 4203), (17_000, 1000), (1000, 17_001)])
def test_whole_rounds_of_large_tiles_and_a_rest(rows, n_out, dt):
    """A little more than 256 tiles of 256 x 256, in either direction, in products of all three layouts."""
    check_forward(rows, 200, n_out, dt, act="silu", bias=True, residual=True, seed=1)
    if dt != "f32":
        check_backward(rows, n_out, 200, dt, act="silu", seed=2)  # dX [rows, n_out]
        check_backward(200, rows, n_out, dt, seed=3)              # dW [n_out, rows]


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("rows, n_in, n_out", [(33, 129, 1001), (48, 70, 33), (64, 515, 2000), (65, 515, 300)])
def test_a_few_dozen_rows(rows, n_in, n_out, dt):
    check_forward(rows, n_in, n_out, dt, act="gelu_tanh", bias=True, residual=True, lay=(3, 1), seed=rows)


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("sizes", [[0, 70, 3, 33, 0, 129], [20, 0, 40, 1], [5, 16, 17, 15]])
def test_groups_of_a_few_dozen_rows(sizes, dt):
    check_forward(sum(sizes), 100, 130, dt, act="silu", bias=True, sizes=sizes, seed=4)


def test_offsets_past_32_bits():
    """70,000 rows that are 40,000 elements apart: more than 2^31 of them, and 5.6 GB, between the first and the last."""
    big = torch.empty(70_000 * 40_000, dtype=torch.bfloat16, device="cuda").view(70_000, 40_000)
    X, Y = big[:, 8:72], big[:, 128:192]
    X.copy_(torch.randn(70_000, 64, device="cuda"))
    W = rand((64, 64), "bf16", 2)
    d.op_linear(X, W, Y, act="relu")
    for rows in (slice(0, 300), slice(53_600, 53_800), slice(69_700, 70_000)):
        x = X[rows].double().cpu()
        close(Y[rows], (x @ W.double().cpu().T).clamp(min=0), x.abs() @ W.double().cpu().abs().T, 64, "bf16")
    dW, dX = torch.zeros_like(W), big[:, 256:320]
    ends = ends_of([69_000, 0, 1_000])
    d.op_linear_backward(Y, X, W, dW=dW, dX=dX)
    a, b = Y.double(), X.double()
    close(dW, a.T @ b, a.T.abs() @ b.abs(), 70_000, "bf16")
    close(dX[-500:], (a[-500:] @ W.double()), a[-500:].abs() @ W.double().abs(), 64, "bf16")
    out = torch.zeros(3, 64, 64, device="cuda")
    d.op_example_grads(Y, X, ends, out)
    close(out[2], a[-1000:].T @ b[-1000:], a[-1000:].T.abs() @ b[-1000:].abs(), 1000, "f32")
    assert not out[1].any()


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_the_widest_layer(dt):
    """2^24 columns, forward and backward; the last ones against the formulas."""
    rows, n_in, n_out = 3, 2, 1 << 24
    X, W = rand((rows, n_in), dt, 1), rand((n_out, n_in), dt, 2)
    dY, Y = rand((rows, n_out), dt, 3), torch.zeros(rows, n_out, dtype=DTYPES[dt], device="cuda")
    d.op_linear(X, W, Y, act="relu")
    dX, dW, db = torch.zeros_like(X), torch.zeros_like(W), torch.zeros(n_out, dtype=DTYPES[dt], device="cuda")
    d.op_linear_backward(dY, X, W, pre=Y, act="relu", dX=dX, dW=dW, dbias=db)
    dZ = dY.double() * (Y > 0)
    for at in (slice(0, 600), slice(8_388_500, 8_388_800), slice(n_out - 600, n_out)):
        w, g = W[at].double(), dZ[:, at]
        close(Y[:, at], (X.double() @ w.T).clamp(min=0), X.double().abs() @ w.abs().T, n_in, dt)
        close(dW[at], g.T @ X.double(), g.abs().T @ X.double().abs(), rows, dt)
        close(db[at], g.sum(0), g.abs().sum(0), rows, dt)
    close(dX, dZ @ W.double(), dZ.abs() @ W.double().abs(), n_out, dt)


def test_more_rows_to_copy_than_a_launch_dimension_holds():
    rows = (1 << 29) + 300
    X = torch.randn(rows, 1, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda", dtype=torch.float16)
    W, Y = rand((1, 1), "f16", 2), torch.full((rows, 1), 7.0, dtype=torch.float16, device="cuda")
    d.op_linear(X, W, Y)
    for i in range(0, rows, 1 << 27):  # (one product, rounded once)
        assert torch.equal(Y[i : i + (1 << 27)], (X[i : i + (1 << 27)].float() * W.float()).half())
    torch.cuda.empty_cache()


def test_column_sums_of_more_rows_than_a_launch_dimension_holds():
    rows = (1 << 30) + (1 << 16)
    dY = torch.ones(rows, 1, device="cuda")
    db = torch.zeros(1, device="cuda")
    room = torch.empty(1 << 27, dtype=torch.uint8, device="cuda")  # (all three gradients would take 768 GB)
    d.op_linear_backward(dY, dY, dY[:1], dbias=db, workspace=room)
    assert db.item() == rows
    torch.cuda.empty_cache()


def test_refusals():
    X, W, Y = torch.zeros(8, 16, device="cuda"), torch.zeros(4, 16, device="cuda"), torch.zeros(8, 4, device="cuda")

    def refused(*a, **k):
        with pytest.raises(d.DnpeffError):
            d.op_linear(*a, **k)

    refused(X, W.half(), Y)
    refused(X.double(), W.double(), Y.double())
    refused(X, W[:, :8], Y)
    refused(X, W, Y[:7])
    refused(X.T.contiguous().T, W, Y)
    refused(X[:1].expand(8, 16), W, Y)
    refused(X, W, Y, act="tanh")
    refused(X, W, Y, bias=torch.zeros(5, device="cuda"))
    refused(X, W, Y, residual=torch.zeros(8, 4))
    refused(X, W, Y, groups=ends_of([8]))
    refused(X, W[None], Y, groups=ends_of([4, 4]))
    refused(X, W[None], Y, groups=ends_of([8]).int())
    refused(X, d.DeviceArray((4, 16)), Y)
    with pytest.raises(d.DnpeffError):
        d.op_linear_backward(Y, X, W, act="silu", dX=torch.zeros_like(X))  # without pre
    big = torch.zeros(100, 5000, device="cuda"), torch.zeros(96, 5000, device="cuda"), torch.zeros(100, 96, device="cuda")
    with pytest.raises(d.DnpeffError, match="workspace"):
        d.op_linear(*big, workspace=torch.zeros(16, dtype=torch.uint8, device="cuda"))
    z = C.c_void_p(0)
    assert d.lib.dnpeff_linear(z, 9, 1, 1, 1, z, 1, z, 1, 1, z, 0, z, 0, z, 1, z, 0, 0, z, z, 0) != 0
    assert b"type" in d.lib.dnpeff_last_error()
    assert d.lib.dnpeff_linear(z, 0, 1, 1, 1, z, 1, z, 1, 1, z, 0, z, 0, z, 1, z, 0, 0, z, z, 0) != 0
    assert b"no X" in d.lib.dnpeff_last_error()
    assert d.lib.dnpeff_linear(z, 0, -1, 1, 1, z, 1, z, 1, 1, z, 0, z, 0, z, 1, z, 0, 0, z, z, 0) != 0
    torch.cuda.synchronize()
