"""Softmax cross entropy over a vocabulary and its gradients, against the formulas in 64 bits.

A logit is a sum of n_in products in fp32: off by (n_in + 8) 2^-24 times the sum of their sizes, s.  lse and the loss are off by at
most twice the worst of a row's logits, and by the rounding of the exponentials and their sum (n_words + 64 operations at
most).  g = (p - label) dloss: p is off by that much relatively, and g is rounded to the type; the products sum those
errors over words or tokens, and are rounded once more."""

import pytest
import torch

import npeff_ref_amd as d

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {k: torch.finfo(t).eps / 2 for k, t in DTYPES.items()}  # relative half unit in the last place
EPS32 = 2.0**-24


def rand(shape, dt, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(DTYPES[dt]).cuda()


def labels_of(rows, words, seed, masked=0.2):
    g = torch.Generator().manual_seed(seed)
    y = torch.randint(0, words, (rows,), generator=g, dtype=torch.int32)
    if rows > 1:
        y[torch.rand(rows, generator=g) < masked] = -1
    if rows:
        y[-1] = words - 1
    return y.cuda()


def padded(t, extra):
    v = torch.full((t.shape[0], t.shape[1] + extra), 5.0, dtype=t.dtype, device="cuda")[:, : t.shape[1]]
    v.copy_(t)
    return v


def check(rows, n_in, words, dt, extra=0, scale=3.0, weight=1.0, seed=0):
    X, E = rand((rows, n_in), dt, seed), rand((words, n_in), dt, seed + 1, scale * n_in**-0.5)
    y = labels_of(rows, words, seed + 2)
    g = torch.Generator().manual_seed(seed + 3)
    dl = (torch.randn(rows, generator=g) * weight).cuda()
    loss, lse = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
    x, e = padded(X, extra), padded(E, extra)
    d.op_vocab_loss(x, e, y, loss, lse)
    gx, ge = padded(torch.zeros_like(X), extra), padded(torch.zeros_like(E), extra)
    d.op_vocab_loss_backward(x, e, y, lse, dl, dX=gx, dE=ge)

    X64, E64, y64, dl64 = X.double().cpu(), E.double().cpu(), y.long().cpu(), dl.double().cpu()
    z = X64 @ E64.T
    logit = (n_in + 8) * EPS32 * (X64.abs() @ E64.abs().T).max(1).values + 4 * EPS32 * z.abs().max(1).values
    want = torch.logsumexp(z, 1)
    off = 2 * logit + (words + 64) * EPS32 + 2 * EPS32 * want.abs()
    assert ((lse.double().cpu() - want).abs() <= off).all()
    has = y64 >= 0
    at = y64.clamp(min=0)[:, None]
    want_loss = torch.where(has, want - z.gather(1, at)[:, 0], 0.0)
    assert ((loss.double().cpu() - want_loss).abs() <= torch.where(has, 2 * off, 0.0)).all()

    p = torch.softmax(z, 1)
    G = p.clone()
    G.scatter_add_(1, at, torch.full((rows, 1), -1.0, dtype=torch.float64))
    weight64 = torch.where(has, dl64, 0.0)[:, None]
    # p's own error, the rounding of g (in fp16 subnormal next to the largest weight), the hardware's exponential
    relative = (2 * off + 32 * EPS32 + 4 * z.abs().max(1).values * EPS32)[:, None]
    err = (p * relative + G.abs() * HALF[dt] * 1.01 + 2 * EPS32) * weight64.abs()
    if dt == "f16":
        err = err + 2.0**-25 * 2 * weight64.abs().max() * has[:, None]
    G = G * weight64
    for got, exact, size, e_sum, k in (
        (gx, G @ E64, G.abs() @ E64.abs(), err @ E64.abs(), words),
        (ge, G.T @ X64, G.abs().T @ X64.abs(), err.T @ X64.abs(), rows),
    ):
        bound = e_sum + (k + 16) * EPS32 * size + HALF[dt] * 1.01 * exact.abs() + (2.0**-25 if dt == "f16" else 0)
        d_ = (got.double().cpu() - exact).abs() - bound
        assert torch.isfinite(got).all() and (d_ <= 0).all(), f"worst {d_.max().item():g} past its bound"


SHAPES = [(1, 1, 1), (1, 64, 1000), (2, 100, 257), (16, 256, 5000), (17, 63, 300), (130, 65, 1001), (128, 128, 128), (300, 200, 2048), (40, 1003, 777)]


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("shape", SHAPES)
def test_sizes(shape, dt):
    check(*shape, dt, seed=sum(shape))


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("extra", [1, 8])
def test_strides(extra, dt):
    check(90, 136, 700, dt, extra=extra)


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("rows, n_in, words, extra", [(1, 4, 700, 0), (3, 257, 9001, 1), (4, 1030, 513, 3), (5, 3, 300, 0), (9, 515, 20_000, 8),
                                                      (16, 1003, 65, 5), (16, 5, 7, 0), (33, 130, 3000, 1), (64, 72, 1000, 0),
                                                      (128, 100, 20_000, 0), (250, 66, 901, 1)])
def test_few_tokens(rows, n_in, words, extra, dt):
    check(rows, n_in, words, dt, extra=extra, seed=rows)


@pytest.mark.parametrize("rows", [0, 3, 40])
def test_one_gradient_alone(rows):
    X, E = rand((rows, 100), "bf16", 1), rand((900, 100), "bf16", 2, 0.3)
    y = labels_of(rows, 900, 3)
    loss, lse, dl = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
    d.op_vocab_loss(X, E, y, loss, lse)
    both, alone = [[torch.full_like(t, 3.0) for t in (X, E)] for _ in range(2)]
    d.op_vocab_loss_backward(X, E, y, lse, dl, dX=both[0], dE=both[1])
    d.op_vocab_loss_backward(X, E, y, lse, dl, dX=alone[0])
    d.op_vocab_loss_backward(X, E, y, lse, dl, dE=alone[1])
    assert torch.equal(both[0], alone[0]) and torch.equal(both[1], alone[1])
    if rows == 0:
        assert not both[1].any()


@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_large_tiles(dt):
    check(1500, 72, 9001, dt)


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("extra", [1, 8])
def test_strided_arrays_on_large_tiles(extra, dt):
    check(1500, 72, 9001, dt, extra=extra)


@pytest.mark.parametrize("rows, n_in, words", [(4200, 200, 4203), (1000, 264, 17_001), (300, 1024, 17_000)])
@pytest.mark.parametrize("dt", list(DTYPES))
def test_whole_rounds_of_large_tiles_and_a_rest(rows, n_in, words, dt):
    check(rows, n_in, words, dt)


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("weight", [1e-7, 1e4])
def test_weights_of_any_size(weight, dt):
    if dt == "f16" and weight < 1:
        # the gradients themselves would be subnormal: what is asked is that they are as good as that
        check(64, 64, 300, dt, weight=weight)
    else:
        check(64, 64, 300, dt, weight=weight if dt != "f16" else 100.0)


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("rows", [3, 64])
@pytest.mark.parametrize("weights", [(1e-36,), (1e-36, 0.0), (4e-35, 0.0, -1e-38), (1e-42, 0.0)])
def test_weights_next_to_nothing(weights, rows, dt):
    """Gradients are at most a weight times the sum of 2 for each row and the size of X or E: zero in fp16, and never more than that."""
    X, E, y = rand((rows, 40), dt, 1), rand((300, 40), dt, 2, 0.3), labels_of(rows, 300, 3, masked=0.0)
    dl = torch.tensor([weights[i % len(weights)] for i in range(rows)]).cuda()
    loss, lse = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
    d.op_vocab_loss(X, E, y, loss, lse)
    gx, ge = torch.ones_like(X), torch.ones_like(E)
    d.op_vocab_loss_backward(X, E, y, lse, dl, dX=gx, dE=ge)
    most = 2 * dl.abs().max().item() * 1.01
    assert gx.abs().max().item() <= most * E.abs().max().item() and ge.abs().max().item() <= most * rows * X.abs().max().item()
    if dt == "f16":
        assert not gx.any() and not ge.any()
    elif max(weights) > 1e-36:
        assert gx.any() and ge.any()


@pytest.mark.parametrize("dt", list(DTYPES))
def test_large_logits(dt):
    check(64, 64, 500, dt, scale=20.0)


def test_pieces_of_the_vocabulary_give_the_whole():
    """More words than one piece holds: the same gradients as from the vocabulary's parts, put together by hand."""
    rows, n_in, words = 4096, 64, 70_000
    X, E = rand((rows, n_in), "bf16", 1), rand((words, n_in), "bf16", 2, 0.3)
    y = labels_of(rows, words, 3)
    loss, lse, dl = (torch.ones(rows, device="cuda") for _ in range(3))
    d.op_vocab_loss(X, E, y, loss, lse)
    gx, ge = torch.zeros_like(X), torch.zeros_like(E)
    d.op_vocab_loss_backward(X, E, y, lse, dl, dX=gx, dE=ge)
    z = X.double() @ E.double().T
    want = torch.logsumexp(z, 1)
    assert (lse - want).abs().max() < 1e-4
    G = torch.exp(z - want[:, None])
    has = (y >= 0).double()[:, None]
    G.scatter_add_(1, y.long().clamp(min=0)[:, None], -torch.ones(rows, 1, dtype=torch.float64, device="cuda"))
    G *= has
    for got, exact in ((gx, G @ E.double()), (ge, G.T @ X.double())):
        assert (got.double() - exact).norm() <= 2 * HALF["bf16"] * exact.norm()
        err = (got.double() - exact).abs()
        assert (err.norm(dim=1) <= 3 * HALF["bf16"] * exact.norm(dim=1) + 1e-6).all()


def gradient_bounds(z, has, dl, dt, n_in, words, size):
    """(p, the rows' weights, p's relative error) from 64-bit logits, as in check(); size: of the products in a row's largest logit."""
    logit = (n_in + 8) * EPS32 * size + 4 * EPS32 * z.abs().max(1).values
    lse = torch.logsumexp(z, 1)
    off = 2 * logit + (words + 64) * EPS32 + 2 * EPS32 * lse.abs()
    p = torch.softmax(z, 1)
    weight = torch.where(has, dl.double(), 0.0)[:, None]
    relative = (2 * off + 32 * EPS32 + 4 * z.abs().max(1).values * EPS32)[:, None]
    return p, weight, relative


@pytest.mark.parametrize("dt", ["f32", "f16"])
@pytest.mark.parametrize("n_in, extra", [(65, 0), (200, 8), (72, 1)])
def test_pieces_of_the_vocabulary_in_other_types_and_widths(n_in, extra, dt):
    """As above, every entry by its own bound: two pieces in fp16, four in fp32."""
    rows, words = 4096, 70_000
    X, E, y = rand((rows, n_in), dt, 1), rand((words, n_in), dt, 2, 2 * n_in**-0.5), labels_of(rows, words, 3)
    dl = torch.randn(rows, generator=torch.Generator().manual_seed(4)).cuda()
    x, e = padded(X, extra), padded(E, extra)
    loss, lse = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
    d.op_vocab_loss(x, e, y, loss, lse)
    gx, ge = padded(torch.zeros_like(X), extra), padded(torch.zeros_like(E), extra)
    d.op_vocab_loss_backward(x, e, y, lse, dl, dX=gx, dE=ge)
    X64, E64, has = X.double(), E.double(), y >= 0
    size = (X64.abs() @ E64.abs().T).max(1).values
    p, weight, relative = gradient_bounds(X64 @ E64.T, has, dl, dt, n_in, words, size)
    G = p.clone()
    G.scatter_add_(1, y.long().clamp(min=0)[:, None], torch.full((rows, 1), -1.0, dtype=torch.float64, device="cuda"))
    err = (p * relative + G.abs() * HALF[dt] * 1.01 + 2 * EPS32) * weight.abs()
    del p
    if dt == "f16":
        err += 2.0**-25 * 2 * weight.abs().max() * has[:, None]
    G *= weight
    for got, exact, all_of, e_sum, k in (
        (gx, G @ E64, G.abs() @ E64.abs(), err @ E64.abs(), words),
        (ge, G.T @ X64, G.abs().T @ X64.abs(), err.T @ X64.abs(), rows),
    ):
        bound = e_sum + (k + 16) * EPS32 * all_of + HALF[dt] * 1.01 * exact.abs() + (2.0**-25 if dt == "f16" else 0)
        assert torch.isfinite(got).all() and ((got.double() - exact).abs() <= bound).all()


@pytest.mark.parametrize("rows", [3, 40])
def test_gradients_of_a_vocabulary_past_32_bits(rows):
    """600,000 words of 4096 and the gradients of all: rows of dE from both ends, and dX, which takes all of E."""
    words, n_in = 600_000, 4096
    g = torch.Generator(device="cuda").manual_seed(1)
    E = torch.empty(words, n_in, dtype=torch.bfloat16, device="cuda")
    for i in range(0, words, 100_000):
        E[i : i + 100_000] = torch.randn(100_000, n_in, generator=g, device="cuda") * 0.03
    X, dl = rand((rows, n_in), "bf16", 2), torch.ones(rows, device="cuda")
    y = torch.randint(0, words, (rows,), generator=torch.Generator().manual_seed(3), dtype=torch.int32).cuda()
    y[0], y[1] = words - 1, 5
    loss, lse = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
    d.op_vocab_loss(X, E, y, loss, lse)
    dX, dE = torch.zeros_like(X), torch.full_like(E, 9.0)
    d.op_vocab_loss_backward(X, E, y, lse, dl, dX=dX, dE=dE)
    X64, parts = X.double(), [slice(i, i + 100_000) for i in range(0, words, 100_000)]
    z = torch.cat([X64 @ E[at].double().T for at in parts], 1)
    size = X64.abs().sum(1) * E.abs().max().double()
    p, _, relative = gradient_bounds(z, y >= 0, dl, "bf16", n_in, words, size)
    G = p.clone()
    G.scatter_add_(1, y.long()[:, None], torch.full((rows, 1), -1.0, dtype=torch.float64, device="cuda"))
    err = p * relative + G.abs() * HALF["bf16"] * 1.01 + 2 * EPS32
    for at in (slice(0, 2000), slice(524_200, 524_400), slice(words - 2000, words)):  # (524,288 x 4096 is 2^31)
        exact, all_of = G[:, at].T @ X64, G[:, at].abs().T @ X64.abs()
        bound = err[:, at].T @ X64.abs() + (rows + 16) * EPS32 * all_of + HALF["bf16"] * 1.01 * exact.abs()
        assert ((dE[at].double() - exact).abs() <= bound).all()
    exact, bound = torch.zeros_like(X64), torch.zeros_like(X64)
    for at in parts:
        e64 = E[at].double()
        exact += G[:, at] @ e64
        bound += err[:, at] @ e64.abs() + (words + 16) * EPS32 * (G[:, at].abs() @ e64.abs())
    assert ((dX.double() - exact).abs() <= bound + HALF["bf16"] * 1.01 * exact.abs()).all()
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows", [3, 40])
def test_a_vocabulary_past_32_bits(rows):
    """600,000 words of 4096: 4.9 GB, its last words past 2^31 elements."""
    g = torch.Generator(device="cuda").manual_seed(1)
    E = torch.empty(600_000, 4096, dtype=torch.bfloat16, device="cuda")
    for i in range(0, 600_000, 100_000):
        E[i : i + 100_000] = torch.randn(100_000, 4096, generator=g, device="cuda") * 0.03
    X = rand((rows, 4096), "bf16", 2)
    y = torch.randint(560_000, 600_000, (rows,), generator=torch.Generator().manual_seed(3), dtype=torch.int32).cuda()
    loss, lse = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
    d.op_vocab_loss(X, E, y, loss, lse)
    z = torch.cat([X.double() @ E[i : i + 100_000].double().T for i in range(0, 600_000, 100_000)], 1)
    want = torch.logsumexp(z, 1)
    size = 4104 * EPS32 * (X.abs().double().sum(1) * E.abs().max().double())
    assert ((lse - want).abs() <= 2 * size + 600_064 * EPS32).all()
    assert ((loss - (want - z.gather(1, y.long()[:, None])[:, 0])).abs() <= 4 * size + 600_064 * EPS32).all()


def test_more_tokens_than_a_launch_has_waves():
    rows = (1 << 26) + 70
    g = torch.Generator(device="cuda").manual_seed(1)
    X = torch.randn(rows, 8, generator=g, device="cuda", dtype=torch.bfloat16)
    E = rand((16, 8), "bf16", 2)
    y = (torch.arange(rows, dtype=torch.int32, device="cuda") % 17) - 1
    loss, lse = torch.full((rows,), 9.0, device="cuda"), torch.full((rows,), 9.0, device="cuda")
    d.op_vocab_loss(X, E, y, loss, lse)
    for at in (slice(0, 500), slice(1 << 24, (1 << 24) + 500), slice(rows - 500, rows)):
        z = X[at].double() @ E.double().T
        want = torch.logsumexp(z, 1)
        size = (16 * EPS32 * (X[at].double().abs() @ E.double().abs().T)).max(1).values + 80 * EPS32 + 2 * EPS32 * want.abs()
        assert ((lse[at] - want).abs() <= 2 * size).all()
        has = y[at] >= 0
        hit = z.gather(1, y[at].long().clamp(min=0)[:, None])[:, 0]
        assert ((loss[at] - torch.where(has, want - hit, 0.0)).abs() <= torch.where(has, 4 * size, 0.0)).all()


def test_more_tiles_than_a_launch_dimension_holds():
    """2 million tokens and 262,400 words: 8.4 million tiles of 256 x 256, of 512 lanes each."""
    rows, words = 1 << 21, (1 << 18) + 256
    X, E = rand((rows, 8), "bf16", 1), rand((words, 8), "bf16", 2)
    y = torch.randint(0, words, (rows,), generator=torch.Generator().manual_seed(3), dtype=torch.int32).cuda()
    loss, lse = torch.full((rows,), 9.0, device="cuda"), torch.full((rows,), 9.0, device="cuda")
    d.op_vocab_loss(X, E, y, loss, lse)
    for at in (slice(0, 150), slice(rows // 3, rows // 3 + 150), slice(rows - 150, rows)):
        z = X[at].double() @ E.double().T
        want = torch.logsumexp(z, 1)
        size = (16 * EPS32 * (X[at].double().abs() @ E.double().abs().T)).max(1).values
        off = 2 * size + (words + 64) * EPS32 + 2 * EPS32 * want.abs()
        assert ((lse[at] - want).abs() <= off).all()
        assert ((loss[at] - (want - z.gather(1, y[at].long()[:, None])[:, 0])).abs() <= 2 * off).all()
    torch.cuda.empty_cache()


def test_all_masked_and_labels_outside():
    X, E = rand((70, 64), "bf16", 1), rand((900, 64), "bf16", 2)
    y = torch.full((70,), -1, dtype=torch.int32, device="cuda")
    loss, lse, dl = (torch.ones(70, device="cuda") for _ in range(3))
    gx, ge = torch.ones_like(X), torch.ones_like(E)
    d.op_vocab_loss(X, E, y, loss, lse)
    assert not loss.any() and torch.isfinite(lse).all()
    d.op_vocab_loss_backward(X, E, y, lse, dl, dX=gx, dE=ge)
    assert not gx.any() and not ge.any()
    y[3], y[4] = 900, 5
    d.op_vocab_loss(X, E, y, loss, lse)
    assert loss[3].isnan() and torch.isfinite(loss[4]) and loss[4] > 0
    d.op_vocab_loss_backward(X, E, y, lse, dl, dX=gx, dE=ge)
    assert gx[3].isnan().all() and torch.isfinite(gx[4]).all() and not gx[5:].any()


def test_masked_rows_may_hold_anything():
    """A row without a label does not reach the gradients, whatever its state holds."""
    X, E = rand((70, 64), "bf16", 1), rand((900, 64), "bf16", 2)
    y = labels_of(70, 900, 3)
    y[10] = -1
    out = []
    for bad in (0.0, float("inf"), float("nan")):
        X[10] = 0
        X[10, 0] = bad
        loss, lse, dl = (torch.ones(70, device="cuda") for _ in range(3))
        gx, ge = torch.ones_like(X), torch.ones_like(E)
        d.op_vocab_loss(X, E, y, loss, lse)
        d.op_vocab_loss_backward(X, E, y, lse, dl, dX=gx, dE=None)
        assert loss[10] == 0 and not gx[10].any()
        out.append((loss.clone(), gx))
    assert all(torch.equal(a, b) for a, b in zip(out[0], out[1])) and all(torch.equal(a, b) for a, b in zip(out[0], out[2]))


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("rows, extra", [(3, 0), (8, 1), (12, 0), (70, 0), (70, 1), (300, 8)])
def test_masked_rows_do_not_reach_the_embeddings(rows, extra, dt):
    """The same bits in all gradients whatever the state of a row without a label holds: infinities and NaN too."""
    X, E = rand((rows, 72), dt, 1), rand((900, 72), dt, 2, 0.3)
    y = labels_of(rows, 900, 3)
    y[1], y[2] = -1, 17
    dl, out = torch.ones(rows, device="cuda"), []
    for bad in (0.0, float("inf"), float("nan")):
        X[1] = 0
        X[1, ::5] = bad
        x, e = padded(X, extra), padded(E, extra)
        loss, lse = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
        d.op_vocab_loss(x, e, y, loss, lse)
        gx, ge, alone = torch.ones_like(X), torch.ones_like(E), torch.ones_like(E)
        d.op_vocab_loss_backward(x, e, y, lse, dl, dX=gx, dE=ge)
        d.op_vocab_loss_backward(x, e, y, lse, dl, dE=alone)
        assert torch.isfinite(ge).all() and not gx[1].any() and loss[1] == 0
        assert torch.equal(ge, alone)
        out.append((loss, gx, ge))
    for other in out[1:]:
        assert all(torch.equal(a, b) for a, b in zip(out[0], other))


def test_gradient_against_differences():
    rows, n_in, words = 5, 7, 11
    X, E, y = rand((rows, n_in), "f32", 1), rand((words, n_in), "f32", 2), labels_of(rows, words, 3)
    loss, lse, dl = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda"), rand((rows,), "f32", 4)
    d.op_vocab_loss(X, E, y, loss, lse)
    gx, ge = torch.zeros_like(X), torch.zeros_like(E)
    d.op_vocab_loss_backward(X, E, y, lse, dl, dX=gx, dE=ge)

    def total(x, e):
        return (torch.nn.functional.cross_entropy(x @ e.T, y.long().cpu(), ignore_index=-1, reduction="none") * dl.double().cpu()).sum()

    x64, e64, h = X.double().cpu(), E.double().cpu(), 1e-6
    for t, got in ((x64, gx), (e64, ge)):
        for i in range(t.shape[0]):
            for j in range(t.shape[1]):
                keep = t[i, j].item()
                t[i, j] = keep + h
                hi = total(x64, e64)
                t[i, j] = keep - h
                lo = total(x64, e64)
                t[i, j] = keep
                assert abs((hi - lo) / (2 * h) - got[i, j].item()) < 1e-5


def test_one_gradient_alone_and_no_rows():
    X, E, y = rand((40, 64), "bf16", 1), rand((300, 64), "bf16", 2), labels_of(40, 300, 3)
    loss, lse, dl = (torch.ones(40, device="cuda") for _ in range(3))
    d.op_vocab_loss(X, E, y, loss, lse)
    both = torch.zeros_like(X), torch.zeros_like(E)
    d.op_vocab_loss_backward(X, E, y, lse, dl, dX=both[0], dE=both[1])
    one = torch.zeros_like(X), torch.zeros_like(E)
    d.op_vocab_loss_backward(X, E, y, lse, dl, dX=one[0])
    d.op_vocab_loss_backward(X, E, y, lse, dl, dE=one[1])
    assert torch.equal(both[0], one[0]) and torch.equal(both[1], one[1])
    none = X[:0]
    d.op_vocab_loss(none, E, y[:0], loss[:0], lse[:0])
    dE = torch.ones_like(E)
    d.op_vocab_loss_backward(none, E, y[:0], lse[:0], dl[:0], dE=dE)
    assert not dE.any()


def test_graph_replays():
    X, E, y = rand((64, 128), "f16", 1), rand((3000, 128), "f16", 2, 0.2), labels_of(64, 3000, 3)
    loss, lse, dl = (torch.ones(64, device="cuda") for _ in range(3))
    gx, ge = torch.zeros_like(X), torch.zeros_like(E)
    ws = torch.empty(max(d.vocab_loss_workspace(64, 128, 3000, "torch.float16")), dtype=torch.uint8, device="cuda")

    def step():
        d.op_vocab_loss(X, E, y, loss, lse, workspace=ws)
        d.op_vocab_loss_backward(X, E, y, lse, dl, dX=gx, dE=ge, workspace=ws)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for k in range(3):
        X.copy_(rand((64, 128), "f16", 10 + k))
        dl.fill_(0.01 * (k + 1))
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (loss, lse, gx, ge)]
        ws.fill_(255)
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (loss, lse, gx, ge)))


def test_refusals():
    X, E = torch.zeros(8, 16, device="cuda"), torch.zeros(40, 16, device="cuda")
    y, f = torch.zeros(8, dtype=torch.int32, device="cuda"), torch.zeros(8, device="cuda")

    def refused(*a, **k):
        with pytest.raises(d.DnpeffError):
            d.op_vocab_loss(*a, **k)

    refused(X, E.half(), y, f, f)
    refused(X, E[:, :8], y, f, f)
    refused(X, E, y.long(), f, f)
    refused(X, E, y[:7], f, f)
    refused(X, E, y, f.half(), f)
    refused(X, E.cpu(), y, f, f)
    refused(X, E, None, f, f)
    refused(X, E, y, f, f, workspace=torch.zeros(8, dtype=torch.uint8, device="cuda"))
    with pytest.raises(d.DnpeffError):
        d.op_vocab_loss_backward(X, E, y, f, None, dX=torch.zeros_like(X))
