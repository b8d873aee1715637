"""What a model answers (log probabilities of given words, entropy, the likeliest words) and distillation from a teacher's listed
words, with their gradients, against the formulas in 64 bits.

A logit is a sum of n_in products in fp32: off by (n_in + 8) 2^-24 times the sum of their sizes, and by its own rounding; lse by twice the
worst of a row's logits and the rounding of the exponentials and their sum (n_words + 64 operations).  A given word's logit is summed
in fp32 too: of the two logit errors in lse's bound one is its own, and logp is rounded.  The entropy log s + sum p (max - z): logits off by d move it by at most
2 H d, exponentials off relatively by r by at most r (1 + log s + sum p (max - z)).  The order of the alternatives is that of 64 bits.
dz = p (a + b log p) + listed: p is off relatively as exp(z - lse) is, a as the entropy; dz is rounded to the type, the products
sum these errors over words or tokens, and are rounded once more."""

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


def words_of(rows, many, words, seed, masked=0.2):
    """Given words, the same ones twice among them; some places and some whole rows without any."""
    g = torch.Generator().manual_seed(seed)
    w = torch.randint(0, words, (rows, many), generator=g, dtype=torch.int32)
    if many > 2:
        w[:, 2] = w[:, 0]
    w[torch.rand((rows, many), generator=g) < masked] = -1
    if rows > 1:
        w[torch.rand(rows, generator=g) < masked] = -1
    if rows and many:
        w[-1, -1] = words - 1
    return w.cuda()


def padded(t, extra):
    v = torch.full((t.shape[0], t.shape[1] + extra), 5.0, dtype=t.dtype, device="cuda")[:, : t.shape[1]]
    v.copy_(t)
    return v


def empty(*shape, dtype=torch.float32):
    return torch.full(shape, 77, device="cuda", dtype=dtype)


class Exact:
    """The row statistics in 64 bits, and how far fp32 may be off."""

    def __init__(self, X, E, heat):
        self.X, self.E, self.heat = X.double(), E.double(), heat
        words, n_in = E.shape
        self.z = z = self.X @ self.E.T / heat
        self.lse = torch.logsumexp(z, 1)
        self.log_p = z - self.lse[:, None]
        self.p = self.log_p.exp()
        self.entropy = torch.special.entr(self.p).sum(1)
        most = z.abs().max(1).values
        size = (self.X.abs() @ self.E.abs().T).max(1).values / heat
        self.logit = (n_in + 8) * EPS32 * size + 6 * EPS32 * most
        self.off = 2 * self.logit + (words + 64) * EPS32 + 2 * EPS32 * self.lse.abs()
        top = z.max(1).values
        spread = z.max(1).values - z.min(1).values
        below = (self.p * (top[:, None] - z)).sum(1)
        self.off_entropy = 2 * self.entropy * self.logit + ((words + 128 + 4 * spread) * EPS32 + 2 * self.logit) * (1 + self.lse - top + below)
        # of p, relatively
        self.relative = (2 * self.off + 32 * EPS32 + 4 * most * EPS32)[:, None]

    def logp(self, words):
        return torch.where(words >= 0, self.log_p.gather(1, words.long().clamp(min=0)), 0.0)

    def logp_off(self, words):
        return torch.where(words >= 0, self.off[:, None] + 4 * EPS32 * (self.logp(words).abs() + self.lse.abs()[:, None]), 0.0)


def near(got, want, off, what):
    worst = ((got.double() - want).abs() - off).max().item() if got.numel() else 0
    assert torch.isfinite(got).all() and worst <= 0, f"{what}: {worst:g} past its bound"


def check_tops(x, top_words, top_logp, n):
    v, at = x.z.sort(dim=1, descending=True, stable=True)
    assert torch.equal(top_words, at[:, :n].to(torch.int32))
    near(top_logp, v[:, :n] - x.lse[:, None], x.off[:, None] + 4 * EPS32 * (v[:, :n].abs() + x.lse.abs()[:, None]), "top_logp")


def check_grads(x, dt, dX, dE, G, err, size, alive):
    """dX = G E and dE = G^T X; err: of G's elements before its rounding, size: the largest a row's can be."""
    rows, words = G.shape
    err = err + G.abs() * HALF[dt] * 1.01
    if dt == "f16" and rows:
        err = err + 2.0**-25 * 2 * size.max() * alive[:, None]
    for got, exact, all_of, e_sum, k in (
        (dX, G @ x.E, G.abs() @ x.E.abs(), err @ x.E.abs(), words),
        (dE, G.T @ x.X, G.abs().T @ x.X.abs(), err.T @ x.X.abs(), rows),
    ):
        near(got, exact, e_sum + (k + 16) * EPS32 * all_of + HALF[dt] * 1.01 * exact.abs() + (2.0**-25 if dt == "f16" else 0), "gradient")


def check_probs(rows, n_in, words, dt, given=3, top=4, heat=1.0, extra=0, scale=3.0, seed=0, train=True):
    X, E = rand((rows, n_in), dt, seed), rand((words, n_in), dt, seed + 1, scale * n_in**-0.5)
    w = words_of(rows, given, words, seed + 2)
    logp, lse, entropy = empty(rows, given), empty(rows), empty(rows)
    tops = dict(top_words=empty(rows, top, dtype=torch.int32), top_logp=empty(rows, top)) if top else {}
    xs, es = padded(X, extra), padded(E, extra)
    d.op_vocab_probs(xs, es, w, logp=logp, lse=lse, entropy=entropy, temperature=heat, **tops)
    x = Exact(X, E, heat)
    near(lse, x.lse, x.off, "lse")
    near(logp, x.logp(w), x.logp_off(w), "logp")
    near(entropy, x.entropy, x.off_entropy, "entropy")
    if top:
        check_tops(x, tops["top_words"], tops["top_logp"], top)
    if not train:
        return
    dlogp, dh = rand((rows, given), "f32", seed + 3), rand((rows,), "f32", seed + 4, 0.3)
    dlogp[::3], dh[::2] = 0, 0
    dX, dE = padded(torch.zeros_like(X), extra), padded(torch.zeros_like(E), extra)
    d.op_vocab_probs_backward(xs, es, w, logp, lse, entropy, dlogp=dlogp, dentropy=dh, dX=dX, dE=dE, temperature=heat)
    dl, dh64 = torch.where(w >= 0, dlogp.double(), 0.0), dh.double()[:, None]
    total = dl.sum(1, keepdim=True)
    inner = total + dh64 * (x.log_p + x.entropy[:, None])
    G = -x.p * inner
    G.scatter_add_(1, w.long().clamp(min=0), dl)
    # (fp32 forms the inner sum from terms of these sizes)
    sizes = dl.abs().sum(1, keepdim=True) + dh64.abs() * (x.log_p.abs() + x.entropy[:, None])
    err = x.p * (x.relative + (given + 16) * EPS32) * sizes + x.p * dh64.abs() * (x.off + x.off_entropy)[:, None]
    err.scatter_add_(1, w.long().clamp(min=0), (given + 8) * EPS32 * dl.abs().sum(1, keepdim=True).expand(rows, given).contiguous())
    size = (dl.abs().sum(1) + 8 * dh64[:, 0].abs()) / heat
    check_grads(x, dt, dX, dE, G / heat, (err + 4 * EPS32 * G.abs()) / heat, size, (size > 0).double())


def teacher_of(rows, many, words, seed):
    w = words_of(rows, many, words, seed)
    logits = rand((rows, many), "f32", seed + 1, 2.0)
    if rows > 3 and many > 1:
        logits[1, 0] = float("-inf")
        logits[2] = float("-inf")
        logits[3, 1] = -3.4e38
        w[3, 0] = 0
    return w, logits


def check_distill(rows, n_in, words, dt, listed=5, heat=1.0, extra=0, scale=3.0, seed=0, train=True):
    X, E = rand((rows, n_in), dt, seed), rand((words, n_in), dt, seed + 1, scale * n_in**-0.5)
    w, logits = teacher_of(rows, listed, words, seed + 2)
    loss, logp, lse = empty(rows), empty(rows, listed), empty(rows)
    xs, es = padded(X, extra), padded(E, extra)
    d.op_vocab_distill(xs, es, w, logits, loss=loss, logp=logp, lse=lse, temperature=heat)
    x = Exact(X, E, heat)
    near(lse, x.lse, x.off, "lse")
    near(logp, x.logp(w), x.logp_off(w), "logp")
    there = (w >= 0) & (logits > float("-inf"))
    alive = there.any(1)
    l = torch.where(there, logits.double(), -float("inf"))
    q = torch.softmax(torch.where(alive[:, None], l, 0.0) / heat, 1) * there
    want = (torch.special.xlogy(q, q) - q * x.logp(w)).sum(1)
    # q is off relatively by its exponentials' arguments and their sum
    range_ = torch.where(there, l.max(1, keepdim=True).values - l, 0.0).clamp(max=200 * heat).max(1).values / heat
    q_off = ((listed + 32 + 4 * range_) * EPS32)[:, None]
    off = (q * (x.logp_off(w) + q_off * (1 + x.logp(w).abs() + torch.where(q > 0, q.clamp(min=1e-300).log().abs(), 0.0)))).sum(1)
    off = off + (listed + 8) * EPS32 * (q * x.logp(w).abs()).sum(1) + 1e-37
    near(loss, want, off * alive, "loss")
    if not train:
        return
    dl = rand((rows,), "f32", seed + 5)
    if rows > 4:
        dl[4] = 0
    dX, dE = padded(torch.zeros_like(X), extra), padded(torch.zeros_like(E), extra)
    d.op_vocab_distill_backward(xs, es, w, logits, logp, lse, dl, dX=dX, dE=dE, temperature=heat)
    weight = torch.where(alive, dl.double(), 0.0)[:, None] / heat
    G = x.p.clone()
    G.scatter_add_(1, w.long().clamp(min=0), -q)
    err = x.p * (x.relative + 8 * EPS32)
    err.scatter_add_(1, w.long().clamp(min=0), q * q_off + (listed + 8) * EPS32 * there)
    check_grads(x, dt, dX, dE, G * weight, (err + 4 * EPS32 * G.abs()) * weight.abs(), weight[:, 0].abs(), alive.double())


SHAPES = [(1, 1, 1), (1, 64, 1000), (2, 100, 257), (16, 256, 5000), (17, 63, 300), (130, 65, 1001), (128, 128, 128), (300, 200, 2048), (40, 1003, 777)]


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("shape", SHAPES)
def test_probs_sizes(shape, dt):
    check_probs(*shape, dt, top=min(4, shape[2]), seed=sum(shape))


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("shape", SHAPES)
def test_distill_sizes(shape, dt):
    check_distill(*shape, dt, seed=sum(shape))


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("extra", [1, 8])
def test_strides(extra, dt):
    check_probs(90, 136, 700, dt, extra=extra)
    check_distill(90, 136, 700, dt, extra=extra)
    check_probs(1500, 72, 9001, dt, extra=extra)


FEW = [(1, 4, 700, 0), (3, 257, 9001, 1), (4, 1030, 513, 3), (5, 3, 300, 0), (9, 515, 20_000, 8), (16, 1003, 65, 5), (16, 5, 7, 0), (33, 130, 3000, 1),
       (64, 72, 1000, 0), (128, 100, 20_000, 0), (250, 66, 901, 1)]


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("rows, n_in, words, extra", FEW)
def test_few_tokens(rows, n_in, words, extra, dt):
    check_probs(rows, n_in, words, dt, extra=extra, seed=rows, heat=0.8)
    check_distill(rows, n_in, words, dt, extra=extra, seed=rows, heat=1.7)


@pytest.mark.parametrize("heat", [0.05, 0.7, 2.0, 30.0])
@pytest.mark.parametrize("rows", [3, 70])
def test_temperatures(heat, rows):
    check_probs(rows, 64, 900, "bf16", heat=heat, scale=min(3.0, 10 * heat))
    check_distill(rows, 64, 900, "f32", heat=heat, scale=min(3.0, 10 * heat))


@pytest.mark.parametrize("rows", [2, 30, 600])
@pytest.mark.parametrize("given, top", [(0, 5), (1, 0), (70, 1), (0, 0), (2, 64), (1, 128), (200, 128)])
def test_how_many_words(given, top, rows):
    check_probs(rows, 72, 4000, "bf16", given=given, top=top, train=given > 0)


@pytest.mark.parametrize("listed", [1, 2, 64, 65, 300])
@pytest.mark.parametrize("rows", [2, 90])
def test_how_many_listed(listed, rows):
    check_distill(rows, 72, 2000, "f16", listed=listed)


@pytest.mark.parametrize("words", [1, 2, 9, 64, 65, 100, 128])
@pytest.mark.parametrize("rows", [2, 70])
def test_all_words_are_alternatives(words, rows):
    check_probs(rows, 48, words, "f32", top=words, train=False)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("rows, n_in, words", [(1500, 72, 9001), (1000, 264, 17_001), (300, 1024, 17_000)])
def test_large_tiles(rows, n_in, words, dt):
    check_probs(rows, n_in, words, dt, top=20)
    check_distill(rows, n_in, words, dt, listed=20)


# Tiles of 128 x 128: reductions of one stage of 32 up to seven, split and whole, of the logits and of both gradients; full rounds of 256 and more.
@pytest.mark.parametrize("rows, n_in, words", [(60, 1, 700), (60, 32, 129), (60, 33, 127), (129, 65, 300), (127, 97, 500), (200, 150, 64), (200, 224, 33), (250, 515, 9000),
                                               (1000, 515, 4000), (1025, 130, 4000), (1500, 72, 9001)])
def test_products_of_fp32(rows, n_in, words):
    check_probs(rows, n_in, words, "f32")
    check_distill(rows, n_in, words, "f32")


@pytest.mark.parametrize("rows, n_in, words, listed, dt", [(1500, 256, 9001, 200, "bf16"), (1500, 255, 9001, 200, "f16"), (700, 515, 3000, 100, "f32")])
def test_long_lists_come_from_the_tiles(rows, n_in, words, listed, dt):
    """Lists whose rows of E are more than 128 MB: their logits are the tiles' own."""
    check_distill(rows, n_in, words, dt, listed=listed)
    check_probs(rows, n_in, words, dt, given=listed, top=20, heat=1.3)


def test_long_lists_and_pieces_of_the_vocabulary():
    """Both, where the logits of all words would be more than 2 GB: three pieces."""
    rows, n_in, words, listed = 60_000, 128, 20_001, 10
    X, E = rand((rows, n_in), "bf16", 1), rand((words, n_in), "bf16", 2, 0.2)
    w, logits = teacher_of(rows, listed, words, 3)
    loss, logp, lse, top_words, top_logp = empty(rows), empty(rows, listed), empty(rows), empty(rows, 9, dtype=torch.int32), empty(rows, 9)
    d.op_vocab_distill(X, E, w, logits, loss=loss, logp=logp, lse=lse, temperature=1.2)
    again, entropy = empty(rows, listed), empty(rows)
    d.op_vocab_probs(X, E, w, logp=again, entropy=entropy, top_words=top_words, top_logp=top_logp, temperature=1.2)
    q = torch.softmax(torch.where((w >= 0) & (logits > -float("inf")), logits.double(), -1e30) / 1.2, 1) * ((w >= 0) & (logits > -float("inf")))
    want = (torch.special.xlogy(q, q) - q * logp.double()).sum(1)
    assert ((loss - want).abs() <= 128 * EPS32 * (1 + (q * logp.abs()).sum(1))).all()
    for i in range(0, rows, 6000):
        at = slice(i, i + 6000)
        x = Exact(X[at], E, 1.2)
        near(lse[at], x.lse, x.off, "lse")
        near(logp[at], x.logp(w[at]), x.logp_off(w[at]), "logp")
        near(again[at], x.logp(w[at]), x.logp_off(w[at]), "logp")  # (summed in other pieces: not the same bits)
        near(entropy[at], x.entropy, x.off_entropy, "entropy")
        check_tops(x, top_words[at], top_logp[at], 9)


def test_the_list_is_at_most_4096_long():
    check_distill(3, 16, 5000, "f32", listed=4096)


@pytest.mark.parametrize("rows", [1, 5, 20, 70])
def test_ties_go_to_the_lower_word(rows):
    """Every embedding twice, and more of one than there are places: in fp32 and in 64 bits the same sums."""
    X, half = rand((rows, 40), "bf16", 1), rand((500, 40), "bf16", 2, 0.5)
    E = torch.cat([half, half])
    top_words, top_logp = empty(rows, 30, dtype=torch.int32), empty(rows, 30)
    d.op_vocab_probs(X, E, top_words=top_words, top_logp=top_logp)
    best = (X.double() @ half.double().T).sort(dim=1, descending=True, stable=True).indices[:, :15]
    assert torch.equal(top_words, torch.stack([best, best + 500], 2).view(rows, 30).to(torch.int32))
    assert torch.equal(top_logp[:, ::2], top_logp[:, 1::2])
    E[100:900] = 0
    X[0] = 0
    d.op_vocab_probs(X, E, top_words=top_words, top_logp=top_logp)
    assert torch.equal(top_words[0].cpu(), torch.arange(30, dtype=torch.int32))
    X[:] = -1
    E[:] = -0.0
    d.op_vocab_probs(X, E, top_words=top_words, top_logp=top_logp)
    assert (top_words.cpu() == torch.arange(30, dtype=torch.int32)).all()


@pytest.mark.parametrize("dt", list(DTYPES))
def test_ties_in_large_tiles_and_the_rest(dt):
    """Words that are alike on both sides of the border between tiles of both sizes, and more of them than there are places."""
    rows, words = 1000, 17_001
    X, E = rand((rows, 264), dt, 1), rand((words, 264), dt, 2, 0.05)
    E[torch.arange(100, words, 450, device="cuda")] = rand((1, 264), dt, 3, 0.3)
    top_words, top_logp = empty(rows, 20, dtype=torch.int32), empty(rows, 20)
    d.op_vocab_probs(X, E, top_words=top_words, top_logp=top_logp)
    z = X.double() @ E.double().T
    z = torch.where(torch.arange(words, device="cuda") % 450 == 100, z[:, 100:101], z)  # (equal, also where a library's sums are not)
    v, at = z.sort(dim=1, descending=True, stable=True)
    assert torch.equal(top_words, at[:, :20].to(torch.int32))


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("order", ["falling", "rising", "one chunk"])
@pytest.mark.parametrize("rows, words", [(1, 20_000), (12, 20_000), (2000, 70_001)])
def test_where_the_likeliest_words_lie(order, rows, words, dt):
    """Logits that fall or rise over the whole vocabulary, or lead in one place, for several pieces of it."""
    g = torch.Generator().manual_seed(1)
    rank = torch.arange(words, dtype=torch.float64)
    level = {"falling": -rank, "rising": rank, "one chunk": ((rank // 64) == 200).double() * words}[order] / words
    E = torch.randn(words, 16, generator=g) * 0.01
    E[:, 0] += level.float() * 8
    X = torch.rand(rows, 16, generator=g) + 0.5
    E, X = E.to(DTYPES[dt]).cuda(), X.to(DTYPES[dt]).cuda()
    top_words, top_logp, lse = empty(rows, 64, dtype=torch.int32), empty(rows, 64), empty(rows)
    d.op_vocab_probs(X, E, lse=lse, top_words=top_words, top_logp=top_logp)
    for i in range(0, rows, 500):
        at = slice(i, i + 500)
        x = Exact(X[at], E, 1.0)
        near(lse[at], x.lse, x.off, "lse")
        v, w = x.z.sort(dim=1, descending=True, stable=True)
        # (16-bit embeddings that rise so slowly are alike by the thousand: what is asked then is that the values are the largest,
        # and that equal ones come in the order of the words)
        assert torch.equal(x.z.gather(1, top_words[at].long()), v[:, :64])
        near(top_logp[at], v[:, :64] - x.lse[:, None], x.off[:, None] + 4 * EPS32 * (v[:, :64].abs() + x.lse.abs()[:, None]), "top_logp")
        got = top_words[at]
        same = v[:, 1:64] == v[:, :63]
        assert (got[:, 1:][same] > got[:, :-1][same]).all()


def test_pieces_of_the_vocabulary():
    """More words than one piece of logits holds."""
    rows, n_in, words = 4096, 64, 70_000
    X, E = rand((rows, n_in), "bf16", 1), rand((words, n_in), "bf16", 2, 0.3)
    w = words_of(rows, 2, words, 3)
    logp, lse, entropy = empty(rows, 2), empty(rows), empty(rows)
    top_words, top_logp = empty(rows, 100, dtype=torch.int32), empty(rows, 100)
    d.op_vocab_probs(X, E, w, logp=logp, lse=lse, entropy=entropy, top_words=top_words, top_logp=top_logp)
    for i in range(0, rows, 512):
        at = slice(i, i + 512)
        x = Exact(X[at], E, 1.0)
        near(lse[at], x.lse, x.off, "lse")
        near(logp[at], x.logp(w[at]), x.logp_off(w[at]), "logp")
        near(entropy[at], x.entropy, x.off_entropy, "entropy")
        check_tops(x, top_words[at], top_logp[at], 100)


@pytest.mark.parametrize("dt", list(DTYPES))
def test_more_rows_than_go_at_once(dt):
    rows, n_in, words = 140_003, 24, 301
    X, E, w = rand((rows, n_in), dt, 1), rand((words, n_in), dt, 2, 0.5), words_of(rows, 2, words, 3)
    logits = rand((rows, 2), "f32", 4)
    logp, lse, entropy, loss = empty(rows, 2), empty(rows), empty(rows), empty(rows)
    top_words, top_logp = empty(rows, 5, dtype=torch.int32), empty(rows, 5)
    d.op_vocab_probs(X, E, w, logp=logp, lse=lse, entropy=entropy, top_words=top_words, top_logp=top_logp)
    again = empty(rows, 2)
    d.op_vocab_distill(X, E, w, logits, loss=loss, logp=again)
    assert torch.equal(again, logp)
    q = torch.softmax(torch.where(w >= 0, logits, -1e30).double(), 1) * (w >= 0)
    want = (torch.special.xlogy(q, q) - q * logp.double()).sum(1)
    assert ((loss - want).abs() <= 64 * EPS32 * (1 + (q * logp.abs()).sum(1))).all()
    for i in range(0, rows, 20_000):
        at = slice(i, i + 20_000)
        x = Exact(X[at], E, 1.0)
        near(lse[at], x.lse, x.off, "lse")
        near(logp[at], x.logp(w[at]), x.logp_off(w[at]), "logp")
        near(entropy[at], x.entropy, x.off_entropy, "entropy")
        check_tops(x, top_words[at], top_logp[at], 5)


@pytest.mark.parametrize("rows", [3, 40])
def test_a_vocabulary_past_32_bits(rows):
    """600,000 words of 4096: 4.9 GB, its last words past 2^31 elements."""
    words, n_in = 600_000, 4096
    g = torch.Generator(device="cuda").manual_seed(1)
    E = torch.empty(words, n_in, dtype=torch.bfloat16, device="cuda")
    for i in range(0, words, 100_000):
        E[i : i + 100_000] = torch.randn(100_000, n_in, generator=g, device="cuda") * 0.03
    X = rand((rows, n_in), "bf16", 2)
    E[words - 3] = X[1] * 0.01
    w = torch.randint(560_000, words, (rows, 2), generator=torch.Generator().manual_seed(3), dtype=torch.int32).cuda()
    logp, lse, top_words, top_logp = empty(rows, 2), empty(rows), empty(rows, 10, dtype=torch.int32), empty(rows, 10)
    d.op_vocab_probs(X, E, w, logp=logp, lse=lse, top_words=top_words, top_logp=top_logp)
    z = torch.cat([X.double() @ E[i : i + 100_000].double().T for i in range(0, words, 100_000)], 1)
    want = torch.logsumexp(z, 1)
    off = 2 * 4104 * EPS32 * X.abs().double().sum(1) * E.abs().max().double() + 600_064 * EPS32
    near(lse, want, off, "lse")
    near(logp, z.gather(1, w.long()) - want[:, None], off[:, None] + 64 * EPS32, "logp")
    v, at = z.sort(dim=1, descending=True, stable=True)
    assert torch.equal(top_words, at[:, :10].to(torch.int32)) and top_words[1, 0] == words - 3
    # the gradients, of both ends of dE and of dX
    dlogp, logits = rand((rows, 2), "f32", 5), rand((rows, 2), "f32", 6)
    dX, dE = torch.zeros_like(X), torch.full_like(E, 9.0)
    d.op_vocab_probs_backward(X, E, w, logp, lse, dlogp=dlogp, dX=dX, dE=dE)
    G = -torch.exp(z - want[:, None]) * dlogp.double().sum(1, keepdim=True)
    G.scatter_add_(1, w.long(), dlogp.double())
    for part in (slice(0, 2000), slice(524_200, 524_400), slice(words - 2000, words)):
        exact = G[:, part].T @ X.double()
        near(dE[part], exact, 4 * HALF["bf16"] * (G[:, part].abs().T @ X.double().abs()) + 1e-9, "dE")
    exact, size = torch.zeros(rows, n_in, dtype=torch.float64, device="cuda"), torch.zeros(rows, n_in, dtype=torch.float64, device="cuda")
    for i in range(0, words, 100_000):
        e = E[i : i + 100_000].double()
        exact += G[:, i : i + 100_000] @ e
        size += G[:, i : i + 100_000].abs() @ e.abs()
    near(dX, exact, 4 * HALF["bf16"] * size, "dX")
    torch.cuda.empty_cache()


def test_words_outside_the_vocabulary():
    X, E = rand((70, 64), "bf16", 1), rand((900, 64), "bf16", 2)
    w, logits = torch.full((70, 2), -1, dtype=torch.int32, device="cuda"), torch.zeros(70, 2, device="cuda")
    logp, lse, loss, dl = empty(70, 2), empty(70), empty(70), torch.ones(70, device="cuda")
    dX, dE = torch.ones_like(X), torch.ones_like(E)
    for rows in (70, 3):
        x, ww, l, lo, ls, g, o = X[:rows], w[:rows], logits[:rows], logp[:rows], lse[:rows], dl[:rows], loss[:rows]
        ww[:] = -1
        d.op_vocab_distill(x, E, ww, l, loss=o, logp=lo, lse=ls)
        assert not lo.any() and not o.any() and torch.isfinite(ls).all()
        dX[:], dE[:] = 1, 1
        d.op_vocab_distill_backward(x, E, ww, l, lo, ls, g, dX=dX[:rows], dE=dE)
        assert not dX[:rows].any() and not dE.any()
        dE[:] = 1
        d.op_vocab_probs_backward(x, E, ww, lo, ls, dlogp=torch.ones_like(lo), dX=dX[:rows], dE=dE)
        assert not dX[:rows].any() and not dE.any()
        ww[1, 1], ww[2, 0] = 900, 899
        d.op_vocab_distill(x, E, ww, l, loss=o, logp=lo, lse=ls)
        assert lo[1, 1].isnan() and o[1].isnan() and torch.isfinite(o[2]) and o[2] > 0 and not o[0]
        d.op_vocab_distill_backward(x, E, ww, l, lo, ls, g, dX=dX[:rows], dE=dE)
        assert dX[1].isnan().all() and torch.isfinite(dX[2]).all() and not dX[0].any() and dE.isnan().any()
        d.op_vocab_probs_backward(x, E, ww, lo, ls, dlogp=torch.ones_like(lo), dX=dX[:rows], dE=dE)
        assert dX[1].isnan().all() and torch.isfinite(dX[2]).all() and not dX[0].any() and dE.isnan().any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("rows", [4, 70])
def test_a_teacher_that_is_not_a_number(rows, bad):
    X, E = rand((rows, 64), "bf16", 1), rand((900, 64), "bf16", 2)
    w, logits = torch.full((rows, 3), 5, dtype=torch.int32, device="cuda"), torch.zeros(rows, 3, device="cuda")
    w[1, 0], logits[1, 0], logits[2, 2] = -1, bad, bad
    logp, lse, loss = empty(rows, 3), empty(rows), empty(rows)
    d.op_vocab_distill(X, E, w, logits, loss=loss, logp=logp, lse=lse)
    assert loss[2].isnan() and torch.isfinite(loss[:2]).all() and torch.isfinite(loss[3:]).all()
    dX = torch.ones_like(X)
    d.op_vocab_distill_backward(X, E, w, logits, logp, lse, torch.ones(rows, device="cuda"), dX=dX)
    assert dX[2].isnan().all() and torch.isfinite(dX[:2]).all() and torch.isfinite(dX[3:]).all()


@pytest.mark.parametrize("rows", [4, 70, 700])
@pytest.mark.parametrize("dt", list(DTYPES))
def test_rows_that_are_not_numbers(rows, dt):
    """NaN and infinities in a row of X stay in its row."""
    X, E = rand((rows, 64), dt, 1), rand((9000, 64), dt, 2, 0.3)
    w = words_of(rows, 2, 9000, 3, masked=0.0)
    outs = []
    for bad in (0.0, float("nan"), float("inf")):
        X[1], X[2, 5] = 0, 0.5
        X[1, 3] = bad
        o = dict(logp=empty(rows, 2), lse=empty(rows), entropy=empty(rows), top_words=empty(rows, 9, dtype=torch.int32), top_logp=empty(rows, 9))
        d.op_vocab_probs(X, E, w, **o)
        if bad:
            assert (o["top_words"][1] == -1).all() and o["top_logp"][1].isnan().all() and o["entropy"][1].isnan() and not torch.isfinite(o["lse"][1])
        else:
            assert (o["top_words"][1].cpu() == torch.arange(9)).all()
        outs.append({k: torch.cat([v[:1], v[2:]]) for k, v in o.items()})
    for other in outs[1:]:
        assert all(torch.equal(other[k], v) for k, v in outs[0].items())


@pytest.mark.parametrize("rows, given", [(4, 2), (70, 2), (1500, 2), (600, 1500)])
@pytest.mark.parametrize("top", [0, 5])
def test_logits_of_infinity_write_nothing_past_the_workspace(rows, given, top):
    """A row whose logits are all infinite, with and without alternatives, lists short and long: the other rows and what lies around
    the workspace stay as they are."""
    X, E, w = rand((rows, 80), "bf16", 1), rand((3000, 80), "bf16", 2, 0.3), words_of(rows, given, 3000, 3, masked=0.0)
    E[:, 7] = E[:, 7].abs() + 0.1
    size = d.vocab_probs_workspace(rows, 80, 3000, given, top, torch.bfloat16, True)[0]
    outs = []
    for big in (0.5, float("inf")):
        X[1, 7] = big
        buf = torch.full((size + (64 << 20),), 123, dtype=torch.uint8, device="cuda")
        o = dict(logp=empty(rows, given), lse=empty(rows), entropy=empty(rows))
        if top:
            o.update(top_words=empty(rows, top, dtype=torch.int32), top_logp=empty(rows, top))
        d.op_vocab_probs(X, E, w, workspace=buf[:size], **o)
        assert (buf[size:] == 123).all()
        if big > 1:
            assert not torch.isfinite(o["lse"][1])
        outs.append({k: torch.cat([v[:1], v[2:]]) for k, v in o.items()})
    assert all(torch.equal(v, outs[1][k]) for k, v in outs[0].items())


@pytest.mark.parametrize("rows", [3, 70, 600])
@pytest.mark.parametrize("words, top", [(700, 128), (8000, 128), (8000, 5), (120, 3)])
@pytest.mark.parametrize("dt", list(DTYPES))
def test_infinities_of_both_signs(rows, words, top, dt):
    """A row of which half the logits are infinity and half minus infinity, and one of minus infinity and NaN: where more of the former are
    there than are wanted, the range of what is looked at ends with the last number that there is."""
    X, E = rand((rows, 64), dt, 1), rand((words, 64), dt, 2, 0.3)
    w = words_of(rows, 2, words, 3, masked=0.0)
    outs = []
    for bad in (0.5, float("inf")):
        X[1:3] = 0
        X[1, 3], X[2, 5], X[2, 6] = bad, bad, bad if dt == "f32" else -bad
        o = dict(logp=empty(rows, 2), lse=empty(rows), entropy=empty(rows), top_words=empty(rows, top, dtype=torch.int32), top_logp=empty(rows, top))
        d.op_vocab_probs(X, E, w, **o)
        if bad > 1:
            assert (o["top_words"][1:3] == -1).all() and o["top_logp"][1:3].isnan().all() and o["entropy"][1:3].isnan().all()
        outs.append({k: torch.cat([v[:1], v[3:]]) for k, v in o.items()})
    assert all(torch.equal(v, outs[1][k]) for k, v in outs[0].items())


@pytest.mark.parametrize("rows", [4, 70])
def test_a_word_that_is_minus_infinity(rows):
    """A word with probability 0: it counts nowhere."""
    X, E = rand((rows, 64), "f32", 1).abs(), rand((300, 64), "f32", 2, 0.3)
    w = torch.tensor([[7, 9]], dtype=torch.int32, device="cuda").repeat(rows, 1)
    o = dict(logp=empty(rows, 2), lse=empty(rows), entropy=empty(rows), top_words=empty(rows, 128, dtype=torch.int32), top_logp=empty(rows, 128))
    E[7, 0] = float("-inf")
    d.op_vocab_probs(X, E, w, **o)
    keep = [i for i in range(300) if i != 7]
    x = Exact(X, E[keep], 1.0)
    near(o["lse"], x.lse, x.off, "lse")
    near(o["entropy"], x.entropy, x.off_entropy, "entropy")
    assert (o["logp"][:, 0] == -float("inf")).all() and not (o["top_words"] == 7).any()
    dX, dE = torch.ones_like(X), torch.ones_like(E)
    d.op_vocab_probs_backward(X, E, w[:, 1:].contiguous(), o["logp"][:, 1:].contiguous(), o["lse"], o["entropy"], dlogp=torch.ones(rows, 1, device="cuda"),
                              dentropy=torch.ones(rows, device="cuda"), dE=dE)
    assert torch.isfinite(dE).all() and not dE[7].any()


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("rows, extra", [(3, 0), (8, 1), (12, 0), (70, 0), (70, 1), (300, 8)])
def test_rows_without_a_gradient_may_hold_anything(rows, extra, dt):
    """The same bits in all gradients whatever the state of a row without listed words, or with weights of zero, holds."""
    X, E = rand((rows, 72), dt, 1), rand((900, 72), dt, 2, 0.3)
    w, logits = words_of(rows, 3, 900, 3), rand((rows, 3), "f32", 4)
    w[1], w[2] = -1, 17
    dl, dlogp, dh = torch.ones(rows, device="cuda"), rand((rows, 3), "f32", 5), rand((rows,), "f32", 6)
    dlogp[2], dh[1], dh[2] = 0, 0, 0
    outs = []
    for bad in (0.0, float("inf"), float("nan")):
        X[1] = 0
        X[1, ::5] = bad
        x, e = padded(X, extra), padded(E, extra)
        loss, logp, lse, entropy = empty(rows), empty(rows, 3), empty(rows), empty(rows)
        d.op_vocab_distill(x, e, w, logits, loss=loss, logp=logp, lse=lse)
        dX, dE, alone = torch.ones_like(X), torch.ones_like(E), torch.ones_like(E)
        d.op_vocab_distill_backward(x, e, w, logits, logp, lse, dl, dX=dX, dE=dE)
        d.op_vocab_distill_backward(x, e, w, logits, logp, lse, dl, dE=alone)
        assert torch.isfinite(dE).all() and not dX[1].any() and loss[1] == 0 and torch.equal(dE, alone)
        d.op_vocab_probs(x, e, w, logp=logp, entropy=entropy, lse=lse)
        pX, pE, alone = torch.ones_like(X), torch.ones_like(E), torch.ones_like(X)
        d.op_vocab_probs_backward(x, e, w, logp, lse, entropy, dlogp=dlogp, dentropy=dh, dX=pX, dE=pE)
        d.op_vocab_probs_backward(x, e, w, logp, lse, entropy, dlogp=dlogp, dentropy=dh, dX=alone)
        assert torch.isfinite(pE).all() and not pX[1].any() and not pX[2].any() and torch.equal(pX, alone)
        outs.append((loss, dX, dE, pX, pE))
    for other in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], other))


@pytest.mark.parametrize("rows", [0, 3, 40])
def test_no_rows_and_gradients_alone(rows):
    X, E = rand((rows, 100), "bf16", 1), rand((900, 100), "bf16", 2, 0.3)
    w = words_of(rows, 2, 900, 3)
    logp, lse, entropy = empty(rows, 2), empty(rows), empty(rows)
    d.op_vocab_probs(X, E, w, logp=logp, lse=lse, entropy=entropy, top_words=empty(rows, 2, dtype=torch.int32), top_logp=empty(rows, 2))
    one = torch.ones(rows, device="cuda")
    both, alone = [[torch.full_like(t, 3.0) for t in (X, E)] for _ in range(2)]
    d.op_vocab_probs_backward(X, E, w, logp, lse, entropy, dentropy=one, dX=both[0], dE=both[1])
    d.op_vocab_probs_backward(X, E, None, None, lse, entropy, dentropy=one, dX=alone[0], dE=alone[1])
    # (each within its own bounds: with words, the scale at which bf16 rounds the logits' gradient may be another)
    x = Exact(X, E, 1.0)
    G, size = -x.p * (x.log_p + x.entropy[:, None]), 8 * one.double()
    err = x.p * (x.relative + 16 * EPS32) * (x.log_p.abs() + x.entropy[:, None]) + x.p * (x.off + x.off_entropy)[:, None]
    for dX, dE in (both, alone):
        check_grads(x, "bf16", dX, dE, G, err + 4 * EPS32 * G.abs(), size, one.double())
    d.op_vocab_probs_backward(X, E, w, logp, lse, dX=both[0], dE=both[1])
    assert not both[0].any() and not both[1].any()


@pytest.mark.parametrize("dt", list(DTYPES))
def test_one_label_is_the_loss(dt):
    """log p of one given word is minus op_vocab_loss, and so are its gradients."""
    X, E = rand((90, 100), dt, 1), rand((2000, 100), dt, 2, 0.3)
    w = words_of(90, 1, 2000, 3)
    logp, lse, loss, lse2 = empty(90, 1), empty(90), empty(90), empty(90)
    d.op_vocab_probs(X, E, w, logp=logp, lse=lse)
    d.op_vocab_loss(X, E, w[:, 0].contiguous(), loss, lse2)
    x = Exact(X, E, 1.0)
    near(loss + logp[:, 0], torch.zeros(90, device="cuda").double(), 4 * x.off, "loss")
    a, b = [[torch.zeros_like(X), torch.zeros_like(E)] for _ in range(2)]
    dl = rand((90,), "f32", 4)
    d.op_vocab_probs_backward(X, E, w, logp, lse, dlogp=-dl[:, None].contiguous(), dX=a[0], dE=a[1])
    d.op_vocab_loss_backward(X, E, w[:, 0].contiguous(), lse2, dl, dX=b[0], dE=b[1])
    for s, t in zip(a, b):
        assert (s.double() - t.double()).norm() <= (2 * HALF[dt] + 1e-5) * t.double().norm()


@pytest.mark.parametrize("rows", [2, 20])
def test_gradients_against_differences(rows):
    n_in, words, heat = 5, 11, 0.9
    X, E = rand((rows, n_in), "f32", 1), rand((words, n_in), "f32", 2)
    w, logits = words_of(rows, 3, words, 3), rand((rows, 3), "f32", 4)
    logp, lse, entropy, loss = empty(rows, 3), empty(rows), empty(rows), empty(rows)
    dlogp, dh, dl = rand((rows, 3), "f32", 5), rand((rows,), "f32", 6), rand((rows,), "f32", 7)
    d.op_vocab_probs(X, E, w, logp=logp, lse=lse, entropy=entropy, temperature=heat)
    d.op_vocab_distill(X, E, w, logits, loss=loss, temperature=heat)
    probs, distill = [[torch.zeros_like(X), torch.zeros_like(E)] for _ in range(2)]
    d.op_vocab_probs_backward(X, E, w, logp, lse, entropy, dlogp=dlogp, dentropy=dh, dX=probs[0], dE=probs[1], temperature=heat)
    d.op_vocab_distill_backward(X, E, w, logits, logp, lse, dl, dX=distill[0], dE=distill[1], temperature=heat)
    host = [t.double().cpu() for t in (dlogp, dh, dl, logits)]
    wc = w.cpu().long()
    q = torch.softmax(torch.where(wc >= 0, host[3] / heat, -1e300), 1) * (wc >= 0)

    def totals(x, e):
        log_p = torch.log_softmax(x @ e.T / heat, 1)
        lp = torch.where(wc >= 0, log_p.gather(1, wc.clamp(min=0)), 0.0)
        return ((lp * host[0]).sum() + (torch.special.entr(log_p.exp()).sum(1) * host[1]).sum(),
                ((torch.special.xlogy(q, q) - q * lp).sum(1) * host[2]).sum())

    x64, e64, h = X.double().cpu(), E.double().cpu(), 1e-6
    for side, t in enumerate((x64, e64)):
        for i in range(t.shape[0]):
            for j in range(t.shape[1]):
                keep = t[i, j].item()
                t[i, j] = keep + h
                hi = totals(x64, e64)
                t[i, j] = keep - h
                lo = totals(x64, e64)
                t[i, j] = keep
                for got, a, b in zip((probs, distill), hi, lo):
                    slope = ((a - b) / (2 * h)).item()
                    assert abs(got[side][i, j].item() - slope) <= 1e-4 * max(1.0, abs(slope))


@pytest.mark.parametrize("rows, dt", [(5, "bf16"), (300, "bf16"), (700, "f16"), (300, "f32")])
def test_captured_and_replayed(rows, dt):
    """A teacher's alternatives, a student's loss and its gradients in one graph; every replay against eager calls."""
    X, S = rand((rows, 128), dt, 1), rand((rows, 128), dt, 2)
    E = rand((9000, 128), dt, 3, 0.3)
    top = dict(top_words=empty(rows, 20, dtype=torch.int32), top_logp=empty(rows, 20))
    loss, logp, lse, one = empty(rows), empty(rows, 20), empty(rows), torch.ones(rows, device="cuda")
    dX, dE = torch.zeros_like(S), torch.zeros_like(E)
    forward, _ = d.vocab_probs_workspace(rows, 128, 9000, 0, 20, DTYPES[dt])
    both = max(forward, *d.vocab_probs_workspace(rows, 128, 9000, 20, 0, DTYPES[dt]))
    ws = torch.empty(both, dtype=torch.uint8, device="cuda")

    def step():
        d.op_vocab_probs(X, E, workspace=ws, **top)
        d.op_vocab_distill(S, E, top["top_words"], top["top_logp"], loss=loss, logp=logp, lse=lse, temperature=1.5, workspace=ws)
        d.op_vocab_distill_backward(S, E, top["top_words"], top["top_logp"], logp, lse, one, dX=dX, dE=dE, temperature=1.5, workspace=ws)
        return [t.clone() for t in (top["top_words"], top["top_logp"], loss, logp, lse, dX, dE)]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        X.copy_(rand((rows, 128), dt, 10 + i))
        S.copy_(rand((rows, 128), dt, 20 + i))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


def test_another_stream_and_arrays_of_the_library():
    X, E, w = rand((50, 64), "f32", 1), rand((700, 64), "f32", 2, 0.4), words_of(50, 2, 700, 3)
    o = dict(logp=empty(50, 2), lse=empty(50), entropy=empty(50), top_words=empty(50, 6, dtype=torch.int32), top_logp=empty(50, 6))
    d.op_vocab_probs(X, E, w, **o)
    want = [t.cpu().numpy() for t in o.values()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = {k: torch.zeros_like(v) for k, v in o.items()}
        d.op_vocab_probs(X, E, w, **other)
    side.synchronize()
    assert all((a.cpu().numpy() == b).all() for a, b in zip(other.values(), want))
    def library(t):
        a = t.cpu().numpy()
        return d.DeviceArray.from_numpy(a, a.dtype)

    own = {k: library(torch.zeros_like(v)) for k, v in o.items()}
    d.op_vocab_probs(library(X), library(E), library(w), **own)
    assert all((a.numpy() == b).all() for a, b in zip(own.values(), want))


def test_a_workspace_as_large_as_asked_for_is_enough_and_all_that_is_written():
    for rows, n_in, words, dt, n, k in ((3, 65, 900, "f32", 2, 7), (70, 72, 4001, "bf16", 3, 20), (40, 65, 3000, "f16", 1, 5), (1500, 72, 9001, "bf16", 2, 128),
                                           (200, 515, 9000, "f32", 2, 5), (1025, 130, 4000, "f32", 2, 5)):
        X, E, w = rand((rows, n_in), dt, 1), rand((words, n_in), dt, 2, 0.3), words_of(rows, n, words, 3)
        logp, lse, entropy = empty(rows, n), empty(rows), empty(rows)
        for aligned in (False, True) if n_in % 8 == 0 else (False,):
            sizes = d.vocab_probs_workspace(rows, n_in, words, n, k, DTYPES[dt], aligned)
            buf = torch.full((max(sizes) + 512,), 123, dtype=torch.uint8, device="cuda")
            top = dict(top_words=empty(rows, k, dtype=torch.int32), top_logp=empty(rows, k))
            d.op_vocab_probs(X, E, w, logp=logp, lse=lse, entropy=entropy, workspace=buf[256 : 256 + sizes[0]], **top)
            dX, dE = torch.zeros_like(X), torch.zeros_like(E)
            d.op_vocab_probs_backward(X, E, w, logp, lse, entropy, dlogp=torch.ones_like(logp), dX=dX, dE=dE, workspace=buf[256 : 256 + sizes[1]])
            assert (buf[:256] == 123).all() and (buf[256 + max(sizes) :] == 123).all()
            check_tops(Exact(X, E, 1.0), top["top_words"], top["top_logp"], k)
        for i in (0, 1):
            short = buf[256 : 256 + sizes[i] - 256]
            with pytest.raises(d.DnpeffError, match="workspace"):
                if i == 0:
                    d.op_vocab_probs(X, E, w, logp=logp, workspace=short, **top)
                else:
                    d.op_vocab_probs_backward(X, E, w, logp, lse, dlogp=logp, dE=dE, workspace=short)


def test_refusals_of_calls():
    X, E, w = rand((10, 64), "bf16", 1), rand((90, 64), "bf16", 2), words_of(10, 2, 90, 3)
    f, i = lambda *s: empty(*s), lambda *s: empty(*s, dtype=torch.int32)
    probs, distill = d.op_vocab_probs, d.op_vocab_distill
    for what, call in {
        "temperature": lambda: probs(X, E, lse=f(10), temperature=0.0),
        "temperature = -1": lambda: probs(X, E, lse=f(10), temperature=-1.0),
        "temperature = nan": lambda: distill(X, E, w, f(10, 2), loss=f(10), temperature=float("nan")),
        "temperature = inf": lambda: distill(X, E, w, f(10, 2), loss=f(10), temperature=float("inf")),
        "alternatives": lambda: probs(X, E, top_words=i(10, 91), top_logp=f(10, 91)),
        "words of a row": lambda: probs(X, E, i(10, 4097), logp=f(10, 4097)),
        "words come with logp": lambda: probs(X, E, w, lse=f(10)),
        "top_logp": lambda: probs(X, E, top_words=i(10, 3)),
        "words is of": lambda: probs(X, E, w.long(), logp=f(10, 2)),
        "logp is": lambda: probs(X, E, w, logp=f(10, 3)),
        "entropy is": lambda: probs(X, E, entropy=f(11)),
        "words has to be dense": lambda: probs(X, E, i(10, 4)[:, :2], logp=f(10, 2)),
        "top_words has to be dense": lambda: probs(X, E, top_words=i(10, 4)[:, :2], top_logp=f(10, 2)),
        "elements of a row": lambda: probs(X.T.contiguous().T, E, lse=f(10)),
        "E is": lambda: probs(X, E[:, :60], lse=f(10)),
        "no words are listed": lambda: distill(X, E, i(10, 0), f(10, 0), loss=f(10)),
        "no words": lambda: distill(X, E, None, None, loss=f(10)),
        "no logits": lambda: distill(X, E, w, None, loss=f(10)),
        "logits is": lambda: distill(X, E, w, f(10, 3), loss=f(10)),
        "no entropy": lambda: d.op_vocab_probs_backward(X, E, w, f(10, 2), f(10), dentropy=f(10)),
        "dlogp without words": lambda: d.op_vocab_probs_backward(X, E, None, None, f(10), dlogp=f(10, 2)),
        "no lse": lambda: d.op_vocab_probs_backward(X, E, w, f(10, 2), None, dlogp=f(10, 2)),
        "no dloss": lambda: d.op_vocab_distill_backward(X, E, w, f(10, 2), f(10, 2), f(10), None),
        "no logp": lambda: d.op_vocab_distill_backward(X, E, w, f(10, 2), None, f(10), f(10)),
        "dE is": lambda: d.op_vocab_distill_backward(X, E, w, f(10, 2), f(10, 2), f(10), f(10), dE=E[:80]),
    }.items():
        with pytest.raises(d.DnpeffError) as told:
            call()
        assert what in str(told.value) or what == "no words", (what, str(told.value))
