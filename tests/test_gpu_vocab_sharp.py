"""What a model answers, distillation and their gradients where logits lie far apart: at temperatures so low that |z| / T goes
up to 1e38, and of logits that are large themselves.

Small whole numbers make the products exact in every type, and powers of two the temperatures, so that what is left are the roundings of
the results: the bounds below hold none that grow with |z| / T but those of a result's own size.  A row's largest logits lead by 2^30 and
more, its probabilities are 1 / (how many are largest) and 0: an exponential, the sum, its logarithm and the result are rounded, 8 half
units in all.  Of arbitrary numbers a word that leads by more than the products' rounding has log p 0 all the same, since the given
words' logits are the same sums as the row's largest."""

import pytest
import torch

import npeff_ref_amd as d
from test_gpu_vocab_answers import DTYPES, EPS32, Exact, check_grads, empty, near, rand, words_of

pytestmark = pytest.mark.gpu

TEMPERATURES = [2.0**-30, 2.0**-63, 2.0**-119]
SHAPES = [(1, 4000), (3, 3000), (12, 3000), (40, 3000), (70, 2500), (200, 9001), (700, 3000), (1500, 9001)]


def whole(shape, dt, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-2, 3, shape, generator=g).to(DTYPES[dt]).cuda()


class Sharp:
    """Of exact logits whose differences are 2^30 and more: the largest share the probability."""

    def __init__(self, X, E, heat):
        self.X, self.E = X.double(), E.double()
        self.raw = self.X @ self.E.T
        self.top = self.raw.max(1, keepdim=True).values
        self.p = (self.raw == self.top).double()
        self.many = self.p.sum(1)
        self.p /= self.many[:, None]
        self.entropy = self.many.log()
        self.log_p = (self.raw - self.top) / heat - self.entropy[:, None]
        self.lse = self.top[:, 0] / heat + self.entropy


def answers(X, E, w, top, heat):
    rows, given = w.shape
    o = dict(logp=empty(rows, given), lse=empty(rows), entropy=empty(rows), top_words=empty(rows, top, dtype=torch.int32), top_logp=empty(rows, top))
    d.op_vocab_probs(X, E, w, temperature=heat, **o)
    return o


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("heat", TEMPERATURES)
@pytest.mark.parametrize("rows, words", SHAPES)
def test_answers_at_low_temperatures(rows, words, heat, dt):
    X, E, w = whole((rows, 40), dt, 1), whole((words, 40), dt, 2), words_of(rows, 3, words, 3)
    x = Sharp(X, E, heat)
    w[0, 0] = int(x.raw[0].argmax())
    o = answers(X, E, w, 9, heat)
    near(o["lse"], x.lse, 8 * EPS32 * (1 + x.lse.abs()), "lse")
    near(o["entropy"], x.entropy, 8 * EPS32 * (1 + x.entropy), "entropy")
    assert torch.equal(o["top_words"], x.raw.sort(dim=1, descending=True, stable=True).indices[:, :9].to(torch.int32))


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("heat", TEMPERATURES)
@pytest.mark.parametrize("rows, words", SHAPES)
def test_log_p_at_low_temperatures(rows, words, heat, dt):
    X, E, w = whole((rows, 40), dt, 1), whole((words, 40), dt, 2), words_of(rows, 3, words, 3)
    x = Sharp(X, E, heat)
    w[0, 0] = int(x.raw[0].argmax())
    o = answers(X, E, w, 9, heat)
    want = torch.where(w >= 0, x.log_p.gather(1, w.long().clamp(min=0)), 0.0)
    near(o["logp"], want, 8 * EPS32 * (1 + want.abs()), "logp")
    v = x.log_p.gather(1, o["top_words"].long())
    near(o["top_logp"], v, 8 * EPS32 * (1 + v.abs()), "top_logp")


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("heat", TEMPERATURES)
@pytest.mark.parametrize("rows, words", SHAPES)
def test_distillation_at_low_temperatures(rows, words, heat, dt):
    X, E, w = whole((rows, 40), dt, 1), whole((words, 40), dt, 2), words_of(rows, 4, words, 3)
    logits = whole((rows, 4), "f32", 4)
    loss, logp, lse = empty(rows), empty(rows, 4), empty(rows)
    d.op_vocab_distill(X, E, w, logits, loss=loss, logp=logp, lse=lse, temperature=heat)
    x = Sharp(X, E, heat)
    there = w >= 0
    l = torch.where(there, logits.double(), -9.0)
    q = ((l == l.max(1, keepdim=True).values) & there).double()
    q /= q.sum(1, keepdim=True).clamp(min=1)
    want = torch.where(there, x.log_p.gather(1, w.long().clamp(min=0)), 0.0)
    near(logp, want, 8 * EPS32 * (1 + want.abs()), "logp")
    exact, size = (torch.special.xlogy(q, q) - q * want).sum(1), (q * want.abs()).sum(1)
    near(loss, exact, 16 * EPS32 * (1 + size), "loss")


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("heat", [0.05, 1e-6, 1e-36])
@pytest.mark.parametrize("rows", [1, 12, 40, 200, 700, 1500])
def test_a_word_that_leads_has_log_p_zero(rows, heat, dt):
    """Logits of arbitrary numbers: one word a row is ahead by 20, all others together have a probability of 9000 exp(-400) at most."""
    X, E, first = leading(rows, dt)
    w = torch.stack([first, torch.zeros_like(first)], 1).contiguous()
    o = answers(X, E, w, 3, heat)
    assert torch.equal(o["top_words"][:, 0], first) and torch.isfinite(o["lse"]).all()
    for name, got in (("logp", o["logp"][:, 0]), ("top_logp", o["top_logp"][:, 0]), ("entropy", o["entropy"])):
        near(got, torch.zeros(rows, device="cuda").double(), torch.full((rows,), 4 * EPS32, device="cuda").double(), name)
    assert (o["logp"][:, 1] < -300).all()


def leading(rows, dt, n_in=264, words=9000):
    X, E = rand((rows, n_in), dt, 1), rand((words, n_in), "f32", 2, 0.1)
    first = torch.arange(rows, device="cuda") * 5 + 2
    x = X.float()
    E[first] += 4 * x / x.norm(dim=1, keepdim=True)
    E = E.to(DTYPES[dt])
    z = X.double() @ E.double().T
    lead = z.gather(1, first[:, None])[:, 0]
    z.scatter_(1, first[:, None], -1e9)
    assert (lead - z.max(1).values > 20).all()
    return X, E, first.to(torch.int32)


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("rows", [1, 12, 40, 200, 700, 1500])
def test_large_logits(rows, dt):
    """At a temperature of 1 and logits of 4e4 and more: alternatives' log p come from products in 64 bits, so the leading one's is 0; given words' are
    off by the rounding of fp32 products, and never above 0."""
    X, E, first = leading(rows, dt)
    E *= 1024
    o = answers(X, E, first[:, None].contiguous(), 3, 1.0)
    x = Exact(X, E, 1.0)
    assert torch.equal(o["top_words"][:, 0], first)
    near(o["top_logp"][:, 0], torch.zeros_like(x.lse), torch.full_like(x.lse, 4 * EPS32), "top_logp")
    near(o["entropy"], torch.zeros_like(x.lse), torch.full_like(x.lse, 4 * EPS32), "entropy")
    near(o["lse"], x.lse, x.off, "lse")
    near(o["logp"][:, 0], torch.zeros_like(x.lse), 2 * x.logit, "logp")
    assert (o["logp"] <= 0).all()


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("heat", TEMPERATURES)
@pytest.mark.parametrize("rows, words", SHAPES)
def test_gradients_at_low_temperatures(rows, words, heat, dt):
    """Weights of the temperature's size, so that the gradients are of the operands' types.  Errors as at other temperatures, but p is off
    by an exponential and a logarithm alone."""
    X, E, w = whole((rows, 40), dt, 1), whole((words, 40), dt, 2), words_of(rows, 3, words, 3)
    x = Sharp(X, E, heat)
    w[0, 0] = int(x.raw[0].argmax())
    o = answers(X, E, w, 1, heat)
    dlogp, dh = rand((rows, 3), "f32", 4) * heat, rand((rows,), "f32", 5, 0.3) * heat
    dlogp[1::3], dh[::2] = 0, 0
    dX, dE = torch.zeros_like(X), torch.zeros_like(E)
    d.op_vocab_probs_backward(X, E, w, o["logp"], o["lse"], o["entropy"], dlogp=dlogp, dentropy=dh, dX=dX, dE=dE, temperature=heat)
    dl, dh64 = torch.where(w >= 0, dlogp.double(), 0.0), dh.double()[:, None]
    # (of the largest words log p + H is 0)
    G = -x.p * dl.sum(1, keepdim=True)
    G.scatter_add_(1, w.long().clamp(min=0), dl)
    err = x.p * 32 * EPS32 * (dl.abs().sum(1, keepdim=True) + 2 * dh64.abs() * x.entropy[:, None])
    err.scatter_add_(1, w.long().clamp(min=0), 16 * EPS32 * dl.abs().sum(1, keepdim=True).expand(rows, 3).contiguous())
    size = (dl.abs().sum(1) + 8 * dh64[:, 0].abs()) / heat
    check_grads(x, dt, dX, dE, G / heat, err / heat, size, (size > 0).double())

    logits, loss = whole((rows, 3), "f32", 6), empty(rows)
    d.op_vocab_distill(X, E, w, logits, loss=loss, logp=o["logp"], lse=o["lse"], temperature=heat)
    dl = rand((rows,), "f32", 7) * heat
    d.op_vocab_distill_backward(X, E, w, logits, o["logp"], o["lse"], dl, dX=dX, dE=dE, temperature=heat)
    there = w >= 0
    l = torch.where(there, logits.double(), -9.0)
    q = ((l == l.max(1, keepdim=True).values) & there).double()
    q /= q.sum(1, keepdim=True).clamp(min=1)
    weight = torch.where(there.any(1), dl.double(), 0.0)[:, None] / heat
    G = x.p.clone()
    G.scatter_add_(1, w.long().clamp(min=0), -q)
    err = x.p * 32 * EPS32
    err.scatter_add_(1, w.long().clamp(min=0), 16 * EPS32 * there.double())
    check_grads(x, dt, dX, dE, G * weight, err * weight.abs(), weight[:, 0].abs(), there.any(1).double())


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("heat", [0.05, 1e-6, 1e-36])
@pytest.mark.parametrize("rows", [1, 5, 12, 40, 200, 700, 1500])
def test_gradients_of_a_word_that_leads(rows, heat, dt):
    """Arbitrary numbers: what one word takes from the leading one is its gradient, and the leading word has none of its own."""
    X, E, first = leading(rows, dt)
    w = torch.stack([first, torch.zeros_like(first)], 1).contiguous()
    o = answers(X, E, w, 1, heat)
    dlogp = rand((rows, 2), "f32", 4) * heat
    dX, dE = torch.zeros_like(X), torch.zeros_like(E)
    d.op_vocab_probs_backward(X, E, w, o["logp"], o["lse"], dlogp=dlogp, dX=dX, dE=dE, temperature=heat)
    x = Sharp(X, E, heat)
    G = torch.zeros_like(x.raw)
    dl = dlogp.double() / torch.tensor(heat, dtype=torch.float32).double().item()
    G[:, 0] = dl[:, 1]
    G.scatter_(1, first.long()[:, None], -dl[:, 1:])
    err = torch.zeros_like(G)
    err.scatter_add_(1, w.long(), 16 * EPS32 * dl.abs().sum(1, keepdim=True).expand(rows, 2).contiguous())
    check_grads(x, dt, dX, dE, G, err, dl.abs().sum(1), torch.ones_like(x.lse))


def test_temperatures_too_low_for_32_bits_are_refused():
    X, E = rand((3, 64), "bf16", 1), rand((90, 64), "bf16", 2)
    for heat in (1e-39, 3e-39, 4.2e-39):  # (1 / T, or 1 / T in units of log 2, is infinite)
        with pytest.raises(d.DnpeffError, match="temperature"):
            d.op_vocab_probs(X, E, lse=empty(3), temperature=heat)
    d.op_vocab_probs(X * 0, E, lse=empty(3), temperature=4.3e-39)


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("rows, words", [(1, 1), (16, 1), (8, 9), (5, 17), (16, 65), (17, 1), (70, 9), (300, 33)])
def test_small_vocabularies_and_exact_workspaces(rows, words, dt):
    """Nothing is written but the results and as much workspace as is asked for: the sums that low temperatures need again lie in it too."""
    heat, top = 2.0**-30, min(words, 4)
    X, E, w = whole((rows, 40), dt, 1), whole((words, 40), dt, 2), words_of(rows, 2, words, 3)
    x = Sharp(X, E, heat)
    sizes = d.vocab_probs_workspace(rows, 40, words, 2, top, DTYPES[dt], True)
    buf = torch.full((max(sizes) + 512,), 123, dtype=torch.uint8, device="cuda")
    o = dict(logp=empty(rows, 2), lse=empty(rows), entropy=empty(rows), top_words=empty(rows, top, dtype=torch.int32), top_logp=empty(rows, top))
    d.op_vocab_probs(X, E, w, temperature=heat, workspace=buf[256 : 256 + sizes[0]], **o)
    assert (buf[:256] == 123).all() and (buf[256 + sizes[0] :] == 123).all()
    want = torch.where(w >= 0, x.log_p.gather(1, w.long().clamp(min=0)), 0.0)
    near(o["logp"], want, 8 * EPS32 * (1 + want.abs()), "logp")
    buf.fill_(123)
    dlogp = rand((rows, 2), "f32", 4) * heat
    dX, dE = torch.zeros_like(X), torch.zeros_like(E)
    d.op_vocab_probs_backward(X, E, w, o["logp"], o["lse"], dlogp=dlogp, dX=dX, dE=dE, temperature=heat, workspace=buf[256 : 256 + sizes[1]])
    assert (buf[:256] == 123).all() and (buf[256 + sizes[1] :] == 123).all()
    dl = torch.where(w >= 0, dlogp.double(), 0.0) / heat
    G = -x.p * dl.sum(1, keepdim=True)
    G.scatter_add_(1, w.long().clamp(min=0), dl)
    err = x.p * 32 * EPS32 * dl.abs().sum(1, keepdim=True)
    err.scatter_add_(1, w.long().clamp(min=0), 16 * EPS32 * dl.abs().sum(1, keepdim=True).expand(rows, 2).contiguous())
    check_grads(x, dt, dX, dE, G, err, dl.abs().sum(1), (dl != 0).any(1).double())


@pytest.mark.parametrize("heat", [1e10, 1e38, 3.4e38])
@pytest.mark.parametrize("rows", [3, 70, 700])
def test_high_temperatures(rows, heat):
    """All words are alike then, the order of the alternatives is that of the products still."""
    X, E, w = whole((rows, 40), "bf16", 1), whole((3000, 40), "bf16", 2), words_of(rows, 3, 3000, 3)
    o = answers(X, E, w, 9, heat)
    v, at = (X.double() @ E.double().T).sort(dim=1, descending=True, stable=True)
    assert torch.equal(o["top_words"], at[:, :9].to(torch.int32))
    even = torch.full((rows, 1), 3000.0, device="cuda").double().log()
    # (sums of 3000 terms)
    near(o["lse"], even[:, 0], 3100 * EPS32 * even[:, 0], "lse")
    near(o["entropy"], even[:, 0], 3100 * EPS32 * even[:, 0], "entropy")
    near(o["logp"], torch.where(w >= 0, -even, 0.0), 3100 * EPS32 * even, "logp")


@pytest.mark.parametrize("rows, dt", [(5, "bf16"), (300, "f16"), (300, "f32")])
def test_captured_at_a_low_temperature(rows, dt):
    X, E, w = whole((rows, 40), dt, 1), whole((9000, 40), dt, 2), words_of(rows, 3, 9000, 3)
    o = dict(logp=empty(rows, 3), lse=empty(rows), entropy=empty(rows), top_words=empty(rows, 5, dtype=torch.int32), top_logp=empty(rows, 5))
    dlogp, dX, dE = rand((rows, 3), "f32", 4) * 1e-3, torch.zeros_like(X), torch.zeros_like(E)
    ws = torch.empty(max(d.vocab_probs_workspace(rows, 40, 9000, 3, 5, DTYPES[dt])), dtype=torch.uint8, device="cuda")

    def step():
        d.op_vocab_probs(X, E, w, temperature=1e-3, workspace=ws, **o)
        d.op_vocab_probs_backward(X, E, w, o["logp"], o["lse"], dlogp=dlogp, dX=dX, dE=dE, temperature=1e-3, workspace=ws)
        return [t.clone() for t in (*o.values(), dX, dE)]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        X.copy_(whole((rows, 40), dt, 10 + i))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
        torch.cuda.synchronize()
