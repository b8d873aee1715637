"""What a model answers and its gradients where the vocabulary goes by in several pieces.  Bounds as for one piece
(test_gpu_vocab_answers)."""

import pytest
import torch

import npeff_ref_amd as d
from test_gpu_vocab_answers import DTYPES, EPS32, Exact, check_grads, empty, near, rand, words_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("rows, words, n_in", [(600, 60_000, 264), (1300, 40_000, 100), (520, 70_000, 515)])
def test_ties_across_pieces(rows, words, n_in, dt):
    """One embedding many times over, more often than a list holds in the small first piece and in what comes after it: the first of
    them lead, whatever products each piece is formed by."""
    X, E = rand((rows, n_in), dt, 1).float(), rand((words, n_in), dt, 2, 0.05)
    v = rand((1, n_in), "f32", 3)
    X = (X + v).to(DTYPES[dt])
    same = torch.cat([torch.arange(70, 1000, 20), torch.arange(1500, words, 701)]).cuda()
    E[same] = (0.3 * v).to(DTYPES[dt])
    top_words, top_logp = empty(rows, 20, dtype=torch.int32), empty(rows, 20)
    d.op_vocab_probs(X, E, top_words=top_words, top_logp=top_logp)
    z = X.double() @ E.double().T
    z[:, same] = z[:, same[:1]]
    at = z.sort(dim=1, descending=True, stable=True).indices[:, :20]
    assert (at == same[:20]).all(1).double().mean() > 0.9
    assert torch.equal(top_words, at.to(torch.int32))
    assert (top_logp[:, :1] == top_logp)[(at == same[:20]).all(1)].all()


def borders(w, piece, words):
    """Some of the listed words are those next to the pieces' borders, the first and the last."""
    at = [0, piece - 1, piece, words - 1] + ([2 * piece - 1, 2 * piece] if 2 * piece < words else [])
    for i, word in enumerate(at):
        w[i::41, i % w.shape[1]] = word
    w[5, :2] = torch.tensor([piece - 1, piece])
    return w


def piece_of(rows, words, planes):
    """Words of a piece of the backward pass, whose gradients of logits take 512 MB at most."""
    most = (512 << 20) // (2 * planes * rows) // 256 * 256
    many = -(-words // most)
    return -(-(-(-words // many)) // 256) * 256


CASES = [(4096, 70_001, 24, "bf16"), (4096, 150_003, 40, "f16"), (2000, 50_001, 20, "f32"), (4100, 47_000, 24, "f32")]


@pytest.mark.parametrize("heat", [0.05, 1.3])
@pytest.mark.parametrize("rows, words, n_in, dt", CASES)
def test_gradients_of_answers_in_pieces(rows, words, n_in, dt, heat):
    piece = piece_of(rows, words, 3 if dt == "f32" else 1)
    assert piece < words and words % piece
    X, E = rand((rows, n_in), dt, 1), rand((words, n_in), dt, 2, min(0.5, 2 * heat))
    w = borders(words_of(rows, 3, words, 3, masked=0.1), piece, words)
    logp, lse, entropy = empty(rows, 3), empty(rows), empty(rows)
    d.op_vocab_probs(X, E, w, logp=logp, lse=lse, entropy=entropy, temperature=heat)
    x = Exact(X, E, heat)
    near(logp, x.logp(w), x.logp_off(w), "logp")
    dlogp, dh = rand((rows, 3), "f32", 4), rand((rows,), "f32", 5, 0.3)
    dlogp[::3], dh[::2] = 0, 0
    dX, dE = torch.zeros_like(X), torch.zeros_like(E)
    d.op_vocab_probs_backward(X, E, w, logp, lse, entropy, dlogp=dlogp, dentropy=dh, dX=dX, dE=dE, temperature=heat)
    dl, dh64 = torch.where(w >= 0, dlogp.double(), 0.0), dh.double()[:, None]
    G = -x.p * (dl.sum(1, keepdim=True) + dh64 * (x.log_p + x.entropy[:, None]))
    G.scatter_add_(1, w.long().clamp(min=0), dl)
    err = x.p * (x.relative + 19 * EPS32) * (dl.abs().sum(1, keepdim=True) + dh64.abs() * (x.log_p.abs() + x.entropy[:, None]))
    err += x.p * dh64.abs() * (x.off + x.off_entropy)[:, None]
    err.scatter_add_(1, w.long().clamp(min=0), 11 * EPS32 * dl.abs().sum(1, keepdim=True).expand(rows, 3).contiguous())
    size = (dl.abs().sum(1) + 8 * dh64[:, 0].abs()) / heat
    check_grads(x, dt, dX, dE, G / heat, (err + 4 * EPS32 * G.abs()) / heat, size, (size > 0).double())


@pytest.mark.parametrize("heat", [0.05, 1.3])
@pytest.mark.parametrize("rows, words, n_in, dt", CASES)
def test_gradients_of_distillation_in_pieces(rows, words, n_in, dt, heat):
    piece = piece_of(rows, words, 3 if dt == "f32" else 1)
    X, E = rand((rows, n_in), dt, 1), rand((words, n_in), dt, 2, min(0.5, 2 * heat))
    w, logits = words_of(rows, 7, words, 3, masked=0.1), rand((rows, 7), "f32", 4, 2.0)
    w = borders(w, piece, words)
    loss, logp, lse = empty(rows), empty(rows, 7), empty(rows)
    d.op_vocab_distill(X, E, w, logits, loss=loss, logp=logp, lse=lse, temperature=heat)
    x = Exact(X, E, heat)
    dl = rand((rows,), "f32", 5)
    dX, dE = torch.zeros_like(X), torch.zeros_like(E)
    d.op_vocab_distill_backward(X, E, w, logits, logp, lse, dl, dX=dX, dE=dE, temperature=heat)
    there = w >= 0
    alive = there.any(1)
    q = torch.softmax(torch.where(there, logits.double(), -1e9) / heat, 1) * there
    spread = torch.where(there, logits.double().max(1, keepdim=True).values - logits, 0.0).clamp(max=200 * heat).max(1).values / heat
    q_off = ((39 + 4 * spread) * EPS32)[:, None]
    weight = torch.where(alive, dl.double(), 0.0)[:, None] / heat
    G = x.p.clone()
    G.scatter_add_(1, w.long().clamp(min=0), -q)
    err = x.p * (x.relative + 8 * EPS32)
    err.scatter_add_(1, w.long().clamp(min=0), q * q_off + 15 * EPS32 * there.double())
    check_grads(x, dt, dX, dE, G * weight, (err + 4 * EPS32 * G.abs()) * weight.abs(), weight[:, 0].abs(), alive.double())
