"""The way from texts to Fishers by the model's own answers and by a teacher's (npeff_ref_amd.lm_fishers), against autograd in 64 bits.

fp32: sums of at most 5000 terms, a few layers deep: relative errors of about 1e-6 of a result's largest entries, so 2e-5 of its
norm bounds them; squares double that."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def plain(p, tokens, c):
    """(log probabilities, h) in 64 bits with h's gradient kept, with the experts that the model's own scores chose; and the weights."""
    q = {k: v.double().cpu().requires_grad_(True) for k, v in p.items()}
    out_emb = p["emb"].double().cpu().requires_grad_(True)
    x = q["emb"].detach()[tokens.cpu()]
    a = torch.nn.functional.silu(x @ q["w1"].T + q["b1"])
    h = x + a @ q["w2"].T
    h.retain_grad()
    order, ends = c["order"].cpu(), c["ends"].tolist()
    y = h.clone()
    for g, (i, j) in enumerate(zip(ends, ends[1:])):
        rows = order[i:j]
        y = y.index_add(0, rows, torch.nn.functional.gelu(h[rows] @ q["we"][g].T))
    return y @ out_emb.T, h, a, q, out_emb


def near(got, exact, bound):
    assert (got.double().cpu() - exact).norm() <= bound * exact.norm()


@pytest.mark.parametrize("dtype,bound", [(torch.float32, 2e-5), (torch.bfloat16, 0.05)])
def test_fishers_by_the_models_own_answers(dtype, bound):
    from npeff_ref_amd import lm_fishers as lm

    s = lm.Sizes(words=700, width=48, inner=72, experts=5, examples=12, tokens=25, keep=300, rank=4, steps=30, answers=3)
    p = lm.init(s, dtype)
    tokens, labels, ends = lm.texts(s)
    _, c = lm.forward(p, tokens, labels)
    rows = lm.answer_fisher_rows(p, c, ends, s.answers)
    z, h, a, _, _ = plain(p, tokens, c)
    log_p, at = torch.log_softmax(z, 1), ends.tolist()
    words = lm.likeliest(p, c, s.answers)[0].cpu().long()
    if dtype == torch.float32:
        assert torch.equal(words, z.topk(s.answers, dim=1).indices)
    exact = torch.zeros(s.examples, 48, 72, dtype=torch.float64)
    for e, (i, j) in enumerate(zip(at, at[1:])):
        for y in words[j - 1]:
            (dh,) = torch.autograd.grad(log_p[j - 1, y], h, retain_graph=True)
            exact[e] += log_p[j - 1, y].exp().detach() * (dh[i:j].T @ a[i:j].detach()) ** 2
    near(rows, exact.flatten(1), 2 * bound)
    W, H, columns, history = lm.factorise(rows, s, log=lambda _line: None)
    assert W.shape == (12, 4) and np.isfinite(W).all() and np.isfinite(H).all() and history[0][1] > history[-1][1] > 0


@pytest.mark.parametrize("dtype,bound", [(torch.float32, 2e-5), (torch.bfloat16, 0.05)])
@pytest.mark.parametrize("heat", [1.0, 1.5])
def test_a_student_learns_from_a_teacher(dtype, bound, heat):
    """The teacher's likeliest words, the student's losses and every gradient, and Fishers from them."""
    from npeff_ref_amd import lm_fishers as lm

    s = lm.Sizes(words=700, width=48, inner=72, experts=5, examples=20, tokens=25, answers=6)
    p, other = lm.init(s, dtype), lm.init(s, dtype, seed=1)
    tokens, labels, ends = lm.texts(s)
    _, c = lm.forward(p, tokens, labels)
    words, logp = lm.likeliest(other, lm.forward(other, tokens, labels)[1], s.answers)
    loss, t = lm.learn_from(p, c, words, logp, heat)
    grads, dh = lm.backward(p, c, torch.ones_like(loss), t)
    rows = lm.fisher_rows(c, dh, ends)

    z, h, a, q, out_emb = plain(p, tokens, c)
    teach = torch.softmax(logp.double().cpu() / heat, 1)
    want = (teach * (teach.log() - torch.log_softmax(z / heat, 1).gather(1, words.long().cpu()))).sum(1)
    want.sum().backward()
    near(loss, want.detach(), bound)
    near(dh, h.grad, bound)
    for k in ("w1", "b1", "w2", "we"):
        near(grads[k], q[k].grad, bound)
    near(grads["emb"], out_emb.grad, bound)
    at = ends.tolist()
    exact = torch.stack([(h.grad[i:j].T @ a[i:j].detach()) ** 2 for i, j in zip(at, at[1:])])
    near(rows, exact.flatten(1), 2 * bound)


@pytest.mark.parametrize("by", ["labels", "answers", "teacher"])
def test_the_command(by, capsys):
    from npeff_ref_amd import lm_fishers as lm

    lm.main(by)
    out = capsys.readouterr().out
    assert out.count("component ") == lm.Sizes().rank and ("teacher" in out) == (by == "teacher")
