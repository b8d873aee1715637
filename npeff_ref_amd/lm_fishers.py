"""From texts to a factorisation: the per-example Fishers of a small token model, made and factorised on the GPU.

What the reference leaves to TensorFlow (npeff/fishers/d_pefs_computer.py:126-145) in one place, with this package's operators:

  forward    x = emb[tokens];  a = silu(x W1^T + b1);  h = x + a W2^T;  experts: y = h + gelu(h_e We^T) of each token's expert;
             token losses of y against the vocabulary
  backward   the gradients of every weight, and of the hidden states on the way
  Fishers    F[e] = (sum over e's tokens of dh_t^T a_t)^2, the row of example e for W2, its largest entries as a PEF
  NMF        rows normalised, empty columns dropped, F ~ W H

    python -m npeff_ref_amd.lm_fishers

The model is a stand-in of random weights (sizes below); a real one calls the same operators with its own arrays."""

from __future__ import annotations

import math
from dataclasses import dataclass

import numpy as np
import torch

from . import binding as d


@dataclass
class Sizes:
    words: int = 5000
    width: int = 128
    inner: int = 256
    experts: int = 4
    examples: int = 48
    tokens: int = 60  # at most, per example
    keep: int = 2048  # entries of a Fisher row that its PEF keeps
    rank: int = 8
    steps: int = 40


def init(s: Sizes, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    return dict(
        emb=normal(s.words, s.width, scale=0.2),
        w1=normal(s.inner, s.width, scale=s.width**-0.5),
        b1=normal(s.inner, scale=0.1),
        w2=normal(s.width, s.inner, scale=s.inner**-0.5),
        router=normal(s.experts, s.width, scale=s.width**-0.5),
        we=normal(s.experts, s.width, s.width, scale=s.width**-0.5),
    )


def texts(s: Sizes, seed=0):
    """(tokens, labels, ends of the examples): every token's label is the one after it, the last has none."""
    host = np.random.default_rng(seed)
    sizes = host.integers(2, s.tokens + 1, s.examples)
    ends = np.concatenate(([0], np.cumsum(sizes))).astype(np.int64)
    tokens = np.exp(host.random(ends[-1]) * math.log(s.words)).astype(np.int64) - 1
    labels = np.append(tokens[1:], -1).astype(np.int32)
    labels[ends[1:] - 1] = -1
    return (torch.from_numpy(a).cuda() for a in (tokens, labels, ends))


def forward(p, tokens, labels):
    """Token losses and what the backward pass needs."""
    x = p["emb"][tokens]
    rows, width = x.shape
    c = dict(x=x, labels=labels)
    c["a"], c["z1"] = x.new_empty(rows, p["w1"].shape[0]), x.new_empty(rows, p["w1"].shape[0])
    d.op_linear(x, p["w1"], c["a"], bias=p["b1"], act="silu", pre=c["z1"])
    c["h"] = torch.empty_like(x)
    d.op_linear(c["a"], p["w2"], c["h"], residual=x)
    # each token to the expert that scores it highest; rows in the order of their experts
    experts = p["router"].shape[0]
    scores = x.new_empty(rows, experts)
    d.op_linear(c["h"], p["router"], scores)
    expert = scores.argmax(1)
    c["order"] = torch.argsort(expert, stable=True)
    count = torch.bincount(expert, minlength=experts)
    c["ends"] = torch.cat([count.new_zeros(1), count.cumsum(0)])
    c["h_e"] = c["h"][c["order"]]
    y_e, c["z_e"] = torch.empty_like(c["h_e"]), torch.empty_like(c["h_e"])
    d.op_linear(c["h_e"], p["we"], y_e, act="gelu", residual=c["h_e"], pre=c["z_e"], groups=c["ends"])
    c["y"] = torch.empty_like(y_e)
    c["y"][c["order"]] = y_e
    loss, c["lse"] = torch.empty(rows, device=x.device), torch.empty(rows, device=x.device)
    d.op_vocab_loss(c["y"], p["emb"], labels, loss, c["lse"])
    return loss, c


def backward(p, c, dloss):
    """Gradients of the weights (the router's choices are taken as given, the embedding's are those of the output side), and of
    the log likelihood by W2's output."""
    g = {k: torch.empty_like(p[k]) for k in ("emb", "w1", "b1", "w2", "we")}
    dy = torch.empty_like(c["y"])
    d.op_vocab_loss_backward(c["y"], p["emb"], c["labels"], c["lse"], dloss, dX=dy, dE=g["emb"])
    dy_e = dy[c["order"]]
    dh_e = torch.empty_like(dy_e)
    d.op_linear_backward(dy_e, c["h_e"], p["we"], pre=c["z_e"], act="gelu", dX=dh_e, dW=g["we"], groups=c["ends"])
    dh = dy.clone()
    dh[c["order"]] += dh_e
    da = torch.empty_like(c["a"])
    d.op_linear_backward(dh, c["a"], p["w2"], dX=da, dW=g["w2"])
    d.op_linear_backward(da, c["x"], p["w1"], pre=c["z1"], act="silu", dW=g["w1"], dbias=g["b1"])
    return g, dh


def fisher_rows(c, dh, ends):
    """[examples, width * inner]: the diagonal Fisher of W2 of every example, by its own labels."""
    out = torch.empty((ends.shape[0] - 1, dh.shape[1], c["a"].shape[1]), device=dh.device)
    d.op_example_grads(dh, c["a"], ends, out, square=True)
    return out.flatten(1)


def factorise(rows, s: Sizes, log=print):
    """PEFs of the rows and their factors: (W [examples, rank], H [rank, kept columns], columns, history)."""
    torch.cuda.current_stream().synchronize()  # the library's calls below are on its own stream
    values, indices, norms = d.topk_rows(d.DeviceArray.view(rows), s.keep)
    A = d.Csr.from_pef(indices, values, rows.shape[1])
    A.normalize_rows(norms)
    A.compact_columns(1)
    nmf = d.MuNmf(A, d.MuNmfParams(rank=s.rank, max_iters=s.steps))
    history = nmf.run(log=log)
    out = nmf.loadWToHostSync(), nmf.loadHToHostSync(), A.kept_indices(), history
    nmf.close()
    A.close()
    return out


def main():
    s = Sizes()
    p = init(s)
    tokens, labels, ends = texts(s)
    loss, c = forward(p, tokens, labels)
    print(f"{s.examples} examples, {len(tokens)} tokens, mean loss {loss.sum().item() / (labels >= 0).sum().item():.4f}")
    # the Fisher of an example is that of its summed log likelihood: every labelled token counts once
    _, dh = backward(p, c, torch.ones_like(loss))
    rows = fisher_rows(c, dh, ends)
    W, H, columns, _ = factorise(rows, s)
    for k in range(s.rank):
        top = np.argsort(-W[:, k])[:4]
        print(f"component {k}: examples {top.tolist()}, {int((H[k] > 0).sum())} of {len(columns)} columns")


if __name__ == "__main__":
    main()
