"""What the operators of a model's answers are timed on: log probabilities of given words with the entropy and the
likeliest alternatives, and distillation from a teacher's likeliest words.

Four kinds of call, all of hidden states X and output embeddings E, at a temperature T (z = X E^T / T):

  probs           log p of given words, log sum exp, entropy, and the n likeliest words with their log p
  probs, train    log p of given words and the entropy, and the gradients of X and E for theirs
  distill         sum_j q_j (log q_j - log p(w_j)), q the softmax over a teacher's listed logits, / T
  distill, train  the same with the gradients of X and E

The plain forms compute in 32 bits with elementary torch operations and round once at the end.  Which of two words next to
each other is the likelier is decided in 64 bits, of equal ones the lower comes first."""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
NEAR = 8  # words past the last alternative whose order is looked at in 64 bits


def listed():
    return [
        # one generated token: its log probability and eight alternatives; the embeddings are all there is to read
        dict(name="probs_1_token", op="probs", rows=1, n_in=4096, vocab=32000, dtype="bf16", given=1, top=8,
             temperature=1.0, train=False),
        # a step of a few sequences in full precision at odd sizes, several candidate words each, a low temperature
        dict(name="probs_13_f32", op="probs", rows=13, n_in=515, vocab=10007, dtype="f32", given=5, top=5,
             temperature=0.7, train=False),
        # an ordinary prompt, scored with twenty alternatives a token
        dict(name="probs_2000", op="probs", rows=2000, n_in=1024, vocab=50001, dtype="f16", given=1, top=20,
             temperature=1.0, train=False),
        # a teacher's batch: the 64 words a token that a student learns from
        dict(name="probs_8192", op="probs", rows=8192, n_in=4096, vocab=131072, dtype="bf16", given=1, top=64,
             temperature=1.0, train=False),
        # training by rewards: log probabilities weighted by them, and a little for the entropy
        dict(name="probs_train_333_f32", op="probs", rows=333, n_in=515, vocab=10007, dtype="f32", given=2, top=0,
             temperature=1.0, train=True),
        dict(name="probs_train_4096", op="probs", rows=4096, n_in=2048, vocab=64000, dtype="bf16", given=1, top=0,
             temperature=1.0, train=True),
        # a student's loss on a handful of tokens
        dict(name="distill_7_tokens", op="distill", rows=7, n_in=2048, vocab=32000, dtype="bf16", listed=32,
             temperature=2.0, train=False),
        # a student's loss on held-out texts
        dict(name="distill_1999_odd", op="distill", rows=1999, n_in=1030, vocab=50001, dtype="f16", listed=100,
             temperature=2.0, train=False),
        # a small head in full precision, forward and backward
        dict(name="distill_train_300_f32", op="distill", rows=300, n_in=768, vocab=10007, dtype="f32", listed=17,
             temperature=1.0, train=True),
        # an ordinary training step of a student, in half precision with a loss scale
        dict(name="distill_train_2000", op="distill", rows=2000, n_in=1024, vocab=50001, dtype="f16", listed=20,
             temperature=1.5, train=True),
        # a large one
        dict(name="distill_train_8192", op="distill", rows=8192, n_in=4096, vocab=131072, dtype="bf16", listed=64,
             temperature=1.0, train=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


ROUND_WIDTHS = (192, 256, 320, 384, 512, 640, 768, 1024, 1280, 1536, 2048, 2560, 4096)


def draw(rng):
    op = rng.choice(["probs", "probs", "distill"])
    train = rng.random() < 0.5
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    n_in = _log_int(rng, 200, 4096) if rng.random() < 0.3 else rng.choice(ROUND_WIDTHS)
    vocab = _log_int(rng, 1000, 131_072)
    # full precision is for the smaller jobs
    budget = 2e11 if dtype == "f32" else 1.5e12
    rows = _log_int(rng, 1, max(1, min(8192, int(budget / (n_in * vocab)))))
    case = dict(op=op, rows=rows, n_in=n_in, vocab=vocab, dtype=dtype, temperature=rng.choice([0.7, 1.0, 1.0, 2.0]),
                train=train)
    if op == "probs":
        case.update(given=rng.choice([1, 1, 2, 5]), top=0 if train else _log_int(rng, 1, 64))
    else:
        case.update(listed=_log_int(rng, 1, 128))
    return case


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _zipf(g, shape, vocab):
    """Words by a Zipf-like law."""
    u = torch.rand(shape, generator=g, device="cuda")
    return torch.exp(u * math.log(vocab)).to(torch.int32).clamp_(max=vocab) - 1


def prepare(case, seed):
    g, dtype = _generator(seed), DTYPES[case["dtype"]]
    rows, n_in, vocab = case["rows"], case["n_in"], case["vocab"]
    e = _normal(g, (vocab, n_in), dtype, 2.0 / math.sqrt(n_in))
    n = case["given"] if case["op"] == "probs" else case["listed"]
    words = _zipf(g, (rows, n), vocab)
    # states after a norm, some channels carrying more than others, that lean to the first of their words
    x = torch.randn((rows, n_in), generator=g, device="cuda")
    x *= torch.exp(0.3 * torch.randn(n_in, generator=g, device="cuda"))
    x += 1.5 * torch.rand((rows, 1), generator=g, device="cuda") * e[words[:, 0].long()].float()
    x = x.to(dtype)
    s = dict(case=case, x=x, e=e, words=words, logp=torch.empty((rows, n), device="cuda"),
             lse=torch.empty(rows, device="cuda"))
    # the mean over the batch, in half precision with a loss scale
    scale = (4096.0 if case["dtype"] == "f16" else 1.0) / rows
    if rows > 1:
        words[torch.rand(rows, generator=g, device="cuda") < 0.125] = -1  # a prompt's tokens
    if case["op"] == "probs":
        s["entropy"] = torch.empty(rows, device="cuda")
        if case["top"]:
            s["top_words"] = torch.empty((rows, case["top"]), device="cuda", dtype=torch.int32)
            s["top_logp"] = torch.empty((rows, case["top"]), device="cuda")
        if case["train"]:
            s["dlogp"] = torch.randn((rows, n), generator=g, device="cuda") * scale
            s["dentropy"] = torch.full((rows,), 0.02 * scale, device="cuda")
    else:
        # a teacher's logits fall off from the first; some lists are shorter
        s["logits"] = (8.0 - 1.2 * torch.randn((rows, n), generator=g, device="cuda").abs().cumsum(1).sqrt())
        length = 1 + (torch.rand(rows, generator=g, device="cuda") * 2 * n).int()
        words[torch.arange(n, device="cuda") >= length[:, None]] = -1
        s["loss"] = torch.empty(rows, device="cuda")
        if case["train"]:
            s["dloss"] = torch.full((rows,), scale, device="cuda")
    if case["train"]:
        s["dx"], s["de"] = torch.empty_like(x), torch.empty_like(e)
    return s


# ---- plain forms -----------------------------------------------------------------------------------------------


def _alternatives(s, z, inv):
    """The likeliest words of z = X E^T / T and their logits: candidates from z, their order from 64 bits."""
    x, e, top = s["x"], s["e"], s["case"]["top"]
    near = z.topk(min(top + NEAR, z.shape[1]), dim=1).indices.sort(1).values
    words, logits = [], []
    step = max(1, (1 << 26) // (near.shape[1] * x.shape[1]))
    for i in range(0, x.shape[0], step):
        at = near[i : i + step]
        v = (e[at].double() * x[i : i + step].double()[:, None]).sum(2)
        v, order = v.sort(dim=1, descending=True, stable=True)
        logits.append(v[:, :top] * inv)
        words.append(at.gather(1, order[:, :top]))
    return torch.cat(words).to(torch.int32), torch.cat(logits)


def _plain(s):
    case = s["case"]
    probs, inv = case["op"] == "probs", 1.0 / case["temperature"]
    x, e = s["x"].float(), s["e"].float()
    held, at = s["words"] >= 0, s["words"].long().clamp(min=0)
    z = x @ e.T
    if case["temperature"] != 1.0:
        z *= inv
    mine, out = z.gather(1, at), {}
    if probs and case["top"]:
        out["top_words"], tops = _alternatives(s, z, inv)
    top = z.max(1, keepdim=True).values
    z -= top
    p = z.exp()
    total = p.sum(1, keepdim=True)
    lse = torch.log(total) + top
    if probs:
        entropy = (torch.log(total) - (p * z).sum(1, keepdim=True) / total)[:, 0]
    p /= total
    logp = torch.where(held, mine - lse, 0.0)
    out["lse"] = lse[:, 0]
    if probs:
        out.update(logp=logp, entropy=entropy)
        if case["top"]:
            out["top_logp"] = (tops - lse).float()
        if not case["train"]:
            return out
        dlogp = torch.where(held, s["dlogp"], 0.0)
        dh = s["dentropy"][:, None]
        # dz = (sum_j dlogp_j ([w_j = v] - p_v) - dH p_v (log p_v + H)) / T
        log_p = z - torch.log(total)
        dz = log_p.add_(entropy[:, None]).mul_(dh).add_(dlogp.sum(1, keepdim=True)).mul_(p).neg_()
        dz.scatter_add_(1, at, dlogp)
    else:
        some = held.any(1)
        # q over the listed words
        logits = torch.where(held, s["logits"] * inv, -math.inf)
        from_top = logits - torch.where(some, logits.max(1).values, 0.0)[:, None]
        weight = from_top.exp()
        total = torch.where(some, weight.sum(1), 1.0)[:, None]
        q = weight / total
        log_q = torch.where(held, from_top - torch.log(total), 0.0)
        out["loss"] = (q * (log_q - logp)).sum(1)
        out["logp"] = logp
        if not case["train"]:
            return out
        p *= some[:, None]
        dz = p.scatter_add_(1, at, -q).mul_(s["dloss"][:, None])
    if case["temperature"] != 1.0:
        dz *= inv
    out["dx"] = (dz @ e).to(s["x"].dtype)
    out["de"] = (dz.T @ x).to(s["e"].dtype)
    return out


def run(s):
    if not own:
        return _plain(s)
    import npeff_ref_amd as d

    case, x, e, words = s["case"], s["x"], s["e"], s["words"]
    out = dict(lse=s["lse"], logp=s["logp"])
    heat = dict(temperature=case["temperature"])
    if case["op"] == "probs":
        tops = dict(top_words=s["top_words"], top_logp=s["top_logp"]) if case["top"] else {}
        d.op_vocab_probs(x, e, words, logp=s["logp"], lse=s["lse"], entropy=s["entropy"], **tops, **heat)
        out.update(entropy=s["entropy"], **tops)
        if case["train"]:
            d.op_vocab_probs_backward(x, e, words, s["logp"], s["lse"], s["entropy"], dlogp=s["dlogp"],
                                      dentropy=s["dentropy"], dX=s["dx"], dE=s["de"], **heat)
    else:
        d.op_vocab_distill(x, e, words, s["logits"], loss=s["loss"], logp=s["logp"], lse=s["lse"], **heat)
        out["loss"] = s["loss"]
        if case["train"]:
            d.op_vocab_distill_backward(x, e, words, s["logits"], s["logp"], s["lse"], s["dloss"], dX=s["dx"],
                                        dE=s["de"], **heat)
    if case["train"]:
        out.update(dx=s["dx"], de=s["de"])
    return out


# ---- the definition in 64 bits ---------------------------------------------------------------------------------


def _exact_rows(case, s, rows):
    """Outputs of some rows, and the gradients of these rows' part of the result."""
    heat = case["temperature"]
    x = s["x"][rows].double().requires_grad_(case["train"])
    e = s["e64"]
    log_p = torch.log_softmax(x @ e.t() / heat, 1)
    words = s["words"][rows].long()
    there = words >= 0
    logp = log_p.gather(1, words.clamp(min=0)).masked_fill(~there, 0.0)
    with torch.no_grad():
        # (log sum exp from a word's logit and its log probability)
        first = words[:, :1].clamp(min=0)
        lse = (x * e[first[:, 0]]).sum(1) / heat - log_p.gather(1, first)[:, 0]
    out = dict(lse=lse, logp=logp.detach())
    if case["op"] == "probs":
        entropy = torch.special.entr(log_p.exp()).sum(1)
        out["entropy"] = entropy.detach()
        if case["top"]:
            v, at = log_p.detach().topk(min(case["top"] + 1, log_p.shape[1]), dim=1)
            at, by_word = at.sort(1)
            v, order = v.gather(1, by_word).sort(dim=1, descending=True, stable=True)
            out["top_logp"] = v[:, : case["top"]]
            out["top_words"] = at.gather(1, order)[:, : case["top"]].to(torch.int32)
        if case["train"]:
            total = (logp * s["dlogp"][rows].double()).sum() + (entropy * s["dentropy"][rows].double()).sum()
    else:
        some = there.any(1, keepdim=True)
        q = torch.softmax((s["logits"][rows].double() / heat).masked_fill(~there & some, -math.inf), 1)
        q = q.masked_fill(~there, 0.0)
        loss = (torch.special.xlogy(q, q) - q * logp).sum(1)
        out["loss"] = loss.detach()
        if case["train"]:
            total = (loss * s["dloss"][rows].double()).sum()
    if case["train"]:
        out["dx"], out["de"] = torch.autograd.grad(total, (x, e))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    s["e64"] = s["e"].double().requires_grad_(case["train"])
    step = max(1, (1 << 27) // case["vocab"])
    parts = [_exact_rows(case, s, slice(i, i + step)) for i in range(0, case["rows"], step)]
    return {k: sum(p[k] for p in parts) if k == "de" else torch.cat([p[k] for p in parts]) for k in parts[0]}


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    rows, k, vocab = case["rows"], case["n_in"], case["vocab"]
    many = case["given"] if case["op"] == "probs" else case["listed"]
    ends = size * (rows * k + vocab * k)
    # words and their log probabilities; log sum exp and the entropy or the loss
    small = rows * (8.0 * many + 8.0)
    if case["op"] == "probs":
        small += rows * 8.0 * case["top"]
    else:
        small += rows * 4.0 * many
    if not case["train"]:
        return dict(bytes=ends + small, flops=2.0 * rows * vocab * k)
    small += rows * (4.0 * many + 4.0 if case["op"] == "probs" else 4.0)
    return dict(bytes=2 * ends + small, flops=6.0 * rows * vocab * k)
