"""What the operators of the Fisher producer are timed on: products, grouped products and the loss of a
language model whose per-example Fishers are then factorised.

Four kinds of call:

  linear     Y = act(X W^T + b) + R, forward alone or with its backward pass
  grouped    the same with a weight per group of rows (experts), ragged and empty groups among them
  examples   per-example squared weight gradients: rows of the Fisher, F[e] = (sum over e's tokens of dY^T X)^2
  loss       softmax cross entropy over a vocabulary: token losses alone, or with the gradients of the hidden
             states and of the output embedding

The plain forms compute in 32 bits with elementary torch operations and round once at the end."""

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one token through an up-projection: little more than a launch
        dict(name="lin_1_token", op="linear", rows=1, n_in=1024, n_out=4096, dtype="bf16", act="silu", bias=True,
             residual=False, train=False),
        # a prompt of odd length at widths that no tile and no 16 bytes divide, with residual
        dict(name="lin_1999_odd", op="linear", rows=1999, n_in=1030, n_out=4101, dtype="f16", act="gelu", bias=True,
             residual=True, train=False),
        # a small layer in full precision, forward and backward
        dict(name="lin_train_777_f32", op="linear", rows=777, n_in=1003, n_out=515, dtype="f32", act="silu",
             bias=True, residual=True, train=True),
        # a training step's up-projection, forward and backward
        dict(name="lin_train_8192", op="linear", rows=8192, n_in=4096, n_out=16384, dtype="bf16", act="gelu_tanh",
             bias=True, residual=False, train=True),
        # eight tokens, two experts each, of 32
        dict(name="grp_16_rows", op="grouped", rows=16, groups=32, n_in=1024, n_out=2048, dtype="bf16", act="silu",
             bias=False, skew=0.5, train=False),
        # a few experts, some of them empty, at odd sizes; the last rows belong to none
        dict(name="grp_train_3001_odd", op="grouped", rows=3001, groups=17, n_in=777, n_out=1025, dtype="f16",
             act="gelu", bias=True, skew=1.5, train=True),
        # a training step of 64 experts
        dict(name="grp_train_16384", op="grouped", rows=16384, groups=64, n_in=2048, n_out=4096, dtype="bf16",
             act="silu", bias=False, skew=0.5, train=True),
        # the Fisher rows of one square layer for a batch of short texts
        dict(name="fisher_64_texts", op="examples", examples=64, tokens=256, n_in=1024, n_out=1024, dtype="bf16"),
        # the log likelihood of one token: the output embedding is all there is to read
        dict(name="loss_1_token", op="loss", rows=1, n_in=4096, vocab=32000, dtype="bf16", train=False),
        # a small head in full precision, odd sizes
        dict(name="loss_train_333_f32", op="loss", rows=333, n_in=515, vocab=10007, dtype="f32", train=True),
        # an ordinary batch
        dict(name="loss_train_2000", op="loss", rows=2000, n_in=1024, vocab=50001, dtype="f16", train=True),
        # a large one: the logits alone would take 4.3 GB in 32 bits
        dict(name="loss_train_8192", op="loss", rows=8192, n_in=4096, vocab=131072, dtype="bf16", train=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


ROUND_WIDTHS = (128, 192, 256, 320, 384, 512, 640, 768, 1024, 1280, 1536, 2048, 2560, 4096, 5120, 8192, 10240, 16384)


def _width(rng, lo, hi):
    """Most widths are round, some are whatever a model has."""
    return _log_int(rng, lo, hi) if rng.random() < 0.3 else rng.choice([w for w in ROUND_WIDTHS if lo <= w <= hi])


def draw(rng):
    op = rng.choice(["linear", "linear", "grouped", "grouped", "examples", "loss", "loss"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    train = rng.random() < 0.6
    n_in = _width(rng, 200, 4096)
    # full precision is for the smaller jobs
    budget = 2e11 if dtype == "f32" else 1.5e12
    if op == "examples":
        n_out = _width(rng, 100, 2048)
        n_in = min(n_in, 2048)
        most = max(1, min(64, 200_000_000 // (n_in * n_out)))
        return dict(op=op, examples=_log_int(rng, 1, most), tokens=_log_int(rng, 1, 512), n_in=n_in, n_out=n_out,
                    dtype=dtype)
    if op == "loss":
        vocab = _log_int(rng, 1000, 131_072)
        rows = _log_int(rng, 1, max(1, min(8192, int(budget / (n_in * vocab)))))
        return dict(op=op, rows=rows, n_in=n_in, vocab=vocab, dtype=dtype, train=train)
    # (relu's slope jumps at zero: in full precision one sum that rounds to the other side of it is all the difference)
    act = rng.choice(["none", "gelu", "gelu_tanh", "silu"] + ["relu"] * (dtype != "f32"))
    bias = rng.random() < 0.6
    if op == "linear":
        n_out = _width(rng, 200, 16_384)
        rows = _log_int(rng, 1, max(1, min(16_384, int(budget / (n_in * n_out)))))
        return dict(op=op, rows=rows, n_in=n_in, n_out=n_out, dtype=dtype, act=act, bias=bias,
                    residual=rng.random() < 0.5, train=train)
    n_in = min(n_in, 2048)
    n_out = _width(rng, 200, 4096)
    groups = _log_int(rng, 2, 64)
    rows = _log_int(rng, 1, max(1, min(16_384, int(budget / (n_in * n_out)))))
    return dict(op=op, rows=rows, groups=groups, n_in=n_in, n_out=n_out, dtype=dtype, act=act, bias=bias,
                skew=rng.choice([0.2, 0.5, 1.0, 1.5]), train=train)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _shares(case):
    """How popular the case's experts are: log-normal shares that are the case's, not the seed's."""
    s = np.exp(case["skew"] * np.random.default_rng(case["groups"]).standard_normal(case["groups"]))
    return s / s.sum()


def _ends(sizes):
    return torch.from_numpy(np.concatenate(([0], np.cumsum(sizes))).astype(np.int64)).cuda()


def prepare(case, seed):
    g, op, dtype = _generator(seed), case["op"], DTYPES[case["dtype"]]
    host = np.random.default_rng(int(seed))
    n_in = case["n_in"]
    if op == "examples":
        sizes = host.integers(1, case["tokens"] + 1, case["examples"])
        rows, n_out = int(sizes.sum()), case["n_out"]
        return dict(case=case, ends=_ends(sizes), most=int(sizes.max()), x=_normal(g, (rows, n_in), dtype),
                    dy=_normal(g, (rows, n_out), dtype, 0.05),
                    out=torch.empty((case["examples"], n_out, n_in), device="cuda"))
    rows = case["rows"]
    # activations after a norm: some channels carry more than others
    x = (torch.randn((rows, n_in), generator=g, device="cuda")
         * torch.exp(0.3 * torch.randn(n_in, generator=g, device="cuda"))).to(dtype)
    if op == "loss":
        vocab = case["vocab"]
        s = dict(case=case, x=x, e=_normal(g, (vocab, n_in), dtype, 2.0 / math.sqrt(n_in)),
                 loss=torch.empty(rows, device="cuda"), lse=torch.empty(rows, device="cuda"))
        # labels by a Zipf-like law; one token in eight is a prompt's and has no loss
        u = torch.rand(rows, generator=g, device="cuda")
        s["labels"] = torch.exp(u * math.log(vocab)).to(torch.int32).clamp_(max=vocab) - 1
        if rows > 1:
            s["labels"][torch.rand(rows, generator=g, device="cuda") < 0.125] = -1
        if case["train"]:
            # the mean over the batch, in half precision with a loss scale
            scale = (4096.0 if case["dtype"] == "f16" else 1.0) / rows
            s["dloss"] = torch.full((rows,), scale, device="cuda")
            s["dx"], s["de"] = torch.empty_like(x), torch.empty_like(s["e"])
        return s
    n_out = case["n_out"]
    s = dict(case=case, x=x, y=torch.empty((rows, n_out), device="cuda", dtype=dtype))
    lead = ()
    if op == "grouped":
        lead = (case["groups"],)
        held = rows - min(5, rows // 100)  # the rest of the buffer is padding
        sizes = host.multinomial(held, _shares(case))
        s["ends"], s["most"] = _ends(sizes), int(sizes.max())
    s["w"] = _normal(g, lead + (n_out, n_in), dtype, 1.0 / math.sqrt(n_in))
    s["bias"] = _normal(g, lead + (n_out,), dtype, 0.1) if case["bias"] else None
    s["residual"] = _normal(g, (rows, n_out), dtype) if case.get("residual") else None
    if case["train"]:
        s["dy"] = _normal(g, (rows, n_out), dtype, 0.05)
        s["pre"] = torch.empty_like(s["y"]) if case["act"] != "none" else None
        s["dx"], s["dw"] = torch.empty_like(x), torch.empty_like(s["w"])
        s["db"] = torch.empty_like(s["bias"]) if case["bias"] else None
    return s


# ---- plain forms -----------------------------------------------------------------------------------------------


def _act(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        t = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def _places(s):
    """(row of each place of a [groups, most] table, whether it holds one)."""
    ends, at = s["ends"], torch.arange(s["most"], device="cuda")
    held = at < (ends[1:] - ends[:-1])[:, None]
    return torch.where(held, ends[:-1, None] + at, 0), held


def _padded(v, places):
    row, held = places
    return v.float()[row] * held[..., None]


def _unpadded(v, places, rows):
    row, held = places
    out = torch.zeros((rows, v.shape[-1]), device="cuda")
    out[row[held]] = v[held]
    return out


def _plain_linear(s, places=None):
    case, dtype = s["case"], s["x"].dtype
    rows = case["rows"]
    x = s["x"].float() if places is None else _padded(s["x"], places)
    w = s["w"].float()
    z = x @ w.transpose(-1, -2)
    if s["bias"] is not None:
        z = z + s["bias"].float().unsqueeze(-2)
    y = _act(z, case["act"])
    if places is not None:
        y = _unpadded(y, places, rows)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = dict(y=y.to(dtype))
    if case["train"]:
        dy = s["dy"].float() if places is None else _padded(s["dy"], places)
        dz = dy * _act_slope(z, case["act"])
        dx = dz @ w
        out["dx"] = (dx if places is None else _unpadded(dx, places, rows)).to(dtype)
        out["dw"] = (dz.transpose(-1, -2) @ x).to(dtype)
        if s["bias"] is not None:
            out["db"] = dz.sum(-2).to(dtype)
    return out


def _plain_loss(s):
    x, e = s["x"].float(), s["e"].float()
    labels = s["labels"].long()
    held, at = labels >= 0, labels.clamp(min=0)[:, None]
    z = x @ e.T
    top = z.max(1, keepdim=True).values
    p = torch.exp(z - top)
    total = p.sum(1, keepdim=True)
    lse = torch.log(total) + top
    out = dict(loss=torch.where(held, (lse - z.gather(1, at))[:, 0], 0.0), lse=lse[:, 0])
    if s["case"]["train"]:
        p /= total
        p.scatter_add_(1, at, torch.full_like(lse, -1.0))
        p *= torch.where(held, s["dloss"], 0.0)[:, None]
        out["dx"] = (p @ e).to(s["x"].dtype)
        out["de"] = (p.T @ x).to(s["e"].dtype)
    return out


def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        if op == "linear":
            return _plain_linear(s)
        if op == "loss":
            return _plain_loss(s)
        places = _places(s)
        if op == "grouped":
            return _plain_linear(s, places)
        return dict(squares=(_padded(s["dy"], places).transpose(1, 2) @ _padded(s["x"], places)).square())
    import npeff_ref_amd as d

    if op == "examples":
        d.op_example_grads(s["dy"], s["x"], s["ends"], s["out"], square=True)
        return dict(squares=s["out"])
    if op == "loss":
        d.op_vocab_loss(s["x"], s["e"], s["labels"], s["loss"], s["lse"])
        out = dict(loss=s["loss"], lse=s["lse"])
        if case["train"]:
            d.op_vocab_loss_backward(s["x"], s["e"], s["labels"], s["lse"], s["dloss"], dX=s["dx"], dE=s["de"])
            out.update(dx=s["dx"], de=s["de"])
        return out
    more = dict(act=case["act"], groups=s.get("ends"))
    d.op_linear(s["x"], s["w"], s["y"], bias=s["bias"], residual=s["residual"], pre=s.get("pre"), **more)
    out = dict(y=s["y"])
    if case["train"]:
        d.op_linear_backward(s["dy"], s["x"], s["w"], pre=s["pre"], dX=s["dx"], dW=s["dw"], dbias=s["db"], **more)
        out.update(dx=s["dx"], dw=s["dw"])
        if s["db"] is not None:
            out["db"] = s["db"]
    return out


# ---- the definition in 64 bits ---------------------------------------------------------------------------------

_EXACT_ACT = {
    "none": lambda z: z,
    "relu": torch.nn.functional.relu,
    "silu": torch.nn.functional.silu,
    "gelu": torch.nn.functional.gelu,
    "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh"),
}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    x = s["x"].double().requires_grad_(True)
    if op == "examples":
        ends = s["ends"].tolist()
        rows = zip(ends, ends[1:])
        return dict(squares=torch.stack([(s["dy"][a:b].double().T @ s["x"][a:b].double()) ** 2 for a, b in rows]))
    if op == "loss":
        e = s["e"].double().requires_grad_(True)
        z = x @ e.t()
        loss = torch.nn.functional.cross_entropy(z, s["labels"].long(), ignore_index=-1, reduction="none")
        out = dict(loss=loss.detach(), lse=torch.logsumexp(z.detach(), 1))
        if case["train"]:
            loss.backward(s["dloss"].double())
            out.update(dx=x.grad, de=e.grad)
        return out
    w = s["w"].double().requires_grad_(True)
    b = None if s["bias"] is None else s["bias"].double().requires_grad_(True)
    act = _EXACT_ACT[case["act"]]
    if op == "linear":
        y = act(torch.nn.functional.linear(x, w, b))
    else:
        ends = s["ends"].tolist()
        parts = [act(torch.nn.functional.linear(x[i:j], w[g], None if b is None else b[g]))
                 for g, (i, j) in enumerate(zip(ends, ends[1:]))]
        y = torch.cat(parts + [x.new_zeros((case["rows"] - ends[-1], case["n_out"]))])
    if s["residual"] is not None:
        y = y + s["residual"].double()
    out = dict(y=y.detach())
    if case["train"]:
        y.backward(s["dy"].double())
        out.update(dx=x.grad, dw=w.grad)
        if b is not None:
            out["db"] = b.grad
    return out


def work(case):
    op, size = case["op"], 4 if case["dtype"] == "f32" else 2
    k = case["n_in"]
    if op == "examples":
        rows, n = case["examples"] * (case["tokens"] + 1) / 2, case["n_out"]
        return dict(bytes=size * rows * (n + k) + 4.0 * case["examples"] * n * k, flops=2.0 * rows * n * k)
    rows = case["rows"]
    if op == "loss":
        n = case["vocab"]
        read = size * (rows * k + n * k) + 4 * rows
        if not case["train"]:
            return dict(bytes=read + 8.0 * rows, flops=2.0 * rows * n * k)
        return dict(bytes=read + 12.0 * rows + size * (rows * k + n * k), flops=6.0 * rows * n * k)
    n, weights = case["n_out"], 1.0
    if op == "grouped":  # the weights of the groups that hold a row
        weights = float((1.0 - (1.0 - _shares(case)) ** rows).sum())
    one = size * (rows * (k + n) + weights * n * (k + (1 if case["bias"] else 0)))
    if case.get("residual"):
        one += size * rows * n
    if not case["train"]:
        return dict(bytes=one, flops=2.0 * rows * n * k)
    every = case.get("groups", 1)
    back = size * (rows * (n + k) + every * n * (k + (1 if case["bias"] else 0)))
    return dict(bytes=one + back, flops=6.0 * rows * n * k)
