"""Performance cases of the operators at the two ends of a language model's vocabulary, and of the norm beside them: embedding, layer_norm and
linear_cross_entropy.

Six kinds of pass:

  embed        rows of an embedding table by token number, times a scale, without gradients
  embed-train  the same, forward and backward: the gradient of the whole table
  norm         layer norm over the last dimension, without gradients
  norm-train   the same, forward and backward: the gradients of the input, the weight and the bias
  loss         softmax cross entropy of a projection to the vocabulary, of each token, without gradients
  loss-train   the same averaged over the labelled tokens, forward and backward: the gradients of the hidden states, the projection and its bias

Ranges: 1 to 65536 tokens, tables of 2 to 131072 rows, 8 to 4096 columns (of the projection multiples of 8), float32, float16 and bfloat16.
`labelled` is the share of the tokens that have a label, the others hold -100; `padded` the share of token numbers that are the padding's.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5
IGNORE = -100
PADDING = 1
EMBED_MOST = 65536 * 512            # numbers of the table and of the rows looked up, of the largest cases
NORM_MOST = 32768 * 1024
LOSS_MOST = 8192 * 50265 * 1024     # (labelled token, row of the projection, column) products
LOGITS_MOST = 32768 * 50265         # the plain form holds them all


def listed():
    embed = dict(kind="embed", padded=0.0, scaled=False)
    train = dict(embed, kind="embed-train")
    return [
        # a decoder's next token in a batch of sixteen, half precision: nothing but latency
        dict(embed, name="embed-16-step", tokens=16, rows=50265, columns=768, dtype="f16"),
        # fine-tuning on a few sentences padded to the longest of them: an odd width, every third token the padding
        dict(train, name="embed-train-385-odd", tokens=385, rows=8191, columns=389, dtype="bf16", padded=0.33, scaled=True),
        # the training configuration of the reference, 64 x 512 tokens, hidden 512, half precision
        dict(train, name="embed-train-32768-512", tokens=32768, rows=50265, columns=512, dtype="f16", padded=0.1),
        # one short sentence through a RoBERTa-base layer's norm
        dict(kind="norm", name="norm-17-base", tokens=17, columns=768, dtype="f32"),
        # 32 x 512 tokens of the benchmark's encoder
        dict(kind="norm", name="norm-16384-base", tokens=16384, columns=768, dtype="f32"),
        # a ragged batch of an odd width, which has no wide loads
        dict(kind="norm-train", name="norm-train-2103-odd", tokens=2103, columns=701, dtype="bf16"),
        # the training configuration of the reference
        dict(kind="norm-train", name="norm-train-32768-512", tokens=32768, columns=512, dtype="f16"),
        # scoring a short text's tokens against the benchmark's vocabulary
        dict(kind="loss", name="loss-64-base", tokens=64, rows=50265, columns=768, dtype="bf16", labelled=1.0),
        # validation of masked language modelling at the benchmark's sizes, 32 x 512 tokens of which 15 % are masked
        dict(kind="loss", name="loss-16384-base", tokens=16384, rows=50265, columns=768, dtype="f16", labelled=0.15),
        # fine-tuning in fp32 on a few sentences, every token labelled, sizes that no tile divides
        dict(kind="loss-train", name="loss-train-385-f32", tokens=385, rows=32003, columns=520, dtype="f32", labelled=1.0),
        # a step of masked language modelling at the training configuration of the reference
        dict(kind="loss-train", name="loss-train-32768-512", tokens=32768, rows=50265, columns=512, dtype="f16", labelled=0.15),
        # a step in which every token predicts the next one
        dict(kind="loss-train", name="loss-train-8192-next", tokens=8192, rows=50265, columns=1024, dtype="bf16", labelled=1.0),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choices(["embed", "embed-train", "norm", "norm-train", "loss", "loss-train"], [1, 3, 2, 3, 3, 5])[0]
    while True:
        case = dict(kind=kind, tokens=_log_int(rng, 1, 65536), dtype=rng.choice(["f32", "f16", "f16", "bf16", "bf16"]))
        if kind.startswith("norm"):
            case["columns"] = rng.choice([512, 768, 1024, _log_int(rng, 8, 4096)])
            if 256 <= case["tokens"] * case["columns"] <= NORM_MOST:
                return case
        elif kind.startswith("embed"):
            case.update(rows=rng.choice([50265, _log_int(rng, 2, 131072)]), columns=rng.choice([512, 768, 1024, _log_int(rng, 8, 4096)]),
                        padded=rng.choice([0.0, 0.0, round(rng.random(), 2)]), scaled=rng.random() < 0.5)
            if case["tokens"] * case["columns"] >= 256 and (case["tokens"] + case["rows"]) * case["columns"] <= EMBED_MOST:
                return case
        else:
            case.update(rows=rng.choice([50265, _log_int(rng, 2, 131072)]), columns=8 * rng.choice([64, 96, 128, _log_int(rng, 1, 512)]),
                        labelled=rng.choice([1.0, 1.0, 0.15, round(rng.random(), 2)]))
            if 1 << 16 <= _labelled(case) * case["rows"] * case["columns"] <= LOSS_MOST and case["tokens"] * case["rows"] <= LOGITS_MOST:
                return case


def _labelled(case):
    return max(1, round(case["labelled"] * case["tokens"]))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, N, D = DTYPES[case["dtype"]], case["tokens"], case["columns"]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def token_numbers():        # by Zipf's law, as words are: the n-th of a vocabulary about 1 / n as often as the first
        u = torch.rand(N, generator=gen, device="cuda", dtype=torch.float64)
        return ((case["rows"] + 1.0) ** u - 1).long().clamp(max=case["rows"] - 1)

    def some(share):            # so many of the tokens, anywhere
        chosen = torch.zeros(N, dtype=torch.bool, device="cuda")
        chosen[torch.randperm(N, generator=gen, device="cuda")[:share]] = True
        return chosen

    state = {"kind": case["kind"]}
    if case["kind"].startswith("embed"):
        state["ids"] = torch.where(some(round(case["padded"] * N)), PADDING, token_numbers())
        state["w"] = (0.02 * randn(case["rows"], D)).to(dtype)
        state["scale"] = math.sqrt(D) if case["scaled"] else 1.0
        wanted = ["w"]
    elif case["kind"].startswith("norm"):
        state["x"] = (0.3 * randn(1, D) + (0.5 + torch.rand(N, 1, generator=gen, device="cuda")) * randn(N, D)).to(dtype)
        state["w"], state["b"] = (1 + 0.1 * randn(D)).to(dtype), (0.1 * randn(D)).to(dtype)
        wanted = ["x", "w", "b"]
    else:
        state["x"] = randn(N, D).to(dtype)              # behind a norm
        state["w"] = (1.5 / math.sqrt(D) * randn(case["rows"], D)).to(dtype)
        state["b"] = (0.1 * randn(case["rows"])).to(dtype)
        state["labels"] = torch.where(some(_labelled(case)), token_numbers(), IGNORE)
        wanted = ["x", "w", "b"]
    if case["kind"].endswith("train"):
        # of a loss half precision trains with a scale, or its gradients would be below the type's numbers
        state["g"] = (torch.tensor(65536.0 if dtype == torch.float16 else 1.0, device="cuda") if "labels" in state else randn(N, D).to(dtype))
        for name in wanted:
            state[name].requires_grad_()
    state["wanted"] = wanted
    return state


def run(state):
    kind = state["kind"].split("-")[0]
    if own:
        out = _own(kind, state)
    else:
        out = {"embed": _plain_embed, "norm": _plain_norm, "loss": _plain_loss}[kind](state)
    if "g" not in state:
        return out
    return {"out": out.detach(), "grad": torch.autograd.grad(out, [state[n] for n in state["wanted"]], state["g"])}


def _own(kind, state):
    import lookupffn_amd
    if kind == "embed":
        return lookupffn_amd.embedding(state["ids"], state["w"], scale=state["scale"], padding_idx=PADDING)
    if kind == "norm":
        return lookupffn_amd.layer_norm(state["x"], state["w"], state["b"], eps=EPS)
    return lookupffn_amd.linear_cross_entropy(state["x"], state["w"], state["b"], state["labels"], ignore_index=IGNORE,
                                              reduction="mean" if "g" in state else "none")


# (the gradient of a conversion is a conversion: sums are in 32 bits, rounded once)

def _plain_embed(state):
    ids, w = state["ids"], state["w"]
    rows = w.float()[ids]
    rows = torch.where((ids == PADDING)[:, None], rows.detach(), rows)
    return (rows * state["scale"]).to(w.dtype)


def _plain_norm(state):
    x = state["x"].float()
    away = x - x.mean(-1, keepdim=True)
    y = away * torch.rsqrt((away * away).mean(-1, keepdim=True) + EPS)
    return (y * state["w"].float() + state["b"].float()).to(state["x"].dtype)


def _plain_loss(state):
    labels = state["labels"]
    logits = state["x"].float() @ state["w"].float().T + state["b"].float()
    away = logits - logits.detach().amax(-1, keepdim=True)
    live = labels != IGNORE
    at_label = away.gather(1, torch.where(live, labels, 0)[:, None])[:, 0]
    losses = torch.where(live, away.exp().sum(-1).log() - at_label, 0.0)
    return losses.sum() / live.sum().clamp(min=1) if "g" in state else losses


def work(case):
    size, N, D = DTYPES[case["dtype"]].itemsize, case["tokens"], case["columns"]
    train = case["kind"].endswith("train")
    if case["kind"].startswith("embed"):
        # rows in, rows out; their gradient in, the table's out
        moved = (min(N, case["rows"]) + N) * D * size + 8 * N
        return {"bytes": moved + ((N + case["rows"]) * D * size if train else 0), "flops": (3 if train else 1) * N * D}
    if case["kind"].startswith("norm"):
        # x in, y out; x and the gradient in, the gradient out; weight and bias in, their gradients out
        return {"bytes": ((5 if train else 2) * N + (4 if train else 2)) * D * size, "flops": (20 if train else 8) * N * D}
    n, V = _labelled(case), case["rows"]
    states, weights = n * D * size, V * (D + 1) * size
    if train:           # every state's gradient is written, also those of the tokens without a label; three products
        return {"bytes": states + N * D * size + 2 * weights + 8 * N, "flops": 6 * n * V * D}
    return {"bytes": states + weights + 12 * N, "flops": 2 * n * V * D}


def exact(case, seed):
    """From the definitions, in 64 bits; the gradients are the formulas'."""
    state = {n: t.detach().double() if isinstance(t, torch.Tensor) and t.is_floating_point() else t for n, t in prepare(case, seed).items()}
    g = state.get("g")
    if case["kind"].startswith("embed"):
        ids, w, scale = state["ids"], state["w"], state["scale"]
        out = scale * torch.index_select(w, 0, ids)
        if g is None:
            return out
        use = ids != PADDING
        # equal token numbers side by side: their sum is what the running sum grows by
        order = torch.argsort(ids[use], stable=True)
        numbers, counts = torch.unique_consecutive(ids[use][order], return_counts=True)
        grad = torch.zeros_like(w)
        ends = counts.cumsum(0)
        running = torch.cat((torch.zeros(1, w.shape[1], dtype=torch.float64, device="cuda"), g[use][order].cumsum(0)))
        grad[numbers] = scale * (running[ends] - running[ends - counts])
        return {"out": out, "grad": (grad,)}
    if case["kind"].startswith("norm"):
        x, w, b = state["x"], state["w"], state["b"]
        variance, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
        r = 1 / torch.sqrt(variance + EPS)
        z = (x - mean) * r
        out = z * w + b
        if g is None:
            return out
        h = g * w
        return {"out": out, "grad": (r * (h - h.mean(-1, keepdim=True) - z * (h * z).mean(-1, keepdim=True)), (g * z).sum(0), g.sum(0))}
    # some labelled tokens at a time
    x, w, b, labels = state["x"], state["w"], state["b"], state["labels"]
    at = (labels != IGNORE).nonzero()[:, 0]
    losses = torch.zeros(len(labels), dtype=torch.float64, device="cuda")
    gx, gw, gb = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
    for part in at.split(2048):
        logp = torch.log_softmax(torch.addmm(b, x[part], w.T), 1)
        rows = torch.arange(len(part), device="cuda")
        losses[part] = -logp[rows, labels[part]]
        if g is not None:
            d = logp.exp_()
            d[rows, labels[part]] -= 1
            d *= g / len(at)
            gx[part] = d @ w
            gw += d.T @ x[part]
            gb += d.sum(0)
    return losses if g is None else {"out": losses.sum() / max(1, len(at)), "grad": (gx, gw, gb)}
