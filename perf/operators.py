"""Performance cases of the operators around the encoder's states: qk_norm_rotary and cross_attention.

Four kinds of pass:

  norm         queries and keys normed for each head and rotated to their positions, without gradients
  norm-train   the same, forward and backward: the gradients of queries, keys and both weights
  attend       attention of queries to the states of an encoder, without gradients; single tokens over kept keys and values are query=1
  attend-train the same, forward and backward: the gradients of queries, keys and values

Ranges: 1 to 32768 rows of queries, 1 to 32768 keys, heads of 16 to 128 columns, one to eight query heads for a key head, float32, float16 and
bfloat16.  `pad` is the share of the keys that the shortest sequence of a batch lacks (1: a sequence with no state at all).
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6
POSITIONS = 8192                # rows of the rotation's table
NORM_MOST = 32768 * 16 * 64     # columns of queries and keys together, of the largest cases
ATTEND_MOST = 64 * 8 * 512 * 2048 * 64
ATTEND_BYTES = 1 << 28          # of keys and values
SCORES_MOST = 4 * 16 * 2048 * 4096
TRAIN_MOST = SCORES_MOST * 128


def listed():
    norm = dict(kind="norm", packed=False, interleaved=False)
    attend = dict(kind="attend", pad=0.0)
    return [
        # a decoder's next token in a batch of sixteen: the queries of one step, half precision
        dict(norm, name="norm-16-step", batch=16, query=1, key=0, heads=12, key_heads=12, columns=64, rotary=64, dtype="f16"),
        # self-attention of the RoBERTa-base encoder, 32 x 512 tokens, from one fused projection
        dict(norm, name="norm-16384-base", batch=32, query=512, key=512, heads=12, key_heads=12, columns=64, rotary=64, dtype="f32", packed=True),
        # a ragged batch of queries against longer states, shared key heads, half of the columns rotated, pairs side by side
        dict(norm, name="norm-train-385-shared", kind="norm-train", batch=5, query=77, key=131, heads=16, key_heads=4, columns=128, rotary=64,
             dtype="bf16", interleaved=True),
        # the training configuration of the reference: 64 x 512 tokens, hidden 512, half precision
        dict(norm, name="norm-train-32768-512", kind="norm-train", batch=64, query=512, key=512, heads=8, key_heads=8, columns=64, rotary=64,
             dtype="f16"),
        # a decoder's next token in a batch of sixteen sentences
        dict(attend, name="attend-16-step", batch=16, query=1, key=512, heads=12, key_heads=12, columns=64, dtype="f16", pad=0.5),
        # the next token over long documents, four query heads for a key head
        dict(attend, name="attend-4-step-long", batch=4, query=1, key=16384, heads=32, key_heads=8, columns=128, dtype="bf16", pad=0.25),
        # a few pooling queries over ragged sentences: an odd length, too few rows to fill the chip
        dict(attend, name="attend-33-701", batch=3, query=11, key=701, heads=12, key_heads=12, columns=64, dtype="f32", pad=1.0),
        # 32 sentences against the states of the benchmark's encoder, fp32
        dict(attend, name="attend-16384-base", batch=32, query=512, key=512, heads=12, key_heads=12, columns=64, dtype="f32", pad=0.3),
        # the training configuration of the reference: 64 targets of 128 tokens against 512 states
        dict(attend, name="attend-train-8192-512", kind="attend-train", batch=64, query=128, key=512, heads=8, key_heads=8, columns=64,
             dtype="f16", pad=0.3),
        # fine-tuning in fp32 at the RoBERTa-base heads, odd lengths
        dict(attend, name="attend-train-f32", kind="attend-train", batch=8, query=333, key=509, heads=12, key_heads=12, columns=64, dtype="f32",
             pad=0.5),
        # long targets against long documents
        dict(attend, name="attend-train-long", kind="attend-train", batch=4, query=2048, key=4096, heads=16, key_heads=16, columns=128,
             dtype="bf16"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choices(["norm", "norm-train", "attend", "attend-train"], [2, 2, 5, 4])[0]
    train = kind.endswith("train")
    while True:
        key_heads, group = rng.choice([1, 2, 3, 4, 8, 12, 16]), rng.choice([1, 1, 1, 2, 4, 8])
        columns = rng.choice([64, 64, 64, 128, 128, 32, 16, 8 * rng.randint(2, 16)])
        case = dict(kind=kind, batch=_log_int(rng, 1, 64), heads=key_heads * group, key_heads=key_heads, columns=columns,
                    dtype=rng.choice(["f32", "f16", "f16", "bf16", "bf16"]))
        if kind.startswith("norm"):
            case.update(query=_log_int(rng, 1, 4096), key=rng.choice([0, _log_int(rng, 1, 4096)]), rotary=rng.choice([0, columns // 16 * 16, 16]),
                        packed=rng.random() < 0.3, interleaved=rng.random() < 0.3)
            if case["packed"]:
                case["key"] = case["query"]
            if 4096 <= _norm_columns(case) <= NORM_MOST:
                return case
        else:
            case.update(query=_log_int(rng, 1, 4096) if train else rng.choice([1, 1, rng.randint(1, 16), _log_int(rng, 1, 4096)]),
                        key=_log_int(rng, 1, 32768), pad=rng.choice([0.0, 0.0, round(rng.random(), 2), 1.0]))
            scores = case["batch"] * case["heads"] * case["query"] * case["key"]
            kept = 2 * case["batch"] * case["key_heads"] * case["key"] * columns * DTYPES[case["dtype"]].itemsize
            if 1 << 16 <= scores * columns <= (TRAIN_MOST if train else ATTEND_MOST) and scores <= SCORES_MOST and kept <= ATTEND_BYTES:
                return case


def _norm_columns(case):
    return case["batch"] * (case["query"] * case["heads"] + case["key"] * case["key_heads"]) * case["columns"]


def _lengths(case):
    """How many of its keys each sequence has: from all to what `pad` leaves, evenly."""
    batch, key = case["batch"], case["key"]
    return [key - int(case["pad"] * key * b / max(1, batch - 1)) for b in range(batch)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, B, D = DTYPES[case["dtype"]], case["batch"], case["columns"]
    Lq, Lk, Hq, Hk = case["query"], case["key"], case["heads"], case["key_heads"]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda").to(dtype)

    state = {"kind": case["kind"]}
    if case["kind"].startswith("norm"):
        if case["packed"]:          # one projection of queries, keys and values, as a fused product leaves them
            qkv = randn(B, Lq, Hq + 2 * Hk, D)
            state["q"], state["k"] = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk]
        else:
            state["q"], state["k"] = randn(B, Lq, Hq, D), randn(B, Lk, Hk, D) if Lk else None
        for name in ("qw", "kw"):
            state[name] = 1 + 0.1 * torch.randn(D, generator=gen, device="cuda")
        state["interleaved"], state["table"] = case["interleaved"], None
        if case["rotary"]:
            half = case["rotary"] // 2
            angle = (torch.arange(POSITIONS, device="cuda", dtype=torch.float64)[:, None]
                     * 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half))
            state["table"] = torch.cat((angle.cos(), angle.sin()), 1).float()
        # every sequence begins somewhere
        first = torch.randint(0, POSITIONS - max(Lq, Lk), (B, 1), generator=gen, device="cuda")
        state["qp"] = first + torch.arange(Lq, device="cuda")
        state["kp"] = first + torch.arange(Lk, device="cuda")
        grads = ["q", "qw"] + (["k", "kw"] if Lk or case["packed"] else [])
        if case["kind"] == "norm-train":
            state["gq"] = randn(B, Lq, Hq, D)
            state["gk"] = None if state["k"] is None else randn(*state["k"].shape)
    else:
        state["q"] = randn(B, Lq, Hq, D)
        kv = randn(B, Lk, 2, Hk, D)                 # one projection of keys and values
        state["k"], state["v"] = kv[:, :, 0], kv[:, :, 1]
        lengths = torch.tensor(_lengths(case))[torch.randperm(B, generator=torch.Generator().manual_seed(seed))].cuda()
        state["mask"] = None if case["pad"] == 0 else torch.arange(Lk, device="cuda") < lengths[:, None]
        grads = ["q", "k", "v"]
        if case["kind"] == "attend-train":
            state["g"] = randn(B, Lq, Hq, D)
    if case["kind"].endswith("train"):
        for name in grads:
            state[name] = state[name].detach().requires_grad_()
    return state


def _norm_rotary(x, weight, table, positions, interleaved):
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
    if table is None:
        return y
    rotary = table.shape[1]
    cos, sin = table[positions][:, :, None].chunk(2, -1)
    first, rest = y[..., :rotary], y[..., rotary:]
    if interleaved:
        a, b = first[..., ::2], first[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = first.chunk(2, -1)
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, rest), -1)


def _attend(q, k, v, mask):
    """In heads-first order; key heads are repeated for the query heads that share them."""
    B, Lq, Hq, D = q.shape
    group = Hq // k.shape[2]
    q = q.permute(0, 2, 1, 3)
    k, v = (t.permute(0, 2, 1, 3).repeat_interleave(group, 1) for t in (k, v))
    s = torch.matmul(q * D ** -0.5, k.transpose(-1, -2))
    if mask is not None:
        s = s.masked_fill(~mask[:, None, None], -math.inf)
    m = s.detach().amax(-1, keepdim=True)
    p = (s - torch.where(m == -math.inf, 0.0, m)).exp()
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)     # a sequence without states: zeros
    return torch.matmul(p, v).permute(0, 2, 1, 3)


def run(state):
    kind = state["kind"]
    if kind.startswith("norm"):
        names = [n for n in ("q", "k", "qw", "kw") if state["k"] is not None or n[0] == "q"]
        outputs = _own_norm(state) if own else _plain_norm(state, names)
        if kind == "norm":
            return outputs
        grads = [state["gq"]] + ([] if state["k"] is None else [state["gk"]])
    else:
        names = ["q", "k", "v"]
        outputs = _own_attend(state) if own else _plain_attend(state)
        if kind == "attend":
            return outputs
        grads = [state["g"]]
    return {"out": [o.detach() for o in outputs], "grad": torch.autograd.grad(outputs, [state[n] for n in names], grads)}


def _own_norm(state):
    import lookupffn_amd
    q, k = lookupffn_amd.qk_norm_rotary(state["q"], state["k"], state["qw"], state["kw"], table=state["table"], q_positions=state["qp"],
                                        k_positions=state["kp"], eps=EPS, interleaved=state["interleaved"])
    return [q] if k is None else [q, k]


def _own_attend(state):
    import lookupffn_amd
    return [lookupffn_amd.cross_attention(state["q"], state["k"], state["v"], state["mask"])]


def _plain_norm(state, names):
    # (the gradient of a conversion is a conversion: sums are in 32 bits, rounded once)
    return [_norm_rotary(state[n].float(), state[n + "w"], state["table"], state[n + "p"], state["interleaved"]).to(state[n].dtype)
            for n in names if len(n) == 1]


def _plain_attend(state):
    q, k, v = (state[n].float() for n in "qkv")
    return [_attend(q, k, v, state["mask"]).to(state["q"].dtype)]


def work(case):
    size, columns = DTYPES[case["dtype"]].itemsize, case["columns"]
    if case["kind"].startswith("norm"):
        n = _norm_columns(case)
        # x in, y out; x and the gradient in, the gradient out; a row of the table for each position
        moved = (5 if case["kind"] == "norm-train" else 2) * n * size + case["batch"] * (case["query"] + case["key"]) * (4 * case["rotary"] + 8)
        return {"bytes": moved, "flops": (25 if case["kind"] == "norm-train" else 8) * n}
    keys = sum(_lengths(case))
    row = case["heads"] * columns * size
    queries, states = case["batch"] * case["query"] * row, keys * case["key_heads"] * columns * size
    products = case["heads"] * case["query"] * keys * columns
    if case["kind"] == "attend":
        return {"bytes": 2 * queries + 2 * states, "flops": 4 * products}
    every = case["batch"] * case["key"] * case["key_heads"] * columns * size       # the gradients of what takes no part are written as well
    return {"bytes": 4 * queries + 2 * states + 2 * every, "flops": 14 * products}


def exact(case, seed):
    """From the definitions, in 64 bits; the gradients are the formulas'."""
    state = {n: t.detach().double() if isinstance(t, torch.Tensor) and t.is_floating_point() else t for n, t in prepare(case, seed).items()}
    if case["kind"].startswith("norm"):
        every = [_exact_norm(state[n], state[n + "w"], state["table"], state[n + "p"], case, state.get("g" + n))
                 for n in ("q", "k") if state[n] is not None]
        outputs = [e[0] for e in every]
        if case["kind"] == "norm":
            return outputs
        return {"out": outputs, "grad": [e[1] for e in every] + [e[2] for e in every]}
    # a sequence at a time: only the keys that take part
    q, k, v, g = state["q"], state["k"], state["v"], state.get("g")
    out, gq, gk, gv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    group, scale = q.shape[2] // k.shape[2], 1 / math.sqrt(q.shape[3])
    for b in range(q.shape[0]):
        use = slice(None) if state["mask"] is None else state["mask"][b]
        kb, vb = k[b][use], v[b][use]
        if not kb.shape[0]:
            continue
        dk, dv = torch.zeros_like(kb), torch.zeros_like(vb)
        for h in range(k.shape[2]):
            for n in range(h * group, (h + 1) * group):
                p = torch.softmax(scale * (q[b, :, n] @ kb[:, h].T), 1)
                out[b, :, n] = p @ vb[:, h]
                if g is not None:
                    dv[:, h] += p.T @ g[b, :, n]
                    dp = g[b, :, n] @ vb[:, h].T
                    ds = p * (dp - (p * dp).sum(1, keepdim=True)) * scale
                    gq[b, :, n] = ds @ kb[:, h]
                    dk[:, h] += ds.T @ q[b, :, n]
        gk[b][use], gv[b][use] = dk, dv
    return [out] if g is None else {"out": [out], "grad": [gq, gk, gv]}


def _exact_norm(x, w, table, positions, case, g):
    n, rotary = x.shape[-1], case["rotary"]
    r = 1 / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / n + EPS)
    y = x * r * w
    if rotary:
        half = rotary // 2
        at = torch.arange(half, device=x.device)
        a, b = (2 * at, 2 * at + 1) if case["interleaved"] else (at, at + half)
        # as complex numbers: a rotation is a product with e^(i angle)
        turn = torch.complex(table[:, :half], table[:, half:])[positions][:, :, None]
        z = torch.complex(y[..., a], y[..., b]) * turn
        y[..., a], y[..., b] = z.real, z.imag
    if g is None:
        return y, None, None
    h = g.clone()
    if rotary:
        z = torch.complex(g[..., a], g[..., b]) * turn.conj()
        h[..., a], h[..., b] = z.real, z.imag
    xr = x * r
    return y, r * (h * w - xr * (h * w * xr).mean(-1, keepdim=True)), (h * xr).sum((0, 1, 2))
