"""linear_cross_entropy and its gradients in 64 bits, some tokens at a time, with bounds in which a token's errors go by its own row, its own gradient and the entries' own rows."""
import torch

E = 2.0 ** -24


def reference(h, w, b, y, c, logits_kept=False, chunk=2048):
    """c: [tokens], what a token's loss is multiplied with; y: a number of the vocabulary, or anything else without a label.
    -> (losses, grad h, grad w, grad b), their bounds.

    A logit: K / 2 + 16 roundings (an instruction adds two products at least) of sums that are at most S, its products' sizes, and of float32 2^-21 S of two terms and 2^-21 of each row's
    largest number times the other row's sizes (a number is held to 2^-22 of its row's largest), of which no more than 2^-18 is the backward's alone.
    An entry that is 105 below the others' sum by more than these errors has an exponential of zero, exactly, and no part in anything.  A token with one entry left has a softmax of one,
    as both directions' logits are off by no more than 2^-18 from each other; with more, the softmax moves by twice the logits' errors, an argument's rounding and 2^-20.
    d: those, and its rounding (2^-21 of two terms, otherwise the type's), float32's to 2^-30 of the token's own gradient, half's to 2^-37 of the largest token's.
    Gradients: d's errors times the other operand, roundings of sums (two products an instruction), of float32 2^-21 of the other operand's row's largest; a rounding to the type."""
    kind, device = h.dtype, h.device
    u, two = torch.finfo(kind).eps / 2, kind == torch.float32
    bu = torch.finfo(kind if b is None else b.dtype).eps / 2
    tiny = torch.finfo(kind).smallest_normal * 2.0 ** -8
    h, w, c = h.detach().double(), w.detach().double(), c.double().to(device)
    (N, K), V = h.shape, len(w)
    b = torch.zeros(V, dtype=torch.float64, device=device) if b is None else b.detach().double()
    y = y.long()
    live = (y >= 0) & (y < V)
    c = torch.where(live, c.expand(N), 0.0)
    most_w, sizes_w = w.abs().amax(1), w.abs().sum(1)
    loss, of_loss, gh, of_gh = (torch.zeros(s, dtype=torch.float64, device=device) for s in ((N,), (N,), (N, K), (N, K)))
    gw, of_gw, gb, of_gb = (torch.zeros(s, dtype=torch.float64, device=device) for s in ((V, K), (V, K), (V,), (V,)))
    for at in live.nonzero()[:, 0].split(chunk):
        x, t, k = h[at], y[at][:, None], c[at][:, None]
        most_x, sizes_x = x.abs().amax(1, keepdim=True), x.abs().sum(1, keepdim=True)
        logits, sizes = x @ w.T + b, x.abs() @ w.abs().T
        of = (K / 2 + 16) * E * sizes + 2 * E * (sizes + b.abs())
        if two:
            of += 2.0 ** -21 * sizes + 2.0 ** -36 * (most_x * sizes_w + sizes_x * most_w)
            of_both = of + (2.0 ** -21 * (most_x * sizes_w + sizes_x * most_w)).clamp(max=2.0 ** -18)
        else:
            of_both = of
        lse = torch.logsumexp(logits, 1, keepdim=True)
        best = logits.argmax(1, keepdim=True)
        near = lse - logits <= 105 + of_both + of_both.gather(1, best)
        p = torch.where(near, (logits - lse).exp(), 0.0)
        span = torch.where(near, lse - logits, 0.0).amax(1, keepdim=True)
        worst = torch.where(near, of, 0.0).amax(1, keepdim=True)
        loss[at] = (lse - logits.gather(1, t))[:, 0]
        # (the rounding of a level is that of both its exponentials and its logarithm)
        of_loss[at] = (worst + of.gather(1, t) + (span + (lse - logits.gather(1, t)).abs()) * 4 * E + 2.0 ** -20)[:, 0]
        moved = torch.expm1(2 * torch.where(near, of_both, 0.0).amax(1, keepdim=True) + span * 4 * E + 2.0 ** -20)
        of_p = torch.where(near.sum(1, keepdim=True) == 1, torch.full_like(moved, 2.0 ** -17), moved)
        # (an entry's share is between 0 and 1, whatever the errors)
        d, of_d = p.clone(), torch.where(near, (p * of_p).nan_to_num(1.0).clamp(max=1.0), 0.0)
        d.scatter_add_(1, t, torch.full_like(t, -1, dtype=torch.float64))
        of_d.scatter_add_(1, t, torch.full_like(t, 1, dtype=torch.float64) * E)
        d, of_d = d * k, of_d * k.abs()
        of_d += (2.0 ** -21 if two else u) * d.abs() + near * (2.0 ** -30 * k.abs() if two else 2.0 ** -37 * c.abs().max() if kind == torch.float16 else 0.0)
        size = d.abs()
        gh[at] = d @ w
        of_gh[at] = of_d @ w.abs() + (V / 2 + 80) * E * (size @ w.abs()) + (2.0 ** -21 * size @ most_w[:, None] if two else 0.0)
        gw += d.T @ x
        of_gw += of_d.T @ x.abs() + (N / 2 + 80) * E * (size.T @ x.abs()) + (2.0 ** -21 * size.T @ most_x if two else 0.0)
        gb += d.sum(0)
        of_gb += of_d.sum(0) + (N / 2 + 80) * E * size.sum(0)
    return (loss, gh, gw, gb), (of_loss + E * loss.abs() + 1e-30, of_gh + u * gh.abs() + tiny, of_gw + u * gw.abs() + tiny, of_gb + bu * gb.abs() + tiny)


def worst(got, want, bound):
    """The largest error, in bounds; infinity where a result is not finite."""
    assert got.shape == want.shape
    if not got.isfinite().all():
        return float("inf")
    return ((got.double() - want).abs() / bound).max().item() if got.numel() else 0.0
