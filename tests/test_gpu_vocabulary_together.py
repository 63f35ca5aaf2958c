"""embedding, layer_norm and linear_cross_entropy together, as a language model's training step has them, and under what stands around PyTorch's operators: captured graphs, streams, forward
mode, hooks on saved tensors, modes, torch.compile, a second gradient."""
import threading
from argparse import Namespace

import pytest
import torch
import torch.autograd.forward_ad as fwAD
import torch.nn.functional as F
from torch.utils.checkpoint import checkpoint

import lookupffn_amd
from lookupffn_amd import embedding, layer_norm, linear_cross_entropy

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True, params=["host", "python"])
def either_path(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(lookupffn_amd._lib, "loaded_host", False)
    else:
        assert lookupffn_amd._lib.host()
    return request.param


def _parts(dtype=torch.float32, seed=0, tokens=(3, 50), rows=700, columns=96):
    """-> (table, norm's weight, norm's bias, bias), (token numbers, labels)"""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    ids, labels = (torch.randint(0, rows, tokens, generator=gen, device=DEV) for _ in range(2))
    labels[torch.rand(tokens, generator=gen, device=DEV) < 0.4] = -100
    return [(0.3 * randn(rows, columns)).to(dtype), 1 + 0.1 * randn(columns), 0.1 * randn(columns), 0.2 * randn(rows)], (ids, labels)


def _model(table, w, b, bias, ids, labels):
    """A table that is both ends of the vocabulary: its gradient is the lookups' and the projection's."""
    return linear_cross_entropy(layer_norm(embedding(ids, table, scale=2.0, padding_idx=3), w, b, eps=1e-5), table, bias, labels)


def _plain(table, w, b, bias, ids, labels):
    rows = torch.where((ids == 3)[..., None], table[ids].detach(), table[ids])
    logits = F.layer_norm(2.0 * rows, (table.shape[1],), w, b, 1e-5) @ table.T + bias
    return F.cross_entropy(logits.flatten(0, 1), labels.flatten())


def _step(call, leaves, rest):
    leaves = [t.detach().clone().requires_grad_() for t in leaves]
    out = call(*leaves, *rest)
    return (out.detach(), *torch.autograd.grad(out, leaves, torch.ones_like(out)))


def _same(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_step_against_64_bits():
    leaves, rest = _parts()
    got = _step(_model, leaves, rest)
    want = _step(_plain, [t.double() for t in leaves], rest)
    # logits of size 6 (columns' norm 10, table rows' 3) are off by some 2^-22 of their products' sizes, 20, and so are a softmax and its gradients, relative to the largest; a norm by 2^-20
    for a, b in zip(got, want):
        assert (a.double() - b).abs().max() <= 2.0 ** -16 * b.abs().max()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_step_of_16_bits(dtype):
    leaves, rest = _parts(dtype)
    got = _step(_model, leaves, rest)
    want = _step(_plain, [t.double() for t in leaves], rest)
    u = torch.finfo(dtype).eps / 2
    # the embedding and the norm round once each: logits of products' sizes 20 move by 2 u 20 at most, the softmax by twice that; d, h's gradient, the norm's and the table's two round once more
    # each; half's gradients (1 / 90 of a token's) also by 2^-25 of 150 tokens
    for a, b in zip(got, want):
        assert (a.double() - b).abs().max() <= (2 * 40 + 8) * u * b.abs().max() + 150 * 2.0 ** -25


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_captured(dtype):
    """Forward and backward in a graph, replayed with other inputs and the program's own work between."""
    leaves, rest = _parts(dtype)
    leaves = [t.requires_grad_() for t in leaves]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(_model(*leaves, *rest), leaves)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _model(*leaves, *rest)
        grads = torch.autograd.grad(out, leaves)
    for seed in range(4):
        new, new_rest = _parts(dtype, seed)
        if seed == 2:
            new_rest[1].fill_(-100)                 # nobody has a label
        with torch.no_grad():
            for a, b in zip((*leaves, *rest), (*new, *new_rest)):
                a.copy_(b)
        want = _step(_model, new, new_rest)
        graph.replay()
        torch.cuda.synchronize()
        assert _same((out, *grads), want)
        torch.randn(1 << 20, device=DEV).sum().item()


def test_two_captured_graphs_replayed_in_turn():
    made = []
    for seed in range(2):
        leaves, rest = _parts(seed=seed, tokens=(2, 1500 + 700 * seed))
        leaves = [t.requires_grad_() for t in leaves]
        want = _step(_model, leaves, rest)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _model(*leaves, *rest)
            got = (out.detach(), *torch.autograd.grad(out, leaves))
        made.append((graph, got, want, leaves, rest))
    for _ in range(3):
        for m in made:
            m[0].replay()
        torch.cuda.synchronize()
        assert all(_same(m[1], m[2]) for m in made)
        torch.randn(1 << 20, device=DEV).sum().item()


def test_a_graph_from_before_the_capture_is_refused():
    (table, w, b, bias), (ids, labels) = _parts()
    leaves = [t.requires_grad_() for t in (table, w, b, bias)]
    x = torch.randn(4, 96, device=DEV).requires_grad_()
    calls = [lambda: embedding(ids, table), lambda: layer_norm(x, w, b), lambda: linear_cross_entropy(x, table, bias, labels.flatten()[:4])]
    eager = [call() for call in calls]
    if lookupffn_amd._lib.host_module() is None:
        pytest.skip("without the host library no forward with gradients is captured")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        for call in calls:
            with pytest.raises(RuntimeError, match="graph from before the capture"):
                call()
        with torch.no_grad():
            inside = [call() for call in calls]
    graph.replay()
    torch.cuda.synchronize()
    assert _same(inside, eager) and leaves


def test_two_streams_and_threads():
    """Calls at once, on streams of their own."""
    jobs = [(_parts(seed=s, tokens=(2, 300 + 100 * s)), torch.cuda.Stream()) for s in range(4)]
    want = [_step(_model, *parts) for parts, _ in jobs]
    torch.cuda.synchronize()
    got = [None] * len(jobs)

    def work(i):
        parts, stream = jobs[i]
        with torch.cuda.stream(stream):
            for _ in range(3):
                got[i] = _step(_model, *parts)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert all(_same(a, b) for a, b in zip(got, want))


def test_a_tangent_is_refused():
    (table, w, b, bias), (ids, labels) = _parts()
    x, y = torch.randn(6, 96, device=DEV), labels.flatten()[:6]
    for recorded in (False, True):
        with torch.set_grad_enabled(recorded), fwAD.dual_level():
            dual = lambda t: fwAD.make_dual(t, torch.ones_like(t))  # noqa: E731
            for call in (lambda: embedding(ids, dual(table)), lambda: layer_norm(dual(x), w, b), lambda: layer_norm(x, dual(w), b), lambda: layer_norm(x, w, dual(b)),
                         lambda: linear_cross_entropy(dual(x), table, bias, y), lambda: linear_cross_entropy(x, dual(table), bias, y),
                         lambda: linear_cross_entropy(x, table, dual(bias), y)):
                with pytest.raises((NotImplementedError, RuntimeError)):
                    call()
            assert torch.equal(layer_norm(x, w, b), layer_norm(x, w, b))


def test_torch_func():
    (table, w, b, bias), (ids, labels) = _parts()
    x, y = torch.randn(3, 5, 96, device=DEV), labels[:, :5].contiguous()
    assert torch.equal(torch.vmap(lambda t: layer_norm(t, w, b))(x), layer_norm(x, w, b))
    assert torch.equal(torch.vmap(lambda i: embedding(i, table))(ids), embedding(ids, table))
    got = torch.vmap(lambda t, u: linear_cross_entropy(t, table, bias, u, reduction="none"))(x, y)
    assert torch.equal(got, torch.stack([linear_cross_entropy(t, table, bias, u, reduction="none") for t, u in zip(x, y)]))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: layer_norm(t, w, b).sum())(x)


def test_hooks_on_saved_tensors_and_checkpoints():
    leaves, rest = _parts(torch.float16)
    want = _step(_model, leaves, rest)
    packed = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(t.cpu()) or packed[-1], lambda t: t.to(DEV)):
        got = _step(_model, leaves, rest)
    assert packed and _same(got, want)
    got = _step(lambda *a: checkpoint(_model, *a, use_reentrant=False), leaves, rest)
    assert _same(got, want)


def test_what_hooks_give_back_in_another_type_or_shape_is_refused():
    leaves, rest = _parts()
    x = torch.randn(6, 96, device=DEV)
    y = rest[1].flatten()[:6]
    # (of int64 numbers: as 16 bits, and fewer of them)
    for change in (lambda t: t.half() if t.is_floating_point() else t.short(), lambda t: t[:-1]):
        for call in (lambda *p: embedding(rest[0], p[0]), lambda *p: layer_norm(x, p[1], p[2]), lambda *p: linear_cross_entropy(x, p[0], p[3], y)):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change), pytest.raises((RuntimeError, AssertionError)):
                _step(lambda *p: call(*p).sum() + sum(t.sum() for t in p), leaves, ())
    torch.cuda.synchronize()


def test_an_input_that_changes_before_the_backward_is_noticed():
    (table, w, b, bias), (ids, labels) = _parts()
    y = labels.flatten()[:6]
    x = torch.randn(6, 96, device=DEV)
    for n, call in ((1, lambda i, t: embedding(i, t)), (2, lambda p, q: layer_norm(p, q, b)), (3, lambda p, q, u: linear_cross_entropy(p, q, bias, u))):
        given = {1: (ids, table), 2: (x, w), 3: (x, table, y)}[n]
        for changed in range(n):
            inputs = [t.clone().requires_grad_() * 1 if t.is_floating_point() else t.clone() for t in given]
            out = call(*inputs)
            inputs[changed].zero_()
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                out.sum().backward()


def test_gradients_of_gradients_are_refused():
    leaves, rest = _parts()
    x, y = torch.randn(6, 96, device=DEV).requires_grad_(), rest[1].flatten()[:6]
    table, w, b, bias = (t.requires_grad_() for t in leaves)
    for call, of in ((lambda: embedding(rest[0], table), table), (lambda: layer_norm(x, w, b), x), (lambda: linear_cross_entropy(x, table, bias, y), x)):
        g, = torch.autograd.grad(call().square().sum(), of, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiated|differentiate twice|once_differentiable"):
            g.square().sum().backward()


def test_watched_calls():
    class Seen(torch.utils._python_dispatch.TorchDispatchMode):
        names = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            Seen.names.append(str(func))
            return func(*args, **(kwargs or {}))

    leaves, rest = _parts()
    want = _step(_model, leaves, rest)
    with Seen():
        got = _step(_model, leaves, rest)
    assert _same(got, want)
    assert {f"lookupffn.{n}.default" for n in ("embedding", "embedding_bwd", "layer_norm", "layer_norm_rows_bwd", "linear_cross_entropy", "linear_cross_entropy_bwd")} <= set(Seen.names)


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled(backend):
    torch._dynamo.reset()
    leaves, rest = _parts()
    compiled = torch.compile(_model, backend=backend, fullgraph=True)
    with torch.no_grad():
        assert torch.equal(compiled(*leaves, *rest), _model(*leaves, *rest))
    want = _step(_model, leaves, rest)
    for _ in range(2):
        assert _same(_step(compiled, leaves, rest), want)


def test_memory_stays_bounded():
    """The logits of 16384 tokens and 30000 entries in fp32 would be 2 GB; the calls stay below their documented workspaces."""
    x, table = torch.randn(16384, 64, device=DEV, dtype=torch.float16).requires_grad_(), torch.randn(30000, 64, device=DEV, dtype=torch.float16).requires_grad_()
    y = torch.randint(0, 30000, (16384,), device=DEV)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    loss = linear_cross_entropy(x, table, None, y)
    torch.cuda.synchronize()
    # 8 bytes for 256 logits, the rows once more, a few numbers a token and entry
    assert torch.cuda.max_memory_allocated() - before <= 16384 * (118 * 8 + 128 * 2 + 100) + 30000 * 8 + (4 << 20)
    torch.autograd.grad(loss, (x, table))
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before <= (1 << 30) + (256 << 20) + (64 << 20)


CONFIG = dict(hidden_size=128, num_attention_heads=2, attention_head_size=64, attention_probs_dropout_prob=0.0, hidden_dropout_prob=0.0, layer_norm_eps=1e-5, num_hidden_layers=2,
              vocab_size=1003, max_position_embeddings=80, type_vocab_size=2, pad_token_id=1, ffn_num_table=16, ffn_table_size=256, projection_type="bh4", block_size=1)


def _batch(config, shape=(3, 40)):
    gen = torch.Generator(device=DEV).manual_seed(5)
    ids = torch.randint(2, config.vocab_size, shape, generator=gen, device=DEV)
    mask = (torch.arange(shape[1], device=DEV) < torch.tensor([[40], [23], [31]], device=DEV)).float()
    ids = torch.where(mask > 0, ids, config.pad_token_id)
    labels = torch.where((torch.rand(shape, generator=gen, device=DEV) < 0.3) & (mask > 0), ids, -100)
    return (ids, torch.zeros_like(ids), torch.arange(shape[1], device=DEV).expand(shape), mask), labels


def test_the_head_against_64_bits():
    torch.manual_seed(0)
    config = Namespace(**CONFIG)
    head = lookupffn_amd.MaskedLMHead(config).to(DEV)
    torch.nn.init.normal_(head.bias, std=0.2)
    states, table = torch.randn(3, 40, 128, device=DEV).requires_grad_(), (0.2 * torch.randn(1003, 128, device=DEV)).requires_grad_()
    _, labels = _batch(config)
    leaves = [states, table, *head.parameters()]
    loss = head(states, table, labels)
    grads = torch.autograd.grad(loss, leaves)
    import copy
    head64, states64, table64 = copy.deepcopy(head).double(), states.detach().double().requires_grad_(), table.detach().double().requires_grad_()
    hidden = head64.LayerNorm(F.gelu(head64.dense(states64)))
    logits = hidden @ table64.T + head64.bias
    want = F.cross_entropy(logits.flatten(0, 1), labels.flatten())
    # a projection, a norm, a projection of 128 columns and a softmax in fp32: logits off by some 2^-19, gradients as much relative to the largest
    assert abs(loss.item() - want.item()) <= 2.0 ** -17
    for a, b in zip(grads, torch.autograd.grad(want, [states64, table64, *head64.parameters()])):
        assert (a.double() - b).abs().max() <= 2.0 ** -16 * b.abs().max()
    out = head(states, table)
    assert out.shape == (3, 40, 1003) and (out.double() - logits).abs().max() <= 2.0 ** -15


def test_the_embeddings_kernels_change_no_number():
    torch.manual_seed(0)
    config = Namespace(**CONFIG)
    plain = lookupffn_amd.RobertaEmbeddings(config).to(DEV)
    kernels = lookupffn_amd.RobertaEmbeddings(config, kernels=True).to(DEV)
    kernels.load_state_dict(plain.state_dict())
    (ids, types, positions, _), _ = _batch(config)
    a, b = plain(ids, types, positions), kernels(ids, types, positions)
    assert torch.equal(a, b)
    g = torch.randn_like(a)
    want = torch.autograd.grad(a, list(plain.parameters()), g)
    for (name, _), x, y in zip(plain.named_parameters(), torch.autograd.grad(b, list(kernels.parameters()), g), want):
        # sums of up to 120 numbers in another order
        assert (x - y).abs().max() <= 120 * 2.0 ** -23 * y.abs().max(), name
    with torch.autocast("cuda", dtype=torch.float16):
        assert torch.equal(plain(ids, types, positions), kernels(ids, types, positions))
    plain.word_embeddings.max_norm = kernels.word_embeddings.max_norm = 1.0          # another lookup: torch's
    assert torch.equal(plain(ids, types, positions), kernels(ids, types, positions))


def test_the_model_trains():
    """Forward, backward and a step of an optimizer, in fp32 and under autocast: every parameter has a finite gradient, and the tied table both ends'."""
    torch.manual_seed(0)
    config = Namespace(**CONFIG)
    model = lookupffn_amd.LookupForMaskedLM(config).to(DEV)
    batch, labels = _batch(config)
    for autocast in (False, True):
        model.zero_grad()
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            loss = model(*batch, labels)
        loss.backward()
        assert loss.isfinite() and all(p.grad is not None and p.grad.isfinite().all() and p.grad.dtype == p.dtype for p in model.parameters())
        table = model.encoder.embeddings.word_embeddings.weight.grad
        seen = torch.zeros(config.vocab_size, dtype=torch.bool, device=DEV)
        seen[batch[0].flatten()] = True
        # (rows that no token has get theirs from the projection alone, zeros where a logit is so far below a token's largest that its share, below 2^-38, is none)
        assert (table[seen].abs().sum(1) > 0).all() and (table[~seen].abs().sum(1) > 0).any() and table[seen].abs().mean() > table[~seen].abs().mean()
        torch.optim.SGD(model.parameters(), lr=0.1).step()
    model.eval()
    with torch.no_grad():
        logits = model(*batch)
        loss = model(*batch, labels)
    assert logits.shape == (3, 40, config.vocab_size)
    assert abs(loss.item() - F.cross_entropy(logits.flatten(0, 1).double(), labels.flatten()).item()) <= 1e-5
