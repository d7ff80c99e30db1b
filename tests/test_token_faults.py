"""Faults found in the token-model operators, one test each: what a call answered wrongly, and what it answers."""
import math

import pytest
import torch

import beyond_deep_ensembles_amd as bde
from tests.test_token_ops import F32, BF16, U, backend, gen, teacher  # noqa: F401  (backend: the fixture)


@pytest.mark.gpu
@pytest.mark.parametrize("path", ["nodes", "python"])
def test_forward_and_backward_captured_into_two_graphs(path, monkeypatch):
    """The backward's graph computes the gradient itself at every replay: the forward's graph may not run in between, the caller
    may have changed the last result in place, and the upstream value may have been another one."""
    if path == "python":
        import beyond_deep_ensembles_amd.bbb_layers as L
        monkeypatch.setattr(L, "_native_nodes", lambda ops: None)
    dev = "cuda:0"
    z, values, indices, rest = (t.to(dev) for t in teacher(20, 2000, 8, F32, 0))

    def eager(logits, factor):
        y = logits.clone().requires_grad_()
        (g,) = torch.autograd.grad(bde.distillation_loss(y, values, indices, rest), y, torch.tensor(factor, device=dev))
        return g
    want = {f: eager(z, f) for f in (1.0, 0.5)}
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        x = z.clone().requires_grad_()                 # (a leaf of this stream's)
        up = torch.ones((), device=dev)
        forward, backward = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        s.synchronize()
        with torch.cuda.graph(forward, stream=s):
            loss = bde.distillation_loss(x, values, indices, rest)
        with torch.cuda.graph(backward, stream=s):
            (g,) = torch.autograd.grad(loss, x, up)
    torch.cuda.current_stream().wait_stream(s)

    def run(graph):
        graph.replay()
        torch.cuda.synchronize()
    run(forward)
    run(backward)
    assert torch.equal(g, want[1.0])
    up.fill_(0.5)
    run(backward)
    assert torch.equal(g, want[0.5])
    up.fill_(1.0)
    run(backward)
    assert torch.equal(g, want[1.0]), "what an upstream value of 0.5 left"
    g.mul_(3.0)
    run(backward)
    assert torch.equal(g, want[1.0]), "what the caller made of the last gradient"
    with torch.no_grad():
        x.add_(torch.randn(x.shape, generator=gen(1)).to(dev))
    run(forward)
    run(backward)
    assert torch.equal(g, eager(x.detach(), 1.0))


@pytest.mark.gpu
def test_two_steps_captured_into_graphs_of_their_own():
    """Each graph holds a forward and its backward: both still take the gradient the forward pass finished, and neither takes the
    other's."""
    dev = "cuda:0"
    sides = [[t.to(dev) for t in teacher(12, 3000, 5, BF16, seed)] for seed in (1, 2)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(s):
        leaves = [side[0].clone().requires_grad_() for side in sides]
        s.synchronize()
        for x, side in zip(leaves, sides):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                loss = bde.distillation_loss(x, *side[1:])
                (g,) = torch.autograd.grad(loss, x)
            graphs.append(graph)
            outs.append((loss, g))
            del loss, g
    torch.cuda.current_stream().wait_stream(s)
    for order in ((0, 1), (1, 0), (1, 1), (0, 0)):
        for i in order:
            graphs[i].replay()
            torch.cuda.synchronize()
            y = sides[i][0].clone().requires_grad_()
            want = bde.distillation_loss(y, *sides[i][1:])
            (gy,) = torch.autograd.grad(want, y)
            assert torch.equal(outs[i][0], want) and torch.equal(outs[i][1], gy)
            outs[i][1].zero_()


# ---- masks of the type's lowest value, temperatures below 1: against a reference that subtracts the row's maximum before it
# divides by the temperature (numbers of 3e38 lose everything else otherwise), with tolerances that no mask widens
def log_shares(x, tau, dim=1):
    """log softmax(x / tau) in 64 bits; -inf where x is -inf, and rows of -inf alone are -inf."""
    x = x.double()
    top = x.amax(dim, keepdim=True)
    y = (x - torch.where(top == -math.inf, 0.0, top)) / tau
    return y - torch.log(torch.exp(y).sum(dim, keepdim=True))


def masked_distill64(z, values, indices, rest, tau):
    """Losses of the rows, d loss / d z and, per row, the largest difference of exponents that a share above 2^-126 comes from."""
    n, v = z.shape
    # the teacher in units of the temperature, relative to its largest entry (rest already is in those units)
    t = values.double()
    top = t.amax(1, keepdim=True)
    r = torch.full((n, 1), -math.inf, dtype=torch.float64) if rest is None else rest.double()[:, None] - top / tau
    t = torch.cat([(t - top) / tau, r], 1)
    t = t - t.amax(1, keepdim=True)
    lp = t - torch.log(torch.exp(t).sum(1, keepdim=True))
    p = lp.exp()
    listed = torch.zeros(n, v, dtype=torch.bool).scatter_(1, indices, True)
    lq = log_shares(z, tau)
    inside = log_shares(z.masked_fill(listed, -math.inf), tau)              # shares among the others alone
    zd = z.double()
    others = zd.masked_fill(listed, -math.inf)
    o_top, top = others.amax(1, keepdim=True), zd.amax(1, keepdim=True)
    l_tail = (o_top - top) / tau + torch.log(torch.exp((others - o_top) / tau).sum(1, keepdim=True)) - torch.log(torch.exp((zd - top) / tau).sum(1, keepdim=True))
    both = torch.cat([lq.gather(1, indices), l_tail], 1)
    terms = torch.where(p > 2.0 ** -126, p * (lp - both), 0.0)
    q = lq.exp()
    spread_p = torch.zeros(n, v, dtype=torch.float64).scatter_add_(1, indices, p[:, :-1])
    other = torch.where(p[:, -1:] > 0, p[:, -1:] * inside.exp(), 0.0)
    grad = torch.where(listed, q - spread_p, q - other) / tau
    size = torch.where(listed, q + spread_p, q + other) / tau

    def reach(x, share):
        return torch.where(share > 2.0 ** -126, (x - x.amax(1, keepdim=True)).abs() / tau, 0.0).amax(1)
    spread = reach(zd, q) + reach(others, inside.exp()) + reach(values.double(), p[:, :-1])
    return terms.sum(1), terms.abs().sum(1), grad, size, spread


def check_masked(backend, z, values, indices, rest, tau):
    ops, dev = backend
    put = lambda t: None if t is None else t.to(dev)                    # noqa: E731
    x = z.to(dev).requires_grad_()
    rows = bde.distillation_loss(x, put(values), put(indices), put(rest), temperature=tau, reduction="none", _ops=ops)
    (got,) = torch.autograd.grad(rows, x, torch.ones_like(rows))
    want, size, grad, gsize, spread = masked_distill64(z, values, indices, rest, tau)
    # exponents: log2(e) / tau three roundings off, a difference and a product one each, relative to the spread of what has a
    # share; exp and log one step (2 u) each and ln 2 one; sums of v <= 64 and K <= 8 terms; the products of a term and their sum
    rel = (5 * spread + 2 * 64 + 40) * U
    rows = rows.detach().cpu().double()
    # where a masked class has a share p, the term is p (relative error rel, as everywhere) times a difference of exponents of
    # 1e38: one rounding for that difference, two for the temperature (its inverse, the product), one for the product with p and
    # three for its place in the sum -- relative to the term, so 8 u of the sizes' sum beside rel
    off = (rows - want).abs()
    bound = rel * (size + 2) + 8 * U * size
    assert torch.isfinite(want).all() and (off <= bound).all(), f"losses {rows.tolist()}, expected {want.tolist()}"
    off = (got.cpu().double() - grad).abs() - (gsize * (rel + 6 * U)[:, None] + grad.abs() * U + 2.0 ** -125)
    assert off.max().item() <= 0, f"gradient {off.max().item():.3e} beyond the tolerance"


LOWEST = torch.finfo(F32).min


@pytest.mark.parametrize("tau", [0.5, 0.6, 1.0, 2.0])
@pytest.mark.parametrize("what", ["some_others", "others", "a_listed", "all", "teacher", "teacher_and_others", "teacher_entry"])
def test_distill_masked_with_the_lowest_value(backend, what, tau):
    """Classes the student masks, classes the teacher masks, and a teacher whose whole list is masked (uniform over the list where
    nothing is left beside it).  Masked classes that the teacher gives something make losses of 1e35 and more: finite as long as
    they fit."""
    z, values, indices, rest = teacher(6, 30, 5, F32, 11, tau)
    # little is left beside the list, so that a loss of the others' masks fits fp32 at every temperature here
    rest = torch.logsumexp(values.double() / tau, 1).float() - 6.0
    listed = torch.zeros(6, 30, dtype=torch.bool).scatter_(1, indices, True)
    if what == "some_others":
        z = z.masked_fill(~listed & (torch.arange(30) % 3 == 0), LOWEST)
    elif what == "others":
        z = z.masked_fill(~listed, LOWEST)
    elif what == "a_listed":
        values[:, 2] = values.amin(1) - 8.0 * tau                       # the masked class has a small share
        z.scatter_(1, indices[:, 2:3], LOWEST)
    elif what == "all":
        z = torch.full_like(z, LOWEST)
    elif what == "teacher_entry":
        values[:, 1:3] = LOWEST
    else:
        values = torch.full_like(values, LOWEST)
        rest = torch.full_like(rest, -math.inf)
        if what == "teacher_and_others":
            z = z.masked_fill(~listed, LOWEST)
    check_masked(backend, z, values, indices, rest, tau)


@pytest.mark.parametrize("tau", [0.5, 1.0])
def test_the_masked_reference_notices_small_mistakes(tau):
    """The oracle's tolerances are those of the kernel, not of the mask: a loss off by 1%, a uniform teacher's share of 1."""
    z, values, indices, rest = teacher(6, 30, 5, F32, 11, tau)
    values, rest = torch.full_like(values, LOWEST), torch.full_like(rest, -math.inf)
    want, size, grad, gsize, spread = masked_distill64(z, values, indices, rest, tau)
    rel = (5 * spread + 2 * 64 + 40) * U
    assert (0.01 * want.abs() > rel * (size + 2)).all()
    p = torch.full((6, 5), 0.2, dtype=torch.float64)
    # the same loss by hand: five classes of a fifth each against the student's log-shares
    lq = log_shares(z, tau).gather(1, indices)
    assert torch.allclose((p * (math.log(0.2) - lq)).sum(1), want, rtol=0, atol=1e-12)
    assert (0.8 / tau > 1000 * (gsize * rel[:, None]).max()).all()


@pytest.mark.parametrize("tau", [0.5, 1.0])
@pytest.mark.parametrize("v,k", [(50, 7), (3001, 20)])
def test_topk_rest_of_rows_masked_with_the_lowest_value(backend, v, k, tau):
    """The masked classes add nothing to the rest, and widen no tolerance."""
    ops, dev = backend
    z = torch.randn(2, v, generator=gen(v))
    z = z.masked_fill(torch.rand(2, v, generator=gen(v + 1)) < 0.5, LOWEST)
    got = bde.topk_logits(z.to(dev), k, temperature=tau, _ops=ops)
    order = torch.sort(z.double(), dim=1, descending=True, stable=True)
    assert torch.equal(got.indices.cpu(), order.indices[:, :k]) and torch.equal(got.values.cpu().double(), order.values[:, :k])
    left = order.values[:, k:]
    top = left[:, :1]
    want = top[:, 0] / tau + torch.log(torch.exp((left - top) / tau).sum(1))
    spread = 2 * 8.0 / tau                             # (the normal numbers here lie within 4 of 0)
    assert ((got.rest.cpu().double() - want).abs() <= U * (56 + v / 8192 + 8 * spread) + 4 * U * want.abs()).all()


# ---- the gradient of large tables (the kernels alone: no autograd node lies between)
@pytest.fixture(params=["emu", pytest.param("hip", marks=pytest.mark.gpu)])
def kernels(request):
    if request.param == "emu":
        from tests.hip_emu import build, emu_ops
        if not build.available():
            pytest.skip("no host clang / HIP headers to build the CPU model with")
        with emu_ops.emulated(emu_ops.ALL) as ops:
            yield ops, torch.device("cpu")
        return
    from beyond_deep_ensembles_amd.ops import HipOps
    yield HipOps(), torch.device("cuda:0")


def check_table_gradient(kernels, n, v, d, dtype, seed, pad):
    """The lookup's gradient over a table of many rows against float64 sums of the touched rows; all other rows are zero."""
    ops, dev = kernels
    g = gen(seed)
    tokens = (v * torch.rand(n, generator=g, dtype=torch.float64) ** 3).long()
    tokens[:4] = torch.tensor([v - 1, 0, -1, v])                        # the ends, and two outside
    tokens[n // 2:n // 2 + n // 8] = v - 2                              # a run of its own
    grad = torch.randn(n, d, generator=g).to(dtype)
    got = torch.full((v, d), 7.0, device=dev)
    ops.embedding_bwd(grad.to(dev), tokens.to(dev), got, scale=0.5, padding_idx=pad)
    if dev.type != "cpu":
        again = torch.full((v, d), 7.0, device=dev)
        ops.embedding_bwd(grad.to(dev), tokens.to(dev), again, scale=0.5, padding_idx=pad)
        assert torch.equal(got, again)
    live = (tokens >= 0) & (tokens < v) & (tokens != pad)
    rows, place = torch.unique(tokens[live], return_inverse=True)
    want = torch.zeros(len(rows), d, dtype=torch.float64).index_add_(0, place, grad[live].double()) * 0.5
    size = torch.zeros(len(rows), d, dtype=torch.float64).index_add_(0, place, grad[live].double().abs()) * 0.5
    count = torch.bincount(place, minlength=len(rows)).double()[:, None]
    # count terms added one by one (parts of a sum only shorten the chain), the scale exact
    assert ((got.cpu()[rows].double() - want).abs() <= size * (count + 1) * U * 1.01).all()
    got[rows.to(dev)] = 0.0
    assert int(torch.count_nonzero(got)) == 0


@pytest.mark.parametrize("n,v,d,dtype", [(700, 131073, 2, F32), (600, 262145, 1, BF16), (600, 262208, 3, F32), (49200, 262208, 1, BF16),
                                         (49999, 530001, 1, F32)])
def test_embedding_gradient_of_large_tables(kernels, n, v, d, dtype):
    """Several launches over more workgroups than the device has at once; many tokens over more groups than they are dealt out
    to."""
    if kernels[1].type == "cpu" and (n, v) not in ((700, 131073), (600, 262208)):
        pytest.skip("on the CPU model two of the five (a minute each), and the dealt case below")
    check_table_gradient(kernels, n, v, d, dtype, n + v, pad=3)


def test_tokens_of_large_tables_are_not_read_by_every_workgroup(kernels):
    """With many tokens each workgroup of the sort reads its share of them, whatever the table's size: the work is not tokens
    times rows (counted on the CPU model)."""
    ops, dev = kernels
    if dev.type != "cpu":
        pytest.skip("the CPU model counts the bytes")
    from tests.hip_emu.emu_ops import Traffic
    n, v = 49200, 300001
    tokens = torch.randint(0, v, (n,), generator=gen(0))
    grad, table = torch.ones(n, 1), torch.empty(v, 1)
    with Traffic(ops) as t:
        ops.embedding_bwd(grad, tokens, table)
    assert t.of(tokens)[0] <= 4 * 8 * n                                 # counted, counted per wave, dealt out
    assert torch.equal(table, torch.bincount(tokens, minlength=v).float()[:, None])
    # nothing else is read in proportion to tokens x workgroups: the lists, the gradient and its parts come to a few words a token
    assert t.read <= 400 * n + 64 * 4 * v


# ---- replacing tables of a model
class _Tied(torch.nn.Module):
    """The output layer shares the input table."""

    def __init__(self):
        super().__init__()
        self.body = torch.nn.Sequential(torch.nn.Embedding(9, 4), torch.nn.Linear(4, 4))
        self.head = torch.nn.Linear(4, 9, bias=False)
        self.head.weight = self.body[0].weight


class _Shared(torch.nn.Module):
    """Two parts of the model look up in one table."""

    def __init__(self):
        super().__init__()
        self.encoder = torch.nn.Sequential(torch.nn.Embedding(9, 4), torch.nn.Linear(4, 4))
        self.decoder = torch.nn.Sequential(self.encoder[0], torch.nn.Linear(4, 4))


@pytest.mark.parametrize("model", [_Tied, _Shared])
def test_make_module_bbb_refuses_to_untie_a_table(backend, model):
    """Each place would get a Gaussian of its own; the model is left as it was."""
    ops, dev = backend
    net = model().to(dev)
    before = [type(m) for m in net.modules()]
    with pytest.raises(ValueError, match="share"):
        bde.make_module_bbb(net, bde.GaussianPrior(0, 1.0), embeddings=True, _ops=ops)
    assert [type(m) for m in net.modules()] == before


def test_make_module_bbb_leaves_tables_it_does_not_take(backend):
    """16-bit tables and lookups that do more than look up stay as they are."""
    ops, dev = backend
    net = torch.nn.ModuleList([torch.nn.Embedding(9, 4, dtype=BF16), torch.nn.Embedding(9, 4, max_norm=1.0),
                               torch.nn.Embedding(9, 4, scale_grad_by_freq=True), torch.nn.Embedding(9, 4)]).to(dev)
    assert bde.make_module_bbb(net, bde.GaussianPrior(0, 1.0), embeddings=True, _ops=ops) == 1
    assert [type(m) is bde.BBBEmbedding for m in net] == [False, False, False, True]


def test_make_module_bbb_takes_a_table_whose_weight_is_computed(backend):
    """A parametrised table's weight is no parameter of its own: it is in one place."""
    ops, dev = backend
    class Twice(torch.nn.Module):
        def forward(self, w):
            return 2.0 * w
    table = torch.nn.Embedding(9, 4)
    torch.nn.utils.parametrize.register_parametrization(table, "weight", Twice())
    net = torch.nn.Sequential(table).to(dev)
    want = table.weight.detach().clone()
    assert bde.make_module_bbb(net, bde.GaussianPrior(0, 1.0), embeddings=True, _ops=ops) == 1
    assert torch.equal(net[0].weight.mean, want)
