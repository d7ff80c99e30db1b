"""The token-model operators -- scaled / Gaussian embedding, a teacher's top logits, the distillation loss -- against plain
implementations in 64 bits.

Every test runs on the CPU model of the kernels ("emu": the kernel sources lane by lane, buffers fenced by guard pages) and
on the device ("hip").  Tolerances count roundings: u = 2^-24 is half an fp32 step, ``half_step(t)`` half a step of the stored
type; v_exp_f32 and v_log_f32 are one step (2 u), softplus and sigmoid are within 2.5e-7 (5 u, bde_common.hpp)."""
import math

import pytest
import torch

import beyond_deep_ensembles_amd as bde
from beyond_deep_ensembles_amd.ops import BdeKernelError

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
NAMES = {F32: "f32", BF16: "bf16", F16: "f16"}


@pytest.fixture(params=["emu", "emu_python", pytest.param("hip", marks=pytest.mark.gpu)])
def backend(request, monkeypatch):
    if request.param != "hip":
        from tests.hip_emu import build, emu_ops
        if not build.available():
            pytest.skip("no host clang / HIP headers to build the CPU model with")
        # "emu": through the C++ autograd nodes, compiled over the model (lib/_bde_host.so binds the device library);
        # "emu_python": through the Python ones
        import beyond_deep_ensembles_amd.bbb_layers as L
        native = build.load_host_nodes(emu_ops.ALL) if request.param == "emu" else None
        monkeypatch.setattr(L, "_native_nodes", lambda ops: native)
        with emu_ops.emulated(emu_ops.ALL) as ops:
            yield ops, torch.device("cpu")
        return
    from beyond_deep_ensembles_amd.ops import HipOps
    yield HipOps(), torch.device("cuda:0")


def half_step(t):
    return torch.finfo(t).eps / 2


def least_step(t):
    """Half the distance of the smallest numbers of the type (what a result near zero is off by at most)."""
    return {F32: 2.0 ** -150, BF16: 2.0 ** -134, F16: 2.0 ** -25}[t] + 2.0 ** -126     # (fp32 results below 2^-126 are flushed)


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def close(got, want, tol, what):
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, what
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, 0.0, (got - want).abs() - tol)
    assert not off.isnan().any() and off.max().item() <= 0 if off.numel() else True, f"{what}: {off.max().item():.3e} beyond the tolerance"


# --------------------------------------------------------------- embedding --
def embedding64(tokens, mean, rho, noise, eps, scale, pad, g):
    """out, d mean, d rho and the sums of absolute values that bound their rounding."""
    v, d = mean.shape
    t = tokens.reshape(-1).long()
    ok = (t >= 0) & (t < v)
    row = torch.where(ok, t, 0)
    live = (ok & (t != (-1 if pad is None else pad))).double()[:, None]
    m = mean.double()[row]
    out, size = m.clone(), m.abs()
    e = None
    if noise is not None:
        e = (eps.double()[row] if noise == "token" else eps.double().reshape(t.numel(), d)) * live
        s = torch.nn.functional.softplus(rho.double())[row] * e
        out, size = out + s, size + s.abs()
    out = torch.where(ok[:, None], out * scale, math.nan)
    res = dict(out=out, size=size * abs(scale))
    if g is not None:
        g = g.double().reshape(t.numel(), d) * live

        def by_token(x):
            return torch.zeros(v, d, dtype=torch.float64).index_add_(0, row, x)
        res.update(gm=by_token(g) * scale, gm_size=by_token(g.abs()) * abs(scale), count=torch.bincount(t[ok], minlength=v).double()[:, None])
        if noise is not None:
            sg = torch.sigmoid(rho.double())
            res.update(gr=by_token(g * e) * scale * sg, gr_size=by_token((g * e).abs()) * abs(scale) * sg)
    return res


def check_embedding(backend, tokens, mean, rho, *, noise=None, eps=None, scale=1.0, pad=None, out_dtype=None, g=None, seed=5):
    ops, dev = backend
    out_dtype = out_dtype or mean.dtype
    m = mean.to(dev).detach().requires_grad_()
    kw = dict(scale=scale, padding_idx=pad, out_dtype=out_dtype, _ops=ops)
    if noise is None:
        r = None
        out = bde.embedding(tokens.to(dev), m, **kw)
    else:
        r = rho.to(dev).detach().requires_grad_()
        out = bde.gaussian_embedding(tokens.to(dev), m, r, noise=noise, eps=eps.to(dev), **kw)
    d = mean.shape[1]
    assert out.dtype == out_dtype and out.shape == tokens.shape + (d,)
    g = torch.randn(out.shape, generator=gen(seed)).to(out_dtype) if g is None else g
    want = embedding64(tokens, mean, rho, noise, eps, scale, pad, g)
    # product, sum, scale: 3 roundings and softplus' 5 u on the way, one to the stored type
    rounded = (1 + half_step(out_dtype)) * 9 * U
    close(out.reshape(-1, d), want["out"], want["size"] * rounded + want["out"].abs() * half_step(out_dtype) + least_step(out_dtype), "out")
    grads = torch.autograd.grad(out, [x for x in (m, r) if x is not None], g.to(dev))
    # count terms added one by one (parts of a sum only shorten the chain), the scale
    close(grads[0], want["gm"], want["gm_size"] * (want["count"] + 2) * U * 1.01 + want["gm"].abs() * half_step(mean.dtype) * (mean.dtype != F32)
          + least_step(mean.dtype), "gradient of the mean")
    if r is not None:
        close(grads[1], want["gr"], want["gr_size"] * (want["count"] + 10) * U * 1.01 + least_step(F32), "gradient of rho")
    return out, grads


TYPES = [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (F16, F16)]


@pytest.mark.parametrize("wtype,otype", TYPES, ids=[f"{NAMES[a]}-{NAMES[b]}" for a, b in TYPES])
@pytest.mark.parametrize("n,v,d", [(1, 1, 1), (1, 300, 64), (37, 7, 24), (65, 600, 301), (130, 3, 8)])
def test_embedding_sizes_and_types(backend, n, v, d, wtype, otype):
    g = gen(n + 31 * v + d)
    tokens = torch.randint(0, v, (n,), generator=g)
    w = torch.randn(v, d, generator=g).to(wtype)
    check_embedding(backend, tokens, w, None, scale=math.sqrt(d), out_dtype=otype)


@pytest.mark.parametrize("tokens", ["one", "two", "falling", "padding_only", "outside", "int32", "empty", "grid"])
def test_embedding_token_patterns(backend, tokens):
    """Runs that cross the pieces of the sorted list, positions without gradient, tokens outside the table, no tokens."""
    v, d, pad = 11, 12, 2
    t = {"one": torch.full((75,), 4), "two": torch.tensor([9, 1] * 40), "falling": torch.arange(99) // 9 % 11,
         "padding_only": torch.full((20,), pad), "outside": torch.tensor([3, -1, 11, 3, 2, -2 ** 40, 2 ** 40, 10]),
         "int32": torch.tensor([3, -1, 11, 3, 2, 10], dtype=torch.int32), "empty": torch.zeros(0, dtype=torch.int64),
         "grid": torch.arange(24).reshape(2, 3, 4) % v}[tokens]
    g = gen(7)
    w, rho = torch.randn(v, d, generator=g), torch.randn(v, d, generator=g) - 2
    check_embedding(backend, t, w, None, scale=3.0, pad=pad)
    check_embedding(backend, t, w, rho, noise="position", eps=torch.randn(tuple(t.shape) + (d,), generator=g), pad=pad)


@pytest.mark.parametrize("wtype,otype", TYPES, ids=[f"{NAMES[a]}-{NAMES[b]}" for a, b in TYPES])
@pytest.mark.parametrize("n,v,d", [(9, 1, 8), (64, 2, 301), (200, 5, 520), (512, 3, 4), (513, 300, 6), (300, 7, 904)])
def test_embedding_gradient_in_one_launch_and_in_several(backend, n, v, d, wtype, otype):
    """Few positions take one launch, more several: sizes on both sides of the bounds; runs that lie within a wave's piece of the
    list, cross one border, or hold whole pieces; columns in several tiles."""
    g = gen(n + d)
    tokens = (v * torch.rand(n, generator=g) ** 2).long()
    check_embedding(backend, tokens, torch.randn(v, d, generator=g).to(wtype), None, scale=0.5, out_dtype=otype)


@pytest.mark.parametrize("noise", ["position", "token"])
@pytest.mark.parametrize("n,v,d", [(90, 3, 264), (90, 3, 67), (520, 4, 8), (300, 40, 900)])
def test_gaussian_embedding_gradient_in_one_launch_and_in_several(backend, n, v, d, noise):
    g = gen(n + d)
    tokens = (v * torch.rand(n, generator=g) ** 2).long()
    mean, rho = torch.randn(v, d, generator=g), torch.randn(v, d, generator=g) - 2
    check_embedding(backend, tokens, mean, rho, noise=noise, eps=torch.randn(n if noise == "position" else v, d, generator=g), pad=1)


@pytest.mark.parametrize("tokens", ["one", "two", "falling", "padding_only", "outside"])
def test_embedding_token_patterns_of_many_positions(backend, tokens):
    v, d, pad, n = 11, 12, 2, 1056
    i = torch.arange(n)
    t = {"one": torch.full((n,), 4), "two": torch.where(i % 2 == 0, 9, 1), "falling": 10 - i // 96, "padding_only": torch.full((n,), pad),
         "outside": torch.tensor([3, -1, 11, 3, 2, -2 ** 40, 2 ** 40, 10]).repeat(n // 8)}[tokens]
    g = gen(8)
    w, rho = torch.randn(v, d, generator=g), torch.randn(v, d, generator=g) - 2
    check_embedding(backend, t, w, None, scale=3.0, pad=pad)
    check_embedding(backend, t, w, rho, noise="position", eps=torch.randn(n, d, generator=g), pad=pad)


@pytest.mark.parametrize("noise", ["position", "token"])
@pytest.mark.parametrize("otype", [F32, BF16, F16], ids=lambda t: NAMES[t])
@pytest.mark.parametrize("n,v,d", [(50, 9, 16), (70, 300, 13)])
def test_gaussian_embedding(backend, n, v, d, otype, noise):
    g = gen(n + d)
    tokens = torch.randint(0, v, (n,), generator=g)
    mean, rho = torch.randn(v, d, generator=g), 4 * torch.randn(v, d, generator=g) - 2
    eps = torch.randn(n if noise == "position" else v, d, generator=g)
    check_embedding(backend, tokens, mean, rho, noise=noise, eps=eps, scale=2.5, pad=1, out_dtype=otype)


def test_embedding_many_positions_of_few_tokens(backend):
    """More matches in one wave's part of the list than it keeps (it reads its part again), runs over many pieces."""
    g = gen(3)
    tokens = torch.where(torch.rand(6000, generator=g) < 0.9, 1, torch.randint(0, 3, (6000,), generator=g))
    check_embedding(backend, tokens, torch.randn(3, 4, generator=g), None, scale=0.5)


def test_embedding_of_many_rows(backend):
    """Enough rows for four to a group of lanes, and a last group that is not full."""
    g = gen(6)
    tokens = torch.randint(0, 9, (16387,), generator=g)
    check_embedding(backend, tokens, torch.randn(9, 8, generator=g).bfloat16(), None, scale=2.0, pad=4)
    mean, rho = torch.randn(9, 3, generator=g), torch.randn(9, 3, generator=g) - 2
    check_embedding(backend, tokens, mean, rho, noise="position", eps=torch.randn(16387, 3, generator=g))


@pytest.mark.parametrize("v", [5, 1500])
def test_embedding_gradient_of_many_tokens(backend, v):
    """Enough tokens to be dealt out to the sort's workgroups first: one frequent token, padding, tokens outside the table."""
    g = gen(v)
    tokens = torch.where(torch.rand(49200, generator=g) < 0.3, 3, torch.randint(-1, v + 1, (49200,), generator=g))
    check_embedding(backend, tokens, torch.randn(v, 4, generator=g), None, pad=1)
    check_embedding(backend, tokens.int(), torch.randn(v, 2, generator=g), None)


def test_embedding_strided_operands(backend):
    """Rows that lie apart, rows off a 16-byte border, a transposed table, a broadcast and a strided gradient."""
    g = gen(11)
    tokens = torch.randint(0, 20, (33,), generator=g)
    wide = torch.randn(20, 40, generator=g)
    for w in (wide[:, :16], wide[:, 1:17], wide[:, 3:16], torch.randn(16, 20, generator=g).t(), wide[:, :1], wide[:1, :16].expand(20, 16)):
        d = w.shape[1]
        check_embedding(backend, tokens, w, None)
        check_embedding(backend, tokens, w, None, g=torch.randn(1, d, generator=g).expand(33, d))
        check_embedding(backend, tokens, w, None, g=torch.randn(d, 33, generator=g).t())
        check_embedding(backend, tokens[::2], w, w - 2, noise="position", eps=torch.randn(17, d, generator=g))
        check_embedding(backend, tokens, w, w - 2, noise="token", eps=torch.randn(20, 2 * d, generator=g)[:, ::2])


@pytest.mark.parametrize("d", [8, 7])
def test_philox_noise_of_the_embedding(backend, d):
    """By token it is the draw GaussianParameter.sample() makes of that stream; by position the stream's normals in element
    order; and the backward pass regenerates what the forward pass used."""
    ops, dev = backend
    g = gen(d)
    v, n = 13, 21
    tokens = torch.randint(0, v, (n,), generator=g).to(dev)
    mean, rho = torch.randn(v, d, generator=g).to(dev), (torch.randn(v, d, generator=g) - 2).to(dev)
    go = torch.randn(n, d, generator=g).to(dev)
    for noise, rows in (("token", v), ("position", n)):
        eps = torch.empty(rows * d, device=dev)
        ops.philox_normal(42, 9, eps_d=eps, d=rows * d)
        eps = eps.view(rows, d)
        got, want = [], []
        for out, e in ((got, None), (want, eps)):
            m, r = mean.clone().requires_grad_(), rho.clone().requires_grad_()
            y = bde.gaussian_embedding(tokens, m, r, noise=noise, eps=e, seed=42, stream_id=9, _ops=ops)
            out += [y.detach(), *torch.autograd.grad(y, (m, r), go)]
        for a, b in zip(got, want):
            assert torch.equal(a, b), noise
    table = torch.empty(v * d, device=dev)
    ops.gauss_draw_fwd(mean.reshape(-1), rho.reshape(-1), table, v * d, seed=42, stream_id=9)
    y = bde.gaussian_embedding(tokens, mean, rho, noise="token", seed=42, stream_id=9, _ops=ops)
    assert torch.equal(y, table.view(v, d)[tokens])


def test_embedding_gradient_against_differences(backend):
    """Central differences in 64 bits of the formula around fp32 operands: the derivative itself, not its formula."""
    ops, dev = backend
    g = gen(1)
    tokens = torch.tensor([0, 2, 2, 1, 4])
    mean, rho, eps, go = (torch.randn(s, generator=g) for s in ((5, 3), (5, 3), (5, 3), (5, 3)))
    m, r = mean.to(dev).requires_grad_(), rho.to(dev).requires_grad_()
    out = bde.gaussian_embedding(tokens.to(dev), m, r, eps=eps.to(dev), scale=1.5, padding_idx=1, _ops=ops)
    gm, gr = torch.autograd.grad(out, (m, r), go.to(dev))

    def objective(mean, rho):
        x = embedding64(tokens, mean, rho, "position", eps, 1.5, 1, None)["out"] * go.double()
        return x[tokens != 1].sum()              # (the padding position has no gradient by definition)
    h = 1e-5
    for t, grad in ((mean, gm), (rho, gr)):
        for i in range(t.numel()):
            lo, hi = t.double().clone(), t.double().clone()
            lo.view(-1)[i] -= h
            hi.view(-1)[i] += h
            a, b = ((hi, rho.double()), (lo, rho.double())) if t is mean else ((mean.double(), hi), (mean.double(), lo))
            diff = (objective(*a) - objective(*b)) / (2 * h)
            # second-order error of the difference h^2 / 6 * third derivative (below 1e-9 here) and the kernel's roundings
            assert abs(diff.item() - grad.view(-1)[i].item()) <= 1e-8 + 40 * U * (abs(diff.item()) + 1)


def test_embedding_is_bit_reproducible(backend):
    ops, dev = backend
    g = gen(2)
    tokens = torch.randint(0, 5, (500,), generator=g).to(dev)
    w = torch.randn(5, 20, generator=g).to(dev).requires_grad_()
    go = torch.randn(500, 20, generator=g).to(dev)
    a, b = (torch.autograd.grad(bde.embedding(tokens, w, _ops=ops), w, go)[0] for _ in range(2))
    assert torch.equal(a, b)


def test_embedding_refusals(backend):
    ops, dev = backend
    w = torch.zeros(4, 8, device=dev)
    t = torch.zeros(3, dtype=torch.int64, device=dev)
    kw = dict(_ops=ops)
    for call in (lambda: bde.embedding(t.float(), w, **kw), lambda: bde.embedding(t, w[0], **kw), lambda: bde.embedding(t, w.double(), **kw),
                 lambda: bde.embedding(t, w, padding_idx=4, **kw), lambda: bde.embedding(t, w, padding_idx=-5, **kw),
                 lambda: bde.embedding(t, w.bfloat16(), out_dtype=F32, **kw), lambda: bde.embedding(t, w, out_dtype=torch.float64, **kw),
                 lambda: bde.embedding(t, torch.zeros(4, 0, device=dev), **kw),
                 lambda: bde.embedding(t, torch.zeros(2, 16385, device=dev), **kw),
                 lambda: bde.gaussian_embedding(t, w, w[:3], **kw), lambda: bde.gaussian_embedding(t, w.half(), w.half(), **kw),
                 lambda: bde.gaussian_embedding(t, w, w, eps=torch.zeros(4, 8, device=dev), **kw),
                 lambda: bde.gaussian_embedding(t, w, w, noise="token", eps=torch.zeros(3, 8, device=dev), **kw),
                 lambda: bde.gaussian_embedding(t, w, w, eps=torch.zeros(3, 8, device=dev, requires_grad=True), **kw)):
        with pytest.raises(BdeKernelError):
            call()
    with pytest.raises(ValueError):
        bde.gaussian_embedding(t, w, w, noise="row", **kw)
    with pytest.raises(RuntimeError):                                   # no second derivative
        x = w.clone().requires_grad_()
        (gx,) = torch.autograd.grad(bde.embedding(t, x, **kw).sum() ** 2, x, create_graph=True)
        gx.sum().backward()


# -------------------------------------------------------------- top logits --
def topk64(z, k, tau):
    x = z.double()
    key = torch.where(x.isnan(), math.inf, x)
    order = torch.sort(key, dim=1, descending=True, stable=True).indices
    if x.isnan().any():                       # a NaN goes ahead of +inf
        order = torch.stack([torch.tensor(sorted(range(x.shape[1]), key=lambda v: (0 if math.isnan(r[v]) else 1, -r[v] if not math.isnan(r[v])
                                                                                  else 0.0, v))) for r in x])
    indices = order[:, :k]
    others = x.scatter(1, indices, -math.inf) if not x.isnan().any() else torch.stack([r.clone().index_fill_(0, i, -math.inf) for r, i in zip(x, indices)])
    return torch.gather(x, 1, indices), indices, torch.logsumexp(others / tau, 1)


def exponent_error(spread, v=0):
    """Relative error of exp of a difference of fp32 logits over tau, summed over a row: the factor log2(e) / tau is three
    roundings off, the product-difference one, exp one step, a sum of v terms a chain of v / 8192 + 8 + 16 + 6 + 16."""
    return U * (56 + v / 8192 + 8 * spread)


def check_topk(backend, z, k, tau=1.0):
    ops, dev = backend
    got = bde.topk_logits(z.to(dev), k, temperature=tau, _ops=ops)
    values, indices, rest = topk64(z, k, tau)
    assert got.values.dtype == z.dtype and got.indices.dtype == torch.int64 and got.rest.dtype == F32
    assert torch.equal(got.indices.cpu(), indices)
    close(got.values, values, 0.0, "values")
    x = z.double()
    finite = torch.where(x.isfinite(), x, 0.0) / tau
    spread = finite.amax(1) - finite.amin(1) + finite.abs().amax(1)
    close(got.rest, rest, torch.where(rest.isfinite(), exponent_error(spread, z.shape[1]) + 4 * U * rest.abs(), 0.0), "rest")
    return got


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=lambda t: NAMES[t])
@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (3, 10, 3), (2, 10, 10), (5, 182, 10), (2, 300, 129), (2, 1000, 40), (2, 4100, 64), (1, 9001, 256),
                                   (1, 40000, 5)])
def test_topk_sizes_and_types(backend, n, v, k, dtype):
    z = (2.5 * torch.randn(n, v, generator=gen(n + v + k))).to(dtype)
    check_topk(backend, z, k, tau=1.0 if v % 2 else 2.0)


def test_topk_rows_longer_than_the_registers(backend):
    """V above what a workgroup holds: fp32 rows of 65,537 .. 262,144 classes stay in memory."""
    z = torch.randn(1, 66001, generator=gen(0))
    check_topk(backend, z, 33)


@pytest.mark.parametrize("row", ["constant", "two_values", "masked", "masked_all", "lowest", "plus_inf", "signed_zeros", "ramp", "few_finite", "nan"])
@pytest.mark.parametrize("v,k", [(50, 7), (3001, 20)])
def test_topk_rows_with_structure(backend, row, v, k):
    """Ties, masks that leave less than k classes, the type's lowest value, infinities, NaN."""
    g = gen(v)
    z = torch.randn(2, v, generator=g)
    z = {"constant": torch.full((2, v), 0.75), "two_values": (z > 0).float(), "masked": z.masked_fill(torch.rand(2, v, generator=g) < 0.7, -math.inf),
         "masked_all": torch.full((2, v), -math.inf), "lowest": z.masked_fill(torch.rand(2, v, generator=g) < 0.9, torch.finfo(F32).min),
         "plus_inf": z.masked_fill(torch.arange(v) == 5, math.inf), "signed_zeros": torch.where(torch.rand(2, v, generator=g) < 0.5, 0.0, -0.0),
         "ramp": torch.arange(v).float().expand(2, v) * 0.01, "few_finite": torch.where(torch.arange(v) % (v // 3) == 1, z, -math.inf),
         "nan": z.masked_fill(torch.arange(v) == v - 2, math.nan)}[row]
    check_topk(backend, z, k)


@pytest.mark.parametrize("top", [math.inf, math.nan, None])
@pytest.mark.parametrize("v,k", [(50, 1), (50, 30), (3001, 3), (3001, 200)])
def test_topk_what_is_left_beside_infinities(backend, v, k, top):
    """Exactly k classes that are +inf (NaN): the others are summed relative to a number of their own, also where their
    exponentials leave the range, and so small that they would vanish.  (None: the same rows without them.)"""
    z = torch.randn(3, v, generator=gen(v + k)) + torch.tensor([[200.0], [-300.0], [0.0]])
    if top is not None:
        z[:, torch.randperm(v, generator=gen(k))[:k]] = top
    check_topk(backend, z, k)


@pytest.mark.parametrize("gap", [40.0, 100.0, 150.0, 1e4, 1e30])
@pytest.mark.parametrize("v,k", [(50, 1), (50, 30), (3001, 3), (3001, 200)])
def test_topk_what_is_left_far_below(backend, v, k, gap):
    """Exactly k classes that lie far above the others: what is left is still the others' sum, not nothing."""
    z = torch.randn(2, v, generator=gen(v + k))
    z[:, torch.randperm(v, generator=gen(k))[:k]] += gap
    ops, dev = backend
    got = bde.topk_logits(z.to(dev), k, _ops=ops)
    values, indices, rest = topk64(z, k, 1.0)
    assert torch.equal(got.indices.cpu(), indices)
    close(got.values, values, 0.0, "values")
    # relative to the k-th value the difference (one rounding of up to gap + 8) is an error of the exponent, below 1e-20 of a sum
    # relative to the largest of the others none
    close(got.rest, rest, exponent_error(min(gap, 60.0) + 16, v) + 4 * U * (gap if gap <= 60 else 16.0), "rest")


def test_topk_strided_rows(backend):
    wide = torch.randn(4, 700, generator=gen(4))
    for z in (wide[:, :301], wide[:, 3:302], wide[::2, 1:400], wide.t()[:90], wide[:1].expand(3, 700)):
        check_topk(backend, z, min(9, z.shape[1]))
    ops, dev = backend
    z3 = torch.randn(2, 3, 50, generator=gen(5))
    got = bde.topk_logits(z3.to(dev), 4, _ops=ops)
    assert got.values.shape == got.indices.shape == (2, 3, 4) and got.rest.shape == (2, 3)
    empty = bde.topk_logits(torch.zeros(0, 50, device=dev), 4, _ops=ops)
    assert empty.values.shape == (0, 4) and empty.rest.shape == (0,)


def test_topk_refusals(backend):
    ops, dev = backend
    z = torch.zeros(2, 300, device=dev)
    for call in (lambda: bde.topk_logits(z, 0, _ops=ops), lambda: bde.topk_logits(z, 257, _ops=ops), lambda: bde.topk_logits(z[:, :5], 6, _ops=ops),
                 lambda: bde.topk_logits(z.double(), 3, _ops=ops), lambda: bde.topk_logits(z[:, :0], 1, _ops=ops),
                 lambda: bde.topk_logits(torch.zeros(1, 262145, device=dev), 3, _ops=ops)):
        with pytest.raises(BdeKernelError):
            call()
    for t in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError):
            bde.topk_logits(z, 3, temperature=t, _ops=ops)


# ------------------------------------------------------------ distillation --
def distill64(z, values, indices, rest, weight, tau, scale, reduction):
    """Row losses (times weight and scale), their reduction, gradient of the reduction, and what bounds the roundings."""
    n, v = z.shape
    x = z.double() / tau
    ok = (indices >= 0) & (indices < v)
    idx = torch.where(ok, indices, 0).long()
    t = torch.where(ok, values.double() / tau, -math.inf)
    t = torch.cat([t, torch.full((n, 1), -math.inf, dtype=torch.float64) if rest is None else rest.double()[:, None]], 1)
    says = (t > -math.inf).any(1) | t.isnan().any(1)
    lp = torch.where(says[:, None], t - torch.logsumexp(t, 1, keepdim=True), -math.inf)
    p = lp.exp()
    listed = torch.zeros(n, v, dtype=torch.bool).scatter_(1, idx, ok) | torch.zeros(n, v, dtype=torch.bool).scatter_add_(1, idx, ok)
    lq = torch.log_softmax(x, 1)
    ltail = torch.logsumexp(lq.masked_fill(listed, -math.inf), 1, keepdim=True)
    lq_t = torch.cat([lq.gather(1, idx), ltail], 1)
    terms = torch.where(p > 0, p * (lp - lq_t), 0.0)
    w = torch.ones(n, dtype=torch.float64) if weight is None else weight.double()
    per = torch.where(w != 0, scale * w, 0.0)
    if reduction == "mean":
        per = per / w.sum() if w.sum() != 0 else per * 0
    dead = (per == 0) | ~says
    rows = torch.where(dead, 0.0, per * terms.sum(1))
    rows_size = torch.where(dead, 0.0, per.abs() * (2 + torch.where(p > 0, p * (lp - lq_t).abs(), 0.0).sum(1)))
    q = lq.exp()
    tail_part = torch.where((p[:, -1:] > 0) & (lq > -math.inf) | lq.isnan(), p[:, -1:] * (lq - ltail).exp(), 0.0)
    spread_p = torch.zeros(n, v, dtype=torch.float64).scatter_add_(1, idx, torch.where(ok, p[:, :-1], 0.0))
    unit = torch.where(listed, q - spread_p, q - tail_part)
    size = torch.where(listed, q + spread_p, q + tail_part)
    k = (per / tau)[:, None]
    grad, size = torch.where(dead[:, None], 0.0, unit * k), torch.where(dead[:, None], 0.0, size * k.abs())
    return dict(rows=rows, rows_size=rows_size, grad=grad, grad_size=size, total=rows.sum())


def spread_of(z, values, rest, tau):
    big = [torch.where(a.double().isfinite(), a.double(), 0.0).abs().reshape(z.shape[0], -1).amax(1) for a in (z, values)]
    s = 2 * big[0] / tau + 2 * big[1] / tau
    return s if rest is None else s + 2 * torch.where(rest.isfinite(), rest.double(), 0.0).abs()


def check_distill(backend, z, values, indices, rest=None, *, weight=None, tau=1.0, scale=1.0, reduction="mean", upstream=1.0):
    ops, dev = backend
    put = lambda t: None if t is None else t.to(dev)                    # noqa: E731
    x = z.to(dev).detach().requires_grad_()
    loss = bde.distillation_loss(x, put(values), put(indices), put(rest), temperature=tau, weight=put(weight), scale=scale, reduction=reduction,
                                 _ops=ops)
    want = distill64(z, values, indices, rest, weight, tau, scale, reduction)
    assert loss.dtype == F32 and loss.shape == ((z.shape[0],) if reduction == "none" else ())
    # the exponents of teacher and student, and the chain over the K terms of a row's loss
    rel = 2 * exponent_error(spread_of(z, values, rest, tau), z.shape[1]) + (values.shape[1] + 8) * U
    tol = want["rows_size"] * rel
    if reduction == "none":
        close(loss, want["rows"], tol, "losses")
    else:
        close(loss, want["total"], (tol + 4 * U * want["rows"].abs()).sum(), "loss")
    g = torch.full_like(loss, upstream) if not torch.is_tensor(upstream) else upstream.to(dev)
    (got,) = torch.autograd.grad(loss, x, g)
    assert got.dtype == z.dtype
    up = g.detach().cpu().double().reshape(-1, 1)
    grad = torch.where(up == 0, 0.0, want["grad"] * up)
    close(got, grad, torch.where(up == 0, 0.0, want["grad_size"] * up.abs()) * (rel + 6 * U)[:, None] + grad.abs() * half_step(z.dtype)
          + least_step(z.dtype), "gradient")
    return loss, got


def teacher(n, v, k, dtype, seed, tau=1.0):
    g = gen(seed)
    indices = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(n)]) if n else torch.zeros(0, k, dtype=torch.int64)
    values = (4 + 2 * torch.randn(n, k, generator=g)).to(dtype)
    rest = torch.logsumexp(values.double() / tau, 1).float() - 0.5 - 2 * torch.rand(n, generator=g)
    z = 2.5 * torch.randn(n, v, generator=g)
    z.scatter_add_(1, indices, 3 + torch.randn(n, k, generator=g))
    return z.to(dtype), values, indices, rest


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=lambda t: NAMES[t])
@pytest.mark.parametrize("n,v,k", [(1, 2, 1), (3, 10, 3), (2, 10, 10), (4, 182, 16), (2, 1000, 64), (2, 2500, 20), (2, 4100, 100), (1, 9001, 33),
                                   (1, 20001, 3), (1, 40000, 7), (1, 70000, 64)])
def test_distill_sizes_and_types(backend, n, v, k, dtype):
    tau = 1.0 if v % 3 else 2.0
    z, values, indices, rest = teacher(n, v, k, dtype, v + k, tau)
    if k == v:
        rest = None
    check_distill(backend, z, values, indices, rest, tau=tau, scale=float(64 * n))


def test_distill_rows_longer_than_the_registers(backend):
    check_distill(backend, *teacher(1, 66001, 40, F32, 1))


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("upstream", [1.0, 0.3, 0.0])
def test_distill_reductions_and_upstream_values(backend, reduction, weighted, upstream):
    z, values, indices, rest = teacher(6, 50, 5, F32, 3)
    weight = torch.tensor([1.0, 0.0, 0.5, 2.0, 0.0, 1.0]) if weighted else None
    if weighted:
        z[1] = math.nan                                # a row of weight 0 is not looked at
    check_distill(backend, z, values, indices, rest, weight=weight, scale=1.7, reduction=reduction, upstream=upstream)
    if reduction == "none":
        check_distill(backend, z, values, indices, rest, weight=weight, reduction=reduction,
                      upstream=torch.tensor([1.0, 1.0, 0.0, -2.0, 0.25, 0.0]))


@pytest.mark.parametrize("v,k", [(40, 6), (2100, 9)])
def test_distill_lists_with_structure(backend, v, k):
    """Short lists, a class twice, entries the teacher gives nothing, rows without any entry, a list with everything."""
    z, values, indices, rest = teacher(7, v, k, F32, 9)
    indices[0, 2:] = -1                                # short
    indices[1, 3] = indices[1, 0]                      # the same class twice
    indices[2, 4] = indices[2, 1]
    indices[2, 2] = indices[2, 1]
    values[3, 1:3] = -math.inf
    indices[4] = -1                                    # nothing listed, something left: any distribution will do
    indices[5] = v + 3
    rest[5] = -math.inf                                # the teacher says nothing
    rest[6] = -math.inf                                # nothing left
    for r in (rest, None):
        check_distill(backend, z, values, indices, r, tau=1.5)
    check_distill(backend, z, values.bfloat16(), indices.int(), rest, tau=0.7, reduction="none")
    z[5] = math.nan                                    # (nothing said: not looked at)
    check_distill(backend, z, values, indices, rest)


@pytest.mark.parametrize("tau", [0.6, 1.0, 2.0])
def test_distill_teachers_masked_with_the_lowest_value(backend, tau):
    """A teacher whose list holds nothing but the type's lowest value: alone it is uniform over the list, beside a finite rest
    nothing."""
    z, values, indices, rest = teacher(4, 40, 5, F32, 7, tau)
    values[:] = torch.finfo(F32).min
    rest[:2] = -math.inf
    check_distill(backend, z, values, indices, rest, tau=tau)


@pytest.mark.parametrize("v,spike", [(3000, 2900), (20001, 19990), (70000, 69000)])
def test_distill_rows_that_rise_late(backend, v, spike):
    """The largest classes lie behind each thread's first granule, so far above it that the provisional reference overflows; and
    rows whose first granules are masked entirely."""
    z, values, indices, rest = teacher(2, v, 5, F32, v)
    z[0, spike:spike + 3] += 150.0
    z[1, :v // 2] = -math.inf
    check_distill(backend, z, values, indices, rest)


@pytest.mark.parametrize("what", ["masked_others", "masked_listed", "masked_all", "lowest", "lowest_others", "lowest_all", "far", "huge", "nan", "inf"])
def test_distill_students_with_structure(backend, what):
    z, values, indices, rest = teacher(3, 30, 4, F32, 5)
    listed = torch.zeros(3, 30, dtype=torch.bool).scatter_(1, indices, True)
    z = {"masked_others": z.masked_fill(~listed & (torch.arange(30) % 2 == 0), -math.inf), "masked_listed": z.masked_fill(listed & (torch.arange(30) < 20), -math.inf),
         "masked_all": torch.full((3, 30), -math.inf), "lowest": z.masked_fill(~listed & (torch.arange(30) % 3 == 0), torch.finfo(F32).min),
         "lowest_others": z.masked_fill(~listed, torch.finfo(F32).min), "lowest_all": torch.full((3, 30), torch.finfo(F32).min),
         "far": torch.where(listed, z + 150.0, z),      # the others' share underflows beside the listed ones'
         "huge": z * 1000.0, "nan": z.masked_fill(torch.arange(30) == 3, math.nan), "inf": z.masked_fill(torch.arange(30) == 3, math.inf)}[what]
    check_distill(backend, z, values, indices, rest)
    if what == "masked_others":                        # no class but the listed ones has any weight
        z = z.masked_fill(~listed, -math.inf)
        check_distill(backend, z, values, indices, None)
        check_distill(backend, z, values, indices, rest)


def test_distill_strided_logits_and_leading_shapes(backend):
    ops, dev = backend
    z, values, indices, rest = teacher(6, 101, 5, BF16, 8)
    wide = torch.randn(6, 160, generator=gen(1)).to(BF16)
    for x in (wide[:, :101], wide[:, 3:104], wide[:1, :101].expand(6, 101), wide[:, :].t()[:101].t()):
        check_distill(backend, x, values, indices, rest)
    a = bde.distillation_loss(z.to(dev), values.to(dev), indices.to(dev), rest.to(dev), reduction="none", _ops=ops)
    b = bde.distillation_loss(z.to(dev).view(2, 3, 101), values.to(dev).view(2, 3, 5), indices.to(dev).view(2, 3, 5), rest.to(dev).view(2, 3),
                              reduction="none", _ops=ops)
    assert b.shape == (2, 3) and torch.equal(a, b.view(6))
    x = z[:0].to(dev).requires_grad_()
    for reduction in ("none", "sum", "mean"):
        empty = bde.distillation_loss(x, values[:0].to(dev), indices[:0].to(dev), rest[:0].to(dev), reduction=reduction, _ops=ops)
        assert float(empty.detach().sum()) == 0.0
        (gx,) = torch.autograd.grad(empty.sum(), x)
        assert gx.shape == x.shape


@pytest.mark.parametrize("dtype", [F32, BF16], ids=lambda t: NAMES[t])
def test_distill_gradient_of_the_forward_pass_is_the_backward_pass(backend, dtype):
    """The buffer the forward pass fills and a later computation from the logits agree bit for bit, a second backward of a
    retained graph does not touch the first one's result, and a factor on the loss gives one rounding, not two."""
    ops, dev = backend
    z, values, indices, rest = (t.to(dev) for t in teacher(5, 300, 7, dtype, 2))
    weight = torch.tensor([1.0, 0.25, 0.0, 3.0, 1.0], device=dev)
    x = z.clone().requires_grad_()
    kw = dict(temperature=1.3, weight=weight, _ops=ops)
    loss = bde.distillation_loss(x, values, indices, rest, **kw)
    (first,) = torch.autograd.grad(loss, x, retain_graph=True)
    kept = first.clone()
    first.mul_(2.0)                                    # the caller's to change
    (second,) = torch.autograd.grad(loss, x, retain_graph=True)
    assert torch.equal(second, kept)
    (half,) = torch.autograd.grad(loss, x, torch.tensor(0.5, device=dev))
    assert torch.equal(half, kept * 0.5)               # a power of two: exact
    (scaled,) = torch.autograd.grad(bde.distillation_loss(x, values, indices, rest, scale=0.5, **kw), x)
    assert torch.equal(scaled, kept * 0.5)
    (third,) = torch.autograd.grad(bde.distillation_loss(x, values, indices, rest, **kw) * 0.5, x)
    assert torch.equal(third, kept * 0.5)
    with torch.no_grad():
        assert torch.equal(bde.distillation_loss(x, values, indices, rest, **kw), loss.detach())


def test_distill_gradient_against_differences(backend):
    ops, dev = backend
    z, values, indices, rest = teacher(2, 9, 3, F32, 12)
    x = z.to(dev).requires_grad_()
    (got,) = torch.autograd.grad(bde.distillation_loss(x, values.to(dev), indices.to(dev), rest.to(dev), temperature=1.5, reduction="sum", _ops=ops), x)
    h = 1e-5
    for i in range(z.numel()):
        lo, hi = z.double().clone(), z.double().clone()
        lo.view(-1)[i] -= h
        hi.view(-1)[i] += h
        diff = (distill64(hi, values, indices, rest, None, 1.5, 1.0, "sum")["total"] - distill64(lo, values, indices, rest, None, 1.5, 1.0, "sum")["total"]) / (2 * h)
        assert abs(diff.item() - got.view(-1)[i].item()) <= 1e-8 + 400 * U


def test_distill_refusals(backend):
    ops, dev = backend
    z, values, indices, rest = (t.to(dev) for t in teacher(3, 20, 4, F32, 1))
    kw = dict(_ops=ops)
    for call in (lambda: bde.distillation_loss(z.double(), values, indices, rest, **kw), lambda: bde.distillation_loss(z, values.double(), indices, rest, **kw),
                 lambda: bde.distillation_loss(z, values, indices.float(), rest, **kw), lambda: bde.distillation_loss(z, values, indices[:, :3], rest, **kw),
                 lambda: bde.distillation_loss(z, values[:2], indices[:2], rest, **kw), lambda: bde.distillation_loss(z, values, indices, rest[:2], **kw),
                 lambda: bde.distillation_loss(z, values, indices, rest, weight=rest[:1], **kw),
                 lambda: bde.distillation_loss(z, values, indices, rest.double(), **kw),
                 lambda: bde.distillation_loss(z, values[:, :0], indices[:, :0], rest, **kw),
                 lambda: bde.distillation_loss(z, values.clone().requires_grad_(), indices, rest, **kw),
                 lambda: bde.distillation_loss(z, values, indices, rest.clone().requires_grad_(), **kw),
                 lambda: bde.distillation_loss(z, z.new_zeros(3, 1025), indices.new_zeros(3, 1025), rest, **kw),
                 lambda: bde.distillation_loss(z.new_zeros(3, 262145), values, indices, rest, **kw)):
        with pytest.raises(BdeKernelError):
            call()
    for bad in (dict(reduction="batchmean"), dict(temperature=0.0), dict(temperature=math.nan)):
        with pytest.raises(ValueError):
            bde.distillation_loss(z, values, indices, rest, **bad, **kw)
