"""The library without the token-model operators: the sources that were there before them build and run on the CPU model by
themselves -- neither bde_init() nor the layers' autograd nodes need the operators' files."""
import pytest

from tests.hip_emu import build, emu_ops

TOKEN_SOURCES = {"embedding.hip", "topk.hip", "distill.hip"}


def test_sources_without_the_token_operators_build_and_run():
    if not build.available():
        pytest.skip("no host clang / HIP headers to build the CPU model with")
    import torch
    import torch.nn.functional as F
    sources = [s for s in emu_ops.ALL if s not in TOKEN_SOURCES]
    assert len(sources) == len(emu_ops.ALL) - 3
    nodes = build.load_host_nodes(sources)                # (loading it resolves every symbol)
    assert hasattr(nodes, "lrt_linear") and not hasattr(nodes, "distillation_loss")
    with emu_ops.emulated(sources) as ops:
        assert ops.lib.bde_init() == 0 and ops.lib.bde_init_optional_failures() == 0
        assert getattr(ops.lib, "bde_distill_fwd", None) is None
        g = torch.Generator()
        g.manual_seed(0)
        mean, rho, out = torch.randn(64, generator=g), torch.randn(64, generator=g), torch.empty(64)
        eps = torch.randn(64, generator=g)
        ops.gauss_draw_fwd(mean, rho, out, 64, eps=eps)
        want = mean.double() + F.softplus(rho.double()) * eps.double()
        # softplus within 2.5e-7, a product and a sum of numbers below 16: three roundings
        assert torch.allclose(out.double(), want, rtol=0, atol=2.5e-7 * 4 + 3 * 16 * 2.0 ** -24)
