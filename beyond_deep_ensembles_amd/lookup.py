"""Scaled embedding lookup, plain and mean-field Gaussian, with its gradient by sorted tokens.

The first layer of a token model (the reference's text classifiers take theirs from torch).  One kernel per direction step:
lookup, scaling, noise and the rounding to the activations' type in one pass over the touched rows
(``bde_embedding_fwd``); the gradient by a stable sort of the positions and sums in their order (``bde_embedding_bwd``) --
bit-reproducible, where ``torch.nn.functional.embedding`` adds with atomics.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from .ops import BdeKernelError, DTYPE_CODES
from .util import _philox_stream

_TOKEN_TYPES = (torch.int64, torch.int32)
_layers = None
_default = None         # the product's one backend, made at the first call that names none


def _backend(ops):
    """(the kernel backend, the C++ nodes of lib/_bde_host.so or None): the nodes (csrc/host_tokens.cpp) are what this module's
    Python path does, without its interpreter time; they exist for the HIP library only."""
    global _layers, _default
    if _layers is None:
        from . import algo, bbb_layers
        _layers = (algo, bbb_layers)
    if ops is None:
        if _default is None:
            _default = _layers[0]._default_ops()
        ops = _default
    native = _layers[1]._native_nodes(ops)
    return ops, native if native is not None and hasattr(native, "distillation_loss") else None


def _table(tokens, weight, padding_idx, out_dtype, scale):
    """Argument checks shared by both lookups -> (padding_idx or -1, out_dtype, scale)."""
    if tokens.dtype not in _TOKEN_TYPES:
        raise BdeKernelError(f"tokens: expected int64 / int32, got {tokens.dtype}")
    if weight.dim() != 2 or weight.dtype not in DTYPE_CODES:
        raise BdeKernelError(f"weight: expected a float32 / bfloat16 / float16 [V, D] tensor, got {weight.dtype} {tuple(weight.shape)}")
    if tokens.device != weight.device:
        raise BdeKernelError(f"tokens: on {tokens.device}, the weight is on {weight.device}")
    out_dtype = weight.dtype if out_dtype is None else out_dtype
    if out_dtype not in DTYPE_CODES or (weight.dtype != torch.float32 and out_dtype != weight.dtype):
        raise BdeKernelError(f"out_dtype: a {weight.dtype} weight gives {weight.dtype}" +
                             (", torch.bfloat16 or torch.float16" if weight.dtype == torch.float32 else "") + f", not {out_dtype}")
    v = weight.shape[0]
    if padding_idx is None:
        padding_idx = -1
    elif not -v <= padding_idx < v:
        raise BdeKernelError(f"padding_idx {padding_idx} is outside the table of {v} rows")
    elif padding_idx < 0:
        padding_idx += v
    return int(padding_idx), out_dtype, float(scale)


def _row_major(t):
    """Rows may lie apart, their elements not."""
    if t.dim() == 2 and t.shape[1] == 1:          # (a column may carry any second stride)
        return t.reshape(-1).contiguous().view(-1, 1)
    if t.dim() == 2 and t.stride(1) == 1 and (t.stride(0) >= t.shape[1] or t.shape[0] == 1):
        return t
    return t.contiguous()


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, rho, tokens, eps, out_dtype, noise, seed, stream_id, scale, padding_idx, ops):
        w = _row_major(weight.detach())
        r = None if rho is None else _row_major(rho.detach())
        t = tokens.contiguous().view(-1)
        out = torch.empty((t.numel(), w.shape[1]), dtype=out_dtype, device=w.device)
        ops.embedding_fwd(t, w, out, rho=r, noise=noise, eps=eps, seed=seed, stream_id=stream_id, scale=scale, padding_idx=padding_idx)
        ctx.save_for_backward(t, rho, eps)
        ctx.meta = (weight.shape, weight.dtype, noise, seed, stream_id, scale, padding_idx, ops)
        return out.view(tokens.shape + (w.shape[1],))

    @staticmethod
    @once_differentiable          # the kernels produce plain tensors: no double backward
    def backward(ctx, grad_out):
        t, rho, eps = ctx.saved_tensors
        shape, dtype, noise, seed, stream_id, scale, padding_idx, ops = ctx.meta
        g = grad_out.reshape(t.numel(), shape[1])
        if shape[1] > 1 and g.stride(1) != 1:
            g = g.contiguous()    # (rows may coincide: a broadcast gradient is read as it is)
        gw = torch.empty(shape, dtype=dtype, device=t.device)
        gr = None
        if rho is not None and ctx.needs_input_grad[1]:
            r = _row_major(rho.detach())
            gr = torch.empty(shape, dtype=torch.float32, device=t.device)
        else:
            r = None              # the mean's gradient is the plain lookup's
        ops.embedding_bwd(g, t, gw, rho=r, g_rho=gr, noise=noise, eps=eps, seed=seed, stream_id=stream_id, scale=scale,
                          padding_idx=padding_idx)
        return (gw if ctx.needs_input_grad[0] else None, gr) + (None,) * 9


def embedding(tokens: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0, padding_idx: Optional[int] = None,
              out_dtype: Optional[torch.dtype] = None, _ops=None) -> torch.Tensor:
    """``scale * weight[tokens]`` for int64 / int32 ``tokens`` of any shape and a [V, D] ``weight`` (float32, bfloat16 or
    float16; a float32 one may give ``out_dtype`` bfloat16 / float16 activations, rounded once).

    The gradient of ``weight`` is dense and leaves out the positions that hold ``padding_idx``.  A token outside [0, V) gives
    a row of NaN and no gradient (the host does not look at the tokens)."""
    _ops, native = _backend(_ops)
    if native is not None:
        return native.embedding(tokens, weight, None, None, 0, 0, 0, scale, padding_idx, out_dtype)
    padding_idx, out_dtype, scale = _table(tokens, weight, padding_idx, out_dtype, scale)
    return _Embedding.apply(weight, None, tokens, None, out_dtype, None, 0, 0, scale, padding_idx, _ops)


def gaussian_embedding(tokens: torch.Tensor, mean: torch.Tensor, rho: torch.Tensor, *, noise: str = "position",
                       eps: Optional[torch.Tensor] = None, seed: int = 0, stream_id: Optional[int] = None, scale: float = 1.0,
                       padding_idx: Optional[int] = None, out_dtype: Optional[torch.dtype] = None, _ops=None) -> torch.Tensor:
    """``scale * (mean[t] + softplus(rho[t]) * e)``: the lookup in a table of independent Gaussians (float32 ``mean`` / ``rho``).

    ``noise="position"``: every position has its own ``e`` -- the local reparameterisation of a linear layer whose input is
    one-hot (``eps`` of the output's shape).  ``noise="token"``: all positions of a token share ``e``, one draw of the table
    of which only the touched rows are evaluated (``eps`` [V, D]).  Without ``eps`` the kernels generate it (Philox stream
    ``stream_id`` of ``seed``, a fresh stream per call by default) and generate it again in the backward pass; by token it is
    the noise ``GaussianParameter.sample()`` of that stream has.  Positions that hold ``padding_idx`` have no noise and no
    gradient."""
    if noise not in ("position", "token"):
        raise ValueError(f"noise: 'position' or 'token', not {noise!r}")
    if eps is None and stream_id is None:
        stream_id = next(_philox_stream)
    _ops, native = _backend(_ops)
    if native is not None:
        return native.embedding(tokens, mean, rho, eps, 1 if noise == "position" else 2, int(seed), int(stream_id or 0), scale, padding_idx, out_dtype)
    padding_idx, out_dtype, scale = _table(tokens, mean, padding_idx, out_dtype, scale)
    if mean.dtype != torch.float32 or rho.dtype != torch.float32 or rho.shape != mean.shape or rho.device != mean.device:
        raise BdeKernelError("gaussian_embedding: mean and rho must be float32 tensors of one shape and device")
    n, (v, d) = tokens.numel(), mean.shape
    if eps is not None:
        want = (v, d) if noise == "token" else tuple(tokens.shape) + (d,)
        if tuple(eps.shape) != want or eps.dtype != torch.float32 or eps.device != mean.device:
            raise BdeKernelError(f"eps: expected a float32 tensor of shape {want} on {mean.device}, got {eps.dtype} {tuple(eps.shape)} on "
                                 f"{eps.device}")
        if eps.requires_grad:
            raise BdeKernelError("eps: the noise is a constant of this operator (no gradient); detach it")
        eps = _row_major(eps.reshape(v if noise == "token" else n, d))
    return _Embedding.apply(mean, rho, tokens, eps, out_dtype, noise, int(seed), int(stream_id or 0), scale, padding_idx, _ops)


class ScaledEmbedding(nn.Embedding):
    """``nn.Embedding`` (same parameter, state_dict and initialisation) whose lookup is ``embedding``: the rows times ``scale``
    (text models multiply by the square root of the dimension), in ``out_dtype``."""

    def __init__(self, num_embeddings: int, embedding_dim: int, padding_idx: Optional[int] = None, *, scale: float = 1.0,
                 out_dtype: Optional[torch.dtype] = None, device=None, dtype=None, _ops=None):
        super().__init__(num_embeddings, embedding_dim, padding_idx, device=device, dtype=dtype)
        self.scale, self.out_dtype, self._ops = float(scale), out_dtype, _ops

    def __getstate__(self):
        from .ops import HipOps
        state = dict(self.__dict__)
        if isinstance(state.get("_ops"), HipOps):          # bound again at the first use (GaussianParameter does the same)
            state["_ops"] = None
        return state

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        return embedding(tokens, self.weight, scale=self.scale, padding_idx=self.padding_idx, out_dtype=self.out_dtype, _ops=self._ops)

    def extra_repr(self) -> str:
        return super().extra_repr() + f", scale={self.scale:g}"
