"""Operators around the routed experts, over the C ABI: token rows sorted by expert and back with their gradients, layer
norm with its gradients, and gradient clipping by the global norm.

Calls enqueue on the current stream of the tensors' device and do not synchronise.  Matrices are [rows, d] with rows
that may lie apart (``stride(0) >= d``, ``stride(1) == 1``), fp32 or bf16.  What a call needs besides its arguments it
takes from the caching allocator, so calls on different streams and captured graphs share nothing.  Autograd records none of them: results are detached, also from
inputs that require gradients, and the backward passes are calls of their own.  What a call writes of its caller's (``out``, gradients
clipped in place, a plan's tensors) counts as modified in place.  Tensors are checked and
the library is called in ``_torch_ops.so`` (csrc/bind/torch_ops.cpp): a small batch is over before Python has looked at its tensors.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import native
from .layer import Layer, Tensor
from .native import OmoeError


def _bind():
    try:
        from . import _torch_ops
    except ImportError as e:
        raise ImportError(f"omega_ai_b200/_torch_ops.so cannot be loaded ({e}): build it with omega_ai_b200.native.build_binding()") from e
    L = native.lib()
    _torch_ops.init({n: C.cast(getattr(L, n), C.c_void_p).value for n in native.OPERATORS}, OmoeError)
    return _torch_ops


_b = _bind()
_plan, _sort, _sort_backward = _b.TokenSort.plan, _b.TokenSort.sort, _b.TokenSort.sort_backward
_unsort, _unsort_backward = _b.TokenSort.unsort, _b.TokenSort.unsort_backward
_norm, _scale, _clip = _b.GradList.norm, _b.GradList.scale, _b.GradList.clip


class TokenSort(_b.TokenSort):
    """Where every pick's row lies once token rows are sorted by expert, and the moves of rows there and back.

    ``plan(topk_idx)`` fills ``pos`` [T, k] (row of each pick, -1 for a pick outside the experts), ``perm`` [rows_cap]
    (flat pick index of each row, -1 where there is none), ``counts`` [E] and ``offsets`` [E + 1] (first row of each
    expert, a multiple of ``row_align``; int32 on the device).  The other methods move rows by the last plan; a plan made
    on one stream is used on another only after the caller has ordered the two.  Sorted buffers have ``rows_cap``
    rows; those behind the last expert's (``offsets[E]`` on) are neither read nor written.
    """

    def __init__(self, tokens: int, top_k: int, n_experts: int, row_align: int = 1, device="cuda"):
        super().__init__(tokens, top_k, n_experts, row_align, torch.device(device))

    def plan(self, topk_idx: torch.Tensor) -> "TokenSort":
        """From the picks [T, k], int32, as the routing leaves them."""
        _plan(self, topk_idx)
        return self

    def sort(self, x: torch.Tensor, out=None, dtype=None) -> torch.Tensor:
        """xs[pos[t, j]] = x[t]; padding rows zero, rows behind the last expert's as they were."""
        return _sort(self, x, out, dtype)

    def sort_backward(self, dxs: torch.Tensor, out=None, dtype=None) -> torch.Tensor:
        """dx[t] = sum over the token's picks of dxs[pos[t, j]]."""
        return _sort_backward(self, dxs, out, dtype)

    def unsort(self, ys: torch.Tensor, weights=None, out=None, dtype=None) -> torch.Tensor:
        """y[t] = sum over the token's picks of weights[t, j] * ys[pos[t, j]]; weights [T, k] fp32, None for 1."""
        return _unsort(self, ys, weights, out, dtype)

    def unsort_backward(self, dy: torch.Tensor, ys: torch.Tensor, weights=None, out=None):
        """(dys, dweights): dys[pos[t, j]] = weights[t, j] * dy[t] of the type of ys, padding rows zero, rows behind the
        last expert's as they were; dweights[t, j] = <dy[t], ys[pos[t, j]]>, None without weights."""
        return _unsort_backward(self, dy, ys, weights, out)


def layer_norm(x: torch.Tensor, gamma=None, beta=None, eps: float = 1e-5, out=None, dtype=None, stats: bool = False):
    """(x - mean) * rstd * gamma + beta per row of x [T, d]; gamma and beta [d] fp32, None for 1 and 0; at addresses
    that are not multiples of 32 bytes they send the rows through the slower kernels for single elements.  With ``stats`` (y, mean, rstd), which
    :func:`layer_norm_backward` takes."""
    return _b.layer_norm(x, gamma, beta, eps, out, dtype, stats)


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, gamma, mean: torch.Tensor, rstd: torch.Tensor, out=None,
                        param_grads: bool = True):
    """(dx, dgamma, dbeta) of :func:`layer_norm`; without ``param_grads`` the last two are None.  dgamma and dbeta share a storage, as
    mean and rstd do."""
    return _b.layer_norm_backward(dy, x, gamma, mean, rstd, out, param_grads)


class LNLayer(Layer):
    """Layer norm behind the engine's operator surface: ``forward(Tensor)``, then ``diff(delta)``, which returns the
    input's gradient and leaves ``diffGamma`` and ``diffBeta``."""

    def __init__(self, width: int, bias: bool = True, eps: float = 1e-5, network=None, device="cuda"):
        super().__init__(network)
        self.width, self.eps = width, eps
        self.gamma = torch.ones(width, dtype=torch.float32, device=device)
        self.beta = torch.zeros(width, dtype=torch.float32, device=device) if bias else None
        self.diffGamma = self.diffBeta = self.mean = self.rstd = None

    def init(self):
        t = self.input
        if self.output_t is None or self.output_t.number != t.number or self.output_t.dtype != t.dtype:
            self.output_t = Tensor(t.number, 1, 1, self.width, dtype=t.dtype, device=t.gpu.device)
        self.number = t.number

    def output(self):
        _, self.mean, self.rstd = layer_norm(self.input.view2d(), self.gamma, self.beta, self.eps,
                                             out=self.output_t.view2d(), stats=True)

    def diff(self, delta: Tensor) -> Tensor:
        dx, self.diffGamma, dbeta = layer_norm_backward(delta.view2d(), self.input.view2d(), self.gamma, self.mean, self.rstd)
        self.diffBeta = dbeta if self.beta is not None else None
        return Tensor.from_device(dx)


class GradList(_b.GradList):
    """Gradient tensors whose global norm is taken and that are clipped by it: contiguous, fp32 or bf16, on one device,
    not overlapping.  Built once per set of tensors, which it keeps; a call after one of them was resized or given another storage is
    refused.  ``out`` (a list of the same sizes and types) receives the clipped gradients; without it they are scaled in place."""

    def __init__(self, grads, out=None):
        super().__init__(list(grads), None if out is None else list(out))

    def norm(self) -> torch.Tensor:
        """The norm of all elements, fp32 on the device."""
        return _norm(self)

    def scale(self, norm: torch.Tensor, max_norm: float) -> None:
        """Times min(1, max_norm / (norm + 1e-6)), for a norm that covers more than this list; 1 where it is not finite."""
        _scale(self, norm, max_norm)

    def clip(self, max_norm: float) -> torch.Tensor:
        """:meth:`norm` and :meth:`scale` in one; returns the norm before clipping."""
        return _clip(self, max_norm)
