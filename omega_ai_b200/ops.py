"""Operators around the routed experts, over the C ABI: token rows sorted by expert and back with their gradients, layer
norm with its gradients, and gradient clipping by the global norm.

Calls enqueue on the current stream of the tensors' device and do not synchronise.  Matrices are [rows, d] with rows
that may lie apart (``stride(0) >= d``, ``stride(1) == 1``), fp32 or bf16.  What a call needs besides its arguments it
takes from the caching allocator, so calls on different streams and captured graphs share nothing.
"""
from __future__ import annotations

import ctypes as C
import functools

import torch

from . import native
from .layer import Layer, Tensor, _dt
from .native import OmoeError


def _bad(message: str):
    raise OmoeError(-1, message)


_current_device = torch._C._cuda_getDevice
_current_stream = torch._C._cuda_getCurrentRawStream  # torch.cuda.current_stream() takes 3 us to say the same


def _call(device, f, *args):
    """The entry point f on the device's current stream, with that device current."""
    index = device.index
    if device.type != "cuda":
        _bad(f"tensors must be on a GPU, got {device}")
    if _current_device() == index:
        rc = f(*args, _current_stream(index))
    else:
        with torch.cuda.device(index):
            rc = f(*args, _current_stream(index))
    if rc != 0:
        raise OmoeError(rc, native.lib().omoe_ops_error().decode())


def _matrix(t: torch.Tensor, rows: int, d: int, name: str, device) -> int:
    """Leading dimension of a [rows, d] matrix on ``device``."""
    if t.shape != (rows, d) or t.device != device:
        _bad(f"{name}: expected [{rows}, {d}] on {device}, got {list(t.shape)} on {t.device}")
    if t.is_contiguous():
        return d
    ld, one = t.stride()
    if one != 1 and d > 1:
        _bad(f"{name}: the elements of a row must be contiguous")
    if rows > 1 and ld < d:
        _bad(f"{name}: rows overlap")
    return ld if rows > 1 else d


def _vector(t, n: int, name: str, device, dtype=torch.float32):
    """Address of a contiguous buffer of n elements, None for None."""
    if t is None:
        return None
    if t.numel() != n or t.dtype != dtype or t.device != device or not t.is_contiguous():
        _bad(f"{name}: expected {n} contiguous {dtype} on {device}")
    return t.data_ptr()


class TokenSort:
    """Where every pick's row lies once token rows are sorted by expert, and the moves of rows there and back.

    ``plan(topk_idx)`` fills ``pos`` [T, k] (row of each pick, -1 for a pick outside the experts), ``perm`` [rows_cap]
    (flat pick index of each row, -1 where there is none), ``counts`` [E] and ``offsets`` [E + 1] (first row of each
    expert, a multiple of ``row_align``; int32 on the device).  The other methods move rows by the last plan; a plan made
    on one stream is used on another only after the caller has ordered the two.  Sorted buffers have ``rows_cap``
    rows; those behind the last expert's (``offsets[E]`` on) are neither read nor written.
    """

    def __init__(self, tokens: int, top_k: int, n_experts: int, row_align: int = 1, device="cuda"):
        self._lib = native.lib()
        cap = self._lib.omoe_sort_rows_cap(tokens, top_k, n_experts, row_align)
        if cap < 0:
            raise OmoeError(int(cap), f"sizes out of range: {tokens} tokens, {top_k} picks, {n_experts} experts, align {row_align}")
        self.tokens, self.top_k, self.n_experts, self.row_align, self.rows_cap = tokens, top_k, n_experts, row_align, int(cap)
        new = lambda *shape: torch.empty(*shape, dtype=torch.int32, device=device)
        self.pos, self.perm = new(tokens, top_k), new(self.rows_cap)
        self.counts, self.offsets = new(n_experts), new(n_experts + 1)
        self.device = self.pos.device
        ptr = lambda t: t.data_ptr()
        self._c = native.Sort(tokens, top_k, n_experts, row_align, self.rows_cap, ptr(self.pos), ptr(self.perm),
                              ptr(self.counts), ptr(self.offsets))
        self._p = C.byref(self._c)

    def plan(self, topk_idx: torch.Tensor) -> "TokenSort":
        """From the picks [T, k], int32, as the routing leaves them."""
        at = _vector(topk_idx, self.tokens * self.top_k, "topk_idx", self.device, torch.int32)
        _call(self.device, self._lib.omoe_sort_plan, self._p, at)
        return self

    def _out(self, out, rows, d, dtype, name):
        if out is None:
            out = torch.empty(rows, d, dtype=dtype, device=self.device)
        return out, _matrix(out, rows, d, name, self.device)

    def sort(self, x: torch.Tensor, out=None, dtype=None) -> torch.Tensor:
        """xs[pos[t, j]] = x[t]; padding rows zero, rows behind the last expert's as they were."""
        d = x.shape[-1]
        ldx = _matrix(x, self.tokens, d, "x", self.device)
        out, ldo = self._out(out, self.rows_cap, d, dtype or x.dtype, "out")
        _call(self.device, self._lib.omoe_sort_rows, self._p, x.data_ptr(), ldx, _dt(x.dtype), out.data_ptr(), ldo,
              _dt(out.dtype), d)
        return out

    def sort_backward(self, dxs: torch.Tensor, out=None, dtype=None) -> torch.Tensor:
        """dx[t] = sum over the token's picks of dxs[pos[t, j]]."""
        d = dxs.shape[-1]
        ldx = _matrix(dxs, self.rows_cap, d, "dxs", self.device)
        out, ldo = self._out(out, self.tokens, d, dtype or dxs.dtype, "out")
        _call(self.device, self._lib.omoe_sort_rows_backward, self._p, dxs.data_ptr(), ldx, _dt(dxs.dtype), out.data_ptr(),
              ldo, _dt(out.dtype), d)
        return out

    def unsort(self, ys: torch.Tensor, weights=None, out=None, dtype=None) -> torch.Tensor:
        """y[t] = sum over the token's picks of weights[t, j] * ys[pos[t, j]]; weights [T, k] fp32, None for 1."""
        d = ys.shape[-1]
        ldy = _matrix(ys, self.rows_cap, d, "ys", self.device)
        w = _vector(weights, self.tokens * self.top_k, "weights", self.device)
        out, ldo = self._out(out, self.tokens, d, dtype or ys.dtype, "out")
        _call(self.device, self._lib.omoe_unsort_rows, self._p, ys.data_ptr(), ldy, _dt(ys.dtype), w, out.data_ptr(), ldo,
              _dt(out.dtype), d)
        return out

    def unsort_backward(self, dy: torch.Tensor, ys: torch.Tensor, weights=None, out=None):
        """(dys, dweights): dys[pos[t, j]] = weights[t, j] * dy[t] of the type of ys, padding rows zero, rows behind the
        last expert's as they were; dweights[t, j] = <dy[t], ys[pos[t, j]]>, None without weights."""
        d = dy.shape[-1]
        lddy = _matrix(dy, self.tokens, d, "dy", self.device)
        ldys = _matrix(ys, self.rows_cap, d, "ys", self.device)
        w = _vector(weights, self.tokens * self.top_k, "weights", self.device)
        out, ldo = self._out(out, self.rows_cap, d, ys.dtype, "out")
        if out.dtype != ys.dtype:
            _bad("out: must have the type of ys")
        dw = None if weights is None else torch.empty(self.tokens, self.top_k, dtype=torch.float32, device=self.device)
        _call(self.device, self._lib.omoe_unsort_rows_backward, self._p, dy.data_ptr(), lddy, _dt(dy.dtype), ys.data_ptr(),
              ldys, _dt(ys.dtype), w, out.data_ptr(), ldo, None if dw is None else dw.data_ptr(), d)
        return out, dw


@functools.lru_cache(maxsize=None)
def _norm_workspace(T: int, d: int) -> int:
    size = native.lib().omoe_layer_norm_backward_workspace(T, d)
    if size < 0:
        _bad(f"x: no rows of width {d}")
    return size


def layer_norm(x: torch.Tensor, gamma=None, beta=None, eps: float = 1e-5, out=None, dtype=None, stats: bool = False):
    """(x - mean) * rstd * gamma + beta per row of x [T, d]; gamma and beta [d] fp32, None for 1 and 0.  With ``stats``
    (y, mean, rstd), which :func:`layer_norm_backward` takes."""
    if x.dim() != 2:
        _bad(f"x: expected [T, d], got {list(x.shape)}")
    T, d = x.shape
    dev = x.device
    ldx = _matrix(x, T, d, "x", dev)
    if out is None:
        out = torch.empty(T, d, dtype=dtype or x.dtype, device=dev)
    ldo = _matrix(out, T, d, "out", dev)
    mean = rstd = None
    if stats:
        mean = torch.empty(T, dtype=torch.float32, device=dev)
        rstd = torch.empty_like(mean)
    _call(dev, native.lib().omoe_layer_norm, x.data_ptr(), ldx, _dt(x.dtype), _vector(gamma, d, "gamma", dev),
          _vector(beta, d, "beta", dev), eps, out.data_ptr(), ldo, _dt(out.dtype), mean.data_ptr() if stats else None,
          rstd.data_ptr() if stats else None, T, d)
    return (out, mean, rstd) if stats else out


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, gamma, mean: torch.Tensor, rstd: torch.Tensor, out=None,
                        param_grads: bool = True):
    """(dx, dgamma, dbeta) of :func:`layer_norm`; without ``param_grads`` the last two are None."""
    if x.dim() != 2:
        _bad(f"x: expected [T, d], got {list(x.shape)}")
    T, d = x.shape
    dev = x.device
    L = native.lib()
    ldx, lddy = _matrix(x, T, d, "x", dev), _matrix(dy, T, d, "dy", dev)
    if out is None:
        out = torch.empty(T, d, dtype=x.dtype, device=dev)
    ldo = _matrix(out, T, d, "out", dev)
    if out.dtype != x.dtype:
        _bad("out: must have the type of x")
    size = _norm_workspace(T, d)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    dgamma = dbeta = None
    if param_grads:
        dgamma = torch.empty(d, dtype=torch.float32, device=dev)
        dbeta = torch.empty_like(dgamma)
    _call(dev, L.omoe_layer_norm_backward, dy.data_ptr(), lddy, _dt(dy.dtype), x.data_ptr(), ldx, _dt(x.dtype),
          _vector(gamma, d, "gamma", dev), _vector(mean, T, "mean", dev), _vector(rstd, T, "rstd", dev), out.data_ptr(), ldo,
          dgamma.data_ptr() if param_grads else None, dbeta.data_ptr() if param_grads else None, T, d, ws.data_ptr(), size)
    return out, dgamma, dbeta


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


class GradList:
    """Gradient tensors whose global norm is taken and that are clipped by it: contiguous, fp32 or bf16, on one device,
    not overlapping.  Built once per set of tensors, which it keeps.  ``out`` (a list of the same shapes and types)
    receives the clipped gradients; without it they are scaled in place."""

    def __init__(self, grads, out=None):
        self.grads, self.out = list(grads), None if out is None else list(out)
        self._lib = native.lib()
        if self.out is not None and [(o.dtype, o.numel()) for o in self.out] != [(g.dtype, g.numel()) for g in self.grads]:
            _bad("out: must have the sizes and types of the gradients")
        every = self.grads + (self.out or [])
        self.device = every[0].device if every else torch.device("cuda", torch.cuda.current_device())
        for t in every:
            if t.device != self.device or not t.is_contiguous():
                _bad("gradients must be contiguous and on one device")
        refs = lambda ts: (native.TensorRef * max(1, len(ts)))(*[native.TensorRef(t.data_ptr(), t.numel(), _dt(t.dtype), 0) for t in ts])
        self._in, self._to = refs(self.grads), None if self.out is None else refs(self.out)

    def _new(self):
        return (torch.empty((), dtype=torch.float32, device=self.device),
                torch.empty(native.GRAD_WORKSPACE_BYTES, dtype=torch.uint8, device=self.device))

    def norm(self) -> torch.Tensor:
        """The norm of all elements, fp32 on the device."""
        norm, ws = self._new()
        _call(self.device, self._lib.omoe_grad_norm, self._in, len(self.grads), norm.data_ptr(), ws.data_ptr(),
              native.GRAD_WORKSPACE_BYTES)
        return norm

    def scale(self, norm: torch.Tensor, max_norm: float) -> None:
        """Times min(1, max_norm / (norm + 1e-6)), for a norm that covers more than this list; 1 where it is not finite."""
        _call(self.device, self._lib.omoe_grad_scale, self._in, self._to, len(self.grads),
              _vector(norm, 1, "norm", self.device), max_norm)

    def clip(self, max_norm: float) -> torch.Tensor:
        """:meth:`norm` and :meth:`scale` in one; returns the norm before clipping."""
        norm, ws = self._new()
        _call(self.device, self._lib.omoe_grad_clip, self._in, self._to, len(self.grads), max_norm, norm.data_ptr(),
              ws.data_ptr(), native.GRAD_WORKSPACE_BYTES)
        return norm
