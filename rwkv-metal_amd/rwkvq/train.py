"""The operators of a training step around the packed products.

    linear_act(x, weight, bias, activation, residual)  act(x W^T + b) + r, one pass, with gradients
    embedding(idx, weight, scale, padding_idx)          scale * W[idx] of a table that is trained
    grad_norm(grads)                                    the 2-norm over a list of gradients
    clip_grad_norm(grads, max_norm, out)                <- mlx.optimizers.clip_grad_norm
    clip_grad_norm_(parameters, max_norm)               the same in place, on .grad
    LinearAct, ScaledEmbedding                          the modules over the first two

Reference call sites: the projections and low-rank tanh / sigmoid branches the
stock quantizer leaves dense (rwkv_metal/lora/finetune.py:40-42,
rwkv_metal/model/rwkv7_x070.py:108-111,142-182), the FFN's relu^2
(rwkv7_x070.py:215-221), the table's lookup (rwkv7_x070.py:302) and the clip of
the fine-tune loop (rwkv_metal/lora/finetune.py:108-205).

Operands of one dtype stay in it; any other mix computes in float32, as in the
packed products, and under torch.autocast linear_act computes in its dtype.  Tensors must live on the ROCm GPU; there is no CPU path.
"""
from __future__ import annotations

import array
import operator
from typing import Iterable, List, Optional, Sequence, Tuple

import torch
from torch import Tensor, nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from ._lib import DTYPE_CODE, check, lib
from .ops import (_DeviceGuard, _eager, _float, _functorch_active, _on_gpu, _ptr, _ready, _stream_on,
                  _tracing)

ACTIVATIONS = (None, "relu", "relu2", "silu", "gelu", "sigmoid", "tanh")
_ACT_CODE = {a: i for i, a in enumerate(ACTIVATIONS)}
_SLOPE_NONE, _SLOPE_Y, _SLOPE_BOUND16, _SLOPE_F32, _SLOPE_WIDE16 = range(5)
# the dtype a tensor of slopes is allocated in; BOUND16 holds float16 values but for
# those below 2^-14, whose bits have a code of their own
_SLOPE_DTYPE = {_SLOPE_BOUND16: torch.float16, _SLOPE_F32: torch.float32, _SLOPE_WIDE16: torch.int16}


def _workspace(device: torch.device, nbytes: int) -> Optional[Tensor]:
    """Scratch memory of one call's launches, from torch's caching allocator and
    back to it when the call returns: the allocator hands it on only to later work of
    the stream that was current here, which is the one launched on.  Nothing is kept
    from call to call (a backward pass takes as much as its output's gradient)."""
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes > 0 else None


_workspace_bytes: dict = {}  # (query, *its arguments) -> bytes


def _queried_workspace(query: str, args: tuple, device: torch.device, what: str) -> Optional[Tensor]:
    """The workspace that the entry point `query` asks for with `args`.  The caller
    holds it until its launches are queued."""
    key = (query, *args)
    nbytes = _workspace_bytes.get(key)
    if nbytes is None:
        nbytes = getattr(lib(), query)(*args)
        check(min(nbytes, 0), what)
        if len(_workspace_bytes) > 4096:
            _workspace_bytes.clear()
        _workspace_bytes[key] = nbytes
    return _workspace(device, nbytes)


def _addr(t: Optional[Tensor]) -> int:
    return 0 if t is None or t.numel() == 0 else t.data_ptr()


def _size(t: Optional[Tensor]) -> int:
    return 0 if t is None else t.numel()


# -------------------------------------------------------------- linear_act

_slope_kinds: dict = {}   # (activation code, dtype code, residual?) -> rq_linear_slope


def _slope_kind(act: int, dt: int, residual: bool) -> int:
    key = (act, dt, residual)
    kind = _slope_kinds.get(key)
    if kind is None:
        kind = lib().rq_linear_slope(act, dt, int(residual))
        check(min(kind, 0), "linear_act")
        _slope_kinds[key] = kind
    return kind


def _linear_impl(x: Tensor, weight: Tensor, bias: Optional[Tensor], residual: Optional[Tensor],
                 act: int, want_slope: bool) -> Tuple[Tensor, Optional[Tensor]]:
    """y, and the slopes where they are wanted and the backward pass reads them."""
    _on_gpu(x, weight, *[t for t in (bias, residual) if t is not None])
    lead, k = x.shape[:-1], x.shape[-1]
    n = weight.shape[0]
    x, weight = _ready(x), _ready(weight)
    bias = None if bias is None else _ready(bias)
    residual = None if residual is None else _ready(residual)
    m = 1
    for s in lead:
        m *= s
    dt = DTYPE_CODE[x.dtype]
    ydt = x.dtype if residual is None else residual.dtype
    y = torch.empty(*lead, n, dtype=ydt, device=x.device)
    kind = _slope_kind(act, dt, residual is not None) if want_slope else _SLOPE_NONE
    slope = None
    if kind >= _SLOPE_BOUND16:
        slope = torch.empty(*lead, n, device=x.device, dtype=_SLOPE_DTYPE[kind])
    if m and n:
        with _DeviceGuard(x.device):
            stream = _stream_on(x.device)
            ws = _queried_workspace("rq_linear_workspace_bytes", (m, n, k, dt), x.device,
                                    "linear_act")
            rc = lib().rq_linear(_ptr(x), _ptr(weight), _addr(bias), dt, _addr(residual),
                                 DTYPE_CODE[ydt], m, n, k, act, y.data_ptr(), _addr(slope),
                                 _addr(ws), _size(ws), stream)
        if rc:
            check(rc, "linear_act")
    return y, slope


def _linear_backward_impl(dy: Tensor, x: Optional[Tensor], weight: Optional[Tensor],
                          saved: Optional[Tensor], act: int, kind: int, want_b: bool,
                          dtype: torch.dtype):
    """(dx, dw, db) of operands of `dtype`: dw where x is given, dx where the weight is."""
    _on_gpu(dy, *[t for t in (x, weight) if t is not None])
    n, k = dy.shape[-1], 0 if x is weight is None else (weight if x is None else x).shape[-1]
    dy = _ready(dy)
    x = None if x is None else _ready(x)
    weight = None if weight is None else _ready(weight)
    m = dy.numel() // n if n else 0
    device = dy.device
    dx = None if weight is None else torch.empty(*dy.shape[:-1], k, dtype=dtype, device=device)
    dw = None if x is None else torch.empty(n, k, dtype=dtype, device=device)
    db = torch.empty(n, dtype=dtype, device=device) if want_b else None
    if n == 0:
        return None if dx is None else dx.zero_(), dw, db
    dt, ydt = DTYPE_CODE[dtype], DTYPE_CODE[dy.dtype]
    with _DeviceGuard(device):
        stream = _stream_on(device)
        ws = _queried_workspace("rq_linear_backward_workspace_bytes",
                                (m, n, k, dt, ydt, kind, dx is not None, dw is not None, want_b),
                                device, "linear_act backward")
        rc = lib().rq_linear_backward(
            _ptr(dy), ydt, _addr(saved) if kind != _SLOPE_NONE else 0, kind, act, _addr(x),
            _addr(weight), dt, m, n, k, _addr(dx), _addr(dw), _addr(db), _addr(ws), _size(ws),
            stream)
    if rc:
        check(rc, "linear_act backward")
    return dx, dw, db


def _save(ctx, x, weight, residual, act, y, slope) -> None:
    """Keeps for the backward pass what the gradients wanted read: x for dw, the weight for
    dx, the slopes (or y) for all of them.  A frozen layer keeps no activations."""
    need_x, need_w = ctx.needs_input_grad[:2]
    ctx.act, ctx.dtype = act, x.dtype
    ctx.kind = _slope_kind(act, DTYPE_CODE[x.dtype], residual is not None)
    saved = y if ctx.kind == _SLOPE_Y else slope if ctx.kind >= _SLOPE_BOUND16 else None
    ctx.save_for_backward(x if need_w else None, weight if need_x else None, saved)


def _linear_op_impl(x: Tensor, weight: Tensor, bias: Optional[Tensor], residual: Optional[Tensor],
                    act: int, want_slope: bool = True) -> Tuple[Tensor, Tensor]:
    y, slope = _linear_impl(x, weight, bias, residual, act, want_slope)
    return y, x.new_empty(0) if slope is None else slope


_linear_op = torch.library.custom_op("rwkvq::linear_act", _linear_op_impl, mutates_args=())


@_linear_op.register_fake
def _(x, weight, bias, residual, act, want_slope=True):
    shape = (*x.shape[:-1], weight.shape[0])
    kind = _slope_kind(act, DTYPE_CODE[x.dtype], residual is not None) if want_slope else _SLOPE_NONE
    slope = x.new_empty(0) if kind < _SLOPE_BOUND16 else x.new_empty(shape, dtype=_SLOPE_DTYPE[kind])
    return x.new_empty(shape, dtype=x.dtype if residual is None else residual.dtype), slope


def _linear_backward_op_impl(dy: Tensor, x: Optional[Tensor], weight: Optional[Tensor],
                             saved: Optional[Tensor], act: int, kind: int, want_b: bool,
                             dtype: torch.dtype) -> Tuple[Tensor, Tensor, Tensor]:
    got = _linear_backward_impl(dy, x, weight, saved, act, kind, want_b, dtype)
    return tuple(dy.new_empty(0, dtype=dtype) if t is None else t for t in got)


_linear_backward_op = torch.library.custom_op("rwkvq::linear_act_backward", _linear_backward_op_impl,
                                              mutates_args=())


@_linear_backward_op.register_fake
def _(dy, x, weight, saved, act, kind, want_b, dtype):
    # row-major whatever the operands' own strides, as the kernels write them
    n = dy.shape[-1]
    return (dy.new_empty(0 if weight is None else (*dy.shape[:-1], weight.shape[-1]), dtype=dtype),
            dy.new_empty(0 if x is None else (n, x.shape[-1]), dtype=dtype),
            dy.new_empty(n if want_b else 0, dtype=dtype))


def _linear_op_setup(ctx, inputs, output):
    x, weight, bias, residual, act, want_slope = inputs
    ctx.set_materialize_grads(False)  # else the unused slopes get a gradient of zeros
    ctx.want_slope = want_slope
    if want_slope:
        _save(ctx, x, weight, residual, act, *output)


def _linear_op_backward(ctx, dy, _dslope):
    need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
    if dy is None:
        return (None,) * 6
    dx = dw = db = None
    if need_x or need_w or need_b:
        if not ctx.want_slope:
            raise RuntimeError("rwkvq::linear_act was called with want_slope=False: only its residual has a "
                               "gradient")
        x, weight, saved = ctx.saved_tensors
        dx, dw, db = _linear_backward_op(dy.contiguous(), x if need_w else None,
                                         weight if need_x else None, saved, ctx.act, ctx.kind, need_b,
                                         ctx.dtype)
    return (dx if need_x else None, dw if need_w else None, db if need_b else None,
            dy if need_r else None, None, None)


_linear_op.register_autograd(_linear_op_backward, setup_context=_linear_op_setup)


class _LinearActFunction(torch.autograd.Function):
    """The registered op's autograd formula without its dispatch, for plain eager
    GPU tensors."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        need_pre = ctx.needs_input_grad[0] or ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        y, slope = _linear_impl(x, weight, bias, residual, act, need_pre)
        if need_pre:
            _save(ctx, x, weight, residual, act, y, slope)
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():  # a graph of this pass is wanted; it has none
            return _LinearActFunction._once(ctx, dy)
        return _LinearActFunction._gradients(ctx, dy)

    @staticmethod
    def _gradients(ctx, dy):
        need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
        dx = dw = db = None
        if need_x or need_w or need_b:
            x, weight, saved = ctx.saved_tensors
            dx, dw, db = _linear_backward_impl(dy, x if need_w else None, weight if need_x else None,
                                               saved, ctx.act, ctx.kind, need_b, ctx.dtype)
        return dx, dw, db, dy if need_r else None, None

    _once = staticmethod(once_differentiable(_gradients.__func__))


def linear_act(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None,
               activation: Optional[str] = None, residual: Optional[Tensor] = None) -> Tensor:
    """act(x @ weight^T + bias) + residual in one pass over the output.

    x [..., k], weight [n, k], bias [n]; residual [..., n] is added after the
    activation and may be float32 beside 16-bit operands: y then is too, a
    float32 residual stream.  Under torch.autocast x, weight and bias are cast to its
    dtype, as nn.Linear casts them.  activation: None, "relu", "relu2" (relu(v)^2),
    "silu", "gelu" (v Phi(v)), "sigmoid" or "tanh".  The sums, the activation and
    the residual's addition are in float32, rounded once.

    The backward pass keeps x where the weight has a gradient, the weight where x has
    one, and the slope act'(v): read off y for relu
    (and float32 relu2) without a residual, else a tensor of its own, 16 bits with
    three more of them significant than bf16's (as many below 2^-14) beside bf16
    operands and float32 beside others.  Its products take g = dy act'(v) rounded to the operands' type
    (past 65504 an infinity beside float16)."""
    if activation not in _ACT_CODE:
        raise ValueError(f"activation must be one of {ACTIVATIONS} (got {activation!r})")
    _float(x, "x")
    _float(weight, "weight")
    if weight.dim() != 2:
        raise ValueError("linear_act expects a 2-D weight")
    if x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x has shape {tuple(x.shape)} but the weight expects an inner dimension of "
                         f"{weight.shape[1]}")
    if bias is not None:
        _float(bias, "bias")
        if bias.shape != (weight.shape[0],):
            raise ValueError(f"bias must have shape {(weight.shape[0],)} (got {tuple(bias.shape)})")
    if residual is not None:
        _float(residual, "residual")
        want = (*x.shape[:-1], weight.shape[0])
        if residual.shape != want:
            raise ValueError(f"residual must have shape {want} (got {tuple(residual.shape)})")
    dt = x.dtype
    if x.is_cuda and torch.is_autocast_enabled("cuda"):
        cast = torch.get_autocast_dtype("cuda")
    elif weight.dtype != dt or (bias is not None and bias.dtype != dt):
        cast = torch.float32
    else:
        cast = None
    if cast is not None:
        dt = cast
        x, weight = x.to(dt), weight.to(dt)
        bias = None if bias is None else bias.to(dt)
    if residual is not None and residual.dtype not in (dt, torch.float32):
        residual = residual.to(torch.float32)
    act = _ACT_CODE[activation]
    ts = [t for t in (x, weight, bias, residual) if t is not None]
    if _eager(*ts):
        if not torch.is_grad_enabled() or not any(t.requires_grad for t in ts):
            return _linear_impl(x, weight, bias, residual, act, False)[0]
        if forward_ad._current_level < 0:
            return _LinearActFunction.apply(x, weight, bias, residual, act)
    return _linear_op(x, weight, bias, residual, act, _records(x, weight, bias))[0]


def _records(*ts: Optional[Tensor]) -> bool:
    """Whether a recorded call has to keep what gradients of these operands take.  A
    functorch transform or torch.jit.trace may ask for them later."""
    if not torch.is_grad_enabled():
        return False
    if any(t is not None and t.requires_grad for t in ts):
        return True
    return not torch.compiler.is_compiling() and (_functorch_active() or _tracing() is not None)


class LinearAct(nn.Linear):
    """nn.Linear with an activation and an optional residual in its product's
    output stage: forward(x, residual=None) = act(x W^T + b) + residual."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True,
                 activation: Optional[str] = None, device=None, dtype=None):
        super().__init__(in_features, out_features, bias, device=device, dtype=dtype)
        if activation not in _ACT_CODE:
            raise ValueError(f"activation must be one of {ACTIVATIONS} (got {activation!r})")
        self.activation = activation

    @classmethod
    def from_linear(cls, linear: nn.Linear, activation: Optional[str] = None) -> "LinearAct":
        """The same parameters (shared, not copied) with an activation behind them."""
        m = cls(linear.in_features, linear.out_features, linear.bias is not None, activation,
                device="meta", dtype=linear.weight.dtype)
        m.weight, m.bias = linear.weight, linear.bias
        return m

    def forward(self, x: Tensor, residual: Optional[Tensor] = None) -> Tensor:
        return linear_act(x, self.weight, self.bias, self.activation, residual)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, activation={self.activation}"


# --------------------------------------------------------------- embedding

_INDEX_TYPES = (torch.int64, torch.int32)


def _embed_impl(idx: Tensor, weight: Tensor, scale: float) -> Tensor:
    _on_gpu(weight, idx)
    idx, weight = idx.contiguous(), weight.contiguous()
    vocab, dim = weight.shape
    out = torch.empty(*idx.shape, dim, dtype=weight.dtype, device=weight.device)
    if out.numel():
        with _DeviceGuard(weight.device):
            rc = lib().rq_embed(_ptr(idx), idx.element_size(), idx.numel(), _ptr(weight),
                                DTYPE_CODE[weight.dtype], vocab, dim, scale, out.data_ptr(),
                                _stream_on(weight.device))
        if rc:
            check(rc, "embedding")
    return out


def _embed_grad_impl(dout: Tensor, idx: Tensor, vocab: int, scale: float, padding_idx: int) -> Tensor:
    _on_gpu(dout, idx)
    dout, idx = dout.contiguous(), idx.contiguous()
    dim, n = dout.shape[-1], idx.numel()
    dw = torch.empty(vocab, dim, dtype=dout.dtype, device=dout.device)
    if dw.numel():
        L = lib()
        with _DeviceGuard(dout.device):
            stream = _stream_on(dout.device)
            ws = _queried_workspace("rq_embed_grad_workspace_bytes", (n, vocab, dim), dout.device,
                                    "embedding backward")
            rc = L.rq_embed_grad(_ptr(idx), idx.element_size(), n, _ptr(dout), DTYPE_CODE[dout.dtype],
                                 vocab, dim, scale, padding_idx, dw.data_ptr(), _addr(ws), _size(ws),
                                 stream)
        if rc:
            check(rc, "embedding backward")
    return dw


def _embed_op_impl(idx: Tensor, weight: Tensor, scale: float, padding_idx: int) -> Tensor:
    return _embed_impl(idx, weight, scale)


_embed_op = torch.library.custom_op("rwkvq::embedding", _embed_op_impl, mutates_args=())
_embed_grad_op = torch.library.custom_op("rwkvq::embedding_grad", _embed_grad_impl, mutates_args=())


@_embed_op.register_fake
def _(idx, weight, scale, padding_idx):
    return weight.new_empty(*idx.shape, weight.shape[1])


@_embed_grad_op.register_fake
def _(dout, idx, vocab, scale, padding_idx):
    return dout.new_empty(vocab, dout.shape[-1])


def _embed_setup(ctx, inputs, output):
    idx, weight, ctx.scale, ctx.padding_idx = inputs
    ctx.vocab = weight.shape[0]
    ctx.save_for_backward(idx)


def _embed_backward(ctx, dout):
    idx, = ctx.saved_tensors
    dw = None
    if ctx.needs_input_grad[1]:
        dw = _embed_grad_op(dout, idx, ctx.vocab, ctx.scale, ctx.padding_idx)
    return None, dw, None, None


_embed_op.register_autograd(_embed_backward, setup_context=_embed_setup)


class _EmbeddingFunction(torch.autograd.Function):
    """The registered op's autograd formula without its dispatch."""

    @staticmethod
    def forward(ctx, idx, weight, scale, padding_idx):
        ctx.save_for_backward(idx)
        ctx.vocab, ctx.scale, ctx.padding_idx = weight.shape[0], scale, padding_idx
        return _embed_impl(idx, weight, scale)

    @staticmethod
    def backward(ctx, dout):
        if torch.is_grad_enabled():  # a graph of this pass is wanted; it has none
            return _EmbeddingFunction._once(ctx, dout)
        return _EmbeddingFunction._gradients(ctx, dout)

    @staticmethod
    def _gradients(ctx, dout):
        idx, = ctx.saved_tensors
        return None, _embed_grad_impl(dout, idx, ctx.vocab, ctx.scale, ctx.padding_idx), None, None

    _once = staticmethod(once_differentiable(_gradients.__func__))


def embedding(idx: Tensor, weight: Tensor, scale: float = 1.0,
              padding_idx: Optional[int] = None) -> Tensor:
    """scale * weight[idx], rounded once: idx integers of any shape, weight
    [vocab, dim].  Indices outside the table give rows of NaN and no gradient.
    The table's gradient is dense: scale times the float32 sum of each token's rows,
    in an order that does not change from run to run; 0 for padding_idx."""
    _float(weight, "weight")
    if weight.dim() != 2:
        raise ValueError("embedding expects a 2-D table")
    if idx.dtype not in _INDEX_TYPES:
        if idx.dtype not in (torch.int16, torch.uint8, torch.int8):
            raise ValueError(f"indices must be an integer tensor (got {idx.dtype})")
        idx = idx.to(torch.int32)
    vocab = weight.shape[0]
    pad = -1
    if padding_idx is not None:
        if not -vocab <= padding_idx < vocab:
            raise ValueError(f"padding_idx {padding_idx} is outside the table of {vocab} rows")
        pad = padding_idx % vocab
    scale = float(scale)
    if _eager(idx, weight):
        if not (weight.requires_grad and torch.is_grad_enabled()):
            return _embed_impl(idx, weight, scale)
        if forward_ad._current_level < 0:
            return _EmbeddingFunction.apply(idx, weight, scale, pad)
    return _embed_op(idx, weight, scale, pad)


class ScaledEmbedding(nn.Embedding):
    """nn.Embedding whose rows are multiplied by `scale` in the lookup."""

    def __init__(self, num_embeddings: int, embedding_dim: int, scale: float = 1.0,
                 padding_idx: Optional[int] = None, device=None, dtype=None):
        super().__init__(num_embeddings, embedding_dim, padding_idx, device=device, dtype=dtype)
        self.scale = scale

    @classmethod
    def from_pretrained(cls, embeddings: Tensor, freeze: bool = True, padding_idx: Optional[int] = None,
                        scale: float = 1.0) -> "ScaledEmbedding":
        """The module over a table that is there (shared, not copied)."""
        if embeddings.dim() != 2:
            raise ValueError("embedding expects a 2-D table")
        m = cls(*embeddings.shape, scale=scale, padding_idx=padding_idx, device="meta", dtype=embeddings.dtype)
        m.weight = nn.Parameter(embeddings, requires_grad=not freeze)
        return m

    def forward(self, idx: Tensor) -> Tensor:
        return embedding(idx, self.weight, self.scale, self.padding_idx)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, scale={self.scale}"


# --------------------------------------------------- gradient norm and clip

_dtype_of = operator.attrgetter("dtype")


def _grad_list(grads: Sequence[Tensor], out: Optional[Sequence[Tensor]], sizes: List[int],
               codes: List[int]) -> array.array:
    """The tensors as an array of rq_grad: (g, out, n, dtype code), 8 bytes each
    (the dtype's upper four are rq_grad's padding).  Column by column: a model has
    hundreds of gradients, and a loop over them would take longer than the launches."""
    a = array.array("q", bytes(32 * len(grads)))
    a[0::4] = array.array("q", map(Tensor.data_ptr, grads))
    a[1::4] = a[0::4] if out is None else array.array("q", map(Tensor.data_ptr, out))
    a[2::4] = array.array("q", sizes)
    a[3::4] = array.array("q", codes)
    return a


def _check_grads(grads: Sequence[Tensor]) -> Tuple[torch.device, List[int]]:
    """The one GPU that holds them all, and their dtype codes, or an error."""
    try:
        devices = set(map(Tensor.get_device, grads))
        if len(devices) == 1 and -1 not in devices:
            return grads[0].device, list(map(DTYPE_CODE.__getitem__, map(_dtype_of, grads)))
    except (TypeError, KeyError):
        pass
    for t in grads:
        if not isinstance(t, Tensor):
            raise ValueError(f"gradients must be tensors (got {type(t).__name__})")
        _float(t, "gradients")
    _on_gpu(*grads)
    raise AssertionError("unreachable")


def _contiguous(ts: Sequence[Tensor]) -> bool:
    try:
        return all(map(Tensor.is_contiguous, ts))
    except RuntimeError:
        raise ValueError("sparse gradients are not supported") from None


def _dense(t: Tensor) -> bool:
    """Whether the tensor's elements fill its memory without gaps, in any order
    of the dimensions: the norm and the factor do not depend on the order."""
    if t.is_contiguous():
        return True
    expect = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != expect:
            return False
        expect *= size
    return True


def _run_norm(grads, out, sizes, codes, max_norm, eps, device) -> Tensor:
    norm = torch.empty((), dtype=torch.float32, device=device)
    a = _grad_list(grads, out, sizes, codes)
    at, n = a.buffer_info()[0], len(grads)
    L = lib()
    with _DeviceGuard(device):
        stream = _stream_on(device)
        nbytes = L.rq_grad_norm_workspace_bytes(at, n)
        check(min(nbytes, 0), "clip_grad_norm")
        ws = _workspace(device, max(nbytes, 16))
        if max_norm is None:
            rc = L.rq_grad_norm(at, n, norm.data_ptr(), ws.data_ptr(), ws.numel(), stream)
        else:
            rc = L.rq_clip_grads(at, n, max_norm, eps, norm.data_ptr(), ws.data_ptr(), ws.numel(),
                                 stream)
    check(rc, "clip_grad_norm")
    return norm


@torch.no_grad()
def grad_norm(grads: Iterable[Tensor]) -> Tensor:
    """sqrt(sum of squares of every element of every tensor), a float32 scalar on
    the GPU (nothing waits for it).  The squares are added in float64.  An empty
    list has norm 0 and gives a CPU tensor."""
    grads = list(grads)
    if not grads:
        return torch.zeros(())
    device, codes = _check_grads(grads)
    if not _contiguous(grads):
        grads = [t if _dense(t) else t.contiguous() for t in grads]
    return _run_norm(grads, None, list(map(Tensor.numel, grads)), codes, None, 0.0, device)


@torch.no_grad()
def clip_grad_norm(grads: Iterable[Tensor], max_norm: float, out: Optional[Sequence[Tensor]] = None,
                   eps: float = 1e-6) -> Tuple[List[Tensor], Tensor]:
    """(clipped, norm): every gradient times min(max_norm / (norm + eps), 1), the
    factor in float32 and one rounding, and the norm over all of them
    (mlx.optimizers.clip_grad_norm).  out: contiguous tensors of the gradients'
    sizes and dtypes to write to (they may be the gradients themselves); by
    default views of one new buffer for each dtype.  A NaN norm makes every
    gradient NaN.  A gradient listed twice with one output counts twice in the norm
    and is scaled once; outputs that overlap otherwise are refused, and so are
    gradients and outputs that overlap in a way that leaves no order."""
    grads = list(grads)
    max_norm, eps = float(max_norm), float(eps)
    if not max_norm >= 0 or not eps >= 0:
        raise ValueError(f"max_norm and eps must not be negative (got {max_norm} and {eps})")
    if out is not None:
        out = list(out)
        if len(out) != len(grads):
            raise ValueError(f"out has {len(out)} tensors for {len(grads)} gradients")
    if not grads:
        return [], torch.zeros(())
    device, codes = _check_grads(grads)
    sizes = list(map(Tensor.numel, grads))
    if out is None:
        out = _new_like(grads)
    else:
        on, kinds = _check_grads(out)
        if on != device:
            raise ValueError(f"rwkvq ops take every operand on one device; got '{device}' and '{on}'")
        if kinds != codes or list(map(Tensor.numel, out)) != sizes or not _contiguous(out):
            raise ValueError("out must hold contiguous tensors of the gradients' sizes and dtypes")
    src = grads if _contiguous(grads) else [t.contiguous() for t in grads]
    return out, _run_norm(src, out, sizes, codes, max_norm, eps, device)


def _new_like(grads: Sequence[Tensor]) -> List[Tensor]:
    """A contiguous tensor for each, cut from one buffer per dtype."""
    out: list = [None] * len(grads)
    by: dict = {}
    for i, t in enumerate(grads):
        by.setdefault(t.dtype, []).append(i)
    for dtype, places in by.items():
        # whole 16-byte lines, so that every view stays on the wide path
        per = 16 // dtype.itemsize
        sizes = [-(-grads[i].numel() // per) * per for i in places]
        flat = torch.empty(sum(sizes), dtype=dtype, device=grads[0].device)
        for i, p in zip(places, flat.split(sizes)):
            out[i] = p[:grads[i].numel()].view(grads[i].shape)
    return out


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm: float, eps: float = 1e-6) -> Tensor:
    """Clips the .grad of the parameters (or one parameter) in place and returns
    the norm over them, a float32 scalar on the GPU; parameters without a
    gradient are left out.  Nothing is written where the norm is within
    max_norm.  A gradient listed twice (tied weights) counts twice in the norm and is
    scaled once; gradients that overlap otherwise are refused.  The gradients are
    written through their memory: autograd's version counters do not see it."""
    if isinstance(parameters, Tensor):
        parameters = [parameters]
    grads = [g for g in (p.grad for p in parameters) if g is not None]
    max_norm, eps = float(max_norm), float(eps)
    if not max_norm >= 0 or not eps >= 0:
        raise ValueError(f"max_norm and eps must not be negative (got {max_norm} and {eps})")
    if not grads:
        return torch.zeros(())
    device, codes = _check_grads(grads)
    sizes = list(map(Tensor.numel, grads))
    if _contiguous(grads):
        return _run_norm(grads, None, sizes, codes, max_norm, eps, device)
    dense = [t if _dense(t) else t.contiguous() for t in grads]
    norm = _run_norm(dense, None, sizes, codes, max_norm, eps, device)
    for t, d in zip(grads, dense):
        if t is not d:
            t.copy_(d)
    return norm
