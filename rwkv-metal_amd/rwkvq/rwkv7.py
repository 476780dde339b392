"""What an RWKV-7 block runs between its products, and the token choice behind its head.

    wkv7(r, w, k, v, a, b, state, cu_seqlens)   the time mixing's recurrence, with gradients
    wkv7_step(r, w, k, v, a, b, state, out)     its form for one token of every sequence
    sample(logits, u, temperature, top_k, top_p, min_p)   tokens from given uniform numbers

Reference call sites: wkv7 / wkv7_train / wkv7_infer (rwkv_metal/kernel/wkv7.py:67-214,
330-381, called at rwkv_metal/model/rwkv7_x070.py:184-187), wkv7_step
(rwkv7_x070.py:174-182) and the carried state (rwkv_metal/model/state.py:33-127).

Inputs of one dtype stay in it; any other mix computes in float32, as in the packed
products.  States are float32.  Tensors must live on the ROCm GPU; there is no CPU path.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch import Tensor
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from ._lib import DTYPE_CODE, check, lib
from .ops import (_PLAIN, _DeviceGuard, _dispatch_modes, _eager, _float, _function_modes, _functorch_active,
                  _is_compiling, _on_gpu, _ptr, _ready, _stream_on, _tracing)
from .train import _addr, _queried_workspace, _records, _size

HEAD_SIZE = 64   # channels of a head
CHUNK = 16       # tokens between two states that are kept for the backward pass


# -------------------------------------------------------------- recurrence

_device_of, _address_of, _contiguous_one = Tensor.get_device, Tensor.data_ptr, Tensor.is_contiguous
_PLAIN_TYPES = frozenset(_PLAIN)


def _operands(ts: list) -> Tuple[list, list]:
    """The tensors as the C entry points take them (on one GPU, contiguous, 16-byte aligned) and their
    addresses.  Column by column: a decode step's launch is shorter than a loop of Python over its operands."""
    devices = set(map(_device_of, ts))
    if len(devices) != 1 or -1 in devices:
        _on_gpu(*ts)
    if not all(map(_contiguous_one, ts)):
        ts = [t.contiguous() for t in ts]
    at = list(map(_address_of, ts))
    low = 0
    for x in at:
        low |= x
    if low & 15:
        ts = list(map(_ready, ts))
        at = list(map(_ptr, ts))
    return ts, at


def _sizes(r: Tensor, cu: Optional[Tensor]) -> Tuple[int, int, int, int]:
    batch, time, heads = r.shape[:3]
    return batch, time, heads, batch if cu is None else cu.numel() - 1


def _chunks(batch: int, time: int, seqs: int, packed: bool) -> int:
    return time // CHUNK + seqs if packed else batch * -(-time // CHUNK)


def _wkv7_impl(r: Tensor, w: Tensor, k: Tensor, v: Tensor, a: Tensor, b: Tensor, state: Optional[Tensor],
               cu: Optional[Tensor], out_dtype: torch.dtype, keep: bool):
    """(y, last state, and where they are kept the states and S a that the backward pass reads)."""
    held, at = _operands([r, w, k, v, a, b] if state is None else [r, w, k, v, a, b, state])
    r = held[0]
    if cu is not None:
        _on_gpu(r, cu)
    batch, time, heads, seqs = _sizes(r, cu)
    f32 = {"dtype": torch.float32, "device": r.device}
    y = torch.empty(r.shape, dtype=out_dtype, device=r.device)
    last = torch.empty(seqs, heads, HEAD_SIZE, HEAD_SIZE, **f32)
    states = sa = None
    if keep:
        n = _chunks(batch, time, seqs, cu is not None)
        states = torch.empty(n, heads, HEAD_SIZE, HEAD_SIZE, **f32)
        sa = torch.empty(n, heads, CHUNK, HEAD_SIZE, **f32)
    L, dt, odt = lib(), DTYPE_CODE[r.dtype], DTYPE_CODE[out_dtype]
    with _DeviceGuard(r.device):
        stream = _stream_on(r.device)
        if time == 1 and cu is None and not keep:
            rc = L.rq_wkv7_step(*at[:6], dt, batch, heads, at[6] if len(at) > 6 else 0, y.data_ptr(), odt,
                                last.data_ptr(), stream)
        else:
            ws = _queried_workspace("rq_wkv7_workspace_bytes", (batch, time, heads, seqs, cu is not None), r.device,
                                    "wkv7")
            rc = L.rq_wkv7(*at[:6], dt, batch, time, heads, 0 if cu is None else cu.data_ptr(), seqs,
                           at[6] if len(at) > 6 else 0, y.data_ptr(), odt, last.data_ptr(), _addr(states), _addr(sa),
                           _addr(ws), _size(ws), stream)
    if rc:
        check(rc, "wkv7")
    return y, last, states, sa


def _wkv7_backward_impl(r, w, k, v, a, b, cu, states, sa, dy, dlast, want_state: bool):
    """The gradients of the six and, where it is wanted, of the first state."""
    ts = [r, w, k, v, a, b, states, sa, dy]
    held, at = _operands(ts if dlast is None else [*ts, dlast])
    r, dy = held[0], held[8]
    if cu is not None:
        _on_gpu(r, cu)
    batch, time, heads, seqs = _sizes(r, cu)
    grads = [torch.empty_like(r) for _ in range(6)]
    dstate = None
    if want_state:
        dstate = torch.empty(seqs, heads, HEAD_SIZE, HEAD_SIZE, dtype=torch.float32, device=r.device)
    with _DeviceGuard(r.device):
        stream = _stream_on(r.device)
        ws = _queried_workspace("rq_wkv7_backward_workspace_bytes", (batch, time, heads, seqs, cu is not None),
                                r.device, "wkv7 backward")
        rc = lib().rq_wkv7_backward(*at[:6], DTYPE_CODE[r.dtype], batch, time, heads,
                                    0 if cu is None else cu.data_ptr(), seqs, *at[6:9], DTYPE_CODE[dy.dtype],
                                    at[9] if len(at) > 9 else 0, *map(_address_of, grads), _addr(dstate), _addr(ws),
                                    _size(ws), stream)
    if rc:
        check(rc, "wkv7 backward")
    return (*grads, dstate)


def _wkv7_op_impl(r: Tensor, w: Tensor, k: Tensor, v: Tensor, a: Tensor, b: Tensor, state: Optional[Tensor],
                  cu: Optional[Tensor], out_dtype: torch.dtype,
                  keep: bool) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
    y, last, states, sa = _wkv7_impl(r, w, k, v, a, b, state, cu, out_dtype, keep)
    none = last.new_empty(0)
    return y, last, none if states is None else states, last.new_empty(0) if sa is None else sa


_wkv7_op = torch.library.custom_op("rwkvq::wkv7", _wkv7_op_impl, mutates_args=())


@_wkv7_op.register_fake
def _(r, w, k, v, a, b, state, cu, out_dtype, keep):
    batch, time, heads, seqs = _sizes(r, cu)
    n = _chunks(batch, time, seqs, cu is not None)
    f32 = {"dtype": torch.float32}
    return (r.new_empty(r.shape, dtype=out_dtype), r.new_empty(seqs, heads, HEAD_SIZE, HEAD_SIZE, **f32),
            r.new_empty((n, heads, HEAD_SIZE, HEAD_SIZE) if keep else 0, **f32),
            r.new_empty((n, heads, CHUNK, HEAD_SIZE) if keep else 0, **f32))


def _wkv7_backward_op_impl(r: Tensor, w: Tensor, k: Tensor, v: Tensor, a: Tensor, b: Tensor,
                           cu: Optional[Tensor], states: Tensor, sa: Tensor, dy: Tensor,
                           dlast: Optional[Tensor], want_state: bool
                           ) -> Tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    *grads, dstate = _wkv7_backward_impl(r, w, k, v, a, b, cu, states, sa, dy, dlast, want_state)
    return (*grads, states.new_empty(0) if dstate is None else dstate)


_wkv7_backward_op = torch.library.custom_op("rwkvq::wkv7_backward", _wkv7_backward_op_impl, mutates_args=())


@_wkv7_backward_op.register_fake
def _(r, w, k, v, a, b, cu, states, sa, dy, dlast, want_state):
    _, _, heads, seqs = _sizes(r, cu)
    return (*[r.new_empty(r.shape) for _ in range(6)],
            states.new_empty((seqs, heads, HEAD_SIZE, HEAD_SIZE) if want_state else 0))


def _gradients(ctx, dy, dlast, backward):
    """The gradients of wkv7's seven tensors from those of its two results (None: 0)."""
    r, w, k, v, a, b, cu, states, sa = ctx.saved_tensors
    if dy is None and dlast is None:
        return (None,) * 7
    if dy is None:
        dy = torch.zeros(r.shape, dtype=ctx.out_dtype, device=r.device)
    got = backward(r, w, k, v, a, b, cu, states, sa, dy.contiguous(), dlast, ctx.needs_input_grad[6])
    return tuple(g if need else None for g, need in zip(got, ctx.needs_input_grad))


def _wkv7_op_setup(ctx, inputs, output):
    r, w, k, v, a, b, state, cu, ctx.out_dtype, ctx.keep = inputs
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(r, w, k, v, a, b, cu, *output[2:])


def _wkv7_op_backward(ctx, dy, dlast, _dstates, _dsa):
    if not ctx.keep:
        raise RuntimeError("rwkvq::wkv7 was called with keep=False: it has no gradients")
    return (*_gradients(ctx, dy, dlast, _wkv7_backward_op), None, None, None)


_wkv7_op.register_autograd(_wkv7_op_backward, setup_context=_wkv7_op_setup)


class _Wkv7Function(torch.autograd.Function):
    """The registered op's autograd formula without its dispatch, for plain eager
    GPU tensors."""

    @staticmethod
    def forward(ctx, r, w, k, v, a, b, state, cu, out_dtype):
        y, last, states, sa = _wkv7_impl(r, w, k, v, a, b, state, cu, out_dtype, True)
        ctx.set_materialize_grads(False)
        ctx.out_dtype = out_dtype
        ctx.save_for_backward(r, w, k, v, a, b, cu, states, sa)
        return y, last

    @staticmethod
    def backward(ctx, dy, dlast):
        if torch.is_grad_enabled():  # a graph of this pass is wanted; it has none
            return _Wkv7Function._once(ctx, dy, dlast)
        return _Wkv7Function._run(ctx, dy, dlast)

    @staticmethod
    def _run(ctx, dy, dlast):
        return (*_gradients(ctx, dy, dlast, _wkv7_backward_impl), None, None)

    _once = staticmethod(once_differentiable(_run.__func__))


def _no_tangents(*ts: Tensor) -> None:
    """Refuses operands with a forward-mode tangent, which would be lost: there is no formula for one."""
    if any(forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise NotImplementedError("wkv7, wkv7_step and sample have no forward-mode derivatives")


def _check_inputs(six: list, dims: int) -> Tuple[torch.Size, list, torch.dtype]:
    """Their shape, and the six in one dtype with it: float32 where they come in several.  Chained
    comparisons: loops over the six took 1 us of a decode step's 10."""
    r, w, k, v, a, b = six
    shape, dt = r.shape, r.dtype
    if not (shape == w.shape == k.shape == v.shape == a.shape == b.shape and dt in DTYPE_CODE
            and dt is w.dtype is k.dtype is v.dtype is a.dtype is b.dtype):
        for name, t in zip("rwkvab", six):
            _float(t, name)
            if t.shape != shape:
                raise ValueError(f"r, w, k, v, a and b must have one shape (got {tuple(shape)} and "
                                 f"{tuple(t.shape)} of {name})")
        dt = torch.float32
        six = [t.to(dt) for t in six]
    if len(shape) != dims or shape[-1] != HEAD_SIZE:
        lead = "[batch, time, heads, 64]" if dims == 4 else "[batch, heads, 64]"
        raise ValueError(f"r, w, k, v, a and b must be {lead} (got {tuple(shape)})")
    return shape, six, dt


def _check_state(state: Tensor, seqs: int, heads: int, name: str = "state") -> None:
    want = (seqs, heads, HEAD_SIZE, HEAD_SIZE)
    if state.dtype != torch.float32 or state.shape != want:
        raise ValueError(f"{name} must be float32 of shape {want} (got {state.dtype} {tuple(state.shape)})")


def _out_dtype(out_dtype: Optional[torch.dtype], dt: torch.dtype) -> torch.dtype:
    if out_dtype is None:
        return dt
    if out_dtype not in (dt, torch.float32):
        raise ValueError(f"out_dtype must be the inputs' {dt} or float32 (got {out_dtype})")
    return out_dtype


def wkv7(r: Tensor, w: Tensor, k: Tensor, v: Tensor, a: Tensor, b: Tensor, state: Optional[Tensor] = None,
         cu_seqlens: Optional[Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> Tuple[Tensor, Tensor]:
    """(y, last state) of the recurrence, for every head with its state S [64, 64]:

        S_t = S_{t-1} diag(exp(-exp(w_t))) + (S_{t-1} a_t) b_t^T + v_t k_t^T,   y_t = S_t r_t

    r, w, k, v, a, b: [batch, time, heads, 64] of any length.  state: float32 [batch, heads,
    64 values, 64 keys] before the first token, 0 by default.  y has the inputs' dtype or
    out_dtype (float32 is the other choice); the state, its products and all sums are float32.

    cu_seqlens: packed sequences in a batch of one; n + 1 int32 or int64 values on the GPU, from 0,
    not decreasing.  Sequence i is the tokens cu_seqlens[i] to cu_seqlens[i + 1] with state i of
    [n, heads, 64, 64] (an empty one keeps its state); y and the gradients are 0 behind the
    last.  Nothing waits for their values: boundaries outside the batch are moved into it, and
    where they decrease the results are undefined.

    In a padded batch a token with w = -inf, k = 0 and b = 0 leaves the state as it was; its r, v and a have to
    be finite.  Tokens are taken in chunks of 16 from a sequence's first: a NaN or an infinity reaches everything
    behind it, and may reach the outputs before it in its own chunk (never another sequence or head).

    Differentiable in all six and the first state, from both results (once).  For the backward pass 1.25 KB
    are kept for each token and head (every 16th state, and S a)."""
    (batch, time, heads, _), six, dt = _check_inputs([r, w, k, v, a, b], 4)
    odt = _out_dtype(out_dtype, dt)
    seqs = batch
    if cu_seqlens is not None:
        if cu_seqlens.dtype not in (torch.int32, torch.int64) or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
            raise ValueError("cu_seqlens must hold the n + 1 boundaries of n sequences as int32 or int64")
        if batch != 1:
            raise ValueError(f"packed sequences take a batch of 1 (got {batch})")
        seqs = cu_seqlens.numel() - 1
        if seqs == 0 and time:
            raise ValueError("cu_seqlens holds no sequence")
        if cu_seqlens.dtype == torch.int64:  # into the batch before the type takes the high bits off
            cu_seqlens = cu_seqlens.clamp(0, time).to(torch.int32)
        cu_seqlens = cu_seqlens.contiguous()
    if state is not None:
        _check_state(state, seqs, heads)
    ts = six if state is None else [*six, state]
    if not _is_compiling() and forward_ad._current_level >= 0:
        _no_tangents(*ts)
    if _eager(*ts):
        if not torch.is_grad_enabled() or not any(t.requires_grad for t in ts):
            return _wkv7_impl(*six, state, cu_seqlens, odt, False)[:2]
        return _Wkv7Function.apply(*six, state, cu_seqlens, odt)
    return _wkv7_op(*six, state, cu_seqlens, odt, _records(*ts))[:2]


# --------------------------------------------------------------- one token

def _plain(ts: list) -> bool:
    """_eager, column by column; that all are on the last one's device is left to _operands."""
    if _is_compiling() or _dispatch_modes() or _function_modes() or _functorch_active() or _tracing() is not None:
        return False
    return _PLAIN_TYPES.issuperset(map(type, ts)) and ts[-1].is_cuda


def _wkv7_step_into(six: list, state: Tensor, out: Tensor, out_dtype: torch.dtype) -> Tensor:
    """y, with the new state in `out`."""
    if not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError("out must be contiguous and 16-byte aligned")
    if out is not state and out.data_ptr() != state.data_ptr() and _overlap(out, state):
        raise ValueError("out may be the state itself, but must not overlap it otherwise")
    held, at = _operands([*six, state, out])
    r = held[0]
    first, size = at[7], r.numel() * r.element_size()
    behind = first + 4 * out.numel()
    if size and min(at[:6]) < behind and max(at[:6]) + size > first:
        # a block writes its head's state while others still read their tokens
        if any(x < behind and x + size > first for x in at[:6]):
            raise ValueError("out must not overlap r, w, k, v, a or b")
    y = torch.empty(r.shape, dtype=out_dtype, device=r.device)
    with _DeviceGuard(r.device):
        rc = lib().rq_wkv7_step(*at[:6], DTYPE_CODE[r.dtype], r.shape[0], r.shape[1], at[6], y.data_ptr(),
                                DTYPE_CODE[out_dtype], at[7], _stream_on(r.device))
    if rc:
        check(rc, "wkv7_step")
    return y


def _wkv7_step_op_impl(r: Tensor, w: Tensor, k: Tensor, v: Tensor, a: Tensor, b: Tensor, state: Tensor,
                       out_dtype: torch.dtype) -> Tuple[Tensor, Tensor]:
    out = torch.empty(state.shape, dtype=torch.float32, device=state.device)
    return _wkv7_step_into([r, w, k, v, a, b], state, out, out_dtype), out


def _wkv7_step_out_op_impl(r: Tensor, w: Tensor, k: Tensor, v: Tensor, a: Tensor, b: Tensor,
                           state: Optional[Tensor], out: Tensor, out_dtype: torch.dtype) -> Tensor:
    return _wkv7_step_into([r, w, k, v, a, b], out if state is None else state, out, out_dtype)


_wkv7_step_op = torch.library.custom_op("rwkvq::wkv7_step", _wkv7_step_op_impl, mutates_args=())
# state None: the one in `out`
_wkv7_step_out_op = torch.library.custom_op("rwkvq::wkv7_step_out", _wkv7_step_out_op_impl, mutates_args=("out",))


@_wkv7_step_op.register_fake
def _(r, w, k, v, a, b, state, out_dtype):
    return r.new_empty(r.shape, dtype=out_dtype), state.new_empty(state.shape)


@_wkv7_step_out_op.register_fake
def _(r, w, k, v, a, b, state, out, out_dtype):
    return r.new_empty(r.shape, dtype=out_dtype)


def wkv7_step(r: Tensor, w: Tensor, k: Tensor, v: Tensor, a: Tensor, b: Tensor, state: Tensor,
              out: Optional[Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> Tuple[Tensor, Tensor]:
    """(y, new state) of one token of every sequence: r .. b [batch, heads, 64], state
    [batch, heads, 64, 64].  out: a contiguous float32 tensor for the new state, `state` itself for an
    update in place; it must not require gradients, nor share memory with r .. b.  Without gradients (wkv7 over a time of 1 has them)."""
    (batch, heads, _), six, dt = _check_inputs([r, w, k, v, a, b], 3)
    odt = _out_dtype(out_dtype, dt)
    _check_state(state, batch, heads)
    ts = [*six, state]
    if out is not None and out is not state:
        _check_state(out, batch, heads, "out")
        ts.append(out)
    if out is not None and out.requires_grad and torch.is_grad_enabled():
        raise ValueError("out is written to without gradients: it must not require them")
    if not _is_compiling() and forward_ad._current_level >= 0:
        _no_tangents(*ts)
    if _plain(ts):
        if out is None:
            out = torch.empty(state.shape, dtype=torch.float32, device=state.device)
            return _wkv7_step_into(six, state, out, odt), out
        y = _wkv7_step_into(six, state, out, odt)
        if not out.is_inference():  # what was saved of it for a backward pass is no longer there
            increment_version(out)
        return y, out
    with torch.no_grad():
        if out is None:
            return _wkv7_step_op(*six, state, odt)
        return _wkv7_step_out_op(*six, None if out is state else state, out, odt), out


def _overlap(x: Tensor, y: Tensor) -> bool:
    """Whether the memory that the two span has bytes in common (x is contiguous)."""
    if y.is_contiguous():
        last = y.numel()
    else:
        last = 1 + sum((n - 1) * s for n, s in zip(y.shape, y.stride()))
    x0, y0 = x.data_ptr(), y.data_ptr()
    return x.numel() > 0 and x0 < y0 + 4 * last and y0 < x0 + 4 * x.numel()


# ------------------------------------------------------------------ sampler

def _sample_impl(logits: Tensor, u: Tensor, temperature: Optional[Tensor], top_k: Optional[Tensor],
                 top_p: Optional[Tensor], min_p: Optional[Tensor], temperature_all: float, top_k_all: int,
                 top_p_all: float, min_p_all: float) -> Tuple[Tensor, Tensor]:
    rows = [None if t is None else t.contiguous() for t in (temperature, top_k, top_p, min_p)]
    _on_gpu(logits, u, *[t for t in rows if t is not None])
    logits, u = logits.contiguous(), u.contiguous()
    token = torch.empty(u.shape, dtype=torch.int64, device=u.device)
    logprob = torch.empty(u.shape, dtype=torch.float32, device=u.device)
    with _DeviceGuard(logits.device):
        rc = lib().rq_sample(_ptr(logits), DTYPE_CODE[logits.dtype], u.numel(), logits.shape[-1], _ptr(u),
                             _addr(rows[0]), temperature_all, _addr(rows[1]), top_k_all, _addr(rows[2]), top_p_all,
                             _addr(rows[3]), min_p_all, _ptr(token), _ptr(logprob), _stream_on(logits.device))
    if rc:
        check(rc, "sample")
    return token, logprob


_sample_op = torch.library.custom_op("rwkvq::sample", _sample_impl, mutates_args=())


@_sample_op.register_fake
def _(logits, u, temperature, top_k, top_p, min_p, temperature_all, top_k_all, top_p_all, min_p_all):
    return u.new_empty(u.shape, dtype=torch.int64), u.new_empty(u.shape, dtype=torch.float32)


def _parameter(x, name: str, lead, whole: bool):
    """(a value for each row, a value for all) of a parameter that is one or the other."""
    if not isinstance(x, Tensor):
        if not whole:
            return None, float(x)
        if int(x) != x:
            raise ValueError(f"{name} must be an integer (got {x})")
        return None, max(-1, min(int(x), 1 << 62))  # any negative number is refused as -1 is
    if x.is_floating_point() if whole else not x.is_floating_point():
        raise ValueError(f"{name} must hold {'integers' if whole else 'floating numbers'} (got {x.dtype})")
    if x.shape != lead:
        if x.dim() > len(lead):
            raise ValueError(f"{name} must be a number or have shape {tuple(lead)} (got {tuple(x.shape)})")
        x = x.expand(lead)
    return x.to(torch.int64 if whole else torch.float32), (0 if whole else 1.0)


def sample(logits: Tensor, u: Tensor, temperature: Union[float, Tensor] = 1.0, top_k: Union[int, Tensor] = 0,
           top_p: Union[float, Tensor] = 1.0, min_p: Union[float, Tensor] = 0.0) -> Tuple[Tensor, Tensor]:
    """(tokens int64, their log-probabilities float32) for logits [..., vocab] and numbers u [...] in
    [0, 1), float32.  With e_i = exp((l_i - max l) / temperature), in this order:

    1. the top_k largest stay (0: all);
    2. of these, from the largest, those before whom less than top_p of their sum lies (1: all);
    3. of these, those with e_i >= min_p;
    4. the token is the first by index at which the running sum of what stays exceeds u times
       the whole.

    Equal logits rank by index.  Each parameter is a number, or a tensor [...] with one for each row
    (numbers of 32 bits).  A temperature of 0, or a top_k of 1, takes the largest.  -inf logits never
    come; a row of nothing else, or with a NaN in it, gives -1 and a NaN.  The sums are exact, of terms of float64
    rounded to 2^-36 of the largest (2^-33 for a vocabulary past 2^17), so the same inputs give the same tokens; one
    whose e_i is below half of that never comes.  Without gradients."""
    _float(logits, "logits")
    if logits.dim() < 1 or u.dtype != torch.float32 or u.shape != logits.shape[:-1]:
        raise ValueError(f"u must be float32 of shape {tuple(logits.shape[:-1])} (got {u.dtype} {tuple(u.shape)})")
    lead = u.shape
    t, t_all = _parameter(temperature, "temperature", lead, False)
    k, k_all = _parameter(top_k, "top_k", lead, True)
    p, p_all = _parameter(top_p, "top_p", lead, False)
    m, m_all = _parameter(min_p, "min_p", lead, False)
    given = [x for x in (t, k, p, m) if x is not None]
    if not _is_compiling() and forward_ad._current_level >= 0:
        _no_tangents(logits, u, *given)
    op = _sample_impl if _eager(logits, u, *given) else _sample_op
    with torch.no_grad():
        return op(logits, u, t, k, p, m, t_all, k_all, p_all, m_all)
