"""Selective state-space operators on MI355X: the recurrence

    S_t = exp(-exp(A_log) d_t) S_{t-1} + (d_t x_t) B_t^T,   y_t = S_t C_t + D x_t,

with ``d_t = softplus(dt_t + dt_bias)``, per head a ``(head_dim, state_dim)``
float32 state, B and C shared by the consecutive heads of a group, and the
short causal conv with SiLU in front of it. The decay is
:func:`gated_delta.forget_gate` of ``dt``; the state layout, the conv taps and
the slot pool (:class:`RecurrentStatePool`) are those of the gated-delta
layer. :func:`gated_rms_norm` behind it is ``silu(z) * rms_norm(y)`` per head, for
layers that normalise first and gate then; those that gate first and normalise
the product, over a head or a group's channels, bring their own norm.

* :func:`conv_silu`       -- conv + SiLU + conv-state roll over packed prompts
* :func:`selective_scan`  -- the recurrence over prompts (batch-first or packed)
* :func:`selective_step`  -- both for one token of ``B`` sequences, in place in
  a slot pool if asked

The reference has no such layer. Every call runs on the GPU that holds its
tensors; none has a gradient (a tensor that needs one, or that forward mode
follows, raises ``RuntimeError``).
"""

from __future__ import annotations

import functools

import torch

from . import _lib
from .config import StateSpaceDims
from .gated_delta import (_FLOATS, _as, _c, _check_cu_seqlens, _check_out, _promote, _require_device,
                          _stream)
from .linear_attention import _index_array, _rows, check_half_bits, check_slots
from .quant import _followed

_MAX_STATE = 256   # state_dim, both kernels
_MAX_HEAD = 256    # head_dim, the step kernel
_MAX_STEP = 1 << 22  # elements between the rows that the scan reads in place
_F32 = torch.float32


class PackedRuns:
    """Checked offsets of ``N`` packed runs (``N + 1`` of them, from 0 to the
    token count, non-decreasing), on the host and on ``device``: what
    ``cu_seqlens`` of :func:`conv_silu` and :func:`selective_scan` may be given
    instead of a sequence, to check and copy the offsets once for all layers
    of a model (and to capture the calls into a graph)."""

    def __init__(self, offsets, device: torch.device | str = "cuda") -> None:
        host = torch.as_tensor(offsets)
        if host.numel() and (host.is_floating_point() or host.is_complex() or host.dtype == torch.bool):
            raise ValueError(f"offsets must be whole numbers, got {host.dtype}")
        host = host.to("cpu", torch.int64)
        if host.ndim != 1 or host.numel() < 2:
            raise ValueError("offsets must be 1-D with at least two entries")
        self.offsets = tuple(_check_cu_seqlens(host, int(host[-1])))
        self.on_device = torch.tensor(self.offsets, dtype=torch.int32).to(device)
        self.longest = max(b - a for a, b in zip(self.offsets, self.offsets[1:]))

    @property
    def tokens(self) -> int:
        return self.offsets[-1]

    def __len__(self) -> int:
        return len(self.offsets) - 1


def _runs(cu_seqlens, T: int, device) -> PackedRuns:
    if not isinstance(cu_seqlens, PackedRuns):
        cu_seqlens = PackedRuns(cu_seqlens, device)
    if cu_seqlens.tokens != T:
        raise ValueError(f"cu_seqlens must run from 0 to the token count {T}")
    if cu_seqlens.on_device.device != device:
        raise ValueError(f"cu_seqlens are on {cu_seqlens.on_device.device}, the tensors on {device}")
    return cu_seqlens


def _operands(*tensors) -> torch.device:
    """The one GPU that holds these tensors (None skipped), floats without a
    gradient all of them. A step or a short prompt is host-bound, hence the
    integer comparisons (a device object each costs more)."""

    index, device = -1, None
    for t in tensors:
        if t is None:
            continue
        i = t.get_device()
        if device is None:
            index, device = i, t.device
        if i != index or i < 0 or t.dtype not in _FLOATS:
            return _require_device(*tensors)  # raises what is wrong
    _no_gradient(*tensors)
    return device


def _no_gradient(*tensors) -> None:
    if _followed(*tensors):
        raise RuntimeError("the state-space operators have no gradient and no forward mode; call them under "
                           "torch.no_grad()")


def _f32_vector(t: torch.Tensor, n: int, name: str) -> torch.Tensor:
    if t.ndim != 1 or t.shape[0] != n:
        raise ValueError(f"{name} must have shape ({n},), got {tuple(t.shape)}")
    return t if t.dtype is _F32 and t.is_contiguous() else t.float().contiguous()


def _token_rows(t: torch.Tensor, T: int, heads: int, dim: int) -> tuple[torch.Tensor, int]:
    """``t (tokens, heads, dim)``, batch-first or packed, as rows that the
    kernels read in 16-byte pieces, and their stride: in place where the rows
    are packed, aligned, no closer than their width and no further apart than
    the kernels address (column slices of one projection or conv output), else a
    copy."""

    st, width = t.stride(), heads * dim
    step, packed = st[-3], st[-1] == 1 and (st[-2] == dim or heads == 1)
    if t.ndim == 4 and t.shape[0] > 1:
        if t.shape[1] == 1:
            step = st[0]
        else:
            packed = packed and st[0] == t.shape[1] * step
    if T <= 1:
        step = width
    if packed and width <= step <= _MAX_STEP and step * t.element_size() % 16 == 0 and t.data_ptr() % 16 == 0:
        return t, step
    return t.clone(memory_format=torch.contiguous_format), width


@functools.lru_cache(maxsize=1024)
def _scan_workspace(*sizes: int) -> int:
    return int(_lib.load().gdn_selective_scan_workspace_size(*sizes))


def conv_silu(x: torch.Tensor, conv_state: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
              cu_seqlens=None, *, conv_out: torch.Tensor | None = None):
    """``silu(bias + causal depthwise conv(x))`` for N packed runs.

    ``x (T, C)`` (rows at any stride, e.g. columns of a stacked projection);
    ``conv_state (N, K-1, C)``, the rows before each run; ``weight (C, K)`` or
    ``(C, K, 1)``, 2 to 4 taps, the last on the current token; ``bias (C,)`` or
    None; ``cu_seqlens`` the N+1 offsets of the runs (a host sequence or
    :class:`PackedRuns`), or None for N equal runs. Returns ``(out (T, C),
    new_conv (N, K-1, C))`` in x's dtype, the state in ``conv_out`` when given
    (contiguous, not overlapping ``conv_state``). float32 arithmetic with one
    rounding; the state is the raw rows."""

    if x.ndim != 2 or conv_state.ndim != 3:
        raise ValueError("x must be (T, C) and conv_state (N, K-1, C)")
    T, C = x.shape
    N, K = conv_state.shape[0], conv_state.shape[1] + 1
    if not 2 <= K <= 4:
        raise ValueError(f"conv_silu takes 2 to 4 taps, got {K}")
    if C == 0 or N == 0 or conv_state.shape[2] != C or weight.numel() != C * K or weight.shape[:2] != (C, K):
        raise ValueError("conv_silu: conv_state and weight do not match x's channels")
    if bias is not None and bias.shape != (C,):
        raise ValueError(f"bias must have shape ({C},), got {tuple(bias.shape)}")
    if T >= 2 ** 31:
        raise ValueError("the token count must fit int32")
    device = _operands(x, conv_state, weight, bias)
    cu = None
    if cu_seqlens is not None:
        runs = _runs(cu_seqlens, T, device)
        if len(runs) != N:
            raise ValueError(f"cu_seqlens hold {len(runs)} runs, conv_state {N}")
        cu = runs.on_device
    elif T % N:
        raise ValueError(f"{T} tokens do not split into {N} equal runs; pass cu_seqlens")
    if x.stride(1) != 1 or (T > 1 and x.stride(0) < C):
        x = x.contiguous()
    stride = x.stride(0) if T > 1 else C
    conv_state = _c(_as(conv_state, x.dtype))
    weight = _c(_as(weight, _F32))
    bias = None if bias is None else _c(_as(bias, _F32))
    out = x.new_empty((T, C))
    if conv_out is None:
        conv_out = x.new_empty((N, K - 1, C))
    else:
        _check_out(conv_out, (N, K - 1, C), x.dtype, device, conv_state, "conv_out")
    _lib.call_on(device, "gdn_conv_silu", _lib.ptr(x), stride, _lib.ptr(conv_state), _lib.ptr(conv_out),
                 _lib.ptr(weight), _lib.ptr(bias), _lib.ptr(cu), N, T, _lib.ptr(out), C, K, _lib.dtype_code(x.dtype),
                 _stream(device))
    return out, conv_out


def selective_scan(x: torch.Tensor, dt: torch.Tensor, B: torch.Tensor, C: torch.Tensor, A_log: torch.Tensor,
                   dt_bias: torch.Tensor, D: torch.Tensor | None = None, state: torch.Tensor | None = None, *,
                   cu_seqlens=None, y_dtype: torch.dtype | None = None, state_out: torch.Tensor | None = None):
    """The selective scan over prompts.

    Batch-first: ``x (R, L, H, P)``, ``dt (R, L, H)``, ``B, C (R, L, G, N)``.
    Packed: with ``cu_seqlens`` (R+1 offsets: a host sequence or
    :class:`PackedRuns`) ``x (T, H, P)``, ``dt (T, H)``, ``B, C (T, G, N)``.
    ``A_log, dt_bias, D (H,)``; head h reads group ``h // (H / G)``. ``state
    (R, H, P, N)`` or None (zeros); each run starts from its own, and an empty
    run returns it. x, B and C may be column slices of one conv output. ``P``
    and ``N`` are multiples of 8, ``N`` at most 256.

    Returns ``(y, new_state)``: y shaped as x in ``y_dtype`` (x's dtype by
    default), the state float32, in ``state_out`` when given (which may be
    ``state`` itself, and must not overlap it otherwise). bfloat16 inputs with
    bfloat16 y run on the bf16 matrix cores with float32 sums and state; the
    decayed scores and a copy of the state are rounded to bfloat16 on their way to
    y (error 1.9e-3 of its norm, 1.7e-3 of it y's own rounding). Every other mix
    runs on the float32 ones, in full: so do bfloat16 inputs under
    ``y_dtype=torch.float32``, at about twice the time. NaN or infinity in a token
    reaches that and the later tokens of its run, none before it."""

    packed = cu_seqlens is not None
    lead = 1 if packed else 2
    if x.ndim != lead + 2 or B.ndim != lead + 2 or C.shape != B.shape:
        raise ValueError("x must be (tokens, H, P) and B, C (tokens, G, N), batch-first or with cu_seqlens")
    if B.shape[:lead] != x.shape[:lead] or dt.shape != x.shape[:-1]:
        raise ValueError("dt, B and C must match x's leading (token) axes, and dt its heads")
    H, P = x.shape[-2:]
    G, N = B.shape[-2:]
    if min(H, P, G, N) <= 0 or H % G:
        raise ValueError("the heads must be a nonzero multiple of the groups")
    if P % 8 or N % 8 or N > _MAX_STATE:
        raise ValueError(f"head_dim and state_dim must be multiples of 8, state_dim at most {_MAX_STATE}; "
                         f"got {P} and {N}")
    device = _operands(x, dt, B, C, A_log, dt_bias, D, state)
    if packed:
        T = x.shape[0]
        runs = _runs(cu_seqlens, T, device)
        R, longest, cu = len(runs), runs.longest, runs.on_device
    else:
        R, longest = x.shape[:2]
        T, cu = R * longest, None
        if R == 0:
            raise ValueError("selective_scan needs at least one sequence")
        if T >= 2 ** 31:
            raise ValueError("the token count must fit int32")
    if y_dtype is None:
        y_dtype = x.dtype
    y_code = _lib.dtype_code(y_dtype)
    if state is not None:
        if tuple(state.shape) != (R, H, P, N):
            raise ValueError(f"state must have shape {(R, H, P, N)}")
        if state_out is state and state.dtype != _F32:
            raise ValueError("a state updated in place must be float32")
    A_log, dt_bias = _f32_vector(A_log, H, "A_log"), _f32_vector(dt_bias, H, "dt_bias")
    D = None if D is None else _f32_vector(D, H, "D")
    act = _promote(x, B, C)
    shape = x.shape
    x, x_step = _token_rows(_as(x, act), T, H, P)
    B, B_step = _token_rows(_as(B, act), T, G, N)
    C, C_step = _token_rows(_as(C, act), T, G, N)
    dt_step = H
    if not dt.is_contiguous():
        if packed and dt.stride(1) == 1 and dt.stride(0) >= H:
            dt_step = dt.stride(0)
        else:
            dt = dt.contiguous()
    in_place = state is not None and state_out is state
    if state is not None and not in_place:
        state = _c(_as(state, _F32))
        state = state if state.data_ptr() % 16 == 0 else state.clone()
    y = x.new_empty(shape) if y_dtype is act else torch.empty(shape, dtype=y_dtype, device=device)
    if state_out is None:
        state_out = A_log.new_empty((R, H, P, N))
    else:
        src = torch.empty(0, device=device) if state is None or in_place else state
        _check_out(state_out, (R, H, P, N), _F32, device, src, "state_out")
        if state_out.data_ptr() % 16:
            raise ValueError("state_out must be 16-byte aligned")
    act_code = _lib.dtype_code(act)
    nbytes = _scan_workspace(act_code, y_code, R, T, longest, G, H, P, N)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    _lib.call_on(device, "gdn_selective_scan", x.data_ptr(), x_step, B.data_ptr(), B_step, C.data_ptr(), C_step,
                 act_code, dt.data_ptr(), dt_step, _lib.dtype_code(dt.dtype), A_log.data_ptr(),
                 dt_bias.data_ptr(), _lib.ptr(D), _lib.ptr(state), state_out.data_ptr(), y.data_ptr(), y_code,
                 _lib.ptr(cu), R, T, longest, G, H, P, N, _lib.ptr(ws), nbytes, _stream(device))
    return y, state_out


def selective_step(xbc: torch.Tensor, dt: torch.Tensor, conv_state: torch.Tensor, ssm_state: torch.Tensor,
                   conv_weight: torch.Tensor, conv_bias: torch.Tensor | None, A_log: torch.Tensor,
                   dt_bias: torch.Tensor, D: torch.Tensor | None, dims: StateSpaceDims, *, conv_out=None,
                   state_out=None, y_dtype: torch.dtype | None = None, slots=None, conv_half=None,
                   conv_arrivals=None):
    """One token for ``B`` sequences in a single kernel launch: conv + SiLU +
    roll, then the recurrence.

    ``xbc (B, C)`` the channels [x; B; C] before the conv and ``dt (B, H)``, in
    one activation dtype (rows at any stride); ``conv_state (B, K-1, C)`` in
    that dtype; ``ssm_state (B, H, P, N)`` float32; ``conv_weight (C, K)``,
    ``conv_bias (C,)`` or None. ``state_out`` may be ``ssm_state`` (in place);
    ``conv_out`` must be another buffer. ``slots``, ``conv_half`` and
    ``conv_arrivals`` are a pool's, as :func:`fused_decode_step` takes them
    (any number of heads here): the states of ``slots[b]`` are updated in
    place and the conv state rolls into the slot's other half. Slots given as
    an int32 device tensor are used as they are and must be distinct; a row
    whose slot lies outside the pool gets NaN and touches no state. Returns
    ``(y (B, H, P), conv_out, state_out)``, y in ``y_dtype`` (the activation
    dtype by default)."""

    if xbc.ndim != 2:
        raise ValueError("xbc must be (B, C)")
    rows, act = xbc.shape[0], xbc.dtype
    C, H, P, N, K = dims.conv_dim, dims.num_heads, dims.head_dim, dims.state_dim, dims.conv_kernel_dim
    if N % 8 or N > _MAX_STATE or P > _MAX_HEAD or not 2 <= K <= 4:
        raise ValueError(f"selective_step needs state_dim a multiple of 8 up to {_MAX_STATE}, head_dim up to "
                         f"{_MAX_HEAD} and 2 to 4 taps; got {N}, {P} and {K}")
    if xbc.shape[1] != C or dt.shape != (rows, H) or conv_weight.shape[:2] != (C, K) or conv_weight.numel() != C * K:
        raise ValueError("selective_step: xbc, dt or conv_weight do not match the dims")
    device = _operands(xbc, dt, conv_state, ssm_state, conv_weight, conv_bias, A_log, dt_bias, D)
    pool = rows
    slot_t = half_t = None
    if slots is not None:
        pool = ssm_state.shape[0]
        slot_t = _index_array(slots, rows, device, lambda v: check_slots(v, rows, pool), "slots")
        if state_out is not None and state_out is not ssm_state:
            raise ValueError("with slots the state is updated in place (state_out=ssm_state)")
        state_out = ssm_state
    conv_rows = pool
    if conv_half is not None:
        if slots is None:
            raise ValueError("conv_half needs slots")
        if conv_out is not None and conv_out is not conv_state:
            raise ValueError("with conv_half the conv state rolls within conv_state (conv_out=conv_state or None)")
        if not conv_state.is_contiguous():
            raise ValueError("with conv_half, conv_state must be contiguous")
        half_t = _index_array(conv_half, pool, device, lambda v: check_half_bits(v, pool), "conv_half")
        conv_rows = 2 * pool
        conv_out = conv_state
    if conv_arrivals is not None:
        if half_t is None or half_t is not conv_half:
            raise ValueError("conv_arrivals needs conv_half as an int32 device tensor")
        if (not isinstance(conv_arrivals, torch.Tensor) or conv_arrivals.device != device
                or conv_arrivals.dtype != torch.int32 or conv_arrivals.shape != (pool,)
                or not conv_arrivals.is_contiguous()):
            raise ValueError(f"conv_arrivals must be a contiguous int32 device tensor of {pool} counters")
    if conv_state.shape != (conv_rows, K - 1, C) or ssm_state.shape != (pool, H, P, N):
        raise ValueError("selective_step: the states do not match the dims, the rows or the pool")
    if conv_state.dtype != act or dt.dtype != act:
        raise ValueError("xbc, dt and conv_state must share the activation dtype")
    if ssm_state.dtype != _F32 or not ssm_state.is_contiguous() or ssm_state.data_ptr() % 16:
        raise ValueError("ssm state must be contiguous, 16-byte aligned float32")
    (xbc, s_x), (dt, s_dt) = _rows(xbc), _rows(dt)
    conv_state = _c(conv_state)
    conv_weight = _c(_as(conv_weight, _F32))
    conv_bias = None if conv_bias is None else _f32_vector(conv_bias, C, "conv_bias")
    A_log, dt_bias = _f32_vector(A_log, H, "A_log"), _f32_vector(dt_bias, H, "dt_bias")
    D = None if D is None else _f32_vector(D, H, "D")
    if conv_out is None:
        conv_out = torch.empty((rows, K - 1, C), dtype=act, device=device)
    elif half_t is None:
        _check_out(conv_out, (rows, K - 1, C), act, device, conv_state, "conv_out")
    if state_out is None:
        state_out = torch.empty_like(ssm_state)
    elif state_out is not ssm_state:
        _check_out(state_out, ssm_state.shape, _F32, device, ssm_state, "state_out")
        if state_out.data_ptr() % 16:
            raise ValueError("state_out must be 16-byte aligned")
    y_dtype = y_dtype or act
    y = xbc.new_empty((rows, H, P)) if y_dtype is act else torch.empty((rows, H, P), dtype=y_dtype, device=device)
    _lib.call_on(device, "gdn_selective_step", _lib.ptr(xbc), s_x, _lib.ptr(dt), s_dt, _lib.ptr(conv_state),
                 _lib.ptr(conv_out), _lib.ptr(conv_weight), _lib.ptr(conv_bias), _lib.ptr(A_log), _lib.ptr(dt_bias),
                 _lib.ptr(D), _lib.ptr(ssm_state), _lib.ptr(state_out), _lib.ptr(y), _lib.dtype_code(y_dtype), rows,
                 dims.num_groups, H, P, N, K, _lib.dtype_code(act), _lib.ptr(slot_t), pool, _lib.ptr(half_t),
                 _lib.ptr(conv_arrivals), _stream(device))
    return y, conv_out, state_out
