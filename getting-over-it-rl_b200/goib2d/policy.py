"""The policy's side of a batch of worlds: a memory per world (the gated delta rule) and gradient clipping.

    memory = torch.zeros(N, heads, K, V, device="cuda")                       # float32, one matrix per world and head
    o = goib2d.delta_step_(memory, q, k, v, g, beta, reset=fell)              # acting: one token per world
    o, last = goib2d.delta_rule(q, k, v, g, beta, state=first, reset=resets)  # training: (N, T, ...) rollouts
    norm = goib2d.clip_grads_([p.grad for p in net.parameters()], 0.5)        # before the optimiser's step

Per world and head the memory is a matrix S (K, V). A token with decay a = exp(g), key k, value v, query q and write
strength b = beta does

    S' = a S;  r = v - S'^T k;  S = S' + k (b r)^T;  o = scale S^T q

and a token whose `reset` is set (the world's reset came before it), or whose decay is 0 in float32, starts from
S' = 0 whatever S held. q and k may have fewer heads than v: value head h reads key head h // (heads // key_heads).
All of q, k, v, g, beta are float32 or all bfloat16; memories and every sum are float32. Acting computes in float32;
rollouts multiply on the matrix units, their operands in two parts each where a state depends on them (2e-6 off in
float32, 3.4e-6 for the states of bfloat16 rollouts) and rounded to bfloat16 where only bfloat16 results do (o 2.0e-3
off, gradients 1.7e-3 to 3.3e-3, of which their own rounding is 1.7e-3; the gradients of at most 4096 tokens are computed
in full). So a replayed o is within about 2e-3 of the one acted on, not equal to it.

The kernels are in libgoib2d.so (csrc/delta_*.cu, csrc/clip.cu; the C calls are goib2d_delta_* and goib2d_clip_grads):
there is no CPU path. Calls run on the current stream of the tensors' device and return without waiting for it. What they
write in place (a memory, a given out, clipped gradients) counts as modified for autograd. No forward-mode derivatives.
"""
import struct
from array import array

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import native

_DTYPE = {torch.float32: 0, torch.bfloat16: 1}
_DESC = struct.Struct("2q5if9P20q")   # goib2d_delta_desc
_GRADS = struct.Struct("8P18q")       # goib2d_delta_grads
_GRAD = struct.Struct("Pqi4x")        # goib2d_grad (as three int64 words in clip_grads_' table)
MAX_DIM = 128                         # largest key_dim and value_dim


def _rows(name, x, shape, dtype, device, channels=True):
    """x's address and element strides, for a tensor of this shape whose channels (last axis) are contiguous."""
    if x.shape != shape or x.dtype != dtype or x.device != device:
        raise ValueError(f"{name} must be {tuple(shape)} {dtype} on {device}, got {tuple(x.shape)} {x.dtype} on {x.device}")
    st = x.stride()
    if channels:
        if st[-1] != 1 and shape[-1] > 1:
            raise ValueError(f"{name}: the last axis must be contiguous")
        st = st[:-1]
    return x.data_ptr(), st


def _state(name, x, shape, device):
    if x.shape != shape or x.dtype != torch.float32 or x.device != device or not x.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {tuple(shape)} float32 tensor on {device}, got "
                         f"{tuple(x.shape)} {x.dtype} on {x.device}")
    return x.data_ptr()


def _reset(x, shape, device):
    if x is None:
        return 0, (0, 0)
    if x.dtype not in (torch.bool, torch.uint8) or x.shape != shape or x.device != device:
        raise ValueError(f"reset must be {tuple(shape)} bool or uint8 on {device}, got {tuple(x.shape)} {x.dtype} on {x.device}")
    return x.data_ptr(), x.stride()


def _like(v):
    """An uninitialised tensor for o: v's order of axes in memory where that leaves o's channels contiguous (of overlapping
    windows torch's choice need not)."""
    out = torch.empty_like(v)
    return out if out.stride()[-1:] == (1,) else torch.empty(v.shape, dtype=v.dtype, device=v.device)


def _sizes(q, v, steps):
    """(worlds, steps, heads, key heads, K, V) of q (N, [T,] key heads, K) and v (N, [T,] heads, V)."""
    dims = 4 if steps else 3
    if not (isinstance(q, torch.Tensor) and isinstance(v, torch.Tensor) and q.is_cuda and v.is_cuda):
        raise TypeError("q and v must be CUDA tensors")
    if q.dim() != dims or v.dim() != dims or v.dtype not in _DTYPE:
        raise ValueError(f"q and v must be float32 or bfloat16 tensors of {dims} axes, got {tuple(q.shape)} {q.dtype} and "
                         f"{tuple(v.shape)} {v.dtype}")
    hk, K = q.shape[-2:]
    if steps:
        n, t, h, V = v.shape
    else:
        (n, h, V), t = v.shape, 1
    if h < 1 or hk < 1 or h % hk:
        raise ValueError(f"{h} value heads over {hk} key heads")
    if not (1 <= K <= MAX_DIM and 1 <= V <= MAX_DIM):
        raise ValueError(f"key and value channels must be 1..{MAX_DIM}, got {K} and {V}")
    return n, t, h, hk, K, V


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _no_tangents(name, *tensors):
    """Raw pointers would drop forward-mode tangents. Asked for within torch.autograd.forward_ad.dual_level() only, outside
    which the level is -1."""
    if any(x is not None and forward_ad.unpack_dual(x).tangent is not None for x in tensors):
        raise ValueError(f"{name} has no forward-mode derivative")


def delta_step_(state, q, k, v, g, beta, reset=None, scale=None, out=None):
    """One token for every world: state (N, H, K, V) float32 is updated in place, and o (N, H, V) in v's type is
    returned. q, k (N, Hk, K), v (N, H, V), g (log decay) and beta (N, H), reset (N,) bool or None; scale defaults
    to K ** -0.5. Inputs may have any strides with contiguous channels. Not differentiable: rollouts train through
    delta_rule."""
    # everything in one expression first: an acting loop calls this once per world step
    device, dt = v.device, v.dtype
    vs, qs, ks, gs, bs = v.stride(), q.stride(), k.stride(), g.stride(), beta.stride()
    written = state
    if out is None:
        out = torch.empty_like(v)
    else:
        written = (state, out)
    shape, heads = v.shape, g.shape
    os_ = out.stride()
    if not (len(vs) == len(qs) == len(os_) == 3 and q.shape == k.shape and heads == beta.shape and heads == shape[:2] and
            out.shape == shape and q.shape[0] == shape[0] and state.shape == (*heads, q.shape[2], shape[2]) and
            vs[2] == qs[2] == ks[2] == os_[2] == 1 and dt in _DTYPE and
            dt is q.dtype is k.dtype is g.dtype is beta.dtype is out.dtype and state.dtype is torch.float32 and
            0 <= v.get_device() == q.get_device() == k.get_device() == g.get_device() == beta.get_device() ==
            out.get_device() == state.get_device() and state.is_contiguous()):
        if written is state:
            out = _like(v)
            os_ = out.stride()
        _check_step(state, q, k, v, g, beta, out)
    n, h, V = shape
    hk, K = q.shape[1:]
    if not (0 < K <= MAX_DIM and 0 < V <= MAX_DIM and hk > 0 and h > 0 and h % hk == 0):
        _sizes(q, v, False)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or g.requires_grad or
                                    beta.requires_grad or state.requires_grad or out.requires_grad):
        raise ValueError("delta_step_ is not differentiable: use delta_rule, or torch.no_grad()")
    if forward_ad._current_level >= 0:
        _no_tangents("delta_step_", state, q, k, v, g, beta, out)
    rp, rs = (0, (0,)) if reset is None else _reset(reset, (n,), device)
    sp = state.data_ptr()
    desc = _DESC.pack(n, 1, h, hk, K, V, _DTYPE[dt], K ** -0.5 if scale is None else scale, q.data_ptr(), k.data_ptr(),
                      v.data_ptr(), g.data_ptr(), beta.data_ptr(), rp, sp, sp, out.data_ptr(),
                      qs[0], 0, qs[1], ks[0], 0, ks[1], vs[0], 0, vs[1], gs[0], 0, gs[1], bs[0], 0, bs[1],
                      os_[0], 0, os_[1], rs[0], 0)
    _call(device, native.load().goib2d_delta_step, desc)
    increment_version(written)  # a graph that saved what was there before raises
    return out


def _check_step(state, q, k, v, g, beta, out):
    """delta_step_'s refusals, one by one (a channel axis of size 1 may have any stride)."""
    n, _, h, hk, K, V = _sizes(q, v, False)
    device, dt = v.device, v.dtype
    _state("state", state, (n, h, K, V), device)
    for name, x, shape in (("q", q, (n, hk, K)), ("k", k, (n, hk, K)), ("v", v, (n, h, V)), ("out", out, (n, h, V))):
        _rows(name, x, shape, dt, device)
    for name, x in (("g", g), ("beta", beta)):
        _rows(name, x, (n, h), dt, device, False)


def _call(device, function, *args):
    """A C call on the tensors' device and its current stream (the last argument)."""
    index = device.index
    if index == torch.cuda.current_device():
        rc = function(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            rc = function(*args, _raw_stream(index))
    if rc:
        native.check(rc)


def _describe(sizes, q, k, v, g, beta, state, reset, scale, last, out):
    """goib2d_delta_desc of a rollout call."""
    n, t, h, hk, K, V = sizes
    device, dt = v.device, v.dtype
    qs, ks, vs, gs, bs, os_ = q.stride(), k.stride(), v.stride(), g.stride(), beta.stride(), out.stride()
    if not (q.shape == k.shape == (n, t, hk, K) and g.shape == beta.shape == (n, t, h) and
            qs[3] == ks[3] == vs[3] == 1 and dt is q.dtype is k.dtype is g.dtype is beta.dtype and
            v.get_device() == q.get_device() == k.get_device() == g.get_device() == beta.get_device()):
        for name, x, shape in (("q", q, (n, t, hk, K)), ("k", k, (n, t, hk, K)), ("v", v, (n, t, h, V))):
            _rows(name, x, shape, dt, device)
        for name, x in (("g", g), ("beta", beta)):
            _rows(name, x, (n, t, h), dt, device, False)
    rp, rs = (0, (0, 0)) if reset is None else _reset(reset, (n, t), device)
    sp = 0 if state is None else _state("state", state, (n, h, K, V), device)
    return _DESC.pack(n, t, h, hk, K, V, _DTYPE[dt], scale, q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(),
                      beta.data_ptr(), rp, sp, last.data_ptr(), out.data_ptr(), qs[0], qs[1], qs[2], ks[0], ks[1], ks[2],
                      vs[0], vs[1], vs[2], *gs, *bs, os_[0], os_[1], os_[2], *rs)


def _forward(q, k, v, g, beta, state, reset, scale, train):
    """(o, last state, what the backward pass reads or None, the bytes that it works in)."""
    sizes = n, _, h, _, K, V = _sizes(q, v, True)
    device = v.device
    lib = native.load()
    out = _like(v)
    last = torch.empty((n, h, K, V), dtype=torch.float32, device=device) if state is None else torch.empty_like(state)
    desc = _describe(sizes, q, k, v, g, beta, state, reset, scale, last, out)
    saved, work = None, 0
    if train:
        size, work = lib.goib2d_delta_saved_bytes(desc), lib.goib2d_delta_workspace_bytes(desc)
        native.check(min(size, work, 0))
        saved = torch.empty(size, dtype=torch.uint8, device=device)
    _call(device, lib.goib2d_delta_forward, desc, saved.data_ptr() if train else None)
    return out, last, saved, work


class _DeltaRule(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, state, reset, scale):
        ctx.set_materialize_grads(False)
        out, last, saved, ctx.work = _forward(q, k, v, g, beta, state, reset, scale, True)
        # neither state is read backwards: the caller may go on with the last one, or with the first one's memory
        ctx.save_for_backward(q, k, v, g, beta, reset, saved)
        ctx.scale = scale
        return out, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dlast):
        q, k, v, g, beta, reset, saved = ctx.saved_tensors
        if dout is None and dlast is None:
            return (None,) * 8
        sizes = n, t, h, hk, K, V = _sizes(q, v, True)
        device, dt = v.device, v.dtype
        lib = native.load()
        work = torch.empty(max(ctx.work, 16), dtype=torch.uint8, device=device)
        desc = _describe(sizes, q, k, v, g, beta, None, reset, ctx.scale, work, v)  # o and the states are not read
        dop, dos = 0, (0, 0, 0)
        if dout is not None:
            dout = dout if dout.stride(-1) == 1 else dout.contiguous()
            dop, dos = dout.data_ptr(), dout.stride()[:3]
        dlast = None if dlast is None else dlast.contiguous()
        dq, dk = (torch.empty((n, t, hk, K), dtype=dt, device=device) for _ in range(2))
        dv = torch.empty((n, t, h, V), dtype=dt, device=device)
        dg, dbeta = (torch.empty((n, t, h), dtype=dt, device=device) for _ in range(2))
        first = None
        if ctx.needs_input_grad[5]:
            first = torch.empty((n, h, K, V), dtype=torch.float32, device=device)
        grads = _GRADS.pack(dop, 0 if dlast is None else dlast.data_ptr(), dq.data_ptr(), dk.data_ptr(),
                            dv.data_ptr(), dg.data_ptr(), dbeta.data_ptr(), 0 if first is None else first.data_ptr(),
                            *dos, *dq.stride()[:3], *dk.stride()[:3], *dv.stride()[:3], *dg.stride(), *dbeta.stride())
        _call(device, lib.goib2d_delta_backward, desc, grads, saved.data_ptr(), work.data_ptr())
        return dq, dk, dv, dg, dbeta, first, None, None


def delta_rule(q, k, v, g, beta, state=None, reset=None, scale=None):
    """Rollouts of T tokens per world: (o (N, T, H, V) in v's type, last state (N, H, K, V) float32). q, k
    (N, T, Hk, K), v (N, T, H, V), g (log decay) and beta (N, T, H), state: the first state (N, H, K, V) float32 or
    None (zeros), reset (N, T) bool or None; scale defaults to K ** -0.5. Any strides with contiguous channels, so a
    rollout recorded step by step goes in as x.transpose(0, 1). Differentiable in q, k, v, g, beta and state."""
    if scale is None:
        scale = q.shape[-1] ** -0.5
    if forward_ad._current_level >= 0:
        _no_tangents("delta_rule", q, k, v, g, beta, state)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or g.requires_grad or
                                    beta.requires_grad or (state is not None and state.requires_grad)):
        return _DeltaRule.apply(q, k, v, g, beta, state, reset, float(scale))
    return _forward(q, k, v, g, beta, state, reset, float(scale), False)[:2]


def _dense(x):
    """Whether x's elements fill one piece of memory, in any order of its axes."""
    n = 1
    for stride, size in sorted((st, sz) for st, sz in zip(x.stride(), x.shape) if sz > 1):
        if stride != n:
            return False
        n *= size
    return True


def clip_grads_(grads, max_norm):
    """Scale all gradients, in place, by min(1, max_norm / (norm + 1e-6)), where norm is the 2-norm of all their
    elements together; returns norm (a float32 scalar on the device). grads: float32 or bfloat16 CUDA tensors on one
    device, dense in memory and not overlapping; None entries are skipped. A NaN or an infinity among them makes the
    result NaN where the formula does."""
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"max_norm must be a number >= 0, got {max_norm}")
    words, written = [], []  # words: address, elements, type, one tensor after the other (goib2d_grad)
    index, type_of, strided = None, _DTYPE.get, torch.strided
    for x in grads:
        if x is None:
            continue
        if index is None:
            device, index = x.device, x.get_device()
            if index < 0:
                raise TypeError("gradients must be CUDA tensors")
        dt = type_of(x.dtype)
        if dt is None or x.get_device() != index or x.layout is not strided:
            raise ValueError(f"gradients must be dense float32 or bfloat16 tensors on {device}, got {x.dtype} on {x.device} "
                             f"({x.layout})")
        if not (x.is_contiguous() or _dense(x)):
            raise ValueError(f"a gradient of shape {tuple(x.shape)} and strides {x.stride()} is not dense in memory")
        n = x.numel()
        if n:
            words += x.data_ptr(), n, dt
            written.append(x)
    if index is None:
        raise ValueError("no gradients")
    if forward_ad._current_level >= 0:
        _no_tangents("clip_grads_", *written)
    count = len(written)
    if len(set(words[::3])) != count:
        raise ValueError("the same gradient twice")
    table = array("q", words)
    packed = table.buffer_info()[0]
    lib = native.load()
    size = lib.goib2d_clip_workspace_bytes(packed, count)
    native.check(min(size, 0))
    result = torch.empty(size // 4 + 4, dtype=torch.float32, device=device)  # the norm, and the workspace 16 bytes on
    at = result.data_ptr()
    _call(device, lib.goib2d_clip_grads, packed, count, max_norm, at, at + 16)
    increment_version(written)
    return result[0]
