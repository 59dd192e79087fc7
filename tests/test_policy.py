"""The policy operators (goib2d.delta_step_, delta_rule, clip_grads_) against their definitions in 64 bits.

Tolerances, on the 2-norm of the difference over the 2-norm of the result. float32: matrix products run on operands
split in two parts (a relative error of 2^-17 a product at most with bfloat16 parts, less with tf32 ones, and independent
from product to product), in chains of at most four products within a chunk: 4 * 2^-17 = 3.1e-5 at most. bfloat16 results: the rounding of the
result (2^-9) and of the two operands of the product that makes it (2^-9 each) at most: 3 * 2^-9 = 5.9e-3. States are
float32 whatever the inputs' type."""
import ctypes as C
import math
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

import goib2d
from goib2d import native, policy

TOL = {torch.float32: 4 * 2.0**-17, torch.bfloat16: 3 * 2.0**-9}
F32, BF16 = torch.float32, torch.bfloat16


def recurrence(q, k, v, g, beta, state, reset, scale=None):
    """The definition, token by token, on (N, T, ...) float64 tensors; differentiable."""
    n, t, h, V = v.shape
    K, group = q.shape[-1], h // q.shape[2]
    scale = K**-0.5 if scale is None else scale
    q, k = q.repeat_interleave(group, 2), k.repeat_interleave(group, 2)
    S = q.new_zeros(n, h, K, V) if state is None else state
    out = []
    for i in range(t):
        decay = torch.exp(g[:, i])
        fresh = torch.exp(g[:, i].float()) == 0
        if reset is not None:
            fresh = fresh | reset[:, i, None].bool()
        S = torch.where(fresh[..., None, None], torch.zeros_like(S), S * decay[..., None, None])
        u = beta[:, i, :, None] * (v[:, i] - torch.einsum("nhkv,nhk->nhv", S, k[:, i]))
        S = S + k[:, i, :, :, None] * u[:, :, None, :]
        out.append(scale * torch.einsum("nhkv,nhk->nhv", S, q[:, i]))
    return (torch.stack(out, 1) if out else v.new_zeros(n, 0, h, V)), S


def rollout(n, t, h, hk, K, V, dtype, seed=0, resets=True, state=True, alike=0.7, decay=0.2):
    r = np.random.default_rng(seed)

    def tokens(*shape):
        return torch.from_numpy(r.standard_normal((n, t) + shape) + alike * r.standard_normal((n, 1) + shape))

    def unit(x):
        return x / x.norm(dim=-1, keepdim=True)

    a = {"q": unit(tokens(hk, K)), "k": unit(tokens(hk, K)), "v": tokens(h, V), "g": -decay * torch.exp(tokens(h) - 1),
         "beta": torch.sigmoid(tokens(h))}
    a = {x: y.to(dtype).cuda() for x, y in a.items()}
    a["state"] = torch.from_numpy(0.3 * r.standard_normal((n, h, K, V))).float().cuda() if state else None
    a["reset"] = torch.from_numpy(r.random((n, t)) < 0.08).cuda() if resets else None
    return a


def wide(a):
    return {x: None if y is None else y.detach().cpu() if y.dtype == torch.bool else y.detach().double().cpu()
            for x, y in a.items()}


def off(got, want):
    got, want = got.detach().double().cpu(), want.detach()
    if not want.numel():
        return 0.0 if got.shape == want.shape else math.inf
    assert got.shape == want.shape
    assert torch.isfinite(got).all()
    return float((got - want).norm() / want.norm().clamp_min(1e-30))


# (worlds, steps, heads, key heads, K, V): one token, part of a chunk, whole chunks, one more; odd and largest channels
SIZES = [(1, 1, 1, 1, 1, 1), (2, 1, 2, 1, 3, 5), (3, 2, 2, 2, 16, 16), (2, 15, 2, 2, 32, 32), (3, 16, 3, 1, 64, 64),
         (2, 17, 4, 2, 64, 32), (1, 31, 1, 1, 32, 64), (5, 33, 6, 3, 40, 71), (2, 64, 2, 1, 128, 128),
         (1, 65, 2, 2, 100, 128), (2, 130, 1, 1, 8, 128), (1, 129, 2, 1, 128, 8), (1, 600, 1, 1, 48, 24),
         (40, 20, 4, 4, 64, 64),
         # as many (worlds, heads) as fill the GPU
         (300, 17, 1, 1, 20, 10), (110, 50, 3, 3, 32, 64), (80, 70, 4, 2, 64, 64), (301, 35, 1, 1, 100, 65),
         (150, 33, 2, 1, 128, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_rollout(size, dtype):
    a = rollout(*size, dtype, seed=size[1])
    out, last = goib2d.delta_rule(**a)
    want, state = recurrence(**wide(a))
    assert out.dtype == dtype and last.dtype == F32
    assert off(out, want) <= TOL[dtype]
    assert off(last, state) <= TOL[F32]


GRADS = ("q", "k", "v", "g", "beta", "state")


def backward(a, dout, dlast, fn=goib2d.delta_rule):
    leaves = [a[x].detach().requires_grad_() for x in GRADS if a[x] is not None]
    named = dict(zip([x for x in GRADS if a[x] is not None], leaves))
    out, last = fn(**{**a, **named})
    outs = [(out, dout)] if dlast is None else [(out, dout), (last, dlast)]
    got = torch.autograd.grad([x for x, _ in outs], leaves, [y for _, y in outs], allow_unused=True)
    return out, last, dict(zip(named, got))


@pytest.mark.gpu
@pytest.mark.parametrize("last", [False, True], ids=["out", "out+state"])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_gradients(size, dtype, last):
    n, t, h, hk, K, V = size
    a = rollout(*size, dtype, seed=7 + t, state=last)
    r = np.random.default_rng(t)
    dout = torch.from_numpy(r.standard_normal((n, t, h, V))).to(dtype).cuda()
    dlast = torch.from_numpy(r.standard_normal((n, h, K, V))).float().cuda() if last else None
    out, state, got = backward(a, dout, dlast)
    w = wide(a)
    want_out, want_state, want = backward(w, dout.double().cpu(), None if dlast is None else dlast.double().cpu(),
                                          recurrence)
    assert off(out, want_out) <= TOL[dtype]
    assert off(state, want_state) <= TOL[F32]
    for name, x in got.items():
        y = want[name] if want[name] is not None else torch.zeros_like(w[name])
        if name == "g" and float(y.abs().max()) == 0:
            assert not x.any()
            continue
        assert x.dtype == (F32 if name == "state" else dtype)
        # the gradient chain runs through the products of the forward and of the backward pass: twice as many
        assert off(x, y) <= 2 * TOL[x.dtype], name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("n,h,hk,K,V", [(1, 1, 1, 1, 1), (3, 2, 1, 3, 5), (7, 4, 2, 16, 16), (33, 2, 2, 32, 32),
                                        (257, 3, 1, 64, 64), (5, 6, 2, 40, 71), (4, 2, 2, 128, 128), (9, 1, 1, 128, 4),
                                        (9, 1, 1, 5, 128), (3, 1, 1, 127, 127), (0, 2, 1, 8, 8), (2100, 1, 1, 64, 64)])
def test_step(n, h, hk, K, V, dtype):
    a = rollout(max(n, 1), 3, h, hk, K, V, dtype, seed=n)
    a = {x: y[:n] for x, y in a.items()}
    state = a["state"].clone()
    want, last = recurrence(**wide(a))
    for t in range(3):
        out = goib2d.delta_step_(state, *(a[x][:, t] for x in ("q", "k", "v", "g", "beta")), reset=a["reset"][:, t])
        assert off(out, want[:, t]) <= TOL[dtype]
    assert off(state, last) <= TOL[F32]


STEP_LAYOUT = r"""
#include <cstdio>
#include <initializer_list>
#include "delta_step.h"
int main() {
    for (int K = 1; K <= 128; ++K)
        for (int V = 1; V <= 128; ++V)
            for (int rows : {16, 8}) {  // rows in fours, others
                const gb::StepShape b(K, V, rows);
                const gb::StepShared at(K, 4 * b.x, b.y, b.z);
                std::printf("%d %d %d %d %d %d %d %d %d %d\n", K, V, rows, b.x, b.y, b.z, at.sums, at.pairs, at.dots, at.end);
            }
}
"""


def test_step_layout(tmp_path):
    """The one-token kernel's shared memory for all 1..128 x 1..128: the row groups' sums, which it reads and writes 16
    bytes at a time, and the pairs of k and q start at whole pieces, and no two parts overlap."""
    (tmp_path / "layout.cpp").write_text(STEP_LAYOUT)
    csrc = Path(native.__file__).resolve().parent.parent / "csrc"
    subprocess.run(["g++", "-std=c++17", "-I", str(csrc), "layout.cpp", "-o", "layout"], cwd=tmp_path, check=True)
    lines = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.splitlines()
    assert len(lines) == 2 * 128 * 128
    for line in lines:
        K, V, rows, x, y, z, sums, pairs, dots, end = map(int, line.split())
        assert 4 * x >= V and rows * y >= K and 1 <= z <= 64 and x * y * z <= 512, line
        assert sums % 4 == 0 and pairs % 2 == 0, f"misaligned: K {K}, V {V}, {z} heads a block"
        parts = sorted([(sums, z * y * 2 * 4 * x), (pairs, 2 * z * K), (dots, z * y), (end, 0)])
        assert all(at + size <= then for (at, size), (then, _) in zip(parts, parts[1:])), line
        assert parts[-1] == (end, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
# odd key channels and value channels in fours, with odd numbers of heads to a block; the last block is in part empty
@pytest.mark.parametrize("n,h,hk,K,V", [(5, 3, 1, 17, 12), (11, 1, 1, 33, 32), (3, 1, 1, 65, 64), (2, 2, 1, 33, 128),
                                        (3, 1, 1, 127, 128), (7, 4, 2, 9, 100), (7, 1, 1, 1, 100), (27, 2, 2, 3, 20),
                                        (2, 1, 1, 81, 16), (4, 1, 1, 65, 32)])
def test_step_odd_keys(n, h, hk, K, V, dtype):
    test_step(n, h, hk, K, V, dtype)


def test_step_reads_no_state_by_the_read_only_path():
    """The kernels' state is read and written by one launch, which the read-only path's loads do not allow."""
    source = (Path(native.__file__).resolve().parent.parent / "csrc" / "delta_step.cu").read_text()
    assert "__ldg" not in source and "ld.global.nc" not in source and "__restrict__" not in source


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("n,h,hk,K,V", [(300, 4, 2, 64, 64), (37, 3, 3, 33, 128), (41, 2, 1, 40, 71), (9, 1, 1, 7, 3)])
def test_step_in_place_equals_apart(n, h, hk, K, V, dtype):
    """The C call on one buffer for the old and the new state, and on two: the same bits."""
    a = rollout(n, 1, h, hk, K, V, dtype, seed=n)
    one = {x: a[x][:, 0].contiguous() for x in ("q", "k", "v", "g", "beta")}
    state, new, out = a["state"].clone(), torch.empty_like(a["state"]), torch.empty_like(one["v"])
    desc = policy._DESC.pack(n, 1, h, hk, K, V, policy._DTYPE[dtype], K ** -0.5, *(x.data_ptr() for x in one.values()), 0,
                             state.data_ptr(), new.data_ptr(), out.data_ptr(), *[hk * K, 0, K] * 2, h * V, 0, V,
                             *[h, 0, 1] * 2, h * V, 0, V, 0, 0)
    native.check(native.load().goib2d_delta_step(desc, torch.cuda.current_stream().cuda_stream))
    assert torch.equal(state, a["state"])
    assert torch.equal(goib2d.delta_step_(state, **one), out) and torch.equal(state, new)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
def test_rollout_in_pieces_equals_whole(dtype):
    a = rollout(3, 77, 4, 2, 64, 48, dtype, seed=5)
    whole, last = goib2d.delta_rule(**a)
    state, outs = a["state"], []
    for lo, hi in ((0, 1), (1, 20), (20, 20), (20, 52), (52, 77)):
        part = {x: y[:, lo:hi] for x, y in a.items() if x != "state"}
        o, state = goib2d.delta_rule(**part, state=state)
        outs.append(o)
    assert off(torch.cat(outs, 1), whole.double().cpu()) <= 2 * TOL[dtype]
    assert off(state, last.double().cpu()) <= 2 * TOL[F32]
    assert torch.equal(goib2d.delta_rule(**a)[0], whole)  # the same inputs, the same bits


def strided(x, kind):
    """x with other strides: steps first in memory, channels out of a wider row (off the 16-byte boundary), or heads
    first."""
    if kind == "time major":
        return x.transpose(0, 1).contiguous().transpose(0, 1)
    if kind == "wide rows":
        y = x.new_full((*x.shape[:-1], x.shape[-1] + 3), math.nan)
        y[..., 1:-2] = x
        return y[..., 1:-2]
    return x.movedim(2, 0).contiguous().movedim(0, 2)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["time major", "wide rows", "heads first"])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
def test_strides(kind, dtype):
    a = rollout(3, 37, 4, 2, 32, 64, dtype, seed=11)
    dout = torch.randn(3, 37, 4, 64, device="cuda").to(dtype)
    b = {x: strided(y, kind) if x in ("q", "k", "v", "g", "beta") else y for x, y in a.items()}
    b["reset"] = a["reset"].t().contiguous().t()
    out, last, grads = backward(a, dout, None)
    out2, last2, grads2 = backward(b, strided(dout, kind), None)
    tol = 2 * TOL[dtype]
    assert off(out2, out.double().cpu()) <= tol and off(last2, last.double().cpu()) <= 2 * TOL[F32]
    for x in grads:
        assert off(grads2[x], grads[x].double().cpu()) <= 2 * tol, x
    state, state2 = a["state"].clone(), a["state"].clone()
    names = ("q", "k", "v", "g", "beta")
    o = goib2d.delta_step_(state, *(a[x][:, 5] for x in names), reset=a["reset"][:, 5])
    o2 = goib2d.delta_step_(state2, *(b[x][:, 5] for x in names), reset=b["reset"][:, 5],
                            out=strided(torch.empty_like(a["v"]), kind)[:, 5])
    assert torch.equal(o, o2) and torch.equal(state, state2)


def windows(n, t, h, V, axis, dtype=F32, device="cpu"):
    """v as overlapping windows of a signal: neighbours along this axis (1: steps, 2: heads) are shifted by one channel."""
    step = {1: (t + V, 1, n * (t + V)), 2: (t * (h + V), h + V, 1)}[axis]
    x = torch.from_numpy(np.random.default_rng(axis).standard_normal(2 * n * (t + V) * (h + V))).to(device, dtype)
    return x.as_strided((n, t, h, V), (*step, 1))


@pytest.mark.parametrize("axis", [1, 2])
def test_outputs_of_overlapping_inputs_have_contiguous_channels(axis):
    """The kernels write o's channels as neighbours."""
    v = windows(3, 5, 4, 8, axis)
    for x in (v, v[:, 0], v.transpose(0, 1), v[0, 0, 0, 0:1], v.expand(3, 5, 4, 8)[:, :1].expand(3, 5, 4, 8), v[..., :1]):
        out = policy._like(x)
        assert out.shape == x.shape and out.dtype == x.dtype and out.stride(-1) == 1
        assert policy._dense(out)


@pytest.mark.gpu
@pytest.mark.parametrize("axis", [1, 2])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
def test_overlapping_inputs(axis, dtype):
    """Values that are sliding windows give what a copy of them gives, and one token of them is not refused."""
    a = rollout(3, 37, 4, 2, 16, 8, dtype, seed=12)
    names = ("q", "k", "v", "g", "beta")
    v = windows(3, 37, 4, 8, axis, dtype, "cuda")
    copied, slid = dict(a, v=v.contiguous()), dict(a, v=v)
    dout = torch.randn(3, 37, 4, 8, device="cuda").to(dtype)
    out, last, grads = backward(copied, dout, None)
    out2, last2, grads2 = backward(slid, dout, None)
    assert out2.stride(3) == 1
    assert off(out2, out.double().cpu()) <= 2 * TOL[dtype] and off(last2, last.double().cpu()) <= 2 * TOL[F32]
    for x in grads:
        assert off(grads2[x], grads[x].double().cpu()) <= 4 * TOL[dtype], x
    want, _ = recurrence(**wide(copied))
    assert off(goib2d.delta_rule(**slid)[0], want) <= TOL[dtype]
    state, state2 = a["state"].clone(), a["state"].clone()
    for t in range(3):
        o = goib2d.delta_step_(state, *(copied[x][:, t] for x in names), reset=a["reset"][:, t])
        o2 = goib2d.delta_step_(state2, *(slid[x][:, t] for x in names), reset=a["reset"][:, t])
        assert torch.equal(o, o2) and torch.equal(state, state2)


@pytest.mark.gpu
def test_broadcast_inputs_and_gradients():
    """One key for all worlds, one decay for all heads and steps: inputs of stride 0, their gradients summed."""
    a = rollout(4, 21, 2, 1, 16, 24, F32, seed=3, resets=False)
    key, decay = a["k"][:1, :, :, :].clone(), a["g"][:, :1, :1].clone()
    dout = torch.randn_like(a["v"])

    def of(fn, a, key, decay, dout):
        key, decay = key.requires_grad_(), decay.requires_grad_()
        out, _ = fn(a["q"], key.expand_as(a["k"]), a["v"], decay.expand_as(a["g"]), a["beta"], a["state"], None)
        return torch.autograd.grad([out], [key, decay], [dout])

    got = of(goib2d.delta_rule, a, key, decay, dout)
    want = of(recurrence, wide(a), key.detach().double().cpu(), decay.detach().double().cpu(), dout.double().cpu())
    assert off(got[0], want[0]) <= 2 * TOL[F32] and off(got[1], want[1]) <= 2 * TOL[F32]
    # a gradient of stride 0 comes in (from a sum)
    a["v"].requires_grad_()
    out, _ = goib2d.delta_rule(**a)
    out.sum().backward()
    w = wide(a)
    w["v"] = w["v"].detach().requires_grad_()
    recurrence(**w)[0].sum().backward()
    assert off(a["v"].grad, w["v"].grad) <= 2 * TOL[F32]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("n", [4, 160])  # few and many worlds
@pytest.mark.parametrize("K,V", [(16, 16), (64, 64), (40, 71), (128, 128)])
def test_states_that_start_afresh(K, V, n, dtype):
    """A reset, a decay of -inf, of the type's lowest value and of -200 all empty the memory, whatever it held:
    infinities and NaN in the old state are not read. Every token of world 0 is a reset (its own write is all that
    its query sees)."""
    t, h = 40, 2
    a = rollout(n, t, h, h, K, V, dtype, seed=1, resets=False)
    reset = torch.zeros(n, t, dtype=torch.bool, device="cuda")
    reset[0] = True
    reset[:, 0] = True
    reset[1, [15, 16, 17, 31, 39]] = True
    a["g"][2, 7] = -math.inf
    a["g"][2, 16] = torch.finfo(dtype).min
    a["g"][2, 32:34] = -200.0
    a["g"][3, 20, 0] = -math.inf  # one head only
    clean = dict(a, reset=reset)
    want, last = recurrence(**wide(dict(clean, g=a["g"].clamp_min(-1e3))))
    dirty = torch.full_like(a["state"], math.nan)
    dirty[:, :, :, ::2] = math.inf
    dout = torch.randn(n, t, h, V, device="cuda").to(dtype)
    for state in (a["state"], dirty):
        out, got_last, grads = backward(dict(clean, state=state), dout, None)
        assert off(out, want) <= TOL[dtype] and off(got_last, last) <= TOL[F32]
        assert not grads["state"].any()
        assert not grads["g"][reset].any() and not grads["g"][2, [7, 16, 32, 33]].any() and not grads["g"][3, 20, 0]
    w = wide(dict(clean, g=a["g"].clamp_min(-1e3)))
    _, _, want_grads = backward(w, dout.double().cpu(), None, recurrence)
    for x in ("q", "k", "v", "beta", "g"):
        assert off(grads[x], want_grads[x]) <= 2 * TOL[dtype], x
    step = dirty.clone()
    o = goib2d.delta_step_(step, *(a[x][:, 0] for x in ("q", "k", "v", "g", "beta")), reset=reset[:, 0])
    assert off(o, want[:, 0]) <= TOL[dtype]


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("n", [6, 300])  # few and many worlds
@pytest.mark.parametrize("V", [16, 40, 64])
def test_a_world_recovers_from_values_that_are_not_finite(V, n, dtype, bad):
    """A world whose simulation blew up sends NaN or infinities until it is reset: what comes after the reset, in the
    same chunk of tokens or later, is as if the memory had been empty, and other worlds do not notice."""
    t, h, K = 70, 2, 32
    a = rollout(n, t, h, 1, K, V, dtype, seed=13, resets=False)
    reset = torch.zeros(n, t, dtype=torch.bool, device="cuda")
    spoilt = torch.zeros(n, t, dtype=torch.bool, device="cuda")
    for world, (name, first, last) in enumerate((("v", 3, 5), ("k", 4, 8), ("q", 7, 8), ("k", 14, 15), ("v", 15, 33))):
        a[name][world, first:last + 1] = bad
        reset[world, [first - 2, last + 1, last + 4]] = True
        spoilt[world, first:last + 1] = True
    out, last = goib2d.delta_rule(**dict(a, reset=reset))
    state, steps = a["state"].clone(), []
    for i in range(t):
        steps.append(goib2d.delta_step_(state, *(a[x][:, i] for x in ("q", "k", "v", "g", "beta")), reset=reset[:, i]))
    clean = {x: torch.where(spoilt.view(n, t, *[1] * (y.dim() - 2)), 0, y) if x in ("q", "k", "v") else y
             for x, y in a.items()}
    want, want_last = recurrence(**wide(dict(clean, reset=reset)))
    for got, got_last in ((out, last), (torch.stack(steps, 1), state)):
        assert off(got[~spoilt], want[~spoilt.cpu()]) <= TOL[dtype]
        assert off(got_last, want_last) <= TOL[F32]
        assert not torch.isfinite(got[spoilt]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
# few and many worlds; bfloat16 in full products (at most 4096 tokens) and not; all heads, or one of the key head's two
@pytest.mark.parametrize("n,h,hk,K,V,heads", [(12, 2, 1, 32, 40, 2), (12, 1, 1, 128, 71, 1), (80, 2, 1, 64, 64, 1),
                                              (40, 2, 2, 128, 128, 2), (150, 1, 1, 20, 16, 1)])
def test_gradients_of_a_world_that_recovers(n, h, hk, K, V, heads, dtype, bad):
    """What is not finite in one episode does not reach the gradients of the episodes before it and after it, in the
    same chunk of tokens or elsewhere, nor other worlds and heads."""
    t = 150
    a = rollout(n, t, h, hk, K, V, dtype, seed=21, resets=False)
    r = np.random.default_rng(5)
    dout = torch.from_numpy(r.standard_normal((n, t, h, V))).to(dtype).cuda()
    dlast = torch.from_numpy(r.standard_normal((n, h, K, V))).float().cuda()
    reset = torch.zeros(n, t, dtype=torch.bool, device="cuda")
    spoilt = torch.zeros(n, t, h, dtype=torch.bool, device="cuda")  # the episodes
    dirty, dirty_dout = {x: y.clone() if y is not None else y for x, y in a.items()}, dout.clone()
    places = [("v", 3, 5), ("k", 4, 8), ("q", 7, 8), ("k", 14, 15), ("v", 15, 73), ("g", 70, 70), ("beta", 63, 64),
              ("dout", 40, 41), ("q", 100, 149), ("k", 2, 2), ("g", 130, 149)]
    for world, (name, first, last) in enumerate(places):
        x = dirty_dout if name == "dout" else dirty[name]
        x[world, first:last + 1, :heads if name not in ("q", "k") else None] = bad
        hit = slice(None) if name in ("q", "k") else slice(heads)
        reset[world, first - 2] = True
        spoilt[world, first - 2:last + 1, hit] = True
        for i in (last + 1, last + 4):
            if i < t:
                reset[world, i] = True
    dirty["reset"] = a["reset"] = reset
    _, _, got = backward(dirty, dirty_dout, dlast)
    _, _, want = backward(wide(a), dout.double().cpu(), dlast.double().cpu(), recurrence)
    key_spoilt = spoilt.view(n, t, hk, h // hk).any(-1)
    for x in ("q", "k", "v", "g", "beta"):
        clean = ~(key_spoilt if x in ("q", "k") else spoilt)
        assert off(got[x][clean], want[x][clean.cpu()]) <= 2 * TOL[dtype], x
        assert not got[x][~clean].float().isfinite().all(), x
    first_clean = ~spoilt[:, 0]
    assert off(got["state"][first_clean], want["state"][first_clean.cpu()]) <= 2 * TOL[F32]


@pytest.mark.gpu
@pytest.mark.parametrize("g", [0.0, -1e-6, -30.0, -90.0, 0.05])
def test_decays_from_none_to_all(g):
    """No decay at all, a chunk whose decays multiply to less than float32 holds, and growth."""
    a = rollout(2, 70, 2, 1, 32, 32, F32, seed=9, resets=False)
    a["g"] = torch.full_like(a["g"], g)
    a["g"][:, ::3] *= 0.5
    dout = torch.randn_like(a["v"])
    out, last, grads = backward(a, dout, None)
    want_out, want_last, want = backward(wide(a), dout.double().cpu(), None, recurrence)
    assert off(out, want_out) <= TOL[F32] and off(last, want_last) <= TOL[F32]
    for x in grads:
        if float(want[x].norm()) > 1e-30:
            assert off(grads[x], want[x]) <= 2 * TOL[F32], x


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
def test_same_key_every_step(dtype):
    """A world at rest: every token has the same key and beta is 1 (or 0: nothing is written), so that the chunk's
    triangular system is as far from the identity as it gets."""
    a = rollout(2, 80, 2, 2, 64, 64, dtype, seed=2, resets=False)
    a["k"] = a["k"][:, :1].expand_as(a["k"])
    a["g"] = torch.zeros_like(a["g"])
    a["beta"] = torch.ones_like(a["beta"])
    a["beta"][:, ::7] = 0
    dout = torch.randn(2, 80, 2, 64, device="cuda").to(dtype)
    out, last, grads = backward(a, dout, None)
    want_out, want_last, want = backward(wide(a), dout.double().cpu(), None, recurrence)
    assert off(out, want_out) <= TOL[dtype] and off(last, want_last) <= TOL[F32]
    for x in grads:
        assert off(grads[x], want[x]) <= 2 * TOL[F32 if x == "state" else dtype], x


@pytest.mark.gpu
def test_gradients_against_differences():
    """The directional derivative of a smooth loss, by central differences of the definition in 64 bits (step 1e-5:
    an error of about 1e-10 of its own), against the gradients."""
    a = rollout(2, 41, 2, 1, 24, 40, F32, seed=4)
    dout, dlast = torch.randn_like(a["v"]), torch.randn_like(a["state"])
    _, _, grads = backward(a, dout, dlast)
    w, wd, wl = wide(a), dout.double().cpu(), dlast.double().cpu()
    for name in GRADS:
        way = torch.from_numpy(np.random.default_rng(8).standard_normal(tuple(w[name].shape)))

        def loss(e):
            o, s = recurrence(**{**w, name: w[name] + e * way})
            return float((o * wd).sum() + (s * wl).sum())

        slope = (loss(1e-5) - loss(-1e-5)) / 2e-5
        got = float((grads[name].double().cpu() * way).sum())
        size = float(grads[name].double().norm().cpu() * way.norm())
        assert abs(got - slope) <= 2 * TOL[F32] * size, name


# What the split operands carry, tighter than TOL. float32: an operand is hi, rounded to tf32's 11 bits, plus lo, at most 2^-11
# of it, of which the product reads 11 bits (2^-21 of the operand); with the two lo parts' product (2^-22) left out a
# product is 2.5 * 2^-21 off, a chain of four 10 * 2^-21, gradients twice as many: two bfloat16 parts (2^-17) would not do.
# bfloat16 gradients of many tokens: four rounded operands or kept rows and the result, each 2^-9 at most and 1.7e-3 of a
# norm, independent: sqrt(5) * 1.7e-3 < 2 * 2^-9.
@pytest.mark.gpu
@pytest.mark.parametrize("size", [(2, 17, 4, 2, 64, 32), (5, 33, 6, 3, 40, 71), (2, 64, 2, 1, 128, 128), (80, 70, 4, 2, 64, 64)],
                         ids=str)
def test_precision_float32(size):
    n, t, h, hk, K, V = size
    a = rollout(*size, F32, seed=61)
    dout = torch.randn(n, t, h, V, generator=torch.Generator("cuda").manual_seed(t), device="cuda")
    out, last, got = backward(a, dout, None)
    want_out, want_last, want = backward(wide(a), dout.double().cpu(), None, recurrence)
    assert off(out, want_out) <= 10 * 2.0**-21 and off(last, want_last) <= 10 * 2.0**-21
    for x in got:
        assert off(got[x], want[x]) <= 20 * 2.0**-21, x


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(80, 70, 4, 2, 64, 64), (110, 50, 3, 3, 32, 64), (301, 35, 1, 1, 100, 65), (150, 33, 2, 1, 128, 128)],
                         ids=str)
def test_precision_bfloat16_of_many_tokens(size):
    n, t, h, hk, K, V = size
    assert n * t * h > 4096
    a = rollout(*size, BF16, seed=62)
    dout = torch.randn(n, t, h, V, generator=torch.Generator("cuda").manual_seed(t), device="cuda").to(BF16)
    _, last, got = backward(a, dout, None)
    _, want_last, want = backward(wide(a), dout.double().cpu(), None, recurrence)
    assert off(last, want_last) <= 2.0**-16  # float32, of operands in two bfloat16 parts (2^-17)
    for x in ("q", "k", "v", "g", "beta"):
        assert off(got[x], want[x]) <= 2 * 2.0**-9, x


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("size", SIZES + [(4096, 2, 1, 1, 16, 16)], ids=str)
def test_outputs_do_not_depend_on_whether_gradients_are_wanted(size, dtype):
    """The same bits with and without, in calls of few tokens and of many."""
    a = rollout(*size, dtype, seed=size[1])
    out, last = goib2d.delta_rule(**a)
    trained, trained_last = goib2d.delta_rule(**dict(a, v=a["v"].clone().requires_grad_()))
    assert trained.requires_grad
    assert torch.equal(trained, out) and torch.equal(trained_last, last)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
def test_states_may_be_written_to_before_the_gradients(dtype):
    """The gradients need neither the first nor the last state: the world goes on acting with the last one's memory (zeroed
    where it was reset), and the first one's buffer takes the next rollout's, while the loss is still to be trained on."""
    a = rollout(5, 40, 2, 2, 32, 24, dtype, seed=31)
    dout = torch.randn(5, 40, 2, 24, device="cuda").to(dtype)
    _, _, want = backward(a, dout, None)
    first = a["state"].clone()
    leaves = {x: a[x].clone().requires_grad_() for x in GRADS if x != "state"}
    out, last = goib2d.delta_rule(**leaves, state=first, reset=a["reset"])
    memory = last.detach()
    memory[2] = 0
    first.copy_(memory)
    with torch.no_grad():
        goib2d.delta_step_(memory, *(leaves[x][:, 0] for x in ("q", "k", "v", "g", "beta")))
    got = torch.autograd.grad([out], list(leaves.values()), [dout])
    for x, y in zip(leaves, got):
        assert torch.equal(y, want[x]), x


@pytest.mark.gpu
def test_zero_steps_and_worlds():
    a = rollout(3, 4, 2, 1, 16, 16, F32)
    none = {x: y[:, :0] if x not in ("state",) else y for x, y in a.items()}
    out, last, grads = backward(none, torch.empty(3, 0, 2, 16, device="cuda"), torch.ones_like(a["state"]))
    assert out.shape == (3, 0, 2, 16) and torch.equal(last, a["state"])
    assert torch.equal(grads["state"], torch.ones_like(a["state"]))
    out, last = goib2d.delta_rule(**dict(none, state=None))
    assert not last.any()
    out, last = goib2d.delta_rule(**{x: y[:0] for x, y in a.items()})
    assert out.shape == (0, 4, 2, 16) and last.shape == (0, 2, 16, 16)
    # only the last state has a gradient
    state = a["state"].clone().requires_grad_()
    _, last = goib2d.delta_rule(**dict(a, state=state))
    got, = torch.autograd.grad([last], [state], [torch.ones_like(last)])
    w = wide(a)
    w["state"] = w["state"].detach().requires_grad_()
    want, = torch.autograd.grad([recurrence(**w)[1].sum()], [w["state"]])
    assert off(got, want) <= 2 * TOL[F32] if want.any() else not got.any()


@pytest.mark.gpu
def test_streams_and_graphs():
    """Calls follow the current stream: inputs made on a side stream are read there; a captured step replays."""
    a = rollout(64, 9, 2, 2, 32, 32, BF16, seed=6)
    want = goib2d.delta_rule(**a)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        b = {x: None if y is None else y.clone() for x, y in a.items()}
        got = goib2d.delta_rule(**b)
        grads = [torch.randn(100_000, device="cuda") for _ in range(3)]
        whole = torch.cat(grads).double().norm()
        norm = goib2d.clip_grads_(grads, 1.0)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert abs(float(norm) - float(whole)) <= 2e-7 * float(whole)
    names = ("q", "k", "v", "g", "beta")
    state, now = a["state"].clone(), {x: a[x][:, 0].clone() for x in names}
    out = torch.empty(64, 2, 32, dtype=BF16, device="cuda")
    with torch.cuda.stream(side):
        goib2d.delta_step_(state, **now, out=out)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    state.copy_(a["state"])
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        goib2d.delta_step_(state, **now, out=out)
    state.copy_(a["state"])
    for t in range(3):
        for x in names:
            now[x].copy_(a[x][:, t])
        graph.replay()
    plain = a["state"].clone()
    for t in range(3):
        last = goib2d.delta_step_(plain, *(a[x][:, t] for x in names))
    assert torch.equal(state, plain) and torch.equal(out, last)


@pytest.mark.gpu
def test_writes_of_a_step_are_seen_by_autograd():
    """A graph that saved the memory, or a buffer given as `out`, before a step wrote to it raises, as after torch's own
    writes, instead of giving gradients of the new contents. Tensors of inference mode have no versions."""
    a = rollout(3, 1, 2, 1, 16, 24, F32, seed=41)
    token = [a[x][:, 0] for x in ("q", "k", "v", "g", "beta")]
    weight = torch.ones(24, device="cuda", requires_grad=True)
    out = torch.zeros(3, 2, 24, device="cuda")
    for kept in ("state", "out"):
        state = a["state"].clone()
        loss = ((state if kept == "state" else out) * weight).sum()
        goib2d.delta_step_(state, *token, out=out if kept == "out" else None)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with pytest.raises(ValueError, match="differentiable"):
        goib2d.delta_step_(state, *token, out=torch.zeros(3, 2, 24, device="cuda", requires_grad=True))
    with torch.inference_mode():
        memory = a["state"].clone()
        o = goib2d.delta_step_(memory, *token, out=torch.empty(3, 2, 24, device="cuda"))
    state = a["state"].clone()
    assert torch.equal(goib2d.delta_step_(state, *token), o) and torch.equal(memory, state)


# ---- clipping


def clip_want(grads, max_norm):
    w = [x.detach().double().cpu() for x in grads]
    norm = math.sqrt(sum(float((x * x).sum()) for x in w))
    return norm, [x * min(1.0, max_norm / (norm + 1e-6)) for x in w]


@pytest.mark.gpu
@pytest.mark.parametrize("max_norm", [0.0, 0.5, 1e9])
@pytest.mark.parametrize("sizes", [[1], [3, 0, 5], [4096, 4097, 1, 8191], [100_003, 7, 1_000_001], [2_500_000, 13],
                                   [3] * 2100], ids=lambda s: f"{len(s)}x{max(s)}")
def test_clip(sizes, max_norm):
    r = torch.Generator(device="cuda").manual_seed(len(sizes))
    grads = [torch.randn(s, generator=r, device="cuda").to(BF16 if i % 3 == 1 else F32) for i, s in enumerate(sizes)]
    norm_want, want = clip_want(grads, max_norm)
    before = [x.clone() for x in grads]
    norm = goib2d.clip_grads_([None] + grads, max_norm)
    # the sum is in 64 bits: the norm and the factor are rounded to float32 (2^-24 each, a few times), elements once
    assert abs(float(norm) - norm_want) <= 4 * 2.0**-24 * norm_want
    for x, y, b in zip(grads, want, before):
        if max_norm > norm_want:
            assert torch.equal(x, b)
        else:
            err = (x.double().cpu() - y).abs() - y.abs() * (2.0**-8 if x.dtype == BF16 else 8 * 2.0**-24)
            assert not x.numel() or float(err.max()) <= 0


def clip_check(grads, max_norm):
    """clip_grads_ against the formula in 64 bits, every element, with test_clip's bounds."""
    wide_grads, before = [x.double() for x in grads], [x.clone() for x in grads]
    norm_want = math.sqrt(sum(float((x * x).sum()) for x in wide_grads))
    factor = min(1.0, max_norm / (norm_want + 1e-6))
    norm = goib2d.clip_grads_(grads, max_norm)
    assert abs(float(norm) - norm_want) <= 4 * 2.0**-24 * norm_want
    for x, w, b in zip(grads, wide_grads, before):
        if factor == 1.0:
            assert torch.equal(x, b)
        else:
            err = (x.double() - w * factor).abs() - (w * factor).abs() * (2.0**-8 if x.dtype == BF16 else 8 * 2.0**-24)
            assert float(err.max()) <= 0


@pytest.mark.gpu
@pytest.mark.parametrize("max_norm", [0.5, 1e9])
@pytest.mark.parametrize("megabytes", [20, 29, 31, 45, 62])
def test_clip_beyond_what_the_blocks_keep(megabytes, max_norm):
    """The blocks keep 148 x 12 tiles of 16 KB (29 MB) between the norm and the scaling and read the rest again: less than
    that, as much, and more, in mixed types, with tensors that begin and end within a block's tiles, one of them off
    the 16-byte boundary. A block's tiles are 8 to 26, whole batches of four and not."""
    gen = torch.Generator(device="cuda").manual_seed(megabytes)
    share = megabytes * 1_000_000 // 10  # of bytes
    sizes = [(3 * share // 4 + 1, F32, 0), (4099, BF16, 1), (2 * share // 2, BF16, 1), (5, F32, 0), (share // 4, F32, 3),
             (3 * share // 2 + 3, BF16, 0), (share // 4 - 7, F32, 0)]
    grads = [torch.randn(n + at, generator=gen, device="cuda").to(dtype)[at:] for n, dtype, at in sizes]
    clip_check(grads, max_norm)


@pytest.mark.gpu
@pytest.mark.parametrize("max_norm", [0.5, 1e9])
@pytest.mark.parametrize("count", [63, 64, 65, 700, 1023, 1024, 1025, 2048, 2049])
def test_clip_numbers_of_tensors(count, max_norm):
    """The table in the launch holds 64 or 1024 tensors: as many, one more, one fewer; more take several launches."""
    gen = torch.Generator(device="cuda").manual_seed(count)
    clip_check([torch.randn(1 + 997 * i % 9001, generator=gen, device="cuda").to(BF16 if i % 3 == 0 else F32)
                for i in range(count)], max_norm)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
def test_training_in_a_graph(dtype):
    """Rollouts, their gradients and the clipping, captured and replayed on other inputs: what the calls give by themselves."""
    a, b = (rollout(70, 33, 2, 1, 32, 24, dtype, seed=s) for s in (51, 52))
    dout = torch.randn(70, 33, 2, 24, device="cuda").to(dtype)

    def update(a):
        leaves = {x: a[x].detach().requires_grad_() for x in GRADS}
        out, last = goib2d.delta_rule(**leaves, reset=a["reset"])
        grads = torch.autograd.grad([out], list(leaves.values()), [dout])
        return [out.detach(), last.detach(), goib2d.clip_grads_(grads, 0.5), *grads]

    want = [x.clone() for x in update(b)]
    now = {x: y.clone() for x, y in a.items()}
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        update(now)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = update(now)
    for x in now:
        now[x].copy_(b[x])
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.gpu
def test_clip_same_bits_and_alignment():
    base = torch.randn(3_000_001, device="cuda")
    cut = [1, 2, 500_000, 500_003, 1_700_001, 3_000_000]
    norms = []
    for _ in range(3):
        x = base.clone()
        norms.append(float(goib2d.clip_grads_([x[a:b] for a, b in zip(cut, cut[1:])], 1.0)))
        assert torch.equal(x[:1], base[:1]) and torch.equal(x[-1:], base[-1:])
        assert abs(float(x[1:-1].double().norm()) - 1) < 1e-5
    assert len(set(norms)) == 1
    m = torch.randn(130, 70, device="cuda").t()  # dense, in another order
    want = m / (m.norm() + 1e-6) * 0.1
    goib2d.clip_grads_([m], 0.1)
    assert torch.allclose(m, want, rtol=1e-5, atol=0)


@pytest.mark.gpu
def test_clip_values_that_are_not_finite_or_extreme():
    big = [torch.full((10,), 1e30, device="cuda"), torch.full((10,), 1e-30, device="cuda")]
    norm = goib2d.clip_grads_(big, 1.0)  # squares beyond float32
    assert abs(float(norm) / (1e30 * math.sqrt(10)) - 1) < 1e-6 and abs(float(big[0][0]) * math.sqrt(10) - 1) < 1e-6
    x, y = torch.tensor([1.0, math.inf], device="cuda"), torch.ones(5000, device="cuda")
    assert float(goib2d.clip_grads_([x, y], 1.0)) == math.inf
    assert float(x[0]) == 0 and math.isnan(float(x[1])) and not y.any()
    x, y = torch.tensor([1.0, math.nan], device="cuda"), torch.ones(5000, device="cuda")
    assert math.isnan(float(goib2d.clip_grads_([x, y], 1.0)))
    assert torch.isnan(y).all()
    z = torch.zeros(10, device="cuda")
    assert float(goib2d.clip_grads_([z], 1.0)) == 0 and not z.any()
    assert float(goib2d.clip_grads_([torch.empty(0, device="cuda")], 1.0)) == 0


@pytest.mark.gpu
def test_writes_of_clipping_are_seen_by_autograd():
    grads = [torch.ones(5, device="cuda"), torch.ones(70, device="cuda", dtype=BF16), torch.ones(0, device="cuda")]
    weights = [x.clone().float().requires_grad_() for x in grads[:2]]
    losses = [(x.float() if x.dtype == BF16 else x).mul(w).sum() for x, w in zip(grads, weights)]
    square = (grads[1] * torch.ones_like(grads[1], requires_grad=True)).sum()
    with torch.no_grad():
        goib2d.clip_grads_(grads, 0.5)
    for loss in (losses[0], square):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    losses[1].backward()  # saved a copy
    assert torch.equal(weights[1].grad, torch.ones(70, device="cuda"))
    with torch.inference_mode():
        x = torch.ones(4, device="cuda")
        assert float(goib2d.clip_grads_([x], 1.0)) == 2.0 and abs(float(x[0]) - 0.5) < 1e-6


# ---- what is refused


@pytest.mark.gpu
def test_refusals():
    a = rollout(2, 5, 4, 2, 16, 16, F32)
    names = ("q", "k", "v", "g", "beta")
    bad = {"k": a["k"][:, :4], "q": a["q"].to(BF16), "g": a["g"][..., :2], "beta": a["beta"].cpu(),
           "state": a["state"].to(BF16), "reset": a["reset"].float(), "v": a["v"].double()}
    for x, y in bad.items():
        with pytest.raises((ValueError, TypeError)):
            goib2d.delta_rule(**{**a, x: y})
    with pytest.raises(ValueError, match="contiguous"):
        goib2d.delta_rule(**{**a, "q": a["q"].transpose(-1, -2).contiguous().transpose(-1, -2)})
    with pytest.raises(ValueError, match="contiguous"):
        goib2d.delta_rule(**{**a, "state": a["state"].transpose(-1, -2)})
    with pytest.raises(ValueError, match="heads"):
        goib2d.delta_rule(**{**a, "q": a["q"].repeat(1, 1, 2, 1)[:, :, :3], "k": a["k"].repeat(1, 1, 2, 1)[:, :, :3]})
    wide_v = torch.zeros(2, 5, 4, 129, device="cuda")
    with pytest.raises(ValueError, match="128"):
        goib2d.delta_rule(**{**a, "v": wide_v, "state": None})
    one = {x: a[x][:, 0] for x in names}
    with pytest.raises(ValueError, match="differentiable"):
        goib2d.delta_step_(a["state"], **{**one, "q": one["q"].clone().requires_grad_()})
    with pytest.raises(ValueError, match="state"):
        goib2d.delta_step_(a["state"][:1], **one)
    with pytest.raises(ValueError, match="out"):
        goib2d.delta_step_(a["state"], **one, out=torch.empty(2, 4, 16, dtype=BF16, device="cuda"))
    x = torch.ones(4, device="cuda")
    for grads, most in (([x.double()], 1.0), ([x], -1.0), ([x], math.nan), ([], 1.0), ([x, x], 1.0), ([x[::2]], 1.0),
                        ([x, torch.ones(2)], 1.0), ([x.to_sparse()], 1.0)):
        with pytest.raises((ValueError, TypeError)):
            goib2d.clip_grads_(grads, most)
    assert torch.equal(x, torch.ones_like(x))


@pytest.mark.gpu
def test_forward_mode_tangents_are_refused():
    """No derivative in forward mode: tangents raise instead of being dropped; without any, the level changes nothing."""
    from torch.autograd import forward_ad
    a = rollout(2, 5, 2, 1, 16, 16, F32)
    want = goib2d.delta_rule(**a)[0]
    names = ("q", "k", "v", "g", "beta")
    for x in names + ("state",):
        for grad in (False, True):
            with forward_ad.dual_level():
                b = dict(a, **{x: forward_ad.make_dual(a[x].clone().requires_grad_(grad), torch.ones_like(a[x]))})
                with pytest.raises((ValueError, NotImplementedError)):
                    goib2d.delta_rule(**b)
                if not grad:
                    with pytest.raises(ValueError, match="forward-mode"):
                        goib2d.delta_step_(b["state"], *(b[y][:, 0] for y in names))
    with forward_ad.dual_level():
        grad = forward_ad.make_dual(torch.ones(3, device="cuda"), torch.ones(3, device="cuda"))
        with pytest.raises(ValueError, match="forward-mode"):
            goib2d.clip_grads_([torch.ones(2, device="cuda"), grad], 1.0)
        assert torch.equal(goib2d.delta_rule(**a)[0], want)
        state = a["state"].clone()
        goib2d.delta_step_(state, *(a[y][:, 0] for y in names))
        assert float(goib2d.clip_grads_([torch.ones(4, device="cuda")], 1.0)) == 2.0
    with pytest.raises(ValueError, match="forward-mode"):
        torch.func.jvp(lambda v: goib2d.delta_rule(**dict(a, v=v))[0], (a["v"],), (torch.ones_like(a["v"]),))


def test_cpu_tensors_are_refused():
    a = {x: torch.zeros(s) for x, s in (("q", (2, 3, 1, 8)), ("k", (2, 3, 1, 8)), ("v", (2, 3, 1, 8)), ("g", (2, 3, 1)),
                                         ("beta", (2, 3, 1)))}
    with pytest.raises(TypeError, match="CUDA"):
        goib2d.delta_rule(**a)
    with pytest.raises(TypeError, match="CUDA"):
        goib2d.delta_step_(torch.zeros(2, 1, 8, 8), *(x[:, 0] for x in a.values()))
    with pytest.raises(TypeError, match="CUDA"):
        goib2d.clip_grads_([torch.ones(3)], 1.0)


def desc(**kw):
    f = dict(n=1, t=1, h=2, hk=1, K=8, V=8, dtype=0, scale=1.0, q=16, k=16, v=16, g=16, beta=16, reset=0, s_in=16, s_out=16,
             out=16)
    f.update(kw)
    return policy._DESC.pack(*f.values(), *[0] * 20)


def test_c_entries_refuse_bad_arguments():
    """The C calls check sizes and pointers before any launch (so these need no GPU)."""
    lib = native.load()
    einval, elimit = -1, -4
    for call in (lambda d: lib.goib2d_delta_step(d, None), lambda d: lib.goib2d_delta_forward(d, None, None),
                 lambda d: lib.goib2d_delta_saved_bytes(d), lambda d: lib.goib2d_delta_workspace_bytes(d),
                 lambda d: lib.goib2d_delta_backward(d, policy._GRADS.pack(*[16] * 8, *[0] * 18), 16, 16, None)):
        assert call(None) == einval
        assert call(desc(n=-1)) == einval and call(desc(t=-1)) == einval and call(desc(dtype=2)) == einval
        assert call(desc(hk=0)) == einval and call(desc(h=3, hk=2)) == einval and call(desc(K=0)) == einval
        assert call(desc(K=129)) == elimit and call(desc(V=129)) == elimit
        assert call(desc(n=1 << 31)) == elimit and call(desc(n=1 << 20, t=1 << 50)) == elimit
        assert call(desc(v=18)) == einval and call(desc(k=17, dtype=1)) == einval and call(desc(s_out=18)) == einval
        assert call(desc(q=0)) == einval and call(desc(beta=0)) == einval and call(desc(s_out=0)) == einval
        assert call(desc(n=0, q=0, s_out=0)) >= 0
    assert lib.goib2d_delta_step(desc(t=2), None) == einval and lib.goib2d_delta_step(desc(s_in=0), None) == einval
    assert lib.goib2d_delta_step(desc(out=0), None) == einval and lib.goib2d_delta_forward(desc(out=0), None, None) == einval
    assert lib.goib2d_delta_forward(desc(), 8, None) == einval
    grads = policy._GRADS.pack(*[16] * 8, *[0] * 18)
    assert lib.goib2d_delta_backward(desc(), None, 16, 16, None) == einval
    assert lib.goib2d_delta_backward(desc(), grads, None, 16, None) == einval
    assert lib.goib2d_delta_backward(desc(), grads, 16, None, None) == einval
    assert lib.goib2d_delta_backward(desc(), policy._GRADS.pack(16, 0, 0, *[16] * 5, *[0] * 18), 16, 16, None) == einval
    assert b"null" in lib.goib2d_last_error()
    one = policy._GRAD.pack
    assert lib.goib2d_clip_grads(None, 1, 1.0, None, 16, None) == einval
    assert lib.goib2d_clip_grads(one(16, 4, 0), -1, 1.0, None, 16, None) == einval
    assert lib.goib2d_clip_grads(one(16, 4, 0), 1, -1.0, None, 16, None) == einval
    assert lib.goib2d_clip_grads(one(16, 4, 0), 1, math.nan, None, 16, None) == einval
    assert lib.goib2d_clip_grads(one(16, 4, 0), 1, 1.0, None, None, None) == einval
    assert lib.goib2d_clip_grads(one(0, 4, 0), 1, 1.0, None, 16, None) == einval
    assert lib.goib2d_clip_grads(one(18, 4, 0), 1, 1.0, None, 16, None) == einval
    assert lib.goib2d_clip_grads(one(16, -4, 0), 1, 1.0, None, 16, None) == einval
    assert lib.goib2d_clip_grads(one(16, 4, 7), 1, 1.0, None, 16, None) == einval
    assert lib.goib2d_clip_workspace_bytes(None, 2) == einval


def test_clipping_refuses_tensors_that_overlap():
    """Before any launch (so this needs no GPU), in any order, with empty tensors between, few and many."""
    lib, one = native.load(), policy._GRAD.pack

    def call(*tensors):
        return lib.goib2d_clip_grads(b"".join(one(*t) for t in tensors), len(tensors), 1.0, None, 16, None)

    many = [(4096 + 64 * i, 16, 0) for i in range(100)]
    for bad in ([(4096, 100, 0), (4096, 100, 0)], [(4096, 100, 0), (4096 + 396, 1, 0)], [(4096 + 198, 5, 1), (4096, 100, 1)],
                [(8192, 10, 0), (4096, 0, 0), (4096, 1025, 0)], many + [(4096 + 64 * 50 + 60, 2, 0)], many[::-1] + [(4096, 1, 1)]):
        assert call(*bad) == -1 and b"overlap" in lib.goib2d_last_error()


@pytest.mark.gpu
def test_clipping_takes_neighbours():
    flat = torch.randn(10_000, device="cuda")
    want = flat.double() / (flat.double().norm() + 1e-6)
    views = [flat[7000:], flat[:1], flat[1:500], flat[500:500], flat[500:7000]]
    goib2d.clip_grads_(views, 1.0)
    assert off(flat, want.cpu()) <= 1e-6
    with pytest.raises(RuntimeError, match="overlap"):
        goib2d.clip_grads_([flat[:100], flat[99:200]], 1.0)
    assert off(flat, want.cpu()) <= 1e-6


def test_struct_layouts():
    """The packed structures are the header's (sizes as a C compiler lays them out)."""
    assert (policy._DESC.size, policy._GRADS.size, policy._GRAD.size) == (272, 208, 24)
    assert C.sizeof(C.c_void_p) == 8


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
def test_example_acts_and_trains(dtype):
    """examples/memory_policy.py: the rollout replayed for training gives the actions that the acting pass gave, and
    the update's clipped gradient moves the weights."""
    import sys
    from pathlib import Path
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
    import memory_policy
    torch.manual_seed(0)
    fresh = memory_policy.MemoryPolicy().cuda().to(dtype)
    policy, results = memory_policy.train(worlds=64, steps=24, updates=2, dtype=dtype, log=lambda line: None)
    for r in results:
        assert all(math.isfinite(x) for x in r.values())
        assert r["norm"] > 0
        # the linear layers run on other shapes in the two passes: their rounding differs too
        assert r["replayed"] <= 4 * TOL[dtype]
    assert all(torch.isfinite(p).all() for p in policy.parameters())
    assert any(not torch.equal(p, q) for p, q in zip(policy.parameters(), fresh.parameters()))


@pytest.mark.gpu
def test_example_carries_resets_from_rollout_to_rollout(monkeypatch):
    """A world that is reset after the last step of a rollout starts the next one with an empty memory."""
    import sys
    from pathlib import Path
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
    import memory_policy
    seen, forward = [], memory_policy.MemoryPolicy.forward

    def recorded(self, x, memory, reset):
        seen.append(reset.clone())
        return forward(self, x, memory, reset)

    monkeypatch.setattr(memory_policy.MemoryPolicy, "forward", recorded)
    monkeypatch.setattr(memory_policy, "FALLEN", 1e6)  # every world, after every step
    memory_policy.train(worlds=32, steps=3, updates=3, dtype=F32, log=lambda line: None)
    first, *others = seen
    assert not first[:, 0].any() and first[:, 1:].all()
    assert all(reset.all() for reset in others)
