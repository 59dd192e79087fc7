"""The policy-side operators as cases to measure: the gated delta rule (one token per world, whole rollouts, training)
and gradient clipping by the global norm.

Sizes: world counts and episode lengths of the benchmark scenes (256 box-drop worlds, 4096 rigs, 8192 bullet worlds,
65536 worlds of the scale sweep; rollouts of 16 to 8192 steps), memories of 1 to 8 heads of 8 to 128 channels."""
import math
import os
import sys

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def delta(op, worlds, steps, heads, key_heads, key_dim, value_dim, dtype, resets, time_major, init):
    return {"op": op, "worlds": worlds, "steps": steps, "heads": heads, "key_heads": key_heads, "key_dim": key_dim,
            "value_dim": value_dim, "dtype": dtype, "resets": resets, "time_major": time_major, "init": init}


def clip(inputs, hidden, layers, dtype, mixed):
    return {"op": "clip", "inputs": inputs, "hidden": hidden, "layers": layers, "dtype": dtype, "mixed": mixed}


def listed():
    cases = [
        # acting: the memory of every world advances by one token per world step
        ("step: 256 worlds, float32", delta("step", 256, 1, 2, 2, 32, 32, "float32", True, False, True)),
        ("step: 1023 worlds, odd sizes", delta("step", 1023, 1, 6, 2, 40, 71, "float32", True, False, True)),
        ("step: 4096 rigs, bfloat16", delta("step", 4096, 1, 4, 4, 64, 64, "bfloat16", False, False, True)),
        ("step: 65536 worlds", delta("step", 65536, 1, 1, 1, 64, 64, "bfloat16", True, False, True)),
        # replaying rollouts without gradients (values for advantages, warming a stored state up)
        ("rollout: 256 worlds, float32", delta("rollout", 256, 16, 2, 2, 32, 32, "float32", True, False, True)),
        ("rollout: 4096 rigs, bfloat16", delta("rollout", 4096, 64, 4, 4, 64, 64, "bfloat16", True, True, True)),
        ("rollout: 8 whole episodes", delta("rollout", 8, 8192, 4, 2, 128, 128, "bfloat16", True, False, False)),
        # training on them: outputs and all gradients
        ("train: 64 worlds, odd sizes", delta("train", 64, 77, 6, 2, 40, 71, "float32", True, True, True)),
        ("train: 1024 worlds, float32", delta("train", 1024, 128, 2, 2, 64, 64, "float32", True, False, True)),
        ("train: 4096 rigs, bfloat16", delta("train", 4096, 64, 4, 4, 64, 64, "bfloat16", True, True, False)),
        # the update's gradient clipping: a small policy, and one of 64 M weights with bfloat16 matrices
        ("clip: small policy", clip(28, 256, 3, "float32", False)),
        ("clip: large policy, mixed types", clip(117, 2047, 15, "bfloat16", True)),
    ]
    return [dict(c, name=name) for name, c in cases]


def log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    op = rng.choice(("step", "rollout", "train", "clip"))
    if op == "clip":
        dtype = rng.choice(("float32", "bfloat16"))
        return clip(rng.randint(6, 160), log_int(rng, 17, 2047), rng.randint(1, 15), dtype, rng.random() < 0.5)
    dtype = rng.choice(("float32", "bfloat16"))
    key_heads = rng.choice((1, 1, 2, 3, 4))
    heads = key_heads * rng.choice((1, 1, 2))
    if rng.random() < 0.5:
        key_dim, value_dim = rng.choice((16, 32, 64, 128)), rng.choice((16, 32, 64, 128))
    else:
        key_dim, value_dim = log_int(rng, 8, 128), log_int(rng, 8, 128)
    steps = 1 if op == "step" else log_int(rng, 2, 8192)
    # as many worlds as the largest listed case of the operator has room for
    room = 65536 * 4096 // (heads * key_dim * value_dim)
    if op != "step":
        tokens = (4096 * 64 * 4 if dtype == "bfloat16" else 1024 * 128 * 2) * 64 // max(key_dim, value_dim)
        room = min(room // 4, tokens // (heads * steps))
    worlds = log_int(rng, 1, max(1, min(65536, room)))
    return delta(op, worlds, steps, heads, key_heads, key_dim, value_dim, dtype, rng.random() < 0.7,
                 rng.random() < 0.5, op == "step" or rng.random() < 0.5)


def shapes(case):
    """The weights of a policy: an encoder of the observations, hidden layers with biases, a head of two actions."""
    h = case["hidden"]
    return [(h, case["inputs"]), (h,)] + [(h, h), (h,)] * case["layers"] + [(2, h), (2,)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if case["op"] == "clip":
        # gradients of uneven size over the layers, ten times the norm that they are clipped to; with `mixed` the
        # biases and the head stay in float32
        grads = [normal(*s) * (0.3 + i % 3) for i, s in enumerate(shapes(case))]
        types = [torch.float32 if case["mixed"] and (x.dim() == 1 or x.shape[0] == 2) else DTYPES[case["dtype"]]
                 for x in grads]
        grads = [x.to(t) for x, t in zip(grads, types)]
        total = sum(x.numel() * (0.3 + i % 3) ** 2 for i, x in enumerate(grads)) ** 0.5
        return {"case": case, "grads": grads, "max_norm": total / 10}
    n, t, h, hk = case["worlds"], case["steps"], case["heads"], case["key_heads"]
    dk, dv, dt = case["key_dim"], case["value_dim"], DTYPES[case["dtype"]]

    def tokens(*shape):
        """A (n, t, ...) tensor whose tokens resemble one another, as observations of one world do."""
        if case["op"] == "step":
            return normal(n, *shape)
        if case["time_major"]:  # as a rollout records them: step by step
            return (normal(t, n, *shape) + 0.7 * normal(1, n, *shape)).transpose(0, 1)
        return normal(n, t, *shape) + 0.7 * normal(n, 1, *shape)

    def unit(x):
        return (x / x.norm(dim=-1, keepdim=True)).to(dt)

    s = {"case": case, "q": unit(tokens(hk, dk)), "k": unit(tokens(hk, dk)), "v": tokens(h, dv).to(dt),
         "beta": torch.sigmoid(tokens(h)).to(dt), "g": (-0.2 * torch.exp(tokens(h) - 1.5)).to(dt),
         "reset": None, "state": None}
    if case["resets"]:
        s["reset"] = torch.rand(s["g"].shape[:-1], generator=gen, device="cuda") < 1 / 64
    if case["init"]:
        s["state"] = 0.3 * normal(n, h, dk, dv)
    if case["op"] == "train":
        s["do"] = normal(n, t, h, dv).to(dt)
        names = ["q", "k", "v", "g", "beta"]
        # a memory carried over from the rollout before is not trained through; a learned first one is (float32 cases)
        s["leaves"] = names + (["state"] if case["init"] and dt == torch.float32 else [])
        for name in s["leaves"]:
            s[name] = s[name].requires_grad_()
    return s


CHUNK = 16


def plain_step(s):
    state, q, k, v = s["state"], s["q"].float(), s["k"].float(), s["v"].float()
    group = v.shape[1] // q.shape[1]
    q, k = q.repeat_interleave(group, 1), k.repeat_interleave(group, 1)
    decay = torch.exp(s["g"].float())
    if s["reset"] is not None:
        decay = torch.where(s["reset"][:, None], torch.zeros_like(decay), decay)
    new = state * decay[..., None, None]
    u = s["beta"].float()[..., None] * (v - (new * k[..., None]).sum(-2))
    new = new + k[..., None] * u[..., None, :]
    out = (new * q[..., None]).sum(-2) * q.shape[-1] ** -0.5
    state.copy_(new)
    return out.to(s["v"].dtype), state


def plain_rollout(q, k, v, g, beta, state, reset):
    """The chunked form: within chunks of CHUNK tokens as small triangular systems, all of them at once; then the
    state from chunk to chunk."""
    dt = v.dtype
    n, t, h, dv = v.shape
    dk, group = q.shape[-1], h // q.shape[2]
    nc = -(-t // CHUNK)

    def chunks(x):
        x = torch.cat([x, x.new_zeros(n, nc * CHUNK - t, *x.shape[2:])], 1) if t % CHUNK else x
        x = x.reshape(n, nc, CHUNK, *x.shape[2:])
        return x.movedim(3, 1)  # (n, heads, chunks, CHUNK, ...)

    q, k, v, g, beta = (chunks(x.float()) for x in (q, k, v, g, beta))
    q, k = q.repeat_interleave(group, 1), k.repeat_interleave(group, 1)
    if reset is None:
        since = torch.zeros(n, 1, nc, CHUNK, dtype=torch.int64, device=v.device)
    else:
        since = chunks(reset[:, :, None].to(torch.int64)).cumsum(-1)  # resets so far in the chunk
        g = torch.where(chunks(reset[:, :, None]), torch.zeros_like(g), g)
    total = g.cumsum(-1)
    below = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=v.device).tril()
    seen = below & (since[..., :, None] == since[..., None, :])
    d = torch.exp(torch.where(seen, total[..., :, None] - total[..., None, :], -math.inf))
    w = k @ k.transpose(-1, -2) * d * beta[..., None, :]
    p = q @ k.transpose(-1, -2) * d * dk ** -0.5
    # rows of (I + strictly lower part of w)^-1
    eye = torch.eye(CHUNK, device=v.device)
    rows = [eye[0].expand(*w.shape[:-2], CHUNK)]
    for i in range(1, CHUNK):
        rows.append(eye[i] - (w[..., i, :i, None] * torch.stack(rows, -2)).sum(-2))
    z = torch.stack(rows, -2)
    a = torch.exp(total) * (since == 0)
    to_end = torch.exp(total[..., -1:] - total) * (since == since[..., -1:])
    state = v.new_zeros(n, h, dk, dv) if state is None else state
    out = []
    for c in range(nc):
        kc, ac = k[:, :, c], a[:, :, c, :, None]
        u = beta[:, :, c, :, None] * (z[:, :, c] @ (v[:, :, c] - ac * (kc @ state)))
        out.append(dk ** -0.5 * ac * (q[:, :, c] @ state) + p[:, :, c] @ u)
        state = a[:, :, c, -1, None, None] * state + kc.transpose(-1, -2) @ (to_end[:, :, c, :, None] * u)
    out = torch.stack(out, 2).movedim(1, 3).reshape(n, nc * CHUNK, h, dv)[:, :t]
    return out.to(dt), state


def plain_clip(grads, max_norm):
    norm = torch.stack([x.float().square().sum() for x in grads]).sum().sqrt()
    coef = torch.clamp(max_norm / (norm + 1e-6), max=1.0)
    return norm, [x.copy_(x.float() * coef) for x in grads]


def package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "getting-over-it-rl_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import goib2d
    return goib2d


def run(s):
    op = s["case"]["op"]
    if own:
        goib2d = sys.modules.get("goib2d") or package()
        if op == "clip":
            return goib2d.clip_grads_(s["grads"], s["max_norm"]), s["grads"]
        if op == "step":
            return goib2d.delta_step_(s["state"], s["q"], s["k"], s["v"], s["g"], s["beta"], reset=s["reset"]), s["state"]
        rollout = goib2d.delta_rule
    else:
        if op == "clip":
            return plain_clip(s["grads"], s["max_norm"])
        if op == "step":
            return plain_step(s)
        rollout = plain_rollout
    args = [s[x] for x in ("q", "k", "v", "g", "beta", "state", "reset")]
    if op == "rollout":
        return rollout(*args)
    out, state = rollout(*args)
    grads = torch.autograd.grad([out], [s[x] for x in s["leaves"]], [s["do"]])
    return out.detach(), state.detach(), grads


def work(case):
    if case["op"] == "clip":
        n = [math.prod(x) for x in shapes(case)]
        width = [4 if case["mixed"] and (len(x) == 1 or x[0] == 2) else DTYPES[case["dtype"]].itemsize for x in shapes(case)]
        return {"bytes": 2 * sum(a * b for a, b in zip(n, width)), "flops": 3 * sum(n)}
    n, t, h, hk = case["worlds"], case["steps"], case["heads"], case["key_heads"]
    dk, dv, size = case["key_dim"], case["value_dim"], DTYPES[case["dtype"]].itemsize
    state = n * h * dk * dv
    read = n * t * (2 * hk * dk + h * dv + 2 * h) * size + (n * t if case["resets"] else 0)
    out = n * t * h * dv * size + 4 * state
    total = read + out + (4 * state if case["init"] else 0)
    flops = 6 * n * t * h * dk * dv
    if case["op"] == "train":
        total += n * t * h * dv * size + n * t * (2 * hk * dk + h * dv + 2 * h) * size
        total += 4 * state if case["init"] and case["dtype"] == "float32" else 0
        flops *= 3
    return {"bytes": total, "flops": flops}


def exact(case, seed):
    """The definition in 64 bits: the recurrence token by token, its gradient by the same recurrence backwards."""
    s = prepare(case, seed)
    if case["op"] == "clip":
        wide = [x.double() for x in s["grads"]]
        norm = torch.sqrt(sum((x * x).sum() for x in wide))
        return norm, [x * min(1.0, s["max_norm"] / (float(norm) + 1e-6)) for x in wide]
    step = case["op"] == "step"
    q, k, v, g, beta = (s[x].detach().double() for x in ("q", "k", "v", "g", "beta"))
    reset = s["reset"]
    if step:
        q, k, v, g, beta = (x[:, None] for x in (q, k, v, g, beta))
        reset = None if reset is None else reset[:, None]
    n, t, h, dv = v.shape
    hk, dk = q.shape[2:]
    q, k = (x.repeat_interleave(h // hk, 2) for x in (q, k))
    decay = g.exp()
    if reset is not None:
        decay = decay.masked_fill(reset[..., None], 0.0)
    scale = 1 / math.sqrt(dk)
    start = torch.zeros(n, h, dk, dv, dtype=torch.float64, device="cuda")
    if s["state"] is not None:
        start = s["state"].detach().double()

    def read(m, x):  # m^T x
        return torch.einsum("nhkv,nhk->nhv", m, x)

    def onto(m, x):  # m x
        return torch.einsum("nhkv,nhv->nhk", m, x)

    def forward(state, i):
        state = state * decay[:, i, :, None, None]
        r = v[:, i] - read(state, k[:, i])
        u = r * beta[:, i, :, None]
        return state, r, u, state + torch.einsum("nhk,nhv->nhkv", k[:, i], u)

    # states are kept every `every` tokens, and those between made again on the way back
    every = max(1, int(math.sqrt(t)))
    if case["op"] == "train" and start.numel() * 8 * (t / every + 4 * every) > 100e9:
        return None
    out, kept, state = torch.empty_like(v), [], start
    for i in range(t):
        if i % every == 0 and case["op"] == "train":
            kept.append(state)
        state = forward(state, i)[3]
        out[:, i] = scale * read(state, q[:, i])
    if step:
        return out[:, 0], state
    if case["op"] == "rollout":
        return out, state
    do = s["do"].double()
    dq, dkey, dval = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    dg, dbeta, ds = torch.empty_like(g), torch.empty_like(beta), torch.zeros_like(start)
    for c in reversed(range(len(kept))):
        now, part = kept[c], []
        for i in range(c * every, min(t, (c + 1) * every)):
            part.append(forward(now, i))
            now = part[-1][3]
        for i in reversed(range(c * every, min(t, (c + 1) * every))):
            old, r, u, new = part.pop()
            ds = ds + scale * torch.einsum("nhk,nhv->nhkv", q[:, i], do[:, i])
            dq[:, i] = scale * onto(new, do[:, i])
            du = read(ds, k[:, i])
            dbeta[:, i] = (du * r).sum(-1)
            dval[:, i] = du * beta[:, i, :, None]
            dkey[:, i] = onto(ds, u) - onto(old, dval[:, i])
            ds = ds - torch.einsum("nhk,nhv->nhkv", k[:, i], dval[:, i])
            dg[:, i] = (old * ds).sum((-1, -2))
            ds = ds * decay[:, i, :, None, None]
    dq, dkey = (x.unflatten(2, (hk, h // hk)).sum(3) for x in (dq, dkey))
    grads = [dq, dkey, dval, dg, dbeta] + ([ds] if "state" in s["leaves"] else [])
    return out, state, grads
